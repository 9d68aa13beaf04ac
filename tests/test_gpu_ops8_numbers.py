"""Numbers that do not fit the library's 32-bit arguments are refused by the Python calls, not cut off."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("change", [dict(window=2**32 + 5), dict(window=2**40), dict(window=2**31), dict(max_q=2**32 + 1),
                                    dict(max_kv=2**32), dict(max_kv=-2**31 - 1)])
def test_attention(change):
    from e2e_browser_voice_agent_b200 import kv8
    kv, sc = kv8.allocate(4, 16, 2, 64)
    a = dict(q=torch.zeros(1, 4, 64, device=DEV), kv=kv, kv_scale=sc, block_table=torch.zeros(1, 2, dtype=torch.int32, device=DEV),
             q_start=i32(0, 1), kv_len=i32(1), max_q=1, max_kv=1)
    kv8.attention(**a)
    with pytest.raises(ValueError, match="32 bits"):
        kv8.attention(**{**a, **change})


@pytest.mark.parametrize("change", [dict(page_size=2**32 + 16), dict(max_tokens=2**32 + 1)])
def test_plan(change):
    from e2e_browser_voice_agent_b200 import kv8
    ring, state = kv8.free_pool(4)
    a = dict(cached=i32(0), total=i32(1), block_table=torch.zeros(1, 2, dtype=torch.int32, device=DEV), free_pages=ring,
             free_state=state, page_size=16, max_tokens=1)
    with pytest.raises(ValueError, match="32 bits"):
        kv8.plan(**{**a, **change})
    kv8.plan(**a)


def test_matrices():
    from e2e_browser_voice_agent_b200 import int8
    w, ws = int8.quantize(torch.ones(1, 16, device=DEV))
    x = torch.ones(1, 16, device=DEV)
    long = torch.ones(1, 16, device=DEV).expand(2**32 + 1, 16)   # (one row of memory)
    for call in (lambda: int8.quantize(long), lambda: int8.matmul(long, w, ws), lambda: int8.matmul(x, w.expand(2**32 + 1, 16), ws)):
        with pytest.raises(ValueError, match="32 bits"):
            call()
