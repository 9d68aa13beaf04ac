"""The C entries of the 8-bit serving operators refuse arguments that do not fit with a status and a message, before
anything touches a device (so these run without one)."""
import ctypes as C

import pytest

from e2e_browser_voice_agent_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


X = 1 << 20  # stands for a device address: never looked at


def message(lib):
    return lib.h2c_last_error(None).decode()


PLAN = dict(n_req=2, page=16, cached=X, total=X, table=X, cols=4, ring=X, n_pages=8, state=X, out=X + 64, kv_len=X,
            q_start=X, slot=X, position=X, max_tokens=4, status=X, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(n_req=-1), "n_req"), (dict(n_req=8193), "n_req"), (dict(page=24), "page_size"), (dict(page=0), "page_size"),
    (dict(cached=None), "null"), (dict(table=None), "null"), (dict(slot=None), "null"), (dict(status=None), "null"),
    (dict(out=X), "free_state_out"), (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 27), "n_pages"), (dict(cols=0), "table_cols"),
    (dict(max_tokens=-1), "max_tokens"), (dict(max_tokens=2**31 - 1), "max_tokens"),
])
def test_plan_refuses(lib, change, word):
    a = {**PLAN, **change}
    assert lib.h2c_kv8_plan(*a.values()) == _lib.ERR_INVALID
    assert message(lib).startswith("h2c_kv8_plan:") and word in message(lib)


APPEND = dict(kv=X, scale=X, n_pages=8, page=16, kv_heads=2, head_dim=64, type=0, k=X, k_row=128, k_head=64, v=X, v_row=128,
              v_head=64, rows=3, slot=X, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(kv=None), "null"), (dict(kv=X + 8), "aligned"), (dict(page=8), "page_size"), (dict(head_dim=96), "head_dim"),
    (dict(kv_heads=0), "kv_heads"), (dict(n_pages=-3), "n_pages"), (dict(rows=-1), "rows"), (dict(k=None), "null"),
    (dict(slot=None), "null"), (dict(k=X + 2), "aligned"), (dict(type=2, v=X + 1), "aligned"),
])
def test_append_refuses(lib, change, word):
    assert lib.h2c_kv8_append(*{**APPEND, **change}.values()) == _lib.ERR_INVALID
    assert message(lib).startswith("h2c_kv8_append:") and word in message(lib)


def test_types_and_empty_calls(lib):
    assert lib.h2c_kv8_append(*{**APPEND, "type": 7}.values()) == _lib.ERR_BAD_TYPE
    assert "element type 7" in message(lib)
    assert lib.h2c_kv8_append(*{**APPEND, "rows": 0, "k": None}.values()) == _lib.OK
    assert lib.h2c_kv8_read(X, X, 8, 16, 2, 64, X, 3, 0, X + 8, X, None) == _lib.ERR_INVALID and "aligned" in message(lib)
    assert lib.h2c_kv8_read(X, X, 8, 16, 2, 64, X, 3, 9, X, X, None) == _lib.ERR_BAD_TYPE
    assert lib.h2c_kv8_read(X, X, 8, 16, 2, 64, None, 0, 0, None, None, None) == _lib.OK


def attention_args(**change):
    a = dict(q=X, q_row=256, q_head=64, out=X, out_row=256, out_head=64, lse=None, kv=X, kv_scale=X, n_pages=8, page_size=16,
             kv_heads=2, head_dim=64, heads=4, type=0, block_table=X, table_cols=4, n_req=2, q_start=X, kv_len=X, rows=2,
             max_q=1, max_kv=60, window=0, scale=0.125, workspace=None, workspace_bytes=0)
    assert set(change) <= set(a)
    return _lib.Kv8AttentionArgs(**{**a, **change})


@pytest.mark.parametrize("change,word", [
    (dict(page_size=48), "page_size"), (dict(head_dim=32), "head_dim"), (dict(n_pages=0), "n_pages"), (dict(heads=5), "multiple"),
    (dict(heads=1), "multiple"), (dict(kv_heads=0), "multiple"), (dict(n_req=9000), "n_req"), (dict(rows=-1), "negative"),
    (dict(max_kv=-1), "negative"), (dict(window=-2), "negative"), (dict(max_q=2**31 - 1), "max_q"), (dict(q=None), "null"),
    (dict(kv_len=None), "null"), (dict(block_table=None), "null"), (dict(kv=X + 4), "aligned"), (dict(out=X + 2), "aligned"),
    (dict(max_kv=4000), "workspace"), (dict(max_kv=4000, workspace=X + 4, workspace_bytes=1 << 30), "workspace"),
])
def test_attention_refuses(lib, change, word):
    a = attention_args(**change)
    assert lib.h2c_kv8_attention(C.byref(a), None) == _lib.ERR_INVALID
    assert message(lib).startswith("h2c_kv8_attention:") and word in message(lib)


def test_attention_of_nothing_and_its_workspace(lib):
    assert lib.h2c_kv8_attention(None, None) == _lib.ERR_INVALID
    assert lib.h2c_kv8_attention(C.byref(attention_args(type=5)), None) == _lib.ERR_BAD_TYPE
    for change in (dict(n_req=0), dict(rows=0), dict(max_q=0)):
        assert lib.h2c_kv8_attention(C.byref(attention_args(q=None, **change)), None) == _lib.OK
    assert lib.h2c_kv8_attention_workspace(C.byref(attention_args())) == 0
    need = lib.h2c_kv8_attention_workspace(C.byref(attention_args(max_kv=4000)))
    assert 0 < need < 1 << 24
    a = attention_args(max_kv=4000, workspace=X, workspace_bytes=need - 1)
    assert lib.h2c_kv8_attention(C.byref(a), None) == _lib.ERR_INVALID and str(need) in message(lib)


MATMUL = dict(x_type=0, x=X, x_row=64, x_scale=None, w=X, w_row=64, w_scale=X, m=2, n=3, k=50, y_type=0, y=X, y_row=3, bias=None,
              workspace=X, workspace_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,word", [
    (dict(m=-1), "sizes"), (dict(k=0), "sizes"), (dict(k=131073, w_row=131088), "sizes"), (dict(w=None), "null"),
    (dict(w_scale=None), "null"), (dict(x_type=3, x_scale=None), "null"), (dict(w=X + 8), "w must"), (dict(w_row=56), "w must"),
    (dict(w_row=48), "w must"), (dict(x_type=3, x_scale=X, x_row=50), "codes must"), (dict(x=X + 2), "x must"),
    (dict(y=X + 2), "y must"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=10), "workspace"),
    (dict(workspace=X + 8), "workspace"),
])
def test_matmul_refuses(lib, change, word):
    assert lib.h2c_i8_matmul(*{**MATMUL, **change}.values()) == _lib.ERR_INVALID
    assert message(lib).startswith("h2c_i8_matmul:") and word in message(lib)


def test_matmul_types_sizes_of_zero_and_quantize(lib):
    assert lib.h2c_i8_matmul(*{**MATMUL, "x_type": 4}.values()) == _lib.ERR_BAD_TYPE
    assert lib.h2c_i8_matmul(*{**MATMUL, "y_type": 3}.values()) == _lib.ERR_BAD_TYPE
    assert lib.h2c_i8_matmul(*{**MATMUL, "m": 0, "x": None}.values()) == _lib.OK
    assert lib.h2c_i8_matmul(*{**MATMUL, "n": 0, "y": None}.values()) == _lib.OK
    assert lib.h2c_i8_matmul_workspace(0, 2, 50) >= 2 * 64 + 8 and lib.h2c_i8_matmul_workspace(3, 2, 50) == 0
    q = dict(type=0, x=X, x_row=50, rows=2, k=50, q=X, q_row=64, scale=X, stream=None)
    for change in (dict(k=0), dict(rows=-1), dict(x=None), dict(q=X + 4), dict(q_row=48), dict(q_row=60), dict(x=X + 1)):
        assert lib.h2c_i8_quantize(*{**q, **change}.values()) == _lib.ERR_INVALID
    assert lib.h2c_i8_quantize(*{**q, "type": 3}.values()) == _lib.ERR_BAD_TYPE
    assert lib.h2c_i8_quantize(*{**q, "rows": 0, "x": None}.values()) == _lib.OK
