"""Outputs in the memory of inputs: what the 8-bit serving operators allow gives the bits that it gives elsewhere."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 2, 3, 33])
@pytest.mark.parametrize("n,k", [(896, 896), (2048, 2048), (100, 896), (896, 100)])
def test_matmul_over_its_tokens(dtype, m, n, k):
    """One token and two are quantized by every CTA of the product for itself elsewhere, but not here."""
    from e2e_browser_voice_agent_b200 import int8
    gen = torch.Generator(device=DEV)
    gen.manual_seed(m + n + k)
    w = torch.randint(-127, 128, (n, (k + 15) // 16 * 16), generator=gen, device=DEV).to(torch.int8)
    ws = 0.001 * torch.exp(torch.randn(n, generator=gen, device=DEV))
    for _ in range(20):
        buf = torch.randn(m, max(n, k) + 7, generator=gen, device=DEV).to(dtype)
        want = int8.matmul(buf[:, :k].clone(), w, ws)
        for at in (0, 3):
            z = buf.clone()
            got = int8.matmul(z[:, :k], w, ws, out=z[:, at:at + n])
            assert torch.equal(got, want)
            assert torch.equal(z[:, at + n:], buf[:, at + n:]) and torch.equal(z[:, :at], buf[:, :at])


def test_columns_of_one_buffer_stay_one_launch():
    """Tokens and outputs side by side share no memory, although their ranges interleave."""
    from e2e_browser_voice_agent_b200 import int8
    x = torch.randn(2, 900, device=DEV)
    w, ws = int8.quantize(torch.randn(128, 400, device=DEV))
    want = int8.matmul(x[:, :400].contiguous(), w, ws)
    assert torch.equal(int8.matmul(x[:, :400], w, ws, out=x[:, 450:578]), want)


def attention_case(dtype, hd, kv_len, n_q, heads=14, kvh=2, seed=0):
    import test_gpu_kv8 as t
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + hd + sum(kv_len))
    kv, sc, table = t.make_cache(gen, kv_len, 16, kvh, hd)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    start = [0]
    for n in n_q:
        start.append(start[-1] + n)
    q = torch.randn(start[-1], heads, hd, generator=gen, device=DEV).to(dtype)
    call = lambda q, **kw: t.kv8().attention(q, kv, sc, table, i32(start), i32(kv_len), max(n_q), max(kv_len), return_lse=True, **kw)
    return q, call


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv_len,n_q", [([700], [1]), ([5000, 90], [1, 1]), ([3000], [200]), ([900, 2000, 30], [1, 150, 30]),
                                        ([300], [9])])
def test_attention_over_its_queries(dtype, hd, kv_len, n_q):
    """One span, a cluster's, spans joined by a second kernel, both kernels in one call."""
    q, call = attention_case(dtype, hd, kv_len, n_q)
    want, want_lse = call(q)
    for _ in range(5):
        z = q.clone()
        got, lse = call(z, out=z)
        assert got is z and torch.equal(z, want) and torch.equal(lse, want_lse)


def test_attention_into_columns_and_interleaved_heads():
    """Layouts that share no memory although the ranges of their tokens or heads do."""
    q, call = attention_case(torch.float32, 64, [500, 40], [3, 2])
    want, _ = call(q)
    wide = torch.zeros(5, 31, 64, device=DEV)
    wide[:, 1:15] = q
    got, _ = call(wide[:, 1:15], out=wide[:, 15:29])     # beside the queries
    assert torch.equal(got, want) and torch.equal(wide[:, 1:15], q) and (wide[:, 29:] == 0).all()
    flat = torch.zeros(5 * 14 * 64 * 3, device=DEV)
    for row, head in ((64, 5 * 64), (3 * 64, 15 * 64), (15 * 64, 64), (29 * 64, 128)):
        out = flat.as_strided((5, 14, 64), (row, head, 1))
        got, _ = call(q, out=out)
        assert torch.equal(got, want)
    q, call = attention_case(torch.float32, 64, [50, 40], [1, 1])
    want, _ = call(q)
    out = flat.as_strided((2, 14, 64), (13 * 64, 128, 1))   # one token's heads between the other's
    got, _ = call(q, out=out)
    assert torch.equal(got, want)
