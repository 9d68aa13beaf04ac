"""Matrix products in 8-bit integers on the GPU: quantize against its formula in float32 (exact), matmul against exact
integer sums in 64 bits. The scaled result is two or three float32 operations from the exact one: off by at most 2^-22 of
its terms, and by the rounding to the output's type."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def int8():
    from e2e_browser_voice_agent_b200 import int8 as m
    return m


def ref_quantize(x):
    x = x.astype(np.float32)
    a = np.abs(x).max(1, keepdims=True)
    with np.errstate(all="ignore"):
        inv = np.where(a > 0, np.minimum(np.float32(127) / a, np.float32(3.4028234663852886e38)), np.float32(0)).astype(np.float32)
    return np.rint(x * inv), (a / np.float32(127))[:, 0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 2), (2, 31), (5, 896), (700, 130), (1, 18944), (9, 4865), (600, 5000)])
def test_quantize_matches_the_formula(dtype, rows, k):
    rng = np.random.default_rng(rows + k)
    x = (rng.standard_normal((rows, k)) * np.exp(2 * rng.standard_normal((rows, 1)))).astype(np.float32)
    x[rows // 2] *= 0 if rows > 2 else 1
    for t in (torch.from_numpy(x).to(DEV).to(dtype), torch.nn.functional.pad(torch.from_numpy(x).to(DEV).to(dtype), (1, 2))[:, 1:k + 1]):
        q, s = int8().quantize(t)
        want_q, want_s = ref_quantize(t.float().cpu().numpy())
        assert q.shape == (rows, (k + 15) // 16 * 16)
        assert np.array_equal(q[:, :k].cpu().numpy(), want_q) and (q[:, k:] == 0).all()
        assert np.array_equal(s.cpu().numpy(), want_s)


def check(x, w, ws, bias, y, out_dtype, xq=None, xs=None):
    k = x.shape[1]
    if xq is None:
        want_q, want_s = ref_quantize(x.float().cpu().numpy())
        xq, xs = torch.from_numpy(want_q).to(DEV), torch.from_numpy(want_s).to(DEV)
    acc = xq[:, :k].double() @ w[:, :k].double().t()             # exact: below 2^53
    want = acc * xs.double()[:, None] * ws.double()
    size = want.abs()
    if bias is not None:
        want = want + bias.double()
        size = size + bias.double().abs()
    off = (y.double() - want).abs()
    assert y.dtype is out_dtype
    bound = 2.0**-22 * size + EPS[out_dtype] * want.abs() + (2.0**-24 if out_dtype is torch.float16 else 0)
    assert (off <= bound).all(), float((off / bound).max())


def make(m, n, k, dtype, bias, seed=0, ldw=None):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + m + n + k)
    x = (torch.randn(m, k, generator=gen, device=DEV) * torch.exp(torch.randn(m, 1, generator=gen, device=DEV))).to(dtype)
    w = torch.randint(-127, 128, (n, ldw or (k + 15) // 16 * 16), generator=gen, device=DEV).to(torch.int8)  # (padding: garbage)
    ws = 0.001 * torch.exp(torch.randn(n, generator=gen, device=DEV))
    b = torch.randn(n, generator=gen, device=DEV) if bias else None
    return x, w, ws, b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 100, 129, 256, 257, 700])
@pytest.mark.parametrize("n,k", [(1152, 896), (130, 33), (1, 1), (128, 128), (1000, 4864)])
def test_matmul(dtype, m, n, k):
    x, w, ws, b = make(m, n, k, dtype, bias=(m + n) % 2 == 0)
    check(x, w, ws, b, int8().matmul(x, w, ws, bias=b), dtype)


@pytest.mark.parametrize("m,n,k", [(1, 37888, 3584), (32, 4608, 3584), (7, 3584, 18944), (300, 3584, 18944), (4099, 896, 896),
                                   (2000, 9728, 896), (1, 151936, 896), (3, 129, 131072)])
def test_matmul_at_model_sizes(m, n, k):
    x, w, ws, b = make(m, n, k, torch.bfloat16, bias=True)
    check(x, w, ws, b, int8().matmul(x, w, ws, bias=b, out_dtype=torch.float32), torch.float32)


def test_largest_sums_stay_exact():
    """Every code at its largest magnitude over the longest rows: the sum is just below 2^31."""
    k = 131072
    for sign in (1, -1):
        x = torch.full((2, k), 3.0, device=DEV)
        w = torch.full((5, k), 127 * sign, dtype=torch.int8, device=DEV)
        ws = torch.ones(5, device=DEV)
        y = int8().matmul(x, w, ws)
        want = sign * 127.0 * 127 * k * float(np.float32(3) / np.float32(127))
        assert ((y.double() - want).abs() <= 2.0**-22 * abs(want)).all()


@pytest.mark.parametrize("out_dtype", TYPES)
def test_codes_given_and_strides(out_dtype):
    m, n, k = 37, 300, 1000
    x, w, ws, b = make(m, n, k, torch.float32, bias=True, ldw=1040)
    xq, xs = int8().quantize(x)
    y = int8().matmul(xq, w, ws, bias=b, x_scale=xs, k=k, out_dtype=out_dtype)
    check(x, w, ws, b, y, out_dtype, xq, xs)
    assert torch.equal(y, int8().matmul(x, w, ws, bias=b, out_dtype=out_dtype))  # as when they are made on the way
    wide = torch.full((m, n + 9), 5.0, dtype=out_dtype, device=DEV)
    odd = torch.nn.functional.pad(x, (3, 2))[:, 3:k + 3]                         # rows that start at odd elements
    assert torch.equal(int8().matmul(odd, w, ws, bias=b, out=wide[:, 4:n + 4]), y)
    assert (wide[:, :4] == 5).all() and (wide[:, n + 4:] == 5).all()


def test_rows_that_are_no_numbers_stay_alone():
    x, w, ws, b = make(20, 200, 100, torch.float32, bias=True)
    good = int8().matmul(x, w, ws, bias=b)
    for bad in (float("nan"), float("inf"), -float("inf")):
        z = x.clone()
        z[7, 50] = bad
        y = int8().matmul(z, w, ws, bias=b)
        assert y[7].isnan().all()
        y[7] = good[7]
        assert torch.equal(y, good)


def test_zero_and_tiny_rows():
    x, w, ws, b = make(6, 200, 100, torch.float32, bias=True)
    x[1] = 0
    x[2] *= 1e-42
    x[3] *= 1e-36
    y = int8().matmul(x, w, ws, bias=b)
    assert torch.equal(y[1], b) and y.isfinite().all()
    check(x, w, ws, b, y, torch.float32)


def test_no_rows_no_outputs():
    x, w, ws, _ = make(3, 20, 50, torch.float32, bias=False)
    assert int8().matmul(x[:0], w, ws).shape == (0, 20)
    assert int8().matmul(x, w[:0], ws[:0]).shape == (3, 0)
    assert int8().quantize(x[:0])[0].shape == (0, 64)


def test_the_same_bits_every_time_in_a_graph_and_on_a_stream():
    for m in (1, 40, 500):
        x, w, ws, b = make(m, 1152, 896, torch.bfloat16, bias=True)
        want = int8().matmul(x, w, ws, bias=b)
        for _ in range(5):
            assert torch.equal(int8().matmul(x, w, ws, bias=b), want)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            got = int8().matmul(x, w, ws, bias=b)
        x.mul_(-2)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, int8().matmul(x, w, ws, bias=b)) and not torch.equal(got, want)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = int8().matmul(x, w, ws, bias=b)
        s.synchronize()
        assert torch.equal(other, got)
    from e2e_browser_voice_agent_b200 import _lib
    _lib.check_ops()


def test_a_weight_matrix_beyond_32_bit_offsets():
    n, k = 40000, 114688
    w = torch.zeros(n, k, dtype=torch.int8, device=DEV)          # 4.6 GB
    w[-1, -3:] = 5
    w[n // 2, 7] = -2
    x = torch.ones(2, k, device=DEV)
    y = int8().matmul(x, w, torch.ones(n, device=DEV))
    assert abs(float(y[1, -1]) - 15) < 1e-5 and abs(float(y[0, n // 2]) + 2) < 1e-5
    assert int(torch.count_nonzero(y)) == 4


def test_refusals_of_the_python_calls():
    from e2e_browser_voice_agent_b200._lib import H2CError
    m = int8()
    x, w, ws, b = make(3, 20, 50, torch.float32, bias=True)
    xq, xs = m.quantize(x)
    for a, kw in (((x.double(), w, ws), {}), ((x, w.float(), ws), {}), ((x, w, ws.double()), {}), ((xq, w, ws), {}),
                  ((x, w, ws), dict(x_scale=xs, k=50)), ((x, w, ws), dict(out_dtype=torch.int32))):
        with pytest.raises((TypeError, ValueError)):
            m.matmul(*a, **kw)
    for a, kw in (((x[0], w, ws), {}), ((x, w[:, :48], ws), {}), ((x, w, ws[:3]), {}), ((x, w, ws), dict(bias=b[:3])),
                  ((x.t().contiguous().t(), w, ws), {}), ((x, w, ws), dict(out=x)), ((x, w, ws), dict(k=49)),
                  ((xq, w, ws), dict(x_scale=xs)), ((x.cpu(), w, ws), {})):
        with pytest.raises(ValueError):
            m.matmul(*a, **kw)
    with pytest.raises(H2CError):      # rows of w that are not a multiple of 16 bytes apart
        m.matmul(x, torch.zeros(20, 51, dtype=torch.int8, device=DEV), ws)
    with pytest.raises(H2CError):
        m.matmul(torch.zeros(1, 131073, device=DEV), torch.zeros(2, 131088, dtype=torch.int8, device=DEV), ws[:2])
