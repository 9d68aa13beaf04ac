"""int8.norm and int8.values: codes and sums against the formula's, at odd sizes, strides, types and extreme rows."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def int8():
    from e2e_browser_voice_agent_b200 import int8 as m
    return m


def formula(x, weight, eps, residual=None):
    """The formula in 64 bits, each operation on a value rounded to float32 as it says: (codes, scale, sum)."""
    f32 = lambda v: v.float().double()
    total = None
    s = x.double()
    if residual is not None:
        total = f32(s + residual.double()).to(residual.dtype)
        s = total.double()
    f = f32(1 / torch.sqrt(s.square().mean(-1, keepdim=True) + eps))
    y = f32(f32(s * f) * weight.double())
    a = y.abs().amax(-1, keepdim=True)
    inv = torch.where(a > 0, f32(127 / a).clamp(max=torch.finfo(torch.float32).max), 0.0)
    return torch.round(f32(y * inv)), f32(a / 127)[:, 0].float(), total


def stream(rows, k, dtype, seed=0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + 31 * rows + k)
    x = torch.randn(rows, k, generator=gen, device=DEV) * torch.exp(torch.randn(rows, 1, generator=gen, device=DEV))
    x[:, :: max(1, k // 5)] *= 9
    return x.to(dtype), 1 + 0.3 * torch.randn(k, generator=gen, device=DEV)


def check(n, want, k):
    codes, scale, total = want
    assert torch.equal(n.codes[:, :k].double(), codes)
    assert not n.codes[:, k:].any() and n.codes.shape[1] == (k + 15) // 16 * 16
    assert torch.equal(n.scale, scale)
    assert (n.sum is None) == (total is None)
    if total is not None:
        assert n.sum.dtype is total.dtype and torch.equal(n.sum, total)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 896), (3, 17), (5, 64), (2, 100), (33, 3584), (2, 4864), (7, 1000), (1, 131072), (2, 40003),
                                    (300, 8), (4099, 896)])
@pytest.mark.parametrize("residual", ["none", "same", "f32"])
def test_codes_are_the_formulas(dtype, rows, k, residual):
    x, w = stream(rows, k, dtype)
    res = None if residual == "none" else stream(rows, k, dtype if residual == "same" else torch.float32, 1)[0]
    check(int8().norm(x, w, 1e-6, residual=res), formula(x, w, 1e-6, res), k)


@pytest.mark.parametrize("dtype,residual", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                            (torch.bfloat16, None)])
@pytest.mark.parametrize("k", [4, 1020, 1024, 1028, 3584, 4096, 4100, 5003, 8192, 8196, 18944, 32768, 32772])
def test_every_division_of_a_row(dtype, residual, k):
    for rows in (444, 445):
        x, w = stream(rows, k, dtype)
        r = None if residual is None else stream(rows, k, residual, 1)[0]
        want = formula(x, w, 1e-6, r)
        n = int8().norm(x, w, 1e-6, residual=r)
        check(n, want, k)
        if r is not None:
            check(int8().norm(x, w, 1e-6, residual=r, out=r), want, k)

@pytest.mark.parametrize("dtype", TYPES)
def test_strides_places_and_in_place(dtype):
    rows, k = 6, 200
    x, w = stream(rows, k, dtype)
    res, _ = stream(rows, k, dtype, 5)
    want = formula(x, w, 1e-5, res)
    wide = torch.zeros(rows, 3 * k + 5, dtype=dtype, device=DEV)
    for at in (0, 1, 8):  # any start, rows of an odd length apart
        v = wide[:, at:at + k]
        v.copy_(x)
        r = wide[:, at + k:at + 2 * k]
        r.copy_(res)
        check(int8().norm(v, w, 1e-5, residual=r), want, k)
        out = torch.full((rows, k + 3), 7.0, dtype=dtype, device=DEV)
        n = int8().norm(v, w, 1e-5, residual=r, out=out[:, 1:k + 1])
        check(n, want, k)
        assert (out[:, 0] == 7).all() and (out[:, k + 1:] == 7).all()
        keep = wide.clone()
        n = int8().norm(v, w, 1e-5, residual=r, out=r)     # the residual stream itself
        check(n, want, k)
        assert torch.equal(v, x) and torch.equal(wide[:, at + 2 * k:], keep[:, at + 2 * k:])
        r.copy_(res)
        check(int8().norm(v, w, 1e-5, residual=r, out=v), want, k)
        v.copy_(x)
    flipped = torch.flip(x, [0])
    y = flipped.as_strided((rows, k), (k, 1))
    got = int8().norm(y, w, 1e-5)
    check(got, formula(flipped, w, 1e-5), k)
    one = x[0].expand(rows, k)                              # the same row for all
    check(int8().norm(one, w, 1e-5, residual=res), formula(one, w, 1e-5, res), k)
    odd = torch.zeros(k + 1, device=DEV)[1:]                # a weight that is not 16-byte aligned
    odd.copy_(w)
    check(int8().norm(x, odd, 1e-5), formula(x, w, 1e-5), k)
    long, w = stream(2, 40000, dtype)
    r, _ = stream(2, 40000, dtype, 9)
    want = formula(long, w, 1e-6, r)
    check(int8().norm(long, w, 1e-6, residual=r, out=r), want, 40000)   # rows longer than the registers hold, in place


@pytest.mark.parametrize("k", [3584, 3585])
def test_rows_more_than_32_bits_apart(k):
    far = 2**31 + 64
    x, w = stream(2, k, torch.bfloat16)
    r, _ = stream(2, k, torch.bfloat16, 1)
    buf = torch.empty(far + 3 * k + 64, dtype=torch.bfloat16, device=DEV)
    a, b, c = (buf[at:].as_strided((2, k), (far, 1)) for at in (0, k + 15 & ~15, 2 * k + 31 & ~15))
    a.copy_(x)
    b.copy_(r)
    want = formula(x, w, 1e-6, r)
    check(int8().norm(a, w, 1e-6, residual=b, out=c), want, k)
    check(int8().norm(a, w, 1e-6, residual=b, out=b), want, k)
    assert torch.equal(a, x) and torch.equal(b, want[2]) and torch.equal(c, want[2])

@pytest.mark.parametrize("dtype", TYPES)
def test_extreme_rows(dtype):
    big = torch.finfo(dtype).max
    k = 48
    x = torch.zeros(8, k, dtype=dtype, device=DEV)
    x[1] = big                                   # squares beyond float32
    x[2] = torch.finfo(dtype).tiny
    x[3, 5] = math.inf
    x[4, 7] = math.nan
    x[5, 1] = -math.inf
    x[6] = torch.arange(k, device=DEV).to(dtype)
    x[7, :] = torch.finfo(dtype).tiny / 8 if dtype is not torch.float16 else 2.0**-24
    w = torch.ones(k, device=DEV)
    for eps in (1e-6, 1e-30):
        n = int8().norm(x, w, eps)
        codes, scale, _ = formula(x, w, eps)
        fine = [0, 1, 2, 6, 7]
        assert torch.equal(n.codes[fine, :k].double(), codes[fine]) and torch.equal(n.scale[fine], scale[fine])
        assert n.scale[[3, 4, 5]].isnan().all()
        assert int8().values(n.codes, n.scale, k)[[3, 4, 5]].isnan().all()
    zero = int8().norm(x[:1], w, 0.0)            # 0 / 0
    assert zero.scale.isnan().all()
    w[3] = math.inf
    assert int8().norm(x[6:7], w, 1e-6).scale.isnan().all()
    r = torch.full((1, k), big, dtype=dtype, device=DEV)
    n = int8().norm(r, torch.ones(k, device=DEV), 1e-6, residual=r)   # the sum overflows
    assert n.sum.isinf().all() and n.scale.isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 17), (40, 896), (5, 8), (1000, 1000), (2, 131072)])
def test_values(dtype, rows, k):
    x, _ = stream(rows, k, torch.float32)
    q, s = int8().quantize(x)
    assert torch.equal(int8().values(q, s, k, dtype), (q[:, :k].float() * s[:, None]).to(dtype))
    assert int8().values(q, s).shape == q.shape
    wide = torch.zeros(rows, q.shape[1] + 32, dtype=torch.int8, device=DEV)
    wide[:, 16:-16] = q
    assert torch.equal(int8().values(wide[:, 16:-16], s, k, dtype), (q[:, :k].float() * s[:, None]).to(dtype))


def test_codes_go_into_products():
    x, w = stream(9, 100, torch.bfloat16)
    w8, ws = int8().quantize(torch.randn(50, 100, device=DEV))
    n = int8().norm(x, w)
    got = int8().matmul(n.codes, w8, ws, x_scale=n.scale, k=100)
    codes, scale, _ = formula(x, w, 1e-6)
    want = (codes @ w8[:, :100].double().t()).float() * scale[:, None] * ws    # (the integer sums are exact)
    assert torch.equal(got, want)


def test_streams_graphs_and_nothing_to_do():
    x, w = stream(70, 896, torch.bfloat16)
    r, _ = stream(70, 896, torch.bfloat16, 2)
    want = int8().norm(x, w, 1e-6, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = int8().norm(x, w, 1e-6, residual=r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = int8().norm(x, w, 1e-6, residual=r)
        back = int8().values(got.codes, got.scale, 896, torch.bfloat16)
    r2, _ = stream(70, 896, torch.bfloat16, 3)
    r.copy_(r2)
    for _ in range(3):
        g.replay()
    want = int8().norm(x, w, 1e-6, residual=r2)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(back, int8().values(want.codes, want.scale, 896, torch.bfloat16))
    n = int8().norm(x[:0], w)
    assert n.codes.shape == (0, 896) and int8().values(n.codes, n.scale).shape == (0, 896)
