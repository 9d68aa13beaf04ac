"""kv8.prefix_attention against a plain implementation in 64 bits, with attention's tolerance: what belongs to a row are the spans of its
prefix and of its own positions, added up in float32 (2^-24 a span, of which the tolerance's d holds many). bfloat16 rows may carry the
weights of a prefix as one float16 number (2^-11 of itself each), whatever their own positions take."""
import math

import numpy as np
import pytest
import torch

import test_gpu_kv8 as t

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]
i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)


def call(q, kv, sc, ptable, plen, gs, table, q_start, kv_len, **kw):
    n_q = [b - a for a, b in zip(q_start, q_start[1:])]
    kw.setdefault("max_q", max(n_q, default=0))
    kw.setdefault("max_kv", max(kv_len, default=0))
    kw.setdefault("max_prefix", max(plen, default=0))
    return t.kv8().prefix_attention(q, kv, sc, ptable, i32(plen), i32(gs), table, i32(q_start), i32(kv_len), return_lse=True, **kw)


def reference(q, kv, sc, ptable, plen, gs, table, q_start, kv_len, scale):
    """(out, lse, largest |score| in powers of two, largest |v|) in 64 bits."""
    page, hd, kvh, H = kv.shape[3], kv.shape[4], kv.shape[2], q.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    top = vmax = 0.0

    def held(row, n):
        pages = row[: -(-n // page)].long()
        x = kv[pages].double() * sc[pages].double()[..., None, None]
        return x.permute(1, 2, 0, 3, 4).reshape(2, kvh, -1, hd)[:, :, :n]
    for r, n in enumerate(kv_len):
        a, b = q_start[r], q_start[r + 1]
        g = next((g for g in range(len(plen)) if gs[g] <= r < gs[g + 1]), None)
        p = 0 if g is None else plen[g]
        if a == b or p + n == 0:
            continue
        x = held(table[r], n)
        if p:
            x = torch.cat([held(ptable[g], p), x], 2)
        k, v = x.repeat_interleave(H // kvh, 1)
        s = torch.einsum("thd,hnd->thn", q[a:b].double(), k) * scale
        key = torch.arange(p + n, device=DEV)
        pos = torch.arange(n - (b - a), n, device=DEV)
        seen = (key < p) | (key - p <= pos[:, None])
        top, vmax = max(top, float(s.abs().max()) * 1.4427), max(vmax, float(v.abs().max()))
        s = s.masked_fill(~seen[:, None], -math.inf)
        m = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(m.isinf(), 0.0, m))
        total = w.sum(-1, keepdim=True)
        out[a:b] = torch.einsum("thn,hnd->thd", w / torch.where(total == 0, 1.0, total), v)
        lse[a:b] = (m + torch.log(total))[..., 0]
    return out, lse, top, vmax


def inputs(dtype, page, H, kvh, hd, plen, kv_len, n_q, seed=0, spread=0.5):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + page + H + hd + sum(plen) + sum(kv_len))
    kv, sc, both = t.make_cache(gen, plen + kv_len, page, kvh, hd, spread)
    cols = lambda lens: max([1] + [-(-n // page) for n in lens])
    ptable, table = both[:len(plen), :cols(plen)].contiguous(), both[len(plen):, :cols(kv_len)].contiguous()
    q = torch.randn(sum(n_q), H, hd, generator=gen, device=DEV)
    q *= torch.exp(torch.randn(sum(n_q), H, 1, generator=gen, device=DEV))
    return q.to(dtype), kv, sc, ptable, table, [0] + np.cumsum(n_q).tolist()


def run_case(dtype, page, H, kvh, hd, plen, gs, kv_len, n_q, scale=None, seed=0, spread=0.5, **kw):
    q, kv, sc, ptable, table, q_start = inputs(dtype, page, H, kvh, hd, plen, kv_len, n_q, seed, spread)
    o, lse = call(q, kv, sc, ptable, plen, gs, table, q_start, kv_len, scale=scale, **kw)
    ref = reference(q, kv, sc, ptable, plen, gs, table, q_start, kv_len, hd ** -0.5 if scale is None else scale)
    t.close(o, lse, ref, dtype, dtype != torch.float32)
    return o, lse


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128), (4, 4, 64), (7, 1, 128), (16, 1, 64)])
def test_single_tokens(dtype, H, kvh, hd):
    for page, p, kv_len in [(16, 1, [1]), (16, 16, [1, 15, 16, 17]), (16, 641, [20, 200, 1, 77]), (32, 301, [300, 2, 63]), (64, 1000, [65, 1200]),
                            (128, 127, [127, 128, 129])]:
        run_case(dtype, page, H, kvh, hd, [p], [0, len(kv_len)], kv_len, [1] * len(kv_len))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,p", [(3, 5000), (40, 1500), (40, 63), (70, 4097), (150, 2000)])
def test_many_single_tokens(dtype, hd, n, p):
    """Both kernels for the prefix, in one span and in many."""
    kv_len = [1 + (37 * i) % 90 for i in range(n)]
    run_case(dtype, 16, 14 if hd == 64 else 28, 2 if hd == 64 else 4, hd, [p], [0, n], kv_len, [1] * n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128), (4, 2, 128)])
def test_ragged_batches(dtype, H, kvh, hd):
    # prompts from the start, continuations, single tokens, requests without queries, without keys, with neither; a prefix that is empty, a
    # group that is, requests of no group
    kv_len = [50, 700, 129, 0, 333, 20, 0, 512, 1, 9]
    n_q = [50, 3, 1, 0, 120, 0, 2, 200, 1, 9]
    run_case(dtype, 16, H, kvh, hd, [77, 0, 300, 1000], [0, 2, 4, 4, 8], kv_len, n_q)
    run_case(dtype, 128, H, kvh, hd, [77, 20, 300], [1, 2, 4, 8], kv_len, n_q, seed=1)
    run_case(dtype, 32, H, kvh, hd, [3000], [0, 10], kv_len, n_q, seed=2)


@pytest.mark.parametrize("dtype", TYPES)
def test_groups_counted_on_the_device(dtype):
    """A few groups of few rows before long prefixes: the division is found by the kernels themselves."""
    for plen, gs in (([4000, 100, 2500], [0, 40, 41, 44]), ([5000, 4000], [0, 22, 44]), ([3000, 3000, 3000, 3000], [0, 20, 20, 21, 43])):
        run_case(dtype, 16, 28, 4, 128, plen, gs, [1 + 7 * i for i in range(44)], [1] * 44)


@pytest.mark.parametrize("dtype", TYPES)
def test_more_groups_and_requests_than_a_warp(dtype):
    sizes = [1 + (5 * i) % 4 for i in range(41)]
    gs = [0] + np.cumsum(sizes).tolist()
    n = gs[-1] + 3
    kv_len = [(11 * i) % 70 for i in range(n)]
    n_q = [min(1, x) for x in kv_len]
    run_case(dtype, 16, 14, 2, 64, [(97 * i) % 400 for i in range(41)], gs, kv_len, n_q)
    n_q[70], kv_len[70] = 300, 333                      # a prompt behind many single tokens
    run_case(dtype, 32, 8, 4, 128, [(97 * i) % 400 for i in range(41)], gs, kv_len, n_q)
    n = 130                                             # a group whose own requests are counted warp by warp
    n_q = [1] * 100 + [40] + [1] * 29
    run_case(dtype, 16, 7, 1, 64, [2100], [0, n], [x + i for i, x in enumerate(n_q)], n_q)

@pytest.mark.parametrize("dtype", TYPES)
def test_prompts_behind_a_prefix(dtype):
    run_case(dtype, 64, 8, 2, 128, [1500], [0, 3], [400, 90, 1000], [400, 90, 300])
    run_case(dtype, 16, 14, 2, 64, [513], [0, 1], [700], [700])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,kvh,hd,plen,gs,kv_len,n_q", [
    (28, 4, 128, [500, 90], [0, 2, 3], [300, 129, 260, 9, 0], [300, 129, 131, 1, 0]),
    (14, 2, 64, [700], [0, 3], [600, 500, 77], [600, 401, 77]),
    (9, 3, 64, [33, 2000], [1, 2, 4], [900, 5, 700, 31], [900, 7, 700, 31])])
def test_turns_of_many_rows(dtype, H, kvh, hd, plen, gs, kv_len, n_q):
    """So many rows that the join takes two at a time; in place, and rows past the last request's stay."""
    q, kv, sc, ptable, table, q_start = inputs(dtype, 16, H, kvh, hd, plen, kv_len, n_q)
    buf = torch.full((len(q) + 37, H, hd), 9.0, dtype=dtype, device=DEV)
    buf[:len(q)] = q
    rest = [ptable, plen, gs, table, q_start, kv_len]
    o, lse = call(buf, kv, sc, *rest, out=buf)
    assert (o[len(q):] == 9).all()
    t.close(o[:len(q)], lse[:len(q)], reference(q, kv, sc, *rest, hd ** -0.5), dtype, dtype != torch.float32)

@pytest.mark.parametrize("dtype", TYPES)
def test_more_queries_than_own_positions(dtype):
    """Queries before the first own position see the prefix alone, and nothing where there is none."""
    o, lse = run_case(dtype, 16, 14, 2, 64, [40], [0, 2], [5, 0, 3], [9, 3, 6])
    assert (lse[12:15] == -math.inf).all() and (o[12:15] == 0).all() and (lse[:12] > -math.inf).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_far_apart(dtype):
    run_case(dtype, 16, 4, 2, 64, [400, 300], [0, 2, 3], [100, 30, 20], [1, 15, 1], spread=3.0, scale=0.004)
    run_case(dtype, 16, 4, 2, 128, [900], [0, 90], [20] * 90, [1] * 90, spread=3.0, scale=0.004)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,p,n_q", [(6, 1000, 1), (50, 3000, 1), (4, 700, 60)])
def test_strides_in_place_and_rows_of_nobody(dtype, n, p, n_q):
    H, kvh, hd = 14, 2, 64
    kv_len = [n_q + 5 * i for i in range(n)]
    q, kv, sc, ptable, table, q_start = inputs(dtype, 16, H, kvh, hd, [p], kv_len, [n_q] * n)
    want, want_lse = call(q, kv, sc, ptable, [p], [0, n], table, q_start, kv_len)
    rest = [ptable, [p], [0, n], table, q_start, kv_len]
    z = q.clone()
    got, lse = call(z, kv, sc, *rest, out=z)
    assert got is z and torch.equal(z, want) and torch.equal(lse, want_lse)
    buf = torch.zeros(len(q) + 3, H + 2 * kvh, hd + 1, dtype=dtype, device=DEV)     # odd starts, rows past the last request's
    buf[:len(q), :H, 1:] = q
    out = torch.full((len(q) + 3, H + 3, hd + 3), 9.0, dtype=dtype, device=DEV)
    got, lse = call(buf[:, :H, 1:], kv, sc, *rest, out=out[:, 2:2 + H, 3:])
    assert torch.equal(got[:len(q)], want) and torch.equal(lse[:len(q)], want_lse)
    assert (out[len(q):] == 9).all() and (out[:, :2] == 9).all() and (out[:, 2 + H:] == 9).all() and (out[..., :3] == 9).all()
    # fewer queries than a request has: the others are not computed
    if n_q > 1:
        out = torch.full_like(q, 9.0)
        got, _ = call(q, kv, sc, *rest, max_q=n_q - 1, out=out)
        last = torch.arange(len(q), device=DEV) % n_q == n_q - 1
        assert (got[last] == 9).all()
        assert float((got[~last].double() - want[~last].double()).abs().max()) <= 2.0**-7 * float(want.double().abs().max())


@pytest.mark.parametrize("n,p,n_q", [(5, 900, 1), (4, 1500, 70)])
def test_pages_and_rows_more_than_32_bits_apart(n, p, n_q):
    """The same pages at the far end of a large cache, the same rows far apart: the same bits."""
    kv_len = [n_q + 50 * i for i in range(n)]
    q, kv, sc, ptable, table, q_start = inputs(torch.bfloat16, 128, 28, 4, 128, [p], kv_len, [n_q] * n)
    want, want_lse = call(q, kv, sc, ptable, [p], [0, n], table, q_start, kv_len)
    off = 2**32 // kv[0].numel()
    big = torch.empty((off + len(kv),) + kv.shape[1:], dtype=torch.int8, device=DEV)
    far_sc = torch.full((off + len(kv),) + sc.shape[1:], math.nan, device=DEV)
    big[off:], far_sc[off:] = kv, sc
    shift = lambda t: torch.where(t >= 0, t + off, t)
    rest = [shift(ptable), [p], [0, n], shift(table), q_start, kv_len]
    got, lse = call(q, big, far_sc, *rest)
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    row = 2**31 // (len(q) - 1) + 64
    far = torch.empty(row * len(q), dtype=torch.bfloat16, device=DEV).as_strided(q.shape, (row, 128, 1))
    far.copy_(q)
    call(far, big, far_sc, *rest, out=far)
    assert torch.equal(far, want)

@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_as_attention_over_tables_that_name_the_prefix(dtype):
    """A prefix that ends with its page can also stand in every request's table. Two computations of the tolerance each."""
    kv_len = [30, 1, 200, 64]
    q, kv, sc, ptable, table, q_start = inputs(dtype, 32, 14, 2, 64, [320], kv_len, [1, 1, 7, 64])
    got, lse = call(q, kv, sc, ptable, [320], [0, 4], table, q_start, kv_len)
    whole = torch.cat([ptable.expand(4, -1), table], 1).contiguous()
    want, want_lse = t.attend(q, kv, sc, whole, q_start, [320 + n for n in kv_len])
    v = 127 * float(torch.nan_to_num(sc).max())
    eps = torch.finfo(dtype).eps
    assert float((got.double() - want.double()).abs().max()) <= v * (eps + 2.0**-14 + (2.0**-10 if dtype is torch.bfloat16 else 0))
    assert float((lse - want_lse).abs().max()) <= 2.0**-13


@pytest.mark.parametrize("dtype", TYPES)
def test_numbers_without_sense(dtype):
    """Starts that decrease or lie outside, negative lengths, lengths beyond the tables: clamped. What groups that overlap give is one of
    their prefixes'; nothing outside is touched (which the rows of the other requests show)."""
    kv_len, plen = [30, 10, 50, 20], [100, 90]
    q, kv, sc, ptable, table, q_start = inputs(dtype, 16, 14, 2, 64, plen, kv_len, [1] * 4)
    args = (q, kv, sc, ptable)
    want, _ = call(*args, plen, [0, 2, 4], table, q_start, kv_len)
    alone, _ = call(*args, [0, 0], [0, 2, 4], table, q_start, kv_len)
    got, _ = call(*args, plen, [-7, 2, 2**31 - 1], table, q_start, kv_len)
    assert torch.equal(got, want)
    got, _ = call(*args, [-3, 90], [0, 2, 4], table, q_start, kv_len)
    assert torch.equal(got[2:], want[2:]) and float((got[:2].double() - alone[:2].double()).abs().max()) < 0.02
    got, _ = call(*args, plen, [4, 2, 0], table, q_start, kv_len)
    assert float((got.double() - alone.double()).abs().max()) < 0.02
    for gs in ([0, 4, 1], [3, 0, 4], [0, 3, 2]):
        call(*args, plen, gs, table, q_start, kv_len)
    call(*args, plen, [0, 2, 4], table, [0, 3, 1, 4, 2], kv_len, max_q=3)
    got, _ = call(*args, [2**31 - 1, 90], [0, 2, 4], table, q_start, kv_len, max_prefix=112)
    assert torch.equal(got[2:], want[2:])
    torch.cuda.synchronize()


def test_no_groups_no_columns_and_nothing_to_do():
    q, kv, sc, ptable, table, q_start = inputs(torch.float32, 16, 14, 2, 64, [64], [30, 10], [1, 1])
    want, want_lse = t.attend(q, kv, sc, table, q_start, [30, 10])
    for plen, gs, pt in (([], [0], ptable[:0]), ([9], [0, 2], ptable[:, :0]), ([0], [0, 2], ptable)):
        got, lse = call(q, kv, sc, pt, plen, gs, table, q_start, [30, 10])
        assert float((got - want).abs().max()) <= 2.0**-18 * 127 * float(torch.nan_to_num(sc).max())
        assert float((lse - want_lse).abs().max()) <= 2.0**-17
    out, _ = call(q[:0], kv, sc, ptable, [64], [0, 0], table[:0], [0], [])
    assert out.shape == (0, 14, 64)
    # only prefixes: no position of their own
    got, _ = call(q, kv, sc, ptable, [64], [0, 2], table[:, :0], q_start, [0, 0])
    two = ptable.expand(2, -1).contiguous()
    want, _ = t.attend(q, kv, sc, two, q_start, [64, 64])
    assert float((got - want).abs().max()) <= 2.0**-18 * 127 * float(torch.nan_to_num(sc).max())


@pytest.mark.parametrize("n,p,n_q", [(6, 1000, 1), (60, 3000, 1), (5, 700, 100)])
def test_streams_and_graphs(n, p, n_q):
    kv_len = [n_q + 5 * i for i in range(n)]
    q, kv, sc, ptable, table, q_start = inputs(torch.bfloat16, 16, 28, 4, 128, [p], kv_len, [n_q] * n)
    plen, gs, start, lens = i32([p]), i32([0, n]), i32(q_start), i32(kv_len)
    go = lambda: t.kv8().prefix_attention(q, kv, sc, ptable, plen, gs, table, start, lens, n_q, max(kv_len), p)
    want = go()
    for _ in range(20):
        assert torch.equal(go(), want)
    sides = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(10):
        for s in sides:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append(go())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = go()
    plen.sub_(17)
    lens.sub_(n_q - 1 if n_q == 1 else 0)
    for _ in range(3):
        g.replay()
    assert torch.equal(got, go())
    t.kv8()._lib.check_ops()
