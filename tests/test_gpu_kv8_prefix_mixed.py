"""kv8.prefix_attention on calls that mix many requests of a row with few of many, behind one prefix and behind many: the parts of all rows lie one
behind the other in the workspace."""
import math

import numpy as np
import pytest
import torch

import test_gpu_kv8 as t
import test_gpu_kv8_prefix as p

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", p.TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128)])
def test_single_tokens_beside_chunks(dtype, H, kvh, hd):
    n_q = [1] * 100 + [130] + [1] * 90 + [7, 0, 61] + [1] * 62
    kv_len = [n + (29 * i) % 300 for i, n in enumerate(n_q)]
    kv_len[100] = 900
    p.run_case(dtype, 16, H, kvh, hd, [1500], [0, 250], kv_len, n_q)
    p.run_case(dtype, 32, H, kvh, hd, [40, 1100, 0, 700, 300], [3, 90, 100, 103, 200, 230], kv_len, n_q, seed=1)


@pytest.mark.parametrize("dtype", p.TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128)])
def test_hundreds_of_groups(dtype, H, kvh, hd):
    sizes = [(7 * i) % 4 for i in range(150)] + [70] + [1] * 50
    gs = [0] + np.cumsum(sizes).tolist()
    n_q = [1 + 4 * (i % 11 == 0) + 40 * (i % 97 == 5) for i in range(gs[-1])]
    kv_len = [n + (13 * i) % 60 for i, n in enumerate(n_q)]
    p.run_case(dtype, 16, H, kvh, hd, [(101 * i) % 700 for i in range(201)], gs, kv_len, n_q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_starts_that_name_rows_many_times(dtype):
    """More rows than there are: what has no room in the workspace is not computed, rows of the first group and request are right, and
    nothing outside is touched."""
    n, each, P = 12, 40, 900
    kv_len = [each + 31 * i for i in range(n)]
    q, kv, sc, ptable, table, q_start = p.inputs(dtype, 16, 28, 4, 128, [P] * n, kv_len, [each] * n)
    want, _ = p.call(q, kv, sc, ptable, [P] * n, list(range(n + 1)), table, q_start, kv_len)
    ref = p.reference(q, kv, sc, ptable, [P] * n, [0] + [n] * n, table, q_start, kv_len, 128 ** -0.5)
    buf = torch.full((len(q) + 9, 28, 128), 9.0, dtype=dtype, device=p.DEV)
    for gs in ([0, n] * 6 + [n], [0] + [n, 0] * 6):  # every second group has all rows
        o, lse = p.call(q, kv, sc, ptable, [P] * n, gs, table, q_start, kv_len, out=buf[:len(q)])
        t.close(o, lse, ref, dtype, dtype != torch.float32)
    starts = [0, each * n] * 6 + [0]                 # every second request has all rows
    o, _ = p.call(q, kv, sc, ptable, [P] * n, list(range(n + 1)), table, starts, kv_len, out=buf[:len(q)], max_q=each * n)
    assert torch.isfinite(o.float()).all() and (buf[len(q):] == 9).all()
    got, _ = p.call(q, kv, sc, ptable, [P] * n, list(range(n + 1)), table, q_start, kv_len)
    assert torch.equal(got, want)
    t.kv8()._lib.check_ops()


@pytest.mark.parametrize("dtype", p.TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128), (8, 1, 128)])
@pytest.mark.parametrize("groups,n,P", [(8, 4, 640), (2, 3, 4096), (12, 3, 640), (3, 5, 1283)])
def test_groups_of_few_rows(dtype, H, kvh, hd, groups, n, P):
    kv_len = [1 + (23 * i) % 150 for i in range(groups * n)]
    plen = [P - 7 * g for g in range(groups)]
    p.run_case(dtype, 16, H, kvh, hd, plen, list(range(0, groups * n + 1, n)), kv_len, [1] * (groups * n))
    gs = [0, 1] + [n * g for g in range(2, groups)] + [groups * n]   # uneven: the first group has one, the second the others of two
    p.run_case(dtype, 32, H, kvh, hd, plen, gs, kv_len, [1] * (groups * n), seed=1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128)])
def test_a_replayed_graph_follows_lengths_groups_and_starts(dtype, H, kvh, hd):
    """Captured once with generous bounds; then own lengths, prefix lengths, groups, starts, tables and queries change in place between replays, so
    that rows go from one kernel to the other and from one group to another. Each replay has the bits of a fresh call with the same bounds."""
    n, rows, max_q, max_kv, max_prefix = 60, 420, 200, 400, 1600
    steps = [  # prefix lengths, groups, queries, own lengths
        ([1600, 300, 0], [0, 40, 50, 60], [7] * 60, [7 + 5 * i for i in range(60)]),
        ([1500, 1600, 70], [0, 5, 58, 60], [1] * 30 + [200] + [1] * 20 + [90] + [0] * 8, [1 + 3 * i for i in range(30)] + [400] + [60] * 20 + [95] + [4] * 8),
        ([16, 1, 1599], [10, 10, 11, 59], [3] * 20 + [0, 17, 130] + [2] * 37, [9 + (31 * i) % 300 for i in range(20)] + [0, 20, 390] + [5] * 37),
        ([0, 0, 0], [0, 0, 0, 0], [1] * 60, [1 + 6 * i for i in range(60)]),
        ([1600, 1600, 1600], [0, 20, 40, 60], [1] * 60, [0] * 60)]
    gen = torch.Generator(device=p.DEV)
    gen.manual_seed(hd)
    kv, sc, both = t.make_cache(gen, [max_prefix] * 3 + [max_kv] * n, 16, kvh, hd)
    ptable, table = both[:3].contiguous(), both[3:, :max_kv // 16].contiguous()
    q = torch.empty(rows, H, hd, dtype=dtype, device=p.DEV)
    plen, gs, start, lens = (torch.zeros(k, dtype=torch.int32, device=p.DEV) for k in (3, 4, n + 1, n))
    out = torch.zeros(rows, H, hd, dtype=dtype, device=p.DEV)
    go = lambda o: t.kv8().prefix_attention(q, kv, sc, ptable, plen, gs, table, start, lens, max_q, max_kv, max_prefix, out=o, return_lse=True)
    graph = torch.cuda.CUDAGraph()
    q.zero_()
    go(out)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _, lse = go(out)
    for i, (a, b, c, d) in enumerate(steps + steps[::-1]):
        assert sum(c) <= rows and max(c) <= max_q and max(d) <= max_kv and max(a) <= max_prefix
        starts = [0] + np.cumsum(c).tolist()
        q.copy_(torch.randn(q.shape, generator=gen, device=p.DEV))
        for x, y in ((plen, a), (gs, b), (start, starts), (lens, d)):
            x.copy_(p.i32(y))
        if i == len(steps):  # other pages of the same pool
            ptable.copy_(ptable.flip(0))
            table.copy_(table.flip(0))
        out.fill_(9.0)
        graph.replay()
        fresh = torch.full_like(out, 9.0)
        _, fresh_lse = go(fresh)
        used = starts[-1]
        assert torch.equal(out, fresh) and torch.equal(lse[:used], fresh_lse[:used]) and (out[used:] == 9).all()
        ref = p.reference(q, kv, sc, ptable, a, b, table, starts, d, hd ** -0.5)
        t.close(out[:used], lse[:used], [x[:used] for x in ref[:2]] + list(ref[2:]), dtype, dtype != torch.float32)
    t.kv8()._lib.check_ops()
