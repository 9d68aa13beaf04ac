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
