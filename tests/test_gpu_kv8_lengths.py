"""Query ranges and lengths on the device that make no sense reach nothing outside the arrays: their rows stay as they were, and the
other requests are served."""
import pytest
import torch

import test_gpu_kv8 as t

pytestmark = pytest.mark.gpu
MOST = 2**31 - 1


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_q", [1, 150])
@pytest.mark.parametrize("before", [MOST, MOST - 5, 10**9])
@pytest.mark.parametrize("after,length", [(-MOST - 1, MOST), (-5, -7), (0, 0), (-10**9, 60)])
def test_ranges_without_sense(hd, n_q, before, after, length):
    """Of three requests the first and the last have ranges that end before they begin."""
    gen = torch.Generator(device=t.DEV)
    gen.manual_seed(hd + n_q)
    kv, sc, table = t.make_cache(gen, [60, 300, 60], 16, 2, hd)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=t.DEV)
    q = torch.randn(n_q + 4, 14, hd, generator=gen, device=t.DEV)
    ref = t.ref_attention(q[:n_q], kv, sc, table[1:2], [0, n_q], [300], hd ** -0.5, 0)
    for max_kv in (300, 20000):
        out = torch.full_like(q, 7.0)
        o, lse = t.kv8().attention(q, kv, sc, table, i32([before, 0, n_q, after]), i32([length, 300, length]), n_q, max_kv, out=out,
                                   return_lse=True)
        t.close(o[:n_q], lse[:n_q], ref, torch.float32, False)
        assert (o[n_q:] == 7).all()
