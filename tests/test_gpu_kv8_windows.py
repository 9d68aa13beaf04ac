"""Windows at the ends of their range: one, and as long as an int32 goes ("no limit"), with queries before the first position."""
import pytest
import torch

import test_gpu_kv8 as t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 3, 2**31 - 300, 2**30, 1])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv_len,n_q", [([5], [9]), ([5, 0, 100], [9, 3, 140]), ([700, 20], [1, 1]), ([5, 3000], [300, 400])])
def test_windows(window, hd, kv_len, n_q):
    """Few rows and prompts (a high max_kv sends them there), the first queries of some before position 0."""
    for kw in ({}, {"max_kv": 20000}):
        o, lse = t.run_case(torch.float32, 16, 14, 2, hd, kv_len, n_q, window=window, **kw)
        if window > 2**20:
            o0, lse0 = t.run_case(torch.float32, 16, 14, 2, hd, kv_len, n_q, **kw)
            assert torch.allclose(o, o0, atol=1e-4) and torch.allclose(lse, lse0, atol=1e-4)
