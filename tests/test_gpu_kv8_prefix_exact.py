"""How exact kv8.prefix_attention is against the formula in 64 bits, beyond the tolerance of each case."""
import pytest
import torch

import test_gpu_kv8 as t
import test_gpu_kv8_prefix as p

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("n,prefix,n_q", [(90, 4097, 1), (4, 1500, 60), (6, 300, 1)])
def test_16_bit_outputs_are_the_rounding_of_a_float32_computation(dtype, H, kvh, hd, n, prefix, n_q):
    """An output that is off by e before its rounding lies a step beside the exact one's rounding with the chance e / step. Weights of 22
    bits and float32 scores and sums: e is below 2^-16 of the standard deviation s of a row's outputs (test_gpu_kv8_sums.py). Those are
    spread around 0; of them 0.8 2^-i at most lie between s 2^-i and s 2^(1-i), where the step is s 2^-i eps / 2 at least: 1.6 2^-16 / eps of
    all are beside it for each such octave down to s 2^-16 / eps, as many at most among those above s, and half as many below the last. bfloat16 (eps
    2^-7): 9 + 1 + 1/2 times 0.31%, 3.3%; float16 (eps 2^-10): 6 + 1 + 1/2 times 2.5%, 19%. Weights of 11 bits, e = 2^-12 / sqrt(3) s, put some
    6% and 40% there."""
    kv_len = [n_q + (37 * i) % 90 for i in range(n)]
    q, kv, sc, ptable, table, q_start = p.inputs(dtype, 16, H, kvh, hd, [prefix], kv_len, [n_q] * n)
    out, _ = p.call(q, kv, sc, ptable, [prefix], [0, n], table, q_start, kv_len)
    want = p.reference(q, kv, sc, ptable, [prefix], [0, n], table, q_start, kv_len, hd ** -0.5)[0]
    beside = float((out != want.to(dtype)).double().mean())
    assert beside < (0.033 if dtype is torch.bfloat16 else 0.19), beside
