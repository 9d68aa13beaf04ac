"""Attention over the paged 8-bit cache: chunks of prompts among many single tokens, and on long histories."""
import pytest
import torch

import test_gpu_kv8 as t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", t.TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("singles", [131, 255, 1000])
def test_chunks_beside_many_single_tokens(dtype, H, kvh, hd, singles):
    """More requests than whose row tiles are counted on the device: the prompts' kernel finds its few tiles among them."""
    lens, n_q = [1 + 37 * i % 300 for i in range(singles)], [1] * singles
    t.run_case(dtype, 16, H, kvh, hd, lens[:9] + [700] + lens[9:] + [0, 410, 5000], n_q[:9] + [130] + n_q[9:] + [0, 60, 300])


@pytest.mark.parametrize("dtype", t.TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (7, 1, 128)])
def test_a_chunk_on_a_long_history_beside_single_tokens(dtype, H, kvh, hd):
    t.run_case(dtype, 64, H, kvh, hd, [50000, 9, 300, 20000], [70, 1, 1, 1])
    t.run_case(dtype, 64, H, kvh, hd, [9, 40000, 12000], [1, 40, 400], window=30000)
