"""Attention over the paged 8-bit cache: short prompts through both of its kernels.

Calls that visit few keys take the kernel for few rows, whatever their queries; max_kv is a bound, so a loose one sends the same
call to the kernel for prompts. The cases of test_gpu_kv8 (with its inputs, references and tolerances) that are small enough for
the first kernel run here on the second; and the other way round, long ones with a low bound.
"""
import pytest
import torch

import test_gpu_kv8 as t

pytestmark = pytest.mark.gpu
FEW = {64: 32, 128: 16}              # rows of a request (queries x heads of a kv head) that always take the first kernel
VISITS = {64: 1 << 19, 128: 1 << 17}  # (row tiles of 8) x keys that still take it


@pytest.fixture
def prompts(monkeypatch):
    """max_kv raised until the kernel for prompts takes the call; how many calls that was."""
    whole, n = t.kv8().attention, [0]

    def attention(q, kv, kv_scale, block_table, q_start, kv_len, max_q, max_kv, **kw):
        kvh, hd = kv.shape[2], kv.shape[4]
        rows = max_q * (q.shape[1] // kvh)
        if rows > FEW[hd] and kv_len.shape[0]:
            tiles = -(-rows // 8) * kv_len.shape[0] * kvh
            if not kw.get("window"):
                max_kv = max(max_kv, VISITS[hd] // tiles + 1)
                n[0] += 1
        return whole(q, kv, kv_scale, block_table, q_start, kv_len, max_q, max_kv, **kw)

    monkeypatch.setattr(t.kv8(), "attention", attention)
    return n


@pytest.mark.parametrize("dtype", t.TYPES)
@pytest.mark.parametrize("n", [5, 17, 33, 127, 128, 129, 255, 256, 300])
def test_prompt_lengths(prompts, dtype, n):
    t.test_prompt_lengths(dtype, n)
    assert prompts[0] == 2


@pytest.mark.parametrize("dtype", t.TYPES)
def test_continuations(prompts, dtype):
    """A few queries after histories of odd lengths: most rows of the kernel's tiles hold nothing."""
    for hd in (64, 128):
        t.run_case(dtype, 16, 14, 2, hd, [641], [6])
        t.run_case(dtype, 64, 28, 4, hd, [1000, 77, 0, 130], [9, 1, 0, 40])
    assert prompts[0] == 4


@pytest.mark.parametrize("dtype", t.TYPES)
@pytest.mark.parametrize("layout", ["slice", "odd"])
def test_strides(prompts, dtype, layout):
    t.run_case(dtype, 32, 14, 2, 64, [70, 5, 300], [1, 5, 130], layout=layout)
    t.run_case(dtype, 16, 28, 4, 128, [70, 5, 300], [1, 5, 130], layout=layout)
    t.run_case(dtype, 16, 28, 4, 128, [200], [11], layout=layout)
    assert prompts[0] == 3


@pytest.mark.parametrize("dtype", t.TYPES)
def test_masks_and_scales(prompts, dtype):
    t.test_more_queries_than_keys(dtype)
    t.test_scales_far_apart(dtype)
    t.test_queries_of_extreme_magnitude(dtype)
    assert prompts[0] >= 5


def test_what_is_no_number(prompts):
    t.test_zero_scales()
    t.test_a_query_that_is_no_number_stays_alone(70)
    gen = torch.Generator(device=t.DEV)
    gen.manual_seed(3)
    kv, sc, table = t.make_cache(gen, [200, 200], 16, 2, 64)
    sc2 = sc.clone()
    sc2[int(table[0, 2]), 1, 1] = float("nan")
    q = torch.randn(140, 4, 64, device=t.DEV)
    good, _ = t.attend(q, kv, sc, table, [0, 70, 140], [200, 200])
    o, _ = t.attend(q, kv, sc2, table, [0, 70, 140], [200, 200])
    assert o[:70, 2:].isnan().all() and torch.equal(o[:70, :2], good[:70, :2]) and torch.equal(o[70:], good[70:])
    assert prompts[0] >= 4


def test_rows_of_no_request_are_left_alone(prompts):
    t.test_rows_of_no_request_are_left_alone()
    assert prompts[0] == 1


@pytest.mark.parametrize("dtype", t.TYPES)
def test_long_prompts_through_the_kernel_for_few_rows(dtype):
    """The other way round: a bound below the real length costs time only."""
    for hd in (64, 128):
        t.run_case(dtype, 16, 14, 2, hd, [1000], [300], max_kv=200)
        t.run_case(dtype, 64, 4, 2, hd, [800, 3, 129], [200, 3, 129], max_kv=100, window=70)


@pytest.mark.parametrize("dtype", t.TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128), (7, 1, 128)])
@pytest.mark.parametrize("singles", [1, 20, 130])
def test_chunks_beside_single_tokens(dtype, H, kvh, hd, singles):
    """A few row tiles over long histories among many requests: their spans are counted on the device (up to 128 requests)."""
    lens, n_q = [1 + 37 * i % 500 for i in range(singles)], [1] * singles
    t.run_case(dtype, 16, H, kvh, hd, lens[:1] + [2500] + lens[1:], n_q[:1] + [130] + n_q[1:])
    t.run_case(dtype, 64, H, kvh, hd, lens + [0, 1800, 1500], n_q + [0, 60, 200], window=900 if hd == 64 else 0)


def test_float32_sums_over_many_keys():
    """64 wide, float32: no sum in the tensor cores takes more than 4 tiles of 64 keys, 32 additions that each cut off less than
    2^-23 of it, so the output is off by less than 2^-18 of its size whatever the length."""
    for kv_len, n_q in (([4000], [60]), ([3000, 4000], [300, 500])):
        gen = torch.Generator(device=t.DEV)
        gen.manual_seed(8)
        kv, sc, table = t.make_cache(gen, kv_len, 16, 2, 64)
        q = torch.randn(sum(n_q), 14, 64, generator=gen, device=t.DEV)
        q_start = [0, n_q[0], sum(n_q)][: len(n_q) + 1]
        o, _ = t.attend(q, kv, sc, table, q_start, kv_len)
        want = t.ref_attention(q, kv, sc, table, q_start, kv_len, 0.125, 0)[0]
        assert float((o.double() - want).norm() / want.norm()) < 2.0**-18
