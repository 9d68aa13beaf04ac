"""How exact attention over the paged 8-bit cache is, relative to the output's size (2-norms), against the formula in 64 bits.

Values of V have a mean, so that the output's size is that of the sum over the keys and what a sum loses shows. With n the keys
of a row, in one span (a low max_kv makes k_att_rows take them so: 4 warps, and 4 lanes each that sum the weights):

* A sum of N terms of like size, each addition rounded to nearest, is off by some 2^-24 sqrt(N) / 3 of itself (the i-th addition
  rounds i / N of it). k_att_rows: 4 sums of n / 64 terms for the output, 16 of n / 16 for the weights, together 2^-24
  sqrt(2 n) / 48. Three times that is allowed.
* Weights of 22 bits, exponentials off by up to 2^-22 and float32 scores near 0: 2^-21 at most, less by averaging.
* Larger scores: with standard deviation 2 and 128 dimensions the sum of the products' magnitudes is about 14; queries of 22 bits
  and sums of up to 16 steps make a score off by less than 14 (2^-23 + 9 x 2^-24), which is 2^-17; twice that is allowed. (Queries of
  11 bits would give 2^-12 of it, some 1e-4.)
"""
import math

import pytest
import torch

import test_gpu_kv8 as t

pytestmark = pytest.mark.gpu
F32 = torch.float32


def attend(dtype, heads, kvh, hd, n, n_q, spread, page=64, seed=0, **kw):
    """(outputs, 64-bit outputs) of a few heads of one request of n positions whose last n_q are the queries; spread: the standard
    deviation of the scores."""
    gen = torch.Generator(device=t.DEV)
    gen.manual_seed(seed + n + hd + n_q)
    pages = -(-n // page)
    kv = torch.randn(pages, 2, kvh, page, hd, generator=gen, device=t.DEV).mul_(34).round_().clamp_(-127, 127).to(torch.int8)
    kv[:, 1] = kv[:, 1].div(2, rounding_mode="floor") + 40
    sc = 0.03 * torch.exp(0.3 * torch.randn(pages, 2, kvh, generator=gen, device=t.DEV))
    q = (torch.randn(n_q, heads, hd, generator=gen, device=t.DEV) * spread).to(dtype)
    table = torch.randperm(pages, generator=gen, device=t.DEV).int()[None]
    out, lse = t.attend(q, kv, sc, table, [0, n_q], [n], **kw)
    some = sorted({0, heads // 2, heads - 1})
    want = torch.empty(n_q, len(some), hd, dtype=torch.float64, device=t.DEV)
    held = kv[table[0].long()].double() * sc[table[0].long()].double()[..., None, None]
    key = torch.arange(n, device=t.DEV)
    for i, h in enumerate(some):
        k, v = (held[:, w, h // (heads // kvh)].reshape(-1, hd)[:n] for w in (0, 1))
        for a in range(0, n_q, 100):
            pos = n - n_q + torch.arange(a, min(n_q, a + 100), device=t.DEV)
            x = (q[a:a + 100, h].double() @ k.t() * hd ** -0.5).masked_fill(key > pos[:, None], -math.inf)
            want[a:a + 100, i] = torch.softmax(x, 1) @ v
            assert float((lse[a:a + 100, h].double() - torch.logsumexp(x, 1)).abs().max()) < 2.0**-17 * max(1, spread)
    return out[:, some], want


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


# ---------------------------------------------------------------------------------------------- the kernel for few rows

@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [300, 1000, 4000, 16000, 64000, 131072])
@pytest.mark.parametrize("n_q", [1, 10])
def test_few_rows_in_one_span(hd, n, n_q):
    got, want = attend(F32, 1, 1, hd, n, n_q, 0.1, max_kv=16)
    assert off(got, want) < 2.0**-21 + 2.0**-24 * math.sqrt(2 * n) / 16


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [700, 1900, 30000])
def test_few_rows_in_spans(hd, n):
    """A cluster's spans, and spans that a second kernel joins: the sums are shorter."""
    for heads, kvh, n_q in ((7, 1, 1), (1, 1, 10)):
        got, want = attend(F32, heads, kvh, hd, n, n_q, 0.1)
        assert off(got, want) < 2.0**-21 + 2.0**-24 * math.sqrt(2 * n) / 16


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kw", [{}, {"max_kv": 16}])
def test_few_rows_with_larger_scores(hd, kw):
    for n in (300, 5000):
        got, want = attend(F32, 2, 1, hd, n, 4, 2.0, **kw)
        assert off(got, want) < 2.0**-16


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
def test_few_16_bit_rows_are_rounded_once(dtype, hd):
    """The error is that of rounding the exact output (what is below 2^-18 before it adds to it in squares, and moves values
    across a rounding boundary as often one way as the other)."""
    for n in (300, 131072):
        got, want = attend(dtype, 7, 1, hd, n, 4, 0.1 if n > 1000 else 2.0, max_kv=16)
        assert off(got, want) < 1.02 * off(want.to(dtype), want)


# ---------------------------------------------------------------------------------------------- the kernel for prompts
#
# Its sums lie in the tensor cores for 4 tiles of 64 keys (64 wide) or 8 (128 wide), 8 additions a tile for float32: each cuts off
# less than 2^-23 of the sum, which grows evenly, so together less than F 2^-24 with F = 32 or 64. What is rounded: n / 16 additions
# of a row's weights and n / 256 or more of its output: 2^-24 sqrt(n) / 12 together, three times that allowed.

def prompt_bound(hd, n):
    return (32 if hd == 64 else 64) * 2.0**-24 + 2.0**-21 + 2.0**-24 * math.sqrt(n) / 4


def prompt_heads(hd):
    """Heads, kv heads and queries whose row tiles fill the SMs, so that a history is one span."""
    return (14, 2, 1400) if hd == 64 else (28, 4, 780)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [1500, 4000, 16000, 64000, 131072])
@pytest.mark.parametrize("kw", [{}, {"max_kv": 0}])
def test_prompts_in_one_span(hd, n, kw):
    heads, kvh, n_q = prompt_heads(hd)
    got, want = attend(F32, heads, kvh, hd, n, n_q, 0.1, **kw)
    assert off(got, want) < prompt_bound(hd, n)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n", [900, 20000, 131072])
def test_prompts_in_spans(hd, n):
    got, want = attend(F32, 14, 2, hd, n, 60, 0.1)
    assert off(got, want) < prompt_bound(hd, n)


@pytest.mark.parametrize("hd", [64, 128])
def test_prompts_with_larger_scores_and_a_window(hd):
    heads, kvh, n_q = prompt_heads(hd)
    got, want = attend(F32, heads, kvh, hd, 5000, n_q, 2.0)
    assert off(got, want) < 2.0**-16
    gen = torch.Generator(device=t.DEV)
    gen.manual_seed(3)
    t.run_case(F32, 16, heads, kvh, hd, [3000, 40], [n_q, 40], window=1100)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
def test_16_bit_prompts_are_rounded_once(dtype, hd):
    """As with few rows. Float16's weights have 22 bits, bfloat16's 11, which adds (1 / 8)^2 of the rounding's square: 1.008."""
    heads, kvh, n_q = prompt_heads(hd)
    for n, spread in ((1500, 2.0), (20000, 0.1), (131072, 0.1)):
        got, want = attend(dtype, heads, kvh, hd, n, n_q, spread)
        exact = want.to(dtype)
        assert off(got, want) < 1.02 * off(exact, want)
        # and does not shrink: 2^-15 of the output more than the rounding does
        lost = float(((got.double() - exact.double()) * want).sum() / (want * want).sum())
        assert abs(lost) < 2.0**-15


def test_sums_that_change_their_scale():
    """128 wide: keys whose scores rise along the history move the maximum between the sums that go to the workspace."""
    gen = torch.Generator(device=t.DEV)
    gen.manual_seed(4)
    n, n_q = 6000, 900
    kv, sc, table = t.make_cache(gen, [n], 64, 2, 128, spread=0.3)
    rise = torch.linspace(0.0, 3.0, table.shape[1], device=t.DEV).exp()
    sc[table[0].long(), 0] *= rise[:, None]
    for dtype in t.TYPES:
        q = torch.randn(n_q, 16, 128, generator=gen, device=t.DEV).mul(0.3).to(dtype)
        out, lse = t.attend(q, kv, sc, table, [0, n_q], [n])
        t.close(out, lse, t.ref_attention(q, kv, sc, table, [0, n_q], [n], 128 ** -0.5, 0), dtype, dtype != F32)


def test_two_streams_at_once():
    """Calls that run together keep their sums apart."""
    gen = torch.Generator(device=t.DEV)
    gen.manual_seed(5)
    calls = []
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=t.DEV)
    for n, n_q in ((9000, 300), (7000, 200)):
        kv, sc, table = t.make_cache(gen, [n], 64, 4, 128)
        q = torch.randn(n_q, 28, 128, generator=gen, device=t.DEV)
        args = (q, kv, sc, table, i32(0, n_q), i32(n), n_q, n)
        calls.append(lambda args=args: t.kv8().attention(*args))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for _ in range(10):
        for s, c, g in zip(streams, calls, got):
            with torch.cuda.stream(s):
                g.append(c())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)
    from e2e_browser_voice_agent_b200 import _lib
    _lib.check_ops()
