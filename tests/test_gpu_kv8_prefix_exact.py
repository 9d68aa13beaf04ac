"""How exact kv8.prefix_attention is against the formula in 64 bits, beyond the tolerance of each case."""
import pytest
import torch

import test_gpu_kv8 as t
import test_gpu_kv8_prefix as p
import test_gpu_kv8_sums as sums

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


def long_case(dtype, H, kvh, hd, prefix, n, own, n_q, spread, seed=0, page=64):
    """q, a cache whose values have a mean (so that what a sum loses shows), one prefix, requests of `own` positions behind it."""
    gen = torch.Generator(device=t.DEV)
    gen.manual_seed(seed + prefix + hd + n)
    have = [-(-x // page) for x in [prefix] + [own] * n]
    pages = sum(have)
    kv = torch.randn(pages, 2, kvh, page, hd, generator=gen, device=t.DEV).mul_(34).round_().clamp_(-127, 127).to(torch.int8)
    kv[:, 1] = kv[:, 1].div(2, rounding_mode="floor") + 40
    sc = 0.03 * torch.exp(0.3 * torch.randn(pages, 2, kvh, generator=gen, device=t.DEV))
    order = torch.randperm(pages, generator=gen, device=t.DEV).int()
    q = (torch.randn(n * n_q, H, hd, generator=gen, device=t.DEV) * spread).to(dtype)
    return q, kv, sc, order[None, :have[0]].contiguous(), order[have[0]:].view(n, -1).contiguous()


def long_reference(q, kv, sc, ptable, table, prefix, own, n_q, heads):
    """64-bit outputs of some heads of the first and the last request, and those requests."""
    H, kvh, hd = q.shape[1], kv.shape[2], q.shape[2]
    held = lambda pages: kv[pages.long()].double() * sc[pages.long()].double()[..., None, None]
    shared = held(ptable[0])
    some = sorted({0, len(table) - 1})
    want = torch.empty(len(some), n_q, len(heads), hd, dtype=torch.float64, device=t.DEV)
    for i, r in enumerate(some):
        mine = held(table[r])
        for j, h in enumerate(heads):
            cut = lambda x, w, n: x[:, w, h // (H // kvh)].reshape(-1, hd)[:n]
            k, v = (torch.cat([cut(shared, w, prefix), cut(mine, w, own)]) for w in (0, 1))
            x = q[r * n_q:(r + 1) * n_q, h].double() @ k.t() * hd ** -0.5
            hidden = torch.arange(prefix + own, device=t.DEV) > prefix + own - n_q + torch.arange(n_q, device=t.DEV)[:, None]
            want[i, :, j] = torch.softmax(x.masked_fill(hidden, -torch.inf), 1) @ v
    return want, some


@pytest.mark.parametrize("dtype", p.TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128)])
@pytest.mark.parametrize("prefix,n,own,n_q", [(16385, 256, 40, 1), (16385, 5, 600, 300), (40001, 80, 9, 1), (131072, 3, 50, 1), (131072, 30, 50, 20),
                                              (70000, 24, 700, 200)])
def test_sums_behind_long_prefixes(dtype, H, kvh, hd, prefix, n, own, n_q):
    """As test_gpu_kv8_sums.py has it for one history: float32 by the bound of the kernel that keeps sums in the tensor cores for up to 8 tiles
    of keys, 16-bit types by the rounding of the exact output, from which they do not shrink by 2^-15 or more. Of N outputs a share f (as above, 3.3%
    and 19%) may lie a step, eps of themselves at most, beside that rounding, above or below it by chance, which moves their sum by eps
    sqrt(f / N) of itself (4 outputs of 384 by 4e-5); four times that is allowed beside the 2^-15."""
    for spread in (0.1, 2.0):
        q, kv, sc, ptable, table = long_case(dtype, H, kvh, hd, prefix, n, own, n_q, spread)
        out, _ = p.call(q, kv, sc, ptable, [prefix], [0, n], table, list(range(0, n * n_q + 1, n_q)), [own] * n)
        heads = sorted({0, H // 2, H - 1})
        want, some = long_reference(q, kv, sc, ptable, table, prefix, own, n_q, heads)
        got = torch.stack([out[r * n_q:(r + 1) * n_q, heads] for r in some])
        if dtype is torch.float32:
            assert sums.off(got, want) < (sums.prompt_bound(hd, prefix + own) if spread < 1 else 2.0**-16)
        else:
            exact = want.to(dtype)
            assert sums.off(got, want) < 1.02 * sums.off(exact, want)
            lost = float(((got.double() - exact.double()) * want).sum() / (want * want).sum())
            chance = torch.finfo(dtype).eps * ((0.033 if dtype is torch.bfloat16 else 0.19) / want.numel()) ** 0.5
            assert abs(lost) < 2.0**-15 + 4 * chance


@pytest.mark.parametrize("dtype", p.TYPES)
def test_streams_whose_sums_go_through_the_workspace(dtype):
    """Both passes of a call and calls on several streams at once, all with sums too long for the tensor cores: 128 wide, row tiles of more keys
    than are kept there in prefixes (many rows) and in requests' own positions. The same bits as one after another."""
    calls = []
    for i, (prefix, n, own, n_q) in enumerate(((9000, 40, 300, 40), (20000, 2, 9000, 300), (600, 3, 20000, 200))):
        q, kv, sc, ptable, table = long_case(dtype, 28, 4, 128, prefix, n, own, n_q, 0.5, seed=i)
        args = (ptable, p.i32([prefix]), p.i32([0, n]), table, p.i32(list(range(0, n * n_q + 1, n_q))), p.i32([own] * n), n_q, own, prefix)
        calls.append(lambda q=q, kv=kv, sc=sc, args=args: t.kv8().prefix_attention(q, kv, sc, *args, return_lse=True))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(6):
        for s, c, g in zip(streams, calls, got):
            with torch.cuda.stream(s):
                g.append(c())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(o, w[0]) and torch.equal(l, w[1]) for o, l in g)
    # and replayed together from two graphs
    graphs = []
    for c in calls[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = c()
        graphs.append((g, o))
    for _ in range(4):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, o), w in zip(graphs, want):
        assert torch.equal(o[0], w[0]) and torch.equal(o[1], w[1])
    t.kv8()._lib.check_ops()
