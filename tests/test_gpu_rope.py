"""rope.rotate against complex multiplication in 64 bits: layouts, part of the head, far positions, strides, in place."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rope():
    from e2e_browser_voice_agent_b200 import rope as m
    return m


def want_of(x, position, f, interleaved, magnitude=1.0):
    r = 2 * len(f)
    part = x[..., :r].double()
    z = part.unflatten(-1, (-1, 2)) if interleaved else part.unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_complex(z.contiguous())
    u = torch.outer(position[: x.shape[0]].double(), f)
    z = z * torch.polar(torch.full_like(u, magnitude), u)[:, None]
    z = torch.view_as_real(z)
    z = (z if interleaved else z.transpose(-1, -2)).flatten(-2)
    return torch.where((position[: x.shape[0]] >= 0)[:, None, None], torch.cat([z, x[..., r:].double()], -1), x.double())


def near(got, want, x, position, f, magnitude=1.0):
    """Cosine and sine are off by the rounding of the angle to float32 turns (2^-25 of a turn of at most a half: 2^-26 turns, 2 pi of that
    in radians), by the function (2^-23) and by the product with the magnitude (2^-24); the 64-bit product that makes the turns is off by
    2^-52 of them. Each of the two products and their sum rounds once more (2^-24): in all below 2^-21 plus the far term of |a| + |b| <=
    1.5 times the pair's larger, then the output's rounding."""
    far = 2 * math.pi * float(position.clamp(min=0).max()) * float(f.abs().max()) / (2 * math.pi) * 2.0**-51
    size = float(x.abs().max()) * 1.5 * abs(magnitude)
    half_step = torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs()
    assert (off <= size * (2.0**-21 + far) + want.abs() * half_step + torch.finfo(got.dtype).tiny).all(), float(off.max())


def case(tokens, heads, kv_heads, hd, dtype, far=5000, seed=0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + tokens + hd)
    q, k = (torch.randn(tokens, h, hd, generator=gen, device=DEV).to(dtype) for h in (heads, kv_heads))
    position = torch.randint(0, far, (tokens,), generator=gen, device=DEV).int()
    return q, k, position


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,hd,rotary", [
    (1, 14, 2, 64, 64), (1, 1, 1, 2, 2), (7, 4, 2, 64, 32), (33, 28, 4, 128, 128), (5, 3, 1, 80, 80), (5, 3, 1, 96, 24), (3, 2, 1, 65, 10),
    (2, 1, 1, 1024, 1024), (1000, 7, 1, 64, 64), (301, 2, 2, 128, 2), (4, 5, 1, 20, 6)])
def test_layouts(dtype, interleaved, tokens, heads, kv_heads, hd, rotary):
    q, k, position = case(tokens, heads, kv_heads, hd, dtype)
    f = rope().frequencies(rotary, 1e6)
    gq, gk = rope().rotate(q, position, f, k=k, interleaved=interleaved)
    for got, x in ((gq, q), (gk, k)):
        near(got, want_of(x, position, f, interleaved), x, position, f)
        assert torch.equal(got[..., rotary:], x[..., rotary:])
    assert torch.equal(rope().rotate(q, position, f, interleaved=interleaved), gq)
    z, y = q.clone(), k.clone()
    a, b = rope().rotate(z, position, f, k=y, interleaved=interleaved, out=z, k_out=y)
    assert a is z and b is y and torch.equal(z, gq) and torch.equal(y, gk)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv_heads,hd,rotary", [
    (1, 200, 9, 64, 64), (3, 65, 0, 128, 96), (40, 71, 3, 16, 16), (2, 130, 130, 8, 4), (300, 5, 2, 1024, 512), (3000, 14, 2, 64, 64),
    (2400, 3, 1, 66, 66), (1, 65536, 1, 16, 16)])
def test_heads_shared_out_among_warps(dtype, interleaved, tokens, heads, kv_heads, hd, rotary):
    q, k, position = case(tokens, heads, kv_heads, hd, dtype, seed=7)
    f = rope().frequencies(rotary, 1e4)
    position[tokens // 2] = -1
    gq, gk = rope().rotate(q, position, f, k=k, interleaved=interleaved)
    for got, x in ((gq, q), (gk, k)):
        if x.numel():
            near(got, want_of(x, position, f, interleaved), x, position, f)
        assert torch.equal(got[..., rotary:], x[..., rotary:]) and torch.equal(got[tokens // 2], x[tokens // 2])
    rope().rotate(q, position, f, k=k, interleaved=interleaved, out=q, k_out=k)
    assert torch.equal(q, gq) and torch.equal(k, gk)

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_slices_of_a_product(dtype, interleaved):
    """q, k and v as columns of one buffer, at any start, turned in place: nothing else is touched."""
    heads, kvh, hd, tokens = 6, 2, 64, 19
    f = rope().frequencies(32)
    for at, more in ((0, 0), (8, 8), (1, 3)):
        width = (heads + 2 * kvh) * hd
        gen = torch.Generator(device=DEV)
        gen.manual_seed(at)
        buf = torch.randn(tokens, width + at + more, generator=gen, device=DEV).to(dtype)
        keep = buf.clone()
        cut = lambda b, i, j: b[:, at + i * hd:at + j * hd].unflatten(1, (-1, hd))
        position = torch.arange(100, 100 + tokens, dtype=torch.int32, device=DEV)
        q, k = cut(buf, 0, heads), cut(buf, heads, heads + kvh)
        wq, wk = rope().rotate(cut(keep, 0, heads).contiguous(), position, f, k=cut(keep, heads, heads + kvh).contiguous(),
                               interleaved=interleaved)
        rope().rotate(q, position, f, k=k, interleaved=interleaved, out=q, k_out=k)
        assert torch.equal(q, wq) and torch.equal(k, wk)
        buf[:, at:at + (heads + kvh) * hd] = keep[:, at:at + (heads + kvh) * hd]
        assert torch.equal(buf, keep)
        # heads outermost
        t = cut(keep, 0, heads).transpose(0, 1).contiguous().transpose(0, 1)
        got = rope().rotate(t, position, f, interleaved=interleaved, out=torch.empty_like(t))
        assert torch.equal(got, wq)


@pytest.mark.parametrize("interleaved", [False, True])
def test_tokens_and_heads_more_than_32_bits_apart(interleaved):
    far = 2**31 + 64
    q, _, position = case(2, 3, 1, 64, torch.bfloat16)
    f = rope().frequencies(64)
    want = rope().rotate(q, position, f, interleaved=interleaved)
    buf = torch.empty(2 * far + 1024, dtype=torch.bfloat16, device=DEV)
    for shape, strides in (((2, 3, 64), (far, 64, 1)), ((2, 3, 64), (64, far, 1))):
        x = buf.as_strided(shape, strides)
        x.copy_(q)
        assert torch.equal(rope().rotate(x, position, f, interleaved=interleaved), want)
        rope().rotate(x, position, f, interleaved=interleaved, out=x)
        assert torch.equal(x, want)

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_far_positions(dtype):
    q, k, _ = case(6, 2, 1, 128, dtype)
    position = torch.tensor([0, 1, 131071, 10_000_000, 2**31 - 1, 2**24 + 1], dtype=torch.int32, device=DEV)
    f = rope().frequencies(128, 1e4)
    got, _ = rope().rotate(q, position, f, k=k)
    for t in range(6):
        near(got[t:t + 1], want_of(q[t:t + 1], position[t:t + 1], f, False), q, position[t:t + 1], f)
    assert torch.equal(got[0], q[0])


def test_tokens_without_a_position_and_more_positions_than_tokens():
    q, k, position = case(9, 4, 2, 64, torch.float32)
    position[3] = -1
    position[8] = -2**31
    f = rope().frequencies(64)
    more = torch.cat([position, position])
    gq, gk = rope().rotate(q, more, f, k=k, magnitude=1.5)
    for got, x in ((gq, q), (gk, k)):
        assert torch.equal(got[3], x[3]) and torch.equal(got[8], x[8])
        near(got, want_of(x, position, f, False, 1.5), x, position, f, 1.5)
    z = q.clone()
    rope().rotate(z, more, f, out=z, magnitude=1.5)
    assert torch.equal(z, gq)


def test_numbers_that_are_none_stay_in_their_pair():
    q, _, position = case(3, 2, 1, 64, torch.float32)
    q[1, 0, 5] = math.nan
    q[2, 1, 40] = math.inf
    got = rope().rotate(q, position, rope().frequencies(64))
    bad = ~torch.isfinite(got)
    assert bad[1, 0, [5, 37]].all() and bad[2, 1, [8, 40]].all() and int(bad.sum()) == 4


def test_frequencies():
    m = rope()
    plain = m.frequencies(64, 1e4, device="cpu")
    assert plain.dtype is torch.float64 and torch.allclose(plain, 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32), rtol=1e-14)
    assert torch.equal(m.frequencies(64, 1e4, "linear", 4.0, device="cpu"), plain / 4)
    ntk = m.frequencies(64, 1e4, "ntk", 4.0, device="cpu")
    assert ntk[0] == 1 and torch.allclose(ntk[-1], plain[-1] / 4, rtol=1e-12)
    yarn = m.frequencies(64, 1e4, "yarn", 4.0, original=4096, device="cpu")
    turns = plain * 4096 / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], plain[turns >= 32]) and torch.allclose(yarn[turns <= 1], plain[turns <= 1] / 4, rtol=1e-14)
    mid = (turns < 32) & (turns > 1)
    assert mid.any() and (yarn[mid] < plain[mid]).all() and (yarn[mid] > plain[mid] / 4).all()
    assert m.yarn_magnitude(1.0) == 1 and abs(m.yarn_magnitude(4.0) - (0.1 * math.log(4) + 1)) < 1e-15


def test_streams_graphs_and_nothing_to_do():
    q, k, position = case(50, 14, 2, 64, torch.bfloat16)
    f = rope().frequencies(64, 1e6)
    want = rope().rotate(q, position, f, k=k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rope().rotate(q, position, f, k=k)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = rope().rotate(q, position, f, k=k)
    position.add_(11)
    g.replay()
    want = rope().rotate(q, position, f, k=k)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert rope().rotate(q[:0], position, f).shape == (0, 14, 64)
    only, _ = rope().rotate(q, position, f, k=k[:, :0])
    assert torch.equal(only, want[0])
