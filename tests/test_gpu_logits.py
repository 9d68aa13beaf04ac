"""logits.adjust against the formula: counts, biases, masks, types and strides. The formula is single float32 operations, so what is
wanted is the formula's bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def adjust(*a, **kw):
    from e2e_browser_voice_agent_b200 import logits
    return logits.adjust(*a, **kw)


def formula(x, tokens=None, length=None, repetition=None, presence=None, frequency=None, bias_id=None, bias=None, allowed=None):
    """On the host, in 64 bits, each operation rounded to float32 as the formula says."""
    f32 = lambda v: v.float().double()
    cpu = lambda t: None if t is None else t.cpu()
    kind, x = x.dtype, x.cpu().double()
    rows, vocab = x.shape
    ones = torch.ones(rows)
    rep, pres, freq = (ones * d if s is None else cpu(s) for s, d in ((repetition, 1.0), (presence, 0.0), (frequency, 0.0)))
    for r in range(rows):
        if tokens is not None:
            n = max(0, min(int(length[r]), tokens.shape[1]))
            said = cpu(tokens)[r, :n].long()
            said = said[(said >= 0) & (said < vocab)]
            c = torch.bincount(said, minlength=vocab).double()
            y = torch.where(x[r] > 0, f32(x[r] / rep[r].double()), f32(x[r] * rep[r].double()))
            y = f32(y - f32(f32(freq[r].double() * c) + pres[r].double()))
            x[r] = torch.where(c > 0, y, x[r])
        if bias_id is not None:
            sums = {}
            for i, b in zip(bias_id[r].tolist(), bias[r].cpu()):
                if 0 <= i < vocab:
                    sums[i] = b.double() if i not in sums else f32(sums[i] + b.double())
            for i, b in sums.items():
                x[r, i] = f32(x[r, i] + b)
        if allowed is not None:
            i = torch.arange(vocab)
            x[r] = torch.where((cpu(allowed)[r][i // 32].long() >> (i % 32)) % 2 == 1, x[r], -math.inf)
    return x.float().to(kind)


def same(got, want):
    got, want = got.cpu(), want.cpu()
    assert got.dtype is want.dtype and torch.equal(got.isnan(), want.isnan())
    assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))


def inputs(rows, vocab, columns, dtype, n_bias=0, mask=None, seed=0):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + rows + vocab + (columns or 0))
    rand = lambda *s: torch.rand(*s, generator=gen, device=DEV)
    a = {"logits": (4 * torch.randn(rows, vocab, generator=gen, device=DEV)).to(dtype)}
    if columns is not None:
        a["tokens"] = (rand(rows, columns) ** 3 * vocab).int()
        a["length"] = (rand(rows) * (columns + 1)).int()
        a["repetition"], a["presence"], a["frequency"] = 0.8 + 0.6 * rand(rows), rand(rows) - 0.2, 0.4 * rand(rows)
    if n_bias:
        a["bias_id"] = (rand(rows, n_bias) * (vocab + 2)).int() - 1     # -1, the same twice, and one past the end among them
        a["bias"] = 5 * torch.randn(rows, n_bias, generator=gen, device=DEV)
    if mask is not None:
        bits = torch.randint(-2**31, 2**31, (rows, (vocab + 31) // 32), generator=gen, device=DEV)
        for _ in range(mask):
            bits &= torch.randint(-2**31, 2**31, bits.shape, generator=gen, device=DEV)
        a["allowed"] = bits.int()
    return a


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,columns,n_bias,mask", [
    (1, 1, 1, 1, 0), (1, 151936, 641, 5, 3), (3, 2048, 0, 0, None), (3, 2048, 50, 0, None), (2, 1000, None, 7, None), (2, 1001, None, 0, 1),
    (5, 33, 200, 40, 0), (4, 32768 + 77, 3000, 300, 1), (2, 5000, 70000, 3, 0), (40, 40000, 100, 2, None), (2, 3000, 30, 1024, 0),
    (600, 1500, 20, 3, 0), (20, 50, None, 0, None)])
def test_formula(dtype, rows, vocab, columns, n_bias, mask):
    a = inputs(rows, vocab, columns, dtype, n_bias, mask)
    want = formula(a["logits"], **{k: v for k, v in a.items() if k != "logits"})
    got = adjust(**a)
    same(got, want)
    assert got.data_ptr() != a["logits"].data_ptr()
    x = a["logits"].clone()
    assert adjust(**{**a, "logits": x}, out=x) is x
    same(x, want)


@pytest.mark.parametrize("only", ["repetition", "presence", "frequency"])
def test_one_penalty_alone(only):
    a = inputs(3, 500, 60, torch.float32)
    a = {k: v for k, v in a.items() if k in ("logits", "tokens", "length", only)}
    same(adjust(**a), formula(a["logits"], **{k: v for k, v in a.items() if k != "logits"}))
    a.pop(only)
    same(adjust(**a), a["logits"])


@pytest.mark.parametrize("dtype", TYPES)
def test_strong_and_weak_penalties(dtype):
    """Logits of all magnitudes over and times strengths of all: single float32 operations, as the host's."""
    some = [0.0, 1e-45, 1e-30, 2.0**-21, 2.0**-20, 0.3, 1 / 3, 0.9999999, 1.0, 1.0000001, 1.3, 3.0, 7.0, 2.0**20, 2.0**21, 1e30, math.inf, -1.3, -math.inf]
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    x = torch.exp2(torch.randint(-149, 128, (len(some), 40000), generator=gen, device=DEV).double())
    x = (x * (1 + torch.rand(x.shape, generator=gen, device=DEV))).float()
    x[:, 20000:] = torch.exp2(8 * torch.rand(len(some), 20000, generator=gen, device=DEV) - 4)
    x[:, ::7] *= -1
    x = x.to(dtype)
    rep = torch.tensor(some, device=DEV)
    tokens = torch.arange(40000, device=DEV).int().expand(len(some), -1)
    got = adjust(x, tokens=tokens, length=torch.full((len(some),), 40000, device=DEV).int(), repetition=rep)
    y, r = x.cpu().float(), rep.cpu()[:, None]
    same(got, torch.where(y > 0, y / r, y * r).sub(torch.zeros(1)).to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,columns,n_bias", [(3, 40000, 9000, 5), (300, 2100, 9000, 3), (2, 3000, 70001, 1024), (450, 4000, 10, 1024)])
def test_long_histories_and_long_lists_in_place(dtype, rows, vocab, columns, n_bias):
    a = inputs(rows, vocab, columns, dtype, n_bias, 0, seed=3)
    a["bias_id"][:, : n_bias // 2] %= 50
    a["tokens"][:, : columns // 2] %= 3
    a["length"][:] = columns
    want = formula(a["logits"], **{k: v for k, v in a.items() if k != "logits"})
    same(adjust(**a), want)
    adjust(**a, out=a["logits"])
    same(a["logits"], want)

@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_starts(dtype):
    a = inputs(5, 3001, 40, dtype, 6, 0)
    want = adjust(**a)
    for at, width in ((0, 3001), (0, 3008), (1, 3010), (8, 3040)):
        buf = torch.full((5, width + 9), 3.0, dtype=dtype, device=DEV)
        x = buf[:, at:at + 3001]
        x.copy_(a["logits"])
        y = torch.full((5, width + 5), 3.0, dtype=dtype, device=DEV)
        out = y[:, at:at + 3001]
        same(adjust(**{**a, "logits": x}, out=out), want)
        assert (y[:, :at] == 3).all() and (y[:, at + 3001:] == 3).all()
        adjust(**{**a, "logits": x}, out=x)
        same(x, want)
        assert (buf[:, :at] == 3).all() and (buf[:, at + 3001:] == 3).all()
    wide = torch.zeros(5, 99, dtype=torch.int32, device=DEV)       # lists that are columns of larger tables
    wide[:, 7:47] = a["tokens"]
    bits = torch.zeros(5, 200, dtype=torch.int32, device=DEV)
    bits[:, 3:97] = a["allowed"]
    same(adjust(**{**a, "tokens": wide[:, 7:47], "allowed": bits[:, 3:97]}), want)
    one = {**a, "tokens": a["tokens"][:1].expand(5, 40), "allowed": a["allowed"][:1].expand(5, -1)}   # shared by all rows
    same(adjust(**one), formula(a["logits"], **{k: v for k, v in one.items() if k != "logits"}))


def test_rows_more_than_32_bits_apart():
    far = 2**31 + 64
    a = inputs(2, 5000, 40, torch.bfloat16, 6, 0)
    want = adjust(**a)
    buf = torch.empty(far + 10048, dtype=torch.bfloat16, device=DEV)
    for at in (0, 1):
        x, y = buf[at:].as_strided((2, 5000), (far, 1)), buf[5024:].as_strided((2, 5000), (far, 1))
        x.copy_(a["logits"])
        adjust(**{**a, "logits": x}, out=y)
        same(y, want)
        adjust(**{**a, "logits": x}, out=x)
        same(x, want)

@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_and_tokens_without_sense(dtype):
    a = inputs(6, 400, 30, dtype)
    a["length"] = torch.tensor([0, -5, 31, 2**31 - 1, 1, 30], dtype=torch.int32, device=DEV)
    a["tokens"][2, 3], a["tokens"][2, 4], a["tokens"][2, 5] = -1, 400, -2**31
    a["tokens"][5] = 17
    want = formula(a["logits"], **{k: v for k, v in a.items() if k != "logits"})
    same(adjust(**a), want)
    assert torch.equal(adjust(**a)[:2], a["logits"][:2])


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_nan_and_rows_left_with_nothing(dtype):
    a = inputs(4, 300, 20, dtype, 4, 0)
    x = a["logits"]
    x[0, :40] = math.inf
    x[0, 40:80] = -math.inf
    x[1, :90] = math.nan
    x[1, 100:150] = torch.finfo(dtype).min
    a["allowed"][2] = 0
    a["tokens"][:2] = torch.arange(20, device=DEV) * 6
    a["bias"][3, 0] = -math.inf
    got = adjust(**a)
    same(got, formula(x, **{k: v for k, v in a.items() if k != "logits"}))
    assert (got[2] == -math.inf).all()


def test_streams_graphs_and_nothing_to_do():
    a = inputs(8, 5000, 100, torch.float32, 5, 0)
    want = adjust(**a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = adjust(**a)
    side.synchronize()
    same(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = adjust(**a)
    a["length"].clamp_(max=50)
    for _ in range(3):
        g.replay()
    same(got, adjust(**a))
    assert adjust(a["logits"][:0]).shape == (0, 5000)
    same(adjust(a["logits"]), a["logits"])
