"""The operators of a serving step beside its cache and its products, and cases that measure them.

Four operators, each with a plain form in elementary torch operations and the call a user makes of this package:

  norm      the residual's addition, the root-mean-square norm and the 8-bit codes that the next product takes (int8.norm), and the
            values that these stand for (int8.values)
  rope      rotary positions of a step's queries and keys (rope.rotate)
  prefix    grouped-query attention of requests that share a long prefix, whose keys are read once for all of them
            (kv8.prefix_attention)
  logits    penalties for repeated tokens, biases and masks of allowed tokens on a step's logits (logits.adjust)
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one session's token between two products of the 0.5B model: latency
        {"name": "norm decode 1", "op": "norm", "rows": 1, "k": 896, "dtype": "f32", "residual": "f32"},
        # a 32-session step of the 7B model
        {"name": "norm decode 32", "op": "norm", "rows": 32, "k": 3584, "dtype": "bf16", "residual": "bf16"},
        # prompts of several sessions, the residual stream kept in 32 bits: bandwidth
        {"name": "norm prompts 16k", "op": "norm", "rows": 16392, "k": 3584, "dtype": "bf16", "residual": "f32"},
        # one token's queries and keys, far into a session (0.5B heads)
        {"name": "rope decode 1", "op": "rope", "tokens": 1, "sessions": 1, "far": 4000, "heads": 14, "kv_heads": 2, "head_dim": 64,
         "rotary": 64, "interleaved": False, "base": 1e6, "factor": 1.0, "magnitude": 1.0, "dtype": "f32"},
        # prompts of 24 sessions (7B heads), positions stretched for long contexts: bandwidth
        {"name": "rope prompts 16k", "op": "rope", "tokens": 16392, "sessions": 24, "far": 100000, "heads": 28, "kv_heads": 4,
         "head_dim": 128, "rotary": 128, "interleaved": False, "base": 1e6, "factor": 4.0, "magnitude": 1.1386, "dtype": "bf16"},
        # a layout of interleaved pairs in the first half of each head
        {"name": "rope interleaved 2050", "op": "rope", "tokens": 2050, "sessions": 3, "far": 2000, "heads": 16, "kv_heads": 4,
         "head_dim": 128, "rotary": 64, "interleaved": True, "base": 1e4, "factor": 1.0, "magnitude": 1.0, "dtype": "f16"},
        # four sessions behind one system prompt (0.5B heads, float32 activations as the engine has them): latency
        {"name": "prefix decode 4", "op": "prefix", "requests": 4, "groups": 1, "loose": 0, "prefix_lo": 641, "prefix_hi": 641, "page": 16,
         "heads": 14, "kv_heads": 2, "head_dim": 64, "lo": 20, "hi": 200, "new": 1, "dtype": "f32"},
        # a step of 256 sessions behind one long prompt (7B heads)
        {"name": "prefix decode 256", "op": "prefix", "requests": 256, "groups": 1, "loose": 0, "prefix_lo": 16385, "prefix_hi": 16385,
         "page": 64, "heads": 28, "kv_heads": 4, "head_dim": 128, "lo": 16, "hi": 2000, "new": 1, "dtype": "bf16"},
        # sessions of three prompts, and some without one, that bring whole turns
        {"name": "prefix turns 3 groups", "op": "prefix", "requests": 26, "groups": 3, "loose": 2, "prefix_lo": 500, "prefix_hi": 4099,
         "page": 16, "heads": 28, "kv_heads": 4, "head_dim": 128, "lo": 40, "hi": 800, "new": 63, "dtype": "f16"},
        # one session's logits, float32, with what was said so far
        {"name": "logits 1", "op": "logits", "rows": 1, "vocab": 151936, "columns": 4096, "lo": 641, "hi": 641, "biases": 5,
         "mask": True, "dtype": "f32"},
        # a 32-session step over the 7B vocabulary
        {"name": "logits 32", "op": "logits", "rows": 32, "vocab": 152064, "columns": 4096, "lo": 100, "hi": 4000, "biases": 16,
         "mask": True, "dtype": "f32"},
        # many sessions with long histories, 16-bit logits: bandwidth
        {"name": "logits 256 long", "op": "logits", "rows": 256, "vocab": 152064, "columns": 16384, "lo": 1000, "hi": 16384, "biases": 64,
         "mask": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rope", "prefix", "prefix", "logits"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "norm":
        k = rng.choice([896, 3584, 1152, _log(rng, 3, 8000)])
        return {"op": op, "rows": _log(rng, 1, 16392 * 3584 // max(3584, k * SIZE[dtype] // 2)), "k": k, "dtype": dtype,
                "residual": rng.choice(["", dtype, "f32"])}
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (28, 4, 128), (4, 2, 64), (7, 1, 64), (16, 4, 128), (4, 2, 128)])
    if op == "rope":
        return {"op": op, "tokens": _log(rng, 1, 8000), "sessions": rng.randint(1, 30), "far": _log(rng, 10, 131072), "heads": heads,
                "kv_heads": kv_heads, "head_dim": dim, "rotary": rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                "interleaved": rng.random() < 0.5, "base": rng.choice([1e4, 1e6, 5e5]), "factor": rng.choice([1.0, 4.0, 8.5]),
                "magnitude": rng.choice([1.0, 1.1386]), "dtype": dtype}
    if op == "logits":
        columns = _log(rng, 1, 16384)
        vocab = rng.choice([151936, 152064, 2048, _log(rng, 33, 100000)])
        return {"op": op, "rows": _log(rng, 1, 120), "vocab": vocab, "columns": columns, "lo": columns // 20, "hi": columns,
                "biases": rng.choice([0, min(vocab, _log(rng, 1, 300))]), "mask": rng.random() < 0.5, "dtype": dtype}
    page = rng.choice([16, 32, 64, 128])
    if rng.random() < 0.6:
        requests, new = _log(rng, 1, 200), 1
        prefix = _log(rng, 10, 16000)
        hi = _log(rng, 10, 2000)
    else:  # turns of some tokens
        requests, new = _log(rng, 1, 24), _log(rng, 2, 48)
        prefix = _log(rng, 10, 3000)
        hi = _log(rng, 10, 600)
    groups = rng.randint(1, min(4, requests))
    return {"op": op, "requests": requests, "groups": groups, "loose": rng.choice([0, 0, min(2, requests - groups)]),
            "prefix_lo": max(1, prefix // 4), "prefix_hi": prefix, "page": page, "heads": heads, "kv_heads": kv_heads, "head_dim": dim,
            "lo": max(1, hi // 20), "hi": hi, "new": new, "dtype": dtype}


def _spread(lo, hi, n, salt):
    """n lengths from lo to hi, spread over their logarithm: by the case alone, so that work() knows them too."""
    r = random.Random("%s %s %s %s" % (lo, hi, n, salt))
    got = [int(round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1 for _ in range(n)]
    got[r.randrange(n)] = hi
    return [min(hi, max(lo, g)) for g in got]


def _pages(n, page):
    return -(-n // page)


def _prefix_lengths(case):
    """Each group's prefix and first request, then each request's own tokens and its new ones among them."""
    prefix = _spread(case["prefix_lo"], case["prefix_hi"], case["groups"], "prefix")
    shared = case["requests"] - case["loose"]
    r = random.Random("groups %s %s" % (shared, case["groups"]))
    cuts = sorted(r.sample(range(1, shared), case["groups"] - 1)) if case["groups"] > 1 else []
    kv = _spread(case["lo"], case["hi"], case["requests"], "own")
    return prefix, [0] + cuts + [shared], kv, [min(n, case["new"]) for n in kv]


# ---------------------------------------------------------------------------------------------- inputs

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return {"norm": _prepare_norm, "rope": _prepare_rope, "prefix": _prepare_prefix, "logits": _prepare_logits}[case["op"]](case, gen)


def _prepare_norm(case, gen):
    rows, k = case["rows"], case["k"]
    x = 0.3 * torch.randn(rows, k, generator=gen, device=DEV)
    # a residual stream: its size differs from token to token, and a few channels lie far above the others
    res = torch.randn(rows, k, generator=gen, device=DEV) * torch.exp(torch.randn(rows, 1, generator=gen, device=DEV))
    res[:, ::max(1, k // 7)] *= 9
    weight = 1 + 0.3 * torch.randn(k, generator=gen, device=DEV)
    if not case["residual"]:
        x, res = x + res, None
    return {"case": case, "x": x.to(DTYPE[case["dtype"]]), "weight": weight,
            "residual": None if res is None else res.to(DTYPE[case["residual"]])}


def _frequencies(case):
    """Radians per position of each pair of dimensions, the slow ones stretched by the factor."""
    half = case["rotary"] // 2
    f = case["base"] ** (-np.arange(half, dtype=np.float64) * 2 / case["rotary"])
    part = np.clip((f * 8192 / (2 * math.pi) - 1) / 31, 0, 1)  # turns within 8192 positions: below 1 stretched, above 32 as they are
    return f * part + f / case["factor"] * (1 - part)


def _prepare_rope(case, gen):
    t, width = case["tokens"], (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
    # queries and keys as a QKV product leaves them: slices of one row per token
    qkv = torch.randn(t, width, generator=gen, device=DEV).to(DTYPE[case["dtype"]])
    q, k, _ = qkv.split([case["heads"] * case["head_dim"]] + [case["kv_heads"] * case["head_dim"]] * 2, 1)
    # each session's new tokens are consecutive positions from where it stands
    start = torch.randint(0, case["far"], (case["sessions"],), generator=gen, device=DEV)
    each = -(-t // case["sessions"])
    at = torch.arange(t, device=DEV)
    position = (start[at // each] + at % each).int()
    return {"case": case, "q": q.view(t, case["heads"], -1), "k": k.view(t, case["kv_heads"], -1), "position": position,
            "frequency": torch.from_numpy(_frequencies(case)).to(DEV)}


def _codes(gen, *shape):
    """8-bit codes as a cache of normal values holds them: the largest of a block near 127."""
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)
    return x.mul_(34).round_().clamp_(-127, 127).to(torch.int8)


def _prepare_prefix(case, gen):
    page, kvh, hd, heads = case["page"], case["kv_heads"], case["head_dim"], case["heads"]
    prefix, group_start, kv_len, new = _prefix_lengths(case)
    have = [_pages(n, page) for n in prefix + kv_len]
    n_pages = sum(have) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)  # pages spread over the pool at random
    first = np.cumsum([0] + have)

    def tables(a, b):
        col = torch.arange(max(have[a:b]), device=DEV)[None, :]
        at = (_ints(first[a:b].tolist(), torch.int64)[:, None] + col).clamp(max=n_pages - 1)
        return torch.where(col < _ints(have[a:b])[:, None], order[at], torch.full_like(order[at], -1)).contiguous()

    scale = torch.exp(0.3 * torch.randn(n_pages, 2, kvh, generator=gen, device=DEV)) * 0.03
    q = torch.randn(sum(new), heads, hd, generator=gen, device=DEV) * 1.7
    g = len(prefix)
    return {"case": case, "q": q.to(DTYPE[case["dtype"]]), "kv": _codes(gen, n_pages, 2, kvh, page, hd), "scale": scale,
            "prefix_table": tables(0, g), "table": tables(g, len(have)), "prefix_len": _ints(prefix), "group_start": _ints(group_start),
            "q_start": _ints(np.cumsum([0] + new).tolist()), "kv_len": _ints(kv_len), "max_q": max(new), "max_kv": max(kv_len),
            "max_prefix": max(prefix)}


def _prepare_logits(case, gen):
    rows, vocab, cols = case["rows"], case["vocab"], case["columns"]
    x = 3 * torch.randn(rows, vocab, generator=gen, device=DEV)
    # what was said: a few hundred tokens of a vocabulary come again and again
    u = torch.rand(rows, cols, generator=gen, device=DEV)
    said = (u ** 4 * vocab).int().clamp(max=vocab - 1)
    length = _ints(_spread(case["lo"], case["hi"], rows, "said"))
    ids = bias = allowed = None
    if case["biases"]:
        ids = torch.rand(rows, vocab, generator=gen, device=DEV).argsort(1)[:, :case["biases"]].int().contiguous()
        bias = 4 * torch.randn(rows, case["biases"], generator=gen, device=DEV)
        bias[:, 0] = -100.0                                        # (a token that is as good as forbidden)
        ids[:, -1] = torch.where(torch.arange(rows, device=DEV) % 3 == 0, -1, ids[:, -1])  # lists of different lengths
    if case["mask"]:  # a grammar's next tokens: some hundred, or nearly all; a row without a grammar allows all
        words = -(-vocab // 32)
        few = torch.rand(rows, vocab, generator=gen, device=DEV) < torch.tensor([0.002, 0.97, 1.0], device=DEV)[
            torch.arange(rows, device=DEV) % 3][:, None]
        bits = torch.zeros(rows, words * 32, dtype=torch.bool, device=DEV)
        bits[:, :vocab] = few
        packed = (bits.view(rows, words, 32).long() << torch.arange(32, device=DEV)).sum(-1)
        allowed = torch.where(packed >= 2**31, packed - 2**32, packed).int()
    strength = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=gen, device=DEV)
    return {"case": case, "logits": x.to(DTYPE[case["dtype"]]), "tokens": said, "length": length, "repetition": strength(1.0, 1.3),
            "presence": strength(0.0, 0.6), "frequency": strength(0.0, 0.3), "bias_id": ids, "bias": bias, "allowed": allowed}


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "rope": _own_rope, "prefix": _own_prefix, "logits": _own_logits}[op](state)
    return {"norm": _plain_norm, "rope": _plain_rope, "prefix": _plain_prefix, "logits": _plain_logits}[op](state)


def _own_norm(s):
    from e2e_browser_voice_agent_b200 import int8
    n = int8.norm(s["x"], s["weight"], EPS, residual=s["residual"])
    return {"values": int8.values(n.codes, n.scale, s["case"]["k"], dtype=s["x"].dtype), "scale": n.scale, "sum": n.sum}


def _own_rope(s):
    from e2e_browser_voice_agent_b200 import rope
    q, k = rope.rotate(s["q"], s["position"], s["frequency"], k=s["k"], interleaved=s["case"]["interleaved"],
                       magnitude=s["case"]["magnitude"])
    return {"q": q, "k": k}


def _own_prefix(s):
    from e2e_browser_voice_agent_b200 import kv8
    out, lse = kv8.prefix_attention(s["q"], s["kv"], s["scale"], s["prefix_table"], s["prefix_len"], s["group_start"], s["table"],
                                    s["q_start"], s["kv_len"], s["max_q"], s["max_kv"], s["max_prefix"], return_lse=True)
    return {"out": out, "lse": lse}


def _own_logits(s):
    from e2e_browser_voice_agent_b200 import logits
    return {"logits": logits.adjust(s["logits"], tokens=s["tokens"], length=s["length"], repetition=s["repetition"],
                                    presence=s["presence"], frequency=s["frequency"], bias_id=s["bias_id"], bias=s["bias"],
                                    allowed=s["allowed"])}


def _plain_norm(s):
    x, res = s["x"].float(), s["residual"]
    total = None
    if res is not None:
        total = (x + res.float()).to(res.dtype)
        x = total.float()
    r = (1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).float()  # (codes lie next to borders: 64 bits up to here)
    y = x * r * s["weight"]
    amax = y.abs().amax(-1, keepdim=True)
    most = torch.full_like(amax, 127)                            # (a tensor: a number would be divided by approximately)
    inv = torch.where(amax > 0, (most / amax).clamp(max=3.4028234663852886e38), 0.0)
    scale = (amax / most)[:, 0]
    return {"values": (torch.round(y * inv) * scale[:, None]).to(s["x"].dtype), "scale": scale, "sum": total}


def _plain_rope(s):
    c = s["case"]
    half, rotary = c["rotary"] // 2, c["rotary"]
    angle = s["position"].double()[:, None] * s["frequency"]       # (float32 does not hold far positions' angles)
    cos, sin = ((f(angle) * c["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        y = x.clone()
        if c["interleaved"]:
            a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
            y[..., 0:rotary:2], y[..., 1:rotary:2] = a * cos - b * sin, b * cos + a * sin
        else:
            a, b = x[..., :half], x[..., half:rotary]
            y[..., :half], y[..., half:rotary] = a * cos - b * sin, b * cos + a * sin
        out[name] = y.to(s[name].dtype)
    return out


def _plain_prefix(s):
    c, q = s["case"], s["q"]
    page, heads, kvh, hd = c["page"], c["heads"], c["kv_heads"], c["head_dim"]
    group, t = heads // kvh, torch.arange(q.shape[0], device=DEV)

    def cache(table):  # [tables][kv heads][positions][dim] of K and of V
        kv = s["kv"][table.long().clamp(min=0)].float() * s["scale"][table.long().clamp(min=0)][..., None, None]
        return (kv[:, :, i].permute(0, 2, 1, 3, 4).reshape(table.shape[0], kvh, -1, hd) for i in (0, 1))

    def scores(k, first, count, most):  # of the rows first .. first + count, padded to `most`, with their own table's keys
        rows = (first[:, None] + torch.arange(most, device=DEV)).clamp(max=q.shape[0] - 1)
        qp = q[rows].float().reshape(len(first), most, kvh, group, hd).permute(0, 2, 3, 1, 4).reshape(len(first), kvh, -1, hd)
        return (qp @ k.transpose(-1, -2)).mul_(1 / math.sqrt(hd)).reshape(len(first), kvh, group, most, -1)

    start, kv_len, gs = s["q_start"].long(), s["kv_len"].long(), s["group_start"].long()
    count = start[1:] - start[:-1]
    g_first = start[gs[:-1]]
    g_count = start[gs[1:]] - g_first
    r = torch.searchsorted(start[1:], t, right=True)                                     # each row's request
    g = torch.searchsorted(gs[1:], r, right=True)                                        # and its group
    inside = g < c["groups"]
    g = g.clamp(max=c["groups"] - 1)
    most = sum(_prefix_lengths(c)[3][: c["requests"] - c["loose"]])                      # rows of a group at most
    pk, pv = cache(s["prefix_table"])
    ok, ov = cache(s["table"])
    i, j = t - start[r], (t - g_first[g]).clamp(max=most - 1)
    xp = scores(pk, g_first, g_count, most)[g, :, :, j]                                  # [rows][kv heads][group][prefix]
    xo = scores(ok, start[:-1], count, s["max_q"])[r, :, :, i]                           # [rows][kv heads][group][own]
    pos = kv_len[r] - count[r] + i
    xp.masked_fill_(~((torch.arange(xp.shape[-1], device=DEV) < s["prefix_len"][g][:, None]) & inside[:, None])[:, None, None], -math.inf)
    xo.masked_fill_((torch.arange(xo.shape[-1], device=DEV) > pos[:, None])[:, None, None], -math.inf)
    top = torch.maximum(xp.amax(-1, keepdim=True), xo.amax(-1, keepdim=True))
    base = torch.where(top == -math.inf, 0.0, top)
    xp, xo = xp.sub_(base).exp_(), xo.sub_(base).exp_()
    total = xp.sum(-1, keepdim=True) + xo.sum(-1, keepdim=True)

    def product(x, v, of, at, most):  # weights of each row with its own table's values, by tables again
        w = torch.zeros(v.shape[0], most, kvh, group, v.shape[2], device=DEV)
        w[of, at] = x
        w = w.permute(0, 2, 3, 1, 4).reshape(v.shape[0], kvh, -1, v.shape[2])
        return (w @ v).reshape(v.shape[0], kvh, group, most, hd)[of, :, :, at]

    xp = xp * inside[:, None, None, None]
    o = product(xp, pv, g, torch.where(inside, j, most), most + 1) + product(xo, ov, r, i, s["max_q"])
    lse = (top + torch.log(total))[..., 0].reshape(-1, heads)
    return {"out": (o / torch.where(total == 0, 1.0, total)).reshape(-1, heads, hd).to(q.dtype), "lse": lse}


def _plain_logits(s):
    x = s["logits"].float()
    vocab = s["case"]["vocab"]
    live = torch.arange(s["tokens"].shape[1], device=DEV) < s["length"][:, None]
    count = torch.zeros_like(x).scatter_add_(1, s["tokens"].long(), live.float())
    said = count > 0
    rep, pres, freq = (s[n][:, None] for n in ("repetition", "presence", "frequency"))
    x = torch.where(said, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(said, x - (freq * count + pres), x)
    if s["bias"] is not None:
        ids = s["bias_id"].long()
        x = x + torch.zeros_like(x).scatter_add_(1, ids.clamp(min=0), torch.where(ids >= 0, s["bias"], 0.0))
    if s["allowed"] is not None:
        at = torch.arange(vocab, device=DEV)
        x = torch.where((s["allowed"][:, at // 32] >> (at % 32)) & 1 == 1, x, -math.inf)
    return {"logits": x.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------------------------- needs

def work(case):
    """Bytes and operations that one pass cannot do without: inputs read once, outputs written once."""
    op, size = case["op"], SIZE[case["dtype"]]
    if op == "norm":
        rows, k = case["rows"], case["k"]
        # (the codes are written and, for the values, read)
        return {"bytes": rows * k * (2 * size + (2 * SIZE[case["residual"]] if case["residual"] else 0)) + rows * (_pages(k, 16) * 32 + 8) + 4 * k,
                "flops": 0}
    if op == "rope":
        return {"bytes": case["tokens"] * ((case["heads"] + case["kv_heads"]) * case["head_dim"] * 2 * size + 4), "flops": 0}
    if op == "logits":
        rows, vocab = case["rows"], case["vocab"]
        said = sum(_spread(case["lo"], case["hi"], rows, "said"))
        return {"bytes": rows * vocab * 2 * size + 4 * said + rows * (8 * case["biases"] + 16 + (_pages(vocab, 32) * 4 if case["mask"] else 0)),
                "flops": 0}
    prefix, group_start, kv_len, new = _prefix_lengths(case)
    heads, kvh, hd, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    keys, rows = sum(prefix) + sum(kv_len), sum(new)
    pairs = sum(n * q - q * (q - 1) // 2 for n, q in zip(kv_len, new))
    pairs += sum(p * sum(new[a:b]) for p, a, b in zip(prefix, group_start, group_start[1:]))
    return {"bytes": keys * 2 * kvh * hd + (keys // page + 1) * (8 * kvh + 4) + rows * heads * (2 * hd * size + 4),
            "flops": 4 * pairs * heads * hd}


# ---------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """What run() returns, from the definition in 64 bits."""
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rope": _exact_rope, "prefix": _exact_prefix, "logits": _exact_logits}[case["op"]](s)


def _exact_norm(s):
    """The definition rounds to float32 after each operation on a value: a code at the border between two goes by that."""
    def f32(v):
        return v.to(torch.float32).to(torch.float64)
    x, total = s["x"].to(torch.float64), None
    if s["residual"] is not None:
        total = f32(s["residual"].to(torch.float64) + x)
        x = total.to(s["residual"].dtype).to(torch.float64)
        total = x
    power = torch.einsum("rk,rk->r", x, x) / x.shape[1]
    y = f32(f32(x * f32((power + EPS) ** -0.5)[:, None]) * s["weight"].to(torch.float64))
    top = y.abs().max(1).values
    scale = f32(top / 127)
    codes = torch.round(f32(y * f32(127 / top)[:, None]))
    return {"values": codes * scale[:, None], "scale": scale, "sum": total}


def _exact_rope(s):
    c = s["case"]
    rotary = c["rotary"]
    turn = torch.polar(torch.full_like(s["frequency"], c["magnitude"]).expand(len(s["position"]), -1).contiguous(),
                       torch.outer(s["position"].to(torch.float64), s["frequency"]))[:, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].to(torch.float64)
        part = x[..., :rotary]
        pairs = part.unflatten(-1, (-1, 2)) if c["interleaved"] else part.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z if c["interleaved"] else z.transpose(-1, -2)
        out[name] = torch.cat([z.flatten(-2), x[..., rotary:]], -1)
    return out


def _exact_prefix(s):
    c, q = s["case"], s["q"]
    page, kvh = c["page"], c["kv_heads"]
    group = c["heads"] // kvh
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    start, kv_len, gs, plen = (s[n].tolist() for n in ("q_start", "kv_len", "group_start", "prefix_len"))

    def held(table, n):  # K and V of n positions, [2][kv heads][n][dim]
        pages = table[: _pages(n, page)].long()
        x = s["kv"][pages].double() * s["scale"][pages].double()[..., None, None]
        return x.permute(1, 2, 0, 3, 4).reshape(2, kvh, -1, c["head_dim"])[:, :, :n]

    shared = [held(s["prefix_table"][g], n) for g, n in enumerate(plen)]
    for r, n in enumerate(kv_len):
        a, b = start[r], start[r + 1]
        mine = held(s["table"][r], n)
        p = 0
        for g in range(len(plen)):
            if gs[g] <= r < gs[g + 1]:
                mine, p = torch.cat([shared[g], mine], 2), plen[g]
        k, v = mine.repeat_interleave(group, 1)
        x = torch.einsum("thd,hnd->htn", q[a:b].double(), k) / c["head_dim"] ** 0.5
        hidden = torch.arange(p + n, device=DEV)[None, :] > torch.arange(p + n - (b - a), p + n, device=DEV)[:, None]
        x = x.masked_fill(hidden, -math.inf)
        lse[a:b] = torch.logsumexp(x, -1).t()
        out[a:b] = torch.einsum("htn,hnd->thd", torch.softmax(x, -1), v)
    return {"out": out, "lse": lse}


def _exact_logits(s):
    x = s["logits"].to(torch.float64)
    rows, vocab = x.shape
    live = torch.arange(s["tokens"].shape[1], device=DEV)[None, :] < s["length"][:, None]
    at = (torch.arange(rows, device=DEV)[:, None] * vocab + s["tokens"].long())[live]
    count = torch.bincount(at, minlength=rows * vocab).view(rows, vocab).to(torch.float64)
    rep, pres, freq = (s[n].to(torch.float64)[:, None] for n in ("repetition", "presence", "frequency"))
    scaled = x * torch.where(x > 0, 1 / rep, rep) - freq * count - pres
    x = torch.where(count != 0, scaled, x)
    if s["bias"] is not None:
        who, col = torch.nonzero(s["bias_id"] >= 0, as_tuple=True)
        x.index_put_((who, s["bias_id"][who, col].long()), s["bias"][who, col].to(torch.float64), accumulate=True)
    if s["allowed"] is not None:
        bits = (s["allowed"].long()[:, :, None] >> torch.arange(32, device=DEV)) % 2
        x[bits.reshape(rows, -1)[:, :vocab] == 0] = -math.inf
    return {"logits": x}
