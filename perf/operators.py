"""The operators of an 8-bit serving step, and cases that measure them.

Four operators, each with a plain form in elementary torch operations and the call a user makes of this package:

  plan       block tables and slot maps on the GPU from request lengths (kv8.plan)
  append     a step's K and V rows into the paged 8-bit cache, one scale per (page, K or V, kv head) (kv8.append), and
             the rows of the touched pages as the cache now holds them (kv8.read)
  attention  grouped-query attention over that cache for a ragged batch of requests, single tokens to whole prompts
             (kv8.attention)
  matmul     x . w^T in 8-bit integers with a scale for each token and each output channel (int8.matmul)

The cache is int8 [pages][2 (K, V)][kv heads][page size][head dim], with float32 scales [pages][2][kv heads].
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SCALE_MIN, SCALE_MAX = 2.0**-62, 2.0**63  # the range of a page's scale
GROW_AT, GROW_BY = 127.5, 1.25            # a page's scale grows when a value passes GROW_AT steps, by GROW_BY at least


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of the 32-session configuration: the smallest plan, where latency is everything
        {"name": "plan decode 32", "op": "plan", "requests": 32, "page": 16, "lo": 100, "hi": 4000, "ctx": 4096,
         "new_hi": 1, "release": 0.0},
        # a large server between two steps: prompts of many lengths arrive, sessions decode, others end or are cut back
        {"name": "plan mixed 2048", "op": "plan", "requests": 2048, "page": 16, "lo": 1, "hi": 4000, "ctx": 8192,
         "new_hi": 300, "release": 0.2},
        # the K and V of one batched decode step (7B heads): every page is in use already
        {"name": "append decode 32", "op": "append", "requests": 32, "page": 16, "kv_heads": 4, "head_dim": 128,
         "lo": 100, "hi": 4000, "new": 1, "dtype": "bf16"},
        # prompts of many sessions at once: bandwidth
        {"name": "append prompts 16k", "op": "append", "requests": 24, "page": 64, "kv_heads": 4, "head_dim": 128,
         "lo": 0, "hi": 500, "new": 683, "dtype": "bf16"},
        # the headline configuration: one session's decode step, 0.5B heads, float32 activations as the engine has them
        {"name": "attention decode 1", "op": "attention", "requests": 1, "page": 16, "heads": 14, "kv_heads": 2,
         "head_dim": 64, "lo": 641, "hi": 641, "new": 1, "window": 0, "dtype": "f32"},
        # a batched decode step of 32 sessions of very different lengths (7B heads)
        {"name": "attention decode 32", "op": "attention", "requests": 32, "page": 16, "heads": 28, "kv_heads": 4,
         "head_dim": 128, "lo": 100, "hi": 4096, "new": 1, "window": 0, "dtype": "bf16"},
        # a few sessions with very long histories: the cache's bandwidth
        {"name": "attention decode long", "op": "attention", "requests": 8, "page": 64, "heads": 28, "kv_heads": 4,
         "head_dim": 128, "lo": 60000, "hi": 131072, "new": 1, "window": 0, "dtype": "bf16"},
        # one prompt chunk of 256 tokens onto a 4096-token history, 0.5B heads, float32
        {"name": "attention chunk 256", "op": "attention", "requests": 1, "page": 16, "heads": 14, "kv_heads": 2,
         "head_dim": 64, "lo": 4096, "hi": 4096, "new": 256, "window": 0, "dtype": "f32"},
        # whole prompts of four sessions (7B heads): the tensor cores
        {"name": "attention prompts", "op": "attention", "requests": 4, "page": 64, "heads": 28, "kv_heads": 4,
         "head_dim": 128, "lo": 1500, "hi": 4099, "new": 4099, "window": 0, "dtype": "bf16"},
        # one token through the 0.5B model's QKV matrix: latency
        {"name": "matmul qkv 1", "op": "matmul", "m": 1, "n": 1152, "k": 896, "bias": True, "dtype": "f32"},
        # a 32-session step through the 7B model's gate and up matrices: the weights' bandwidth
        {"name": "matmul gate+up 32", "op": "matmul", "m": 32, "n": 37888, "k": 3584, "bias": False, "dtype": "bf16"},
        # a prompt through the 7B model's down matrix: the tensor cores
        {"name": "matmul down 4099", "op": "matmul", "m": 4099, "n": 3584, "k": 18944, "bias": False, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "matmul"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        hi = _log(rng, 10, 4000)
        return {"op": op, "requests": _log(rng, 1, 2048), "page": page, "lo": 1 + hi // 50, "hi": hi, "ctx": 8192,
                "new_hi": _log(rng, 1, 300), "release": rng.choice([0.0, 0.1, 0.3])}
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (28, 4, 128), (4, 2, 64), (7, 1, 64), (16, 4, 128), (4, 2, 128)])
    if op == "append":
        requests = _log(rng, 1, 64)
        return {"op": op, "requests": requests, "page": page, "kv_heads": kv_heads, "head_dim": dim, "lo": 0,
                "hi": _log(rng, 1, 4000), "new": _log(rng, 1, max(2, 16000 // requests)), "dtype": dtype}
    if op == "matmul":
        n, k = rng.choice([(1152, 896), (896, 896), (9728, 896), (896, 4864), (4608, 3584), (3584, 3584), (3584, 18944),
                           (_log(rng, 17, 4000), _log(rng, 33, 5000))])
        return {"op": op, "m": _log(rng, 1, 4099), "n": n, "k": k, "bias": rng.random() < 0.5, "dtype": dtype}
    shape = rng.choice(["decode", "few", "prompt"])
    window = rng.choice([0, 0, _log(rng, 16, 2000)])
    if shape == "decode":  # up to the long case's cache
        requests = _log(rng, 1, 64)
        hi = _log(rng, 16, min(131072, 500000 // requests))
        new = 1
    elif shape == "few":   # a few tokens at once: a drafted continuation, a short turn
        requests, hi, new = _log(rng, 1, 16), _log(rng, 32, 8000), rng.randint(2, 20)
    else:
        requests = rng.randint(1, 4)
        hi = _log(rng, 100, 4000)
        new = _log(rng, 21, hi)
    return {"op": op, "requests": requests, "page": page, "heads": heads, "kv_heads": kv_heads, "head_dim": dim,
            "lo": max(1, hi // 8), "hi": hi, "new": new, "window": window, "dtype": dtype}


def _spread(lo, hi, n, salt):
    """n lengths from lo to hi, spread over their logarithm: by the case alone, so that work() knows them too."""
    r = random.Random("%s %s %s %s" % (lo, hi, n, salt))
    got = [int(round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1 for _ in range(n)]
    got[r.randrange(n)] = hi
    return [min(hi, max(lo, g)) for g in got]


def _plan_lengths(case):
    """(tokens in the cache, tokens after the step) of each request."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    cached = _spread(case["lo"], case["hi"], case["requests"], "cached")
    total = []
    for c in cached:
        if r.random() < case["release"]:
            total.append(r.choice([0, r.randint(0, c)]))  # ends, or is cut back to a shared prefix
        else:
            total.append(min(case["ctx"], c + _log(r, 1, case["new_hi"])))
    return cached, total


def _pages(n, page):
    return -(-n // page)


def _append_lengths(case):
    return _spread(case["lo"], case["hi"], case["requests"], "append")


def _attention_lengths(case):
    kv = _spread(case["lo"], case["hi"], case["requests"], "kv")
    return kv, [min(k, case["new"]) for k in kv]


# ---------------------------------------------------------------------------------------------- inputs

def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _codes(gen, *shape):
    """8-bit codes as a cache of normal values holds them: the largest of a block near 127."""
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)
    return x.mul_(34).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return {"plan": _prepare_plan, "append": _prepare_append, "attention": _prepare_attention,
            "matmul": _prepare_matmul}[case["op"]](case, gen)


def _tables(gen, lengths, page, columns, n_pages):
    """Block tables whose pages are spread over the pool at random, and the pages left, in random order."""
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    have = _ints([_pages(n, page) for n in lengths], torch.int64)
    first = torch.cumsum(have, 0) - have
    col = torch.arange(columns, device=DEV)[None, :]
    at = (first[:, None] + col).clamp(max=n_pages - 1)
    table = torch.where(col < have[:, None], order[at], torch.full_like(order[at], -1))
    return table.contiguous(), order, int(sum(_pages(n, page) for n in lengths))


def _prepare_plan(case, gen):
    cached, total = _plan_lengths(case)
    page, columns = case["page"], _pages(case["ctx"], case["page"])
    used = sum(_pages(c, page) for c in cached)
    n_pages = used + sum(_pages(t, page) for t in total) + 17
    table, order, _ = _tables(gen, cached, page, columns, n_pages)
    start = int(torch.randint(0, n_pages, (1,), generator=gen, device=DEV))  # the free ring starts anywhere
    ring = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
    free = n_pages - used
    ring[(start + torch.arange(free, device=DEV)) % n_pages] = order[used:]
    tokens = sum(max(0, t - c) for c, t in zip(cached, total))
    return {"case": case, "cached": _ints(cached), "total": _ints(total), "table": table, "ring": ring,
            "state": _ints([start, start + free], torch.int64), "max_tokens": tokens + 5}


def _prepare_append(case, gen):
    page, kvh, hd = case["page"], case["kv_heads"], case["head_dim"]
    cached = _append_lengths(case)
    total = [c + case["new"] for c in cached]
    columns = max(_pages(t, page) for t in total)
    n_pages = sum(_pages(t, page) for t in total) + 3
    table, _, _ = _tables(gen, total, page, columns, n_pages)
    slots, touched = [], []
    host = table.cpu().numpy()
    for r, (c, t) in enumerate(zip(cached, total)):
        pos = np.arange(c, t)
        slots.append(host[r, pos // page] * page + pos % page)
        pos = np.arange(c // page * page, t)  # every row of the touched pages
        touched.append(host[r, pos // page] * page + pos % page)
    rows = sum(t - c for c, t in zip(cached, total))
    # K and V as a QKV product leaves them: slices of one row per token; a few channels of K far above the others
    qkv = torch.randn(rows, 3 * kvh * hd, generator=gen, device=DEV)
    qkv[:, kvh * hd:2 * kvh * hd:hd // 4] *= 6
    qkv = qkv.to(DTYPE[case["dtype"]])
    scale = 0.03 * torch.exp(0.2 * torch.randn(n_pages, 2, kvh, generator=gen, device=DEV))
    return {"case": case, "kv": _codes(gen, n_pages, 2, kvh, page, hd), "scale": scale,
            "k": qkv[:, kvh * hd:2 * kvh * hd].view(rows, kvh, hd), "v": qkv[:, 2 * kvh * hd:].view(rows, kvh, hd),
            "slot": _ints(np.concatenate(slots).tolist()), "touched": _ints(np.concatenate(touched).tolist())}


def _prepare_attention(case, gen):
    page, kvh, hd, heads = case["page"], case["kv_heads"], case["head_dim"], case["heads"]
    kv_len, new = _attention_lengths(case)
    columns = max(_pages(n, page) for n in kv_len)
    n_pages = sum(_pages(n, page) for n in kv_len) + 3
    table, _, _ = _tables(gen, kv_len, page, columns, n_pages)
    scale = torch.exp(0.3 * torch.randn(n_pages, 2, kvh, generator=gen, device=DEV)) * 0.03
    rows = sum(new)
    q = torch.randn(rows, heads, hd, generator=gen, device=DEV) * 1.7
    q_start = np.concatenate([[0], np.cumsum(new)])
    return {"case": case, "q": q.to(DTYPE[case["dtype"]]), "kv": _codes(gen, n_pages, 2, kvh, page, hd), "scale": scale,
            "table": table, "q_start": _ints(q_start.tolist()), "kv_len": _ints(kv_len), "max_q": max(new),
            "max_kv": max(kv_len)}


def _prepare_matmul(case, gen):
    m, n, k = case["m"], case["n"], case["k"]
    x = torch.randn(m, k, generator=gen, device=DEV) * torch.exp(0.5 * torch.randn(m, 1, generator=gen, device=DEV))
    x[:, ::max(1, k // 7)] *= 8  # a few large channels, as activations have them
    w = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device=DEV)  # rows padded to 16 bytes, as laid out once
    w[:, :k] = _codes(gen, n, k)
    ws = 0.0006 * torch.exp(0.2 * torch.randn(n, generator=gen, device=DEV))
    bias = torch.randn(n, generator=gen, device=DEV) * 0.02 if case["bias"] else None
    return {"case": case, "x": x.to(DTYPE[case["dtype"]]), "w": w, "w_scale": ws, "bias": bias}


# ---------------------------------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attention": _own_attention, "matmul": _own_matmul}[op](state)
    return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "matmul": _plain_matmul}[op](state)


def _own_plan(s):
    from e2e_browser_voice_agent_b200 import kv8
    p = kv8.plan(s["cached"], s["total"], s["table"], s["ring"], s["state"], s["case"]["page"], s["max_tokens"])
    return {"kv_len": p.kv_len, "q_start": p.q_start, "slot": p.slot, "position": p.position, "state": p.free_state,
            "status": p.status, "table": s["table"], "ring": s["ring"]}


def _own_append(s):
    from e2e_browser_voice_agent_b200 import kv8
    kv8.append(s["kv"], s["scale"], s["k"], s["v"], s["slot"])
    k, v = kv8.read(s["kv"], s["scale"], s["touched"])
    return {"k": k, "v": v, "scale": s["scale"]}


def _own_attention(s):
    from e2e_browser_voice_agent_b200 import kv8
    out, lse = kv8.attention(s["q"], s["kv"], s["scale"], s["table"], s["q_start"], s["kv_len"], s["max_q"], s["max_kv"],
                             window=s["case"]["window"], return_lse=True)
    return {"out": out, "lse": lse}


def _own_matmul(s):
    from e2e_browser_voice_agent_b200 import int8
    return {"y": int8.matmul(s["x"], s["w"], s["w_scale"], bias=s["bias"])}


def _plain_plan(s):
    page, table, ring = s["case"]["page"], s["table"], s["ring"]
    cached, total = s["cached"].long(), s["total"].long()
    n, cols = ring.numel(), table.shape[1]
    head, tail = s["state"][0], s["state"][1]
    have, want = (cached + page - 1) // page, (total + page - 1) // page
    new, take, rel = (total - cached).clamp(min=0), (want - have).clamp(min=0), (have - want).clamp(min=0)
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    q_start, take_start, rel_start = (torch.cat([zero, torch.cumsum(x, 0)]) for x in (new, take, rel))
    bad = ((cached < 0) | (total < 0) | (have > cols) | (want > cols)).any() | (q_start[-1] > s["max_tokens"])
    short = (take_start[-1] - rel_start[-1] - (tail - head)).clamp(min=0)
    ok = ~bad & (short == 0)
    d = torch.arange(n, device=DEV)
    who = torch.searchsorted(rel_start[1:], d, right=True).clamp(max=cached.numel() - 1)
    released = table[who, (want[who] + d - rel_start[who]).clamp(0, cols - 1)]       # the d-th page given back
    # the pages to take, in order: those free before, then those given back
    k = torch.arange(n, device=DEV)
    queue = torch.where(k < tail - head, ring[(head + k) % n], released[(k - (tail - head)).clamp(0, n - 1)])
    col = torch.arange(cols, device=DEV)[None, :]
    taken = (col >= have[:, None]) & (col < want[:, None]) & ok
    at = (take_start[:-1, None] + col - have[:, None]).clamp(0, n - 1)
    table.copy_(torch.where(taken, queue[at], table))
    back = (k - tail) % n
    ring.copy_(torch.where((back < rel_start[-1]) & ok, released[back], ring))
    t = torch.arange(s["max_tokens"], device=DEV)
    r = torch.searchsorted(q_start[1:], t, right=True).clamp(max=cached.numel() - 1)
    live = (t < q_start[-1]) & ok
    pos = torch.where(live, cached[r] + t - q_start[r], -1)
    slot = torch.where(live, table[r, (pos // page).clamp(0, cols - 1)].long() * page + pos % page, -1)
    return {"kv_len": torch.where(ok, total, cached).int(), "q_start": torch.where(ok, q_start, 0).int(), "slot": slot.int(),
            "position": pos.int(), "state": torch.where(ok, torch.stack([head + take_start[-1], tail + rel_start[-1]]), s["state"]),
            "status": torch.stack([torch.where(bad, 2, torch.where(short > 0, 1, 0)), torch.where(bad, 0, short)]).int(),
            "table": table, "ring": ring}


def _plain_append(s):
    kv, scale, slot = s["kv"], s["scale"], s["slot"].long()
    page = s["case"]["page"]
    x = torch.stack([s["k"], s["v"]], 1).float()                      # [rows][2][kv heads][head dim]
    pg, off = slot // page, slot % page
    lead = torch.cat([torch.ones_like(pg[:1], dtype=torch.bool), pg[1:] != pg[:-1]])
    run_of = torch.cumsum(lead, 0) - 1
    at = lead.nonzero()[:, 0]                                         # one run of rows for each page
    pages, first = pg[at], off[at]
    amax = torch.zeros(at.numel(), 2, x.shape[2], device=DEV)
    row = x.abs().amax(-1)
    amax.scatter_reduce_(0, run_of[:, None, None].expand_as(row), row, "amax")
    old = torch.where((first == 0)[:, None, None], 0.0, scale[pages])
    grown = torch.maximum(torch.maximum(amax / torch.full_like(amax, 127), GROW_BY * old), torch.full_like(old, SCALE_MIN)).clamp(max=SCALE_MAX)
    now = torch.where((amax > GROW_AT * old) | (old == 0), grown, old)
    scale[pages] = now
    before = kv[pages].float()
    kept = torch.round(before * (old / now)[..., None, None])
    earlier = torch.arange(page, device=DEV)[None, :] < first[:, None]
    kv[pages] = torch.where(earlier[:, None, None, :, None], kept, before).to(torch.int8)
    kv[pg, :, :, off] = torch.round(x * (1.0 / now)[run_of][..., None]).clamp(-127, 127).to(torch.int8)
    at = s["touched"].long()
    values = kv[at // page, :, :, at % page].float() * scale[at // page][..., None]
    return {"k": values[:, 0], "v": values[:, 1], "scale": scale}


def _plain_attention(s):
    c, q, table = s["case"], s["q"], s["table"].long().clamp(min=0)
    page, heads, kvh, hd = c["page"], c["heads"], c["kv_heads"], c["head_dim"]
    n, mq, mk = table.shape[0], s["max_q"], table.shape[1] * page
    kv = s["kv"][table].float() * s["scale"][table][..., None, None]  # [requests][pages][2][kv heads][page][dim]
    k, v = (kv[:, :, i].permute(0, 2, 1, 3, 4).reshape(n, kvh, mk, hd) for i in (0, 1))
    start, kv_len = s["q_start"].long(), s["kv_len"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(mq, device=DEV)
    rows = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)           # each request's queries, padded to the longest
    qp = q[rows].float().reshape(n, mq, kvh, heads // kvh, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, -1, hd)
    pos = (kv_len - count)[:, None] + i
    key = torch.arange(mk, device=DEV)
    seen = (key <= pos[..., None]) & (key < kv_len[:, None, None])
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    seen = seen[:, None, None].expand(n, kvh, heads // kvh, mq, mk).reshape(n, kvh, -1, mk)
    x = (qp @ k.transpose(-1, -2)).mul_(1 / math.sqrt(hd)).masked_fill_(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).reshape(n, heads, mq)
    o = o.reshape(n, heads, mq, hd).permute(0, 2, 1, 3)
    t = torch.arange(q.shape[0], device=DEV)
    r = torch.searchsorted(start[1:], t, right=True)
    return {"out": o[r, t - start[r]].to(q.dtype), "lse": lse[r, :, t - start[r]]}


def _plain_matmul(s):
    x, w = s["x"].float(), s["w"][:, : s["case"]["k"]].float()
    amax = x.abs().amax(-1, keepdim=True)
    most = torch.full_like(amax, 127)                                 # (a tensor: a number would be divided by approximately)
    inv = torch.where(amax > 0, (most / amax).clamp(max=3.4028234663852886e38), 0.0)
    y = (torch.round(x * inv) @ w.t()) * (amax / most) * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return {"y": y.to(s["x"].dtype)}


# ---------------------------------------------------------------------------------------------- needs

def work(case):
    """Bytes and operations that one pass cannot do without: inputs read once, outputs written once."""
    op = case["op"]
    if op == "plan":
        cached, total = _plan_lengths(case)
        moved = sum(abs(_pages(t, case["page"]) - _pages(c, case["page"])) for c, t in zip(cached, total))
        tokens = sum(max(0, t - c) for c, t in zip(cached, total))
        return {"bytes": 16 * len(cached) + 8 * tokens + 8 * moved, "flops": 0}
    if op == "append":
        page, width = case["page"], 2 * case["kv_heads"] * case["head_dim"]
        cached = _append_lengths(case)
        rows = len(cached) * case["new"]
        back = sum(c + case["new"] - c // page * page for c in cached)   # rows of the touched pages, read back
        pages = sum(_pages(c + case["new"], page) - c // page for c in cached)
        return {"bytes": rows * width * (SIZE[case["dtype"]] + 1) + back * width * (1 + 4) + pages * case["kv_heads"] * 8 * 2,
                "flops": 0}
    if op == "matmul":
        m, n, k, size = case["m"], case["n"], case["k"], SIZE[case["dtype"]]
        return {"bytes": n * k + m * (k + n) * size + 4 * n * (2 if case["bias"] else 1), "flops": 2 * m * n * k}
    kv_len, new = _attention_lengths(case)
    heads, kvh, hd, window = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    keys = rows = pairs = 0
    for n, q in zip(kv_len, new):
        first = max(0, n - q + 1 - window) if window else 0              # the first key any of the queries sees
        keys += n - first
        rows += q
        pairs += sum(min(p + 1, window) if window else p + 1 for p in range(n - q, n))
    size = SIZE[case["dtype"]]
    return {"bytes": keys * 2 * kvh * hd + (keys // case["page"] + 1) * (8 * kvh + 4) + rows * heads * (2 * hd * size + 4),
            "flops": 4 * pairs * heads * hd}


# ---------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """What run() returns, from the definition in 64 bits; the whole numbers of a plan have no such value."""
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "matmul":
        x = s["x"].double()
        top = x.abs().max(1, keepdim=True).values
        codes = torch.round(torch.where(top > 0, x * 127 / top, 0.0))
        w = s["w"][:, : case["k"]].double() * s["w_scale"].double()[:, None]
        y = torch.nn.functional.linear(codes * (top / 127), w, None if s["bias"] is None else s["bias"].double())
        return {"y": y}
    return _exact_attention(s)


def _exact_append(s):
    page, kv, scale = s["case"]["page"], s["kv"].double(), s["scale"].double()
    slot = s["slot"].tolist()
    x = torch.stack([s["k"].double(), s["v"].double()])               # [2][rows][kv heads][dim]
    held = {}
    t = 0
    while t < len(slot):
        pg, off = divmod(slot[t], page)
        end = t + 1
        while end < len(slot) and slot[end] == slot[end - 1] + 1 and slot[end] // page == pg:
            end += 1
        part = x[:, t:end].permute(0, 2, 1, 3)                        # [2][kv heads][run][dim]
        top = part.abs().amax((2, 3))
        old = torch.zeros_like(top) if off == 0 else scale[pg]
        need = torch.maximum(torch.maximum(top / 127, GROW_BY * old), torch.full_like(top, SCALE_MIN))
        step = torch.where((old == 0) | (top > GROW_AT * old), need, old)
        rows = kv[pg].clone()
        rows[:, :, :off] = torch.round(rows[:, :, :off] * (old / step)[..., None, None])
        rows[:, :, off:off + end - t] = torch.round(part / step[..., None, None]).clamp(-127, 127)
        held[pg] = rows * step[..., None, None]
        scale[pg] = step
        t = end
    at = s["touched"].tolist()
    both = torch.stack([held[a // page][:, :, a % page] for a in at])
    return {"k": both[:, 0], "v": both[:, 1], "scale": scale}


def _exact_attention(s):
    c, q = s["case"], s["q"]
    page, heads, kvh = c["page"], c["heads"], c["kv_heads"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    start, kv_len, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["table"]
    for r, n in enumerate(kv_len):
        a, b = start[r], start[r + 1]
        pages = table[r, : _pages(n, page)].long()
        pos = torch.arange(n - (b - a), n, device=DEV)[:, None]
        key = torch.arange(n, device=DEV)[None, :]
        hidden = key > pos
        if c["window"]:
            hidden = hidden | (key <= pos - c["window"])
        for h in range(heads):
            g = h // (heads // kvh)
            held = s["kv"][pages][:, :, g].double() * s["scale"][pages][:, :, g].double()[..., None, None]
            k, v = (held[:, i].reshape(-1, c["head_dim"])[:n] for i in (0, 1))
            x = torch.einsum("td,nd->tn", q[a:b, h].double(), k) * c["head_dim"] ** -0.5
            x = torch.where(hidden, -math.inf, x)
            lse[a:b, h] = torch.logsumexp(x, 1)
            out[a:b, h] = torch.softmax(x, 1) @ v
    return {"out": out, "lse": lse}
