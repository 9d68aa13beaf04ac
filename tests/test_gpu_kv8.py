"""The paged 8-bit KV cache on the GPU against plain implementations in 64 bits: plan (whole numbers, exact), append and
read (the formulas of include/h2cuda.h in float32, exact, and their error bound), attention.

Attention's tolerance. With x the largest |score| in powers of two, the computed scores are off by less than
(x + 1) 2^-20 (22-bit queries, float32 sums of exact products) and exp2 by 2^-22 of itself, so every softmax weight is
off by less than a fraction d = (x + 2) 2^-20 of itself, and the output, an average of values of at most v, by less than
2 d v; rounding to the output's type adds 2^-24, 2^-11 or 2^-8 of it. Float16 or bfloat16 prompt rows may carry their
weights as one float16 number (2^-11 of itself each).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def kv8():
    from e2e_browser_voice_agent_b200 import kv8 as m
    return m


# ---------------------------------------------------------------------------------------------- plan

def ref_plan(cached, total, table, ring, state, page, max_tokens):
    cached, total, table, ring = list(cached), list(total), table.copy(), ring.copy()
    n, cols = len(ring), table.shape[1]
    head, tail = state
    room = cols * page
    pages = lambda x: -(-x // page)
    R = len(cached)
    no = [-1] * max_tokens

    def refuse(code, missing):
        keep = [c if 0 <= c <= room else 0 for c in cached]
        return dict(kv_len=keep, q_start=[0] * (R + 1), slot=no, position=no, state=[head, tail], status=[code, missing],
                    table=table, ring=ring)
    new = [max(0, t - c) for c, t in zip(cached, total)]
    if any(c < 0 or t < 0 or c > room or t > room for c, t in zip(cached, total)) or sum(new) > max_tokens:
        return refuse(2, 0)
    back = [(r, j) for r in range(R) for j in range(pages(total[r]), pages(cached[r]))]
    take = [(r, j) for r in range(R) for j in range(pages(cached[r]), pages(total[r]))]
    if head < 0 or tail < head or tail - head + len(back) > n:
        return refuse(2, 0)
    queue = [ring[i % n] for i in range(head, tail)] + [table[r, j] for r, j in back]
    if len(take) > len(queue):
        return refuse(1, len(take) - len(queue))
    for i, (r, j) in enumerate(back):
        ring[(tail + i) % n] = table[r, j]
    for (r, j), pg in zip(take, queue):
        table[r, j] = pg
    slot, position = [], []
    for r in range(R):
        for p in range(cached[r], total[r]):
            slot.append(table[r, p // page] * page + p % page)
            position.append(p)
    pad = [-1] * (max_tokens - len(slot))
    return dict(kv_len=total, q_start=[0] + list(np.cumsum(new)) if R else [0], slot=slot + pad, position=position + pad,
                state=[head + len(take), tail + len(back)], status=[0, 0], table=table, ring=ring)


def run_plan(cached, total, table, ring, state, page, max_tokens, out=None):
    t, r = torch.tensor(table, dtype=torch.int32, device=DEV), torch.tensor(ring, dtype=torch.int32, device=DEV)
    ten = lambda x, d=torch.int32: torch.tensor(list(x), dtype=d, device=DEV)
    p = kv8().plan(ten(cached), ten(total), t, r, ten(state, torch.int64), page, max_tokens, out=out)
    return dict(kv_len=p.kv_len, q_start=p.q_start, slot=p.slot, position=p.position, state=p.free_state, status=p.status,
                table=t, ring=r), p


def same_plan(got, want):
    for k, w in want.items():
        g = got[k].cpu().numpy()
        assert np.array_equal(g, np.asarray(w, dtype=np.int64).reshape(g.shape)), k


def pool(rng, cached, page, cols, spare, start):
    used = sum(-(-c // page) for c in cached)
    n = used + spare
    order = rng.permutation(n)
    table = np.full((len(cached), cols), -1)
    at = 0
    for r, c in enumerate(cached):
        k = -(-c // page)
        table[r, :k] = order[at:at + k]
        at += k
    ring = np.full(n, -7)
    for i, pg in enumerate(order[used:]):
        ring[(start + i) % n] = pg
    return table, ring, [start, start + n - used]


@pytest.mark.parametrize("R,page,hi", [(1, 16, 40), (3, 16, 70), (32, 32, 300), (513, 64, 700), (2100, 128, 500), (8192, 16, 40)])
@pytest.mark.parametrize("kind", ["decode", "mixed"])
def test_plan_matches_the_formula(R, page, hi, kind):
    rng = np.random.default_rng(R + page)
    cached = rng.integers(0, hi, R).tolist()
    cols = -(-2 * hi // page)
    if kind == "decode":
        total = [c + 1 for c in cached]
    else:
        total = [int(rng.choice([0, c, rng.integers(0, c + 1), min(2 * hi, c + rng.integers(0, hi))])) for c in cached]
    tokens = sum(max(0, t - c) for c, t in zip(cached, total))
    need = sum(-(-t // page) for t in total)
    table, ring, state = pool(rng, cached, page, cols, need + 3, start=int(rng.integers(0, 10**6)))
    want = ref_plan(cached, total, table, ring, state, page, tokens + 4)
    assert want["status"] == [0, 0]
    got, p = run_plan(cached, total, table, ring, state, page, tokens + 4)
    same_plan(got, want)
    got2, _ = run_plan(cached, total, table, ring, state, page, tokens + 4, out=p)  # the same tensors written again
    same_plan(got2, want)


def test_plan_twice_on_the_same_inputs_gives_the_same():
    rng = np.random.default_rng(5)
    cached, total = [40, 3, 64, 0], [20, 100, 0, 17]
    table, ring, state = pool(rng, cached, 16, 8, 9, start=5)
    ten = lambda x, d=torch.int32: torch.tensor(x, dtype=d, device=DEV)
    t, r = ten(table), ten(ring)
    want = ref_plan(cached, total, table, ring, state, 16, 200)
    for _ in range(3):
        p = kv8().plan(ten(cached), ten(total), t, r, ten(state, torch.int64), 16, 200)
        same_plan(dict(kv_len=p.kv_len, q_start=p.q_start, slot=p.slot, position=p.position, state=p.free_state,
                       status=p.status, table=t, ring=r), want)


def test_plan_takes_pages_given_back_in_the_same_call():
    rng = np.random.default_rng(6)
    cached, total = [160, 0, 33, 5], [0, 100, 1, 60]       # 10 + 2 pages given back, 7 + 3 taken, 1 free before
    table, ring, state = pool(rng, cached, 16, 10, 1, start=4)
    want = ref_plan(cached, total, table, ring, state, 16, 200)
    assert want["status"] == [0, 0]
    same_plan(run_plan(cached, total, table, ring, state, 16, 200)[0], want)


@pytest.mark.parametrize("cached,total,spare,tokens,state_add,code", [
    ([16, 16], [17, 400], 3, 500, 0, 1),      # pages are missing
    ([16, 16], [16, 33], 30, 16, 0, 2),       # more tokens than max_tokens
    ([16, -1], [16, 3], 30, 50, 0, 2),        # lengths without sense
    ([16, 16], [16, 16 * 26], 40, 500, 0, 2),
    ([16, 5], [16, -2147483648], 40, 500, 0, 2),
    ([16, 16], [0, 16], 4, 500, 3, 2),        # a ring that holds more than all pages
])
def test_plan_refuses_on_the_device_and_changes_nothing(cached, total, spare, tokens, state_add, code):
    rng = np.random.default_rng(7)
    table, ring, state = pool(rng, [max(0, c) for c in cached], 16, 25, spare, start=2)
    state = [state[0], state[1] + state_add]
    want = ref_plan(cached, total, table, ring, state, 16, tokens)
    assert want["status"][0] == code
    same_plan(run_plan(cached, total, table, ring, state, 16, tokens)[0], want)


def test_plan_without_requests_or_tokens():
    p = run_plan([], [], np.zeros((0, 4)), [0, 1], [0, 2], 16, 3)[1]
    assert p.q_start.tolist() == [0] and p.slot.tolist() == [-1] * 3 and p.status.tolist() == [0, 0]
    assert p.free_state.tolist() == [0, 2] and p.kv_len.numel() == 0
    got, p = run_plan([7], [7], np.array([[1, -1]]), [0, 1], [0, 1], 16, 0)
    assert p.q_start.tolist() == [0, 0] and p.kv_len.tolist() == [7] and p.slot.numel() == 0


# ---------------------------------------------------------------------------------------------- append, read

def ref_append(codes, scale, k, v, slot, page):
    """The header's formula in float32, one run of rows at a time."""
    f = np.float32
    codes, scale = codes.copy(), scale.copy()
    x = np.stack([k, v], 1).astype(f)     # [rows][2][heads][dim]
    n_slots = codes.shape[0] * page
    t = 0
    while t < len(slot):
        s = slot[t]
        if s < 0 or s >= n_slots:
            t += 1
            continue
        pg, off = divmod(s, page)
        e = t + 1
        while e < len(slot) and slot[e] == slot[e - 1] + 1 and slot[e] // page == pg:
            e += 1
        for w in range(2):
            for h in range(x.shape[2]):
                part = x[t:e, w, h]
                s0 = f(0) if off == 0 else scale[pg, w, h]
                if not np.isfinite(part).all() or np.isnan(s0):
                    scale[pg, w, h] = np.nan
                    codes[pg, w, h, off:off + e - t] = 0
                    continue
                a = np.abs(part).max()
                s1 = s0
                if s0 == 0 or a > f(127.5) * s0:
                    s1 = min(max(f(a) / f(127), f(1.25) * s0, f(2.0**-62)), f(2.0**63))
                    old = codes[pg, w, h, :off].astype(f)
                    if off:
                        codes[pg, w, h, :off] = np.rint(old * (s0 / s1))
                scale[pg, w, h] = s1
                codes[pg, w, h, off:off + e - t] = np.clip(np.rint(part * (f(1) / s1)), -127, 127)
        t = e
    return codes, scale


def slots_of(rng, n_pages, page, lengths, cached):
    """Slots of requests that go from cached to lengths, on random pages; and the block table's rows."""
    order = rng.permutation(n_pages)
    slots, rows, at = [], [], 0
    for c, n in zip(cached, lengths):
        k = -(-n // page)
        pages = order[at:at + k]
        at += k
        rows.append(pages)
        pos = np.arange(c, n)
        slots.append(pages[pos // page] * page + pos % page)
    return np.concatenate(slots).astype(np.int32), rows


def to_gpu(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x)).to(DEV)
    return t if dtype is None else t.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,heads,hd,layout", [(16, 2, 64, "dense"), (32, 1, 128, "slice"), (64, 4, 128, "odd"),
                                                  (128, 3, 64, "slice"), (128, 2, 128, "dense"), (16, 7, 128, "odd")])
def test_append_and_read_match_the_formula(dtype, page, heads, hd, layout):
    rng = np.random.default_rng(page + heads + hd)
    cached = [0, 5, page - 1, page, 0, 3 * page + 1, page // 2]
    lengths = [1, 6, page + 40, page + 1, 2 * page, 6 * page + 9, page // 2 + 3]
    n_pages = sum(-(-n // page) for n in lengths) + 2
    slot, _ = slots_of(rng, n_pages, page, lengths, cached)
    slot = np.concatenate([slot[:4], [-1, n_pages * page, -5], slot[4:]]).astype(np.int32)
    T = len(slot)
    codes = rng.integers(-127, 128, (n_pages, 2, heads, page, hd)).astype(np.int8)
    scale = np.exp(rng.standard_normal((n_pages, 2, heads))).astype(np.float32) * np.float32(0.01)
    scale[slot[0] // page] = np.nan       # whatever an unused page held: the first run starts it anew
    x = (rng.standard_normal((T, 3 * heads, hd)) * np.exp(rng.standard_normal((T, 1, 1)))).astype(np.float32)
    x[min(9, T - 1)] = 0
    if layout == "dense":
        k, v = (to_gpu(x[:, i * heads:(i + 1) * heads], dtype) for i in (1, 2))
    elif layout == "slice":
        xt = to_gpu(x, dtype)
        k, v = xt[:, heads:2 * heads], xt[:, 2 * heads:]
    else:  # rows and heads that start at odd elements
        buf = torch.zeros(T, 3 * heads, hd + 1, dtype=dtype, device=DEV)
        buf[:, :, 1:] = to_gpu(x, dtype)
        k, v = buf[:, heads:2 * heads, 1:], buf[:, 2 * heads:, 1:]
    kv, sc = to_gpu(codes), to_gpu(scale)
    kv8().append(kv, sc, k, v, to_gpu(slot))
    want_c, want_s = ref_append(codes, scale, k.float().cpu().numpy(), v.float().cpu().numpy(), slot.tolist(), page)
    assert np.array_equal(sc.cpu().numpy(), want_s)
    assert np.array_equal(kv.cpu().numpy(), want_c)
    rk, rv = kv8().read(kv, sc, to_gpu(slot))
    ok = (slot >= 0) & (slot < n_pages * page)
    safe = np.where(ok, slot, 0)
    both = want_c[safe // page, :, :, safe % page].astype(np.float32) * want_s[safe // page][..., None]
    both[~ok] = 0
    assert np.array_equal(rk.cpu().numpy(), both[:, 0]) and np.array_equal(rv.cpu().numpy(), both[:, 1])
    hk, _ = kv8().read(kv, sc, to_gpu(slot), dtype=torch.bfloat16)
    assert torch.equal(hk, to_gpu(both[:, 0]).to(torch.bfloat16))


@pytest.mark.parametrize("order", ["random", "rising"])
def test_appended_one_by_one_stays_within_its_bound(order):
    """Rows appended one at a time, where each growth of the scale re-rounds the earlier codes: off by at most 2.5 steps
    (rising magnitudes make the scale grow with every row)."""
    rng = np.random.default_rng(3)
    page, heads, hd = 64, 2, 64
    x = rng.standard_normal((page, heads, hd)).astype(np.float32)
    if order == "rising":
        x *= (1.02 ** np.arange(page, dtype=np.float32))[:, None, None]
    k = to_gpu(x)
    kv, sc = kv8().allocate(2, page, heads, hd)
    for t in range(page):
        kv8().append(kv, sc, k[t:t + 1], -k[t:t + 1], torch.tensor([page + t], dtype=torch.int32, device=DEV))
    rk, rv = kv8().read(kv, sc, torch.arange(page, 2 * page, dtype=torch.int32, device=DEV))
    step = sc[1].double()                                  # [2][heads]
    off_k = ((rk.double() - k.double()).abs() / step[0][None, :, None]).max()
    off_v = ((rv.double() + k.double()).abs() / step[1][None, :, None]).max()
    assert off_k <= 2.5 * (1 + 1e-5) and off_v <= 2.5 * (1 + 1e-5)
    assert float(step[0].max()) <= 1.25 * np.abs(x).max() / 127 * (1 + 1e-6)
    kv2, sc2 = kv8().allocate(2, page, heads, hd)          # the same rows in one call: half a step
    kv8().append(kv2, sc2, k, k, torch.arange(page, dtype=torch.int32, device=DEV))
    rk2, _ = kv8().read(kv2, sc2, torch.arange(page, dtype=torch.int32, device=DEV))
    assert ((rk2.double() - k.double()).abs() / sc2[0, 0].double()[None, :, None]).max() <= 0.5 * (1 + 1e-5)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_append_of_a_value_that_is_no_number(bad):
    page, heads, hd = 16, 2, 64
    kv, sc = kv8().allocate(3, page, heads, hd)
    x = torch.randn(20, heads, hd, device=DEV)
    k = x.clone()
    k[3, 1, 7] = bad
    slot = torch.arange(16, 36, dtype=torch.int32, device=DEV)
    kv8().append(kv, sc, k, x, slot)
    rk, rv = kv8().read(kv, sc, slot)
    assert rk[:16, 1].isnan().all() and rk[:16, 0].isfinite().all() and rk[16:].isfinite().all() and rv.isfinite().all()
    kv8().append(kv, sc, x[:1], x[:1], torch.tensor([31], dtype=torch.int32, device=DEV))   # the page stays lost
    assert kv8().read(kv, sc, slot)[0][:16, 1].isnan().all()
    kv8().append(kv, sc, x[:1], x[:1], torch.tensor([16], dtype=torch.int32, device=DEV))   # until it is new again
    assert kv8().read(kv, sc, slot[:1])[0].isfinite().all()


def test_append_of_extreme_magnitudes():
    kv, sc = kv8().allocate(3, 16, 1, 64)
    x = torch.zeros(3, 1, 64, device=DEV)
    x[0] = 1e-30
    x[1] = 3e38
    x[2] = 0
    kv8().append(kv, sc, x, x, torch.tensor([0, 16, 32], dtype=torch.int32, device=DEV))
    assert sc[:, 0, 0].tolist() == [2.0**-62, 2.0**63, 2.0**-62]
    rk, _ = kv8().read(kv, sc, torch.tensor([0, 16, 32], dtype=torch.int32, device=DEV))
    assert rk[0].abs().max() <= 2.0**-62 and (rk[1] == 127 * 2.0**63).all() and (rk[2] == 0).all()


def test_append_and_read_of_no_rows():
    kv, sc = kv8().allocate(1, 16, 1, 64)
    e = torch.zeros(0, 1, 64, device=DEV)
    s = torch.zeros(0, dtype=torch.int32, device=DEV)
    kv8().append(kv, sc, e, e, s)
    assert kv8().read(kv, sc, s)[0].shape == (0, 1, 64)


# ---------------------------------------------------------------------------------------------- attention

def make_cache(gen, kv_len, page, kvh, hd, spread=0.5, extra=2):
    """A cache whose pages are spread over the pool; what lies past a request's length, and in pages of nobody, is
    garbage, with NaN scales where no request's token is."""
    n_pages = sum(-(-n // page) for n in kv_len) + extra
    order = torch.randperm(n_pages, generator=gen, device=DEV).to(torch.int32)
    cols = max([1] + [-(-n // page) for n in kv_len])
    table = torch.full((len(kv_len), cols), 2**31 - 1, dtype=torch.int32, device=DEV)
    at = 0
    for r, n in enumerate(kv_len):
        k = -(-n // page)
        table[r, :k] = order[at:at + k]
        at += k
    kv = torch.randint(-127, 128, (n_pages, 2, kvh, page, hd), generator=gen, device=DEV, dtype=torch.int32).to(torch.int8)
    sc = 0.02 * torch.exp(spread * torch.randn(n_pages, 2, kvh, generator=gen, device=DEV))
    sc[order[at:].long()] = float("nan")
    return kv, sc, table


def ref_attention(q, kv, sc, table, q_start, kv_len, scale, window):
    """64 bits, one request and head at a time. Also the largest |score| in powers of two and the largest |v|."""
    page, hd, kvh, H = kv.shape[3], kv.shape[4], kv.shape[2], q.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    top = vmax = 0.0
    for r, n in enumerate(kv_len):
        a, b = q_start[r], q_start[r + 1]
        if n == 0 or a == b:
            continue
        pages = table[r, : -(-n // page)].long()
        pos = torch.arange(n - (b - a), n, device=DEV)[:, None]
        key = torch.arange(n, device=DEV)[None, :]
        seen = key <= pos
        if window:
            seen &= key > pos - window
        held = kv[pages].double() * sc[pages].double()[..., None, None]
        for h in range(H):
            g = h // (H // kvh)
            k, v = (held[:, i, g].reshape(-1, hd)[:n] for i in (0, 1))
            x = (q[a:b, h].double() @ k.t()) * scale
            top, vmax = max(top, float(x.abs().max()) * 1.4427), max(vmax, float(v.abs().max()))
            x = x.masked_fill(~seen, -math.inf)
            m = x.amax(1, keepdim=True)
            p = torch.exp(x - torch.where(m.isinf(), 0.0, m))
            total = p.sum(1, keepdim=True)
            out[a:b, h] = (p @ v) / torch.where(total == 0, 1.0, total)
            lse[a:b, h] = (m + torch.log(total))[:, 0]
    return out, lse, top, vmax


def close(out, lse, ref, dtype, one_term):
    want, want_lse, top, vmax = ref
    d = (top + 2) * 2.0**-20
    tol = 2 * d * vmax + EPS[dtype] * vmax + (2.0**-11 * vmax if one_term else 0)
    assert float((out.double() - want).abs().max()) <= tol
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (out[empty] == 0).all()
    assert float(torch.where(empty, 0.0, lse.double() - want_lse).abs().max()) <= d + 2.0**-22 * (top + 8)


def attend(q, kv, sc, table, q_start, kv_len, **kw):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    n_q = [b - a for a, b in zip(q_start, q_start[1:])]
    kw.setdefault("max_q", max(n_q, default=0))
    kw.setdefault("max_kv", max(kv_len, default=0))
    return kv8().attention(q, kv, sc, table, i32(q_start), i32(kv_len), return_lse=True, **kw)


def run_case(dtype, page, H, kvh, hd, kv_len, n_q, window=0, scale=None, spread=0.5, layout="dense", seed=0, **kw):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + page + H + hd + sum(kv_len))
    kv, sc, table = make_cache(gen, kv_len, page, kvh, hd, spread)
    T = sum(n_q)
    q_start = [0] + np.cumsum(n_q).tolist()
    q32 = torch.randn(T, H, hd, generator=gen, device=DEV)
    q32 *= torch.exp(torch.randn(T, H, 1, generator=gen, device=DEV))
    if layout == "dense":
        q, out = q32.to(dtype), None
    elif layout == "slice":   # the Q part of a QKV product's rows; the output into a wider row
        buf = torch.zeros(T, H + 2 * kvh, hd, dtype=dtype, device=DEV)
        buf[:, :H] = q32.to(dtype)
        q, out = buf[:, :H], torch.full((T, H + 3, hd), 9.0, dtype=dtype, device=DEV)[:, 2:2 + H]
    else:                     # odd starts, heads outermost
        buf = torch.zeros(H, T, hd + 1, dtype=dtype, device=DEV)
        buf[:, :, 1:] = q32.to(dtype).transpose(0, 1)
        q = buf.transpose(0, 1)[:, :, 1:]
        out = torch.full((H, T, hd + 3), 9.0, dtype=dtype, device=DEV).transpose(0, 1)[:, :, 3:]
    o, lse = attend(q, kv, sc, table, q_start, kv_len, window=window, scale=scale, out=out, **kw)
    ref = ref_attention(q, kv, sc, table, q_start, kv_len, hd ** -0.5 if scale is None else scale, window)
    close(o, lse, ref, dtype, dtype != torch.float32)
    return o, lse


HEADS = [(14, 2, 64), (28, 4, 128), (4, 4, 64), (7, 1, 128), (16, 1, 64), (12, 4, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,kvh,hd", HEADS)
def test_single_tokens(dtype, H, kvh, hd):
    for page, kv_len in [(16, [1]), (16, [1, 15, 16, 17, 31, 33, 64, 100, 257]), (32, [300, 2, 63]), (64, [65, 1200]), (128, [127, 128, 129])]:
        run_case(dtype, page, H, kvh, hd, kv_len, [1] * len(kv_len))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,kvh,hd", [(14, 2, 64), (28, 4, 128), (4, 2, 128)])
@pytest.mark.parametrize("window", [0, 1, 37, 4096])
def test_ragged_batches(dtype, H, kvh, hd, window):
    # prompts from the start, continuations, single tokens, a request without queries, one without keys, one with neither
    kv_len = [50, 700, 129, 0, 333, 20, 0, 512, 1]
    n_q = [50, 3, 1, 0, 120, 0, 2, 200, 1]
    run_case(dtype, 16, H, kvh, hd, kv_len, n_q, window=window)
    run_case(dtype, 128, H, kvh, hd, kv_len, n_q, window=window, seed=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["slice", "odd"])
def test_strides(dtype, layout):
    run_case(dtype, 32, 14, 2, 64, [70, 5, 300], [1, 5, 130], layout=layout)
    run_case(dtype, 16, 28, 4, 128, [70, 5, 300], [1, 5, 130], layout=layout)
    run_case(dtype, 16, 28, 4, 128, [70, 1500], [1, 1], layout=layout)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 127, 128, 129, 255, 256, 300, 641, 1025])
def test_prompt_lengths(dtype, n):
    run_case(dtype, 16, 14, 2, 64, [n], [n])
    run_case(dtype, 64, 8, 2, 128, [n + 77], [n])


@pytest.mark.parametrize("dtype", TYPES)
def test_more_queries_than_keys(dtype):
    """Queries before the first cached position have nothing to attend to: zeros and lse -infinity."""
    o, lse = run_case(dtype, 16, 14, 2, 64, [5, 0, 100], [9, 3, 140])
    assert (lse[:4] == -math.inf).all() and (lse[9:12] == -math.inf).all() and (o[9:12] == 0).all()
    run_case(dtype, 64, 28, 4, 128, [5, 0, 100], [300, 3, 1], window=3)


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_far_apart(dtype):
    """Pages whose scales differ by many powers of two, in K and V; weights that underflow next to the largest."""
    run_case(dtype, 16, 4, 2, 64, [400, 300], [1, 150], spread=3.0, scale=0.004)
    run_case(dtype, 16, 4, 2, 128, [400, 900], [1, 150], spread=3.0, scale=0.004)
    run_case(dtype, 16, 4, 2, 64, [333], [40], scale=2.0)


def test_a_tiny_v_page_under_a_large_weight():
    """Nearly all weight on a page whose V is 2^-20 of the others': the output is that page's V and keeps its precision."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1)
    kv, sc, table = make_cache(gen, [64], 16, 1, 64, spread=0.0)
    first = int(table[0, 0])
    kv[:, 0] = 0
    kv[first, 0, 0, 0] = 127            # K: only key 0 has a score
    sc[:] = 1.0
    sc[first, 1] = 2.0**-20
    for n_q in (1, 40):
        q = torch.full((n_q, 1, 64), 0.05, device=DEV)
        o, _ = attend(q, kv, sc, table, [0, n_q], [64], scale=1.0)
        want, _, top, _ = ref_attention(q, kv, sc, table, [0, n_q], [64], 1.0, 0)
        assert top > 500 and float((o.double() - want).abs().max()) <= 127 * 2.0**-20 * 2.0**-10


def test_zero_scales():
    gen = torch.Generator(device=DEV)
    gen.manual_seed(2)
    kv, sc, table = make_cache(gen, [100, 40], 16, 2, 64)
    sc[table[0, 1].long(), 1] = 0
    sc[table[0, 2].long(), 0] = 0
    sc[table[1, :3].long()] = 0
    for n_q in ([1, 1], [90, 33]):
        q = torch.randn(sum(n_q), 4, 64, device=DEV)
        q_start = [0, n_q[0], sum(n_q)]
        o, lse = attend(q, kv, sc, table, q_start, [100, 40])
        close(o, lse, ref_attention(q, kv, sc, table, q_start, [100, 40], 0.125, 0), torch.float32, False)


@pytest.mark.parametrize("n_q", [1, 70])
def test_a_lost_page_stays_with_its_request_and_head(n_q):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    kv, sc, table = make_cache(gen, [200, 200], 16, 2, 64)
    for w in (0, 1):
        sw = sc.clone()
        sw[int(table[0, 2]), w, 1] = float("nan")
        q = torch.randn(2 * n_q, 4, 64, device=DEV)
        o, lse = attend(q, kv, sw, table, [0, n_q, 2 * n_q], [200, 200])
        assert o[:n_q, 2:].isnan().all()
        good, good_lse = attend(q, kv, sc, table, [0, n_q, 2 * n_q], [200, 200])
        assert torch.equal(o[:n_q, :2], good[:n_q, :2]) and torch.equal(o[n_q:], good[n_q:])
        assert torch.equal(lse[n_q:], good_lse[n_q:])
    # outside the window it is not looked at
    sw = sc.clone()
    sw[int(table[0, 0]), :, 1] = float("nan")
    o, lse = attend(q, kv, sw, table, [0, n_q, 2 * n_q], [200, 200], window=16)
    assert o.isfinite().all() and lse.isfinite().all()


@pytest.mark.parametrize("n_q", [1, 70])
def test_a_query_that_is_no_number_stays_alone(n_q):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(4)
    kv, sc, table = make_cache(gen, [200], 16, 2, 64)
    q = torch.randn(n_q, 4, 64, device=DEV)
    good, _ = attend(q, kv, sc, table, [0, n_q], [200])
    for bad in (float("nan"), float("inf")):
        b = q.clone()
        b[n_q // 2, 1, 3] = bad
        o, _ = attend(b, kv, sc, table, [0, n_q], [200])
        assert o[n_q // 2, 1].isnan().all()
        o[n_q // 2, 1] = good[n_q // 2, 1]
        assert torch.equal(o, good)


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_of_extreme_magnitude(dtype):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(5)
    kv, sc, table = make_cache(gen, [150], 16, 2, 64)
    for n_q in (1, 40):
        big = 60000.0 if dtype == torch.float16 else 1e30
        q = torch.randn(n_q, 4, 64, device=DEV)
        tiny = (q * 1e-30).to(dtype)   # (zero in float16): every score is 0 or nearly
        o, lse = attend(tiny, kv, sc, table, [0, n_q], [150])
        close(o, lse, ref_attention(tiny, kv, sc, table, [0, n_q], [150], 0.125, 0), dtype, dtype != torch.float32)
        large = (q / q.abs().amax() * big).to(dtype)
        o, lse = attend(large, kv, sc, table, [0, n_q], [150], scale=1.0 / big)
        close(o, lse, ref_attention(large, kv, sc, table, [0, n_q], [150], 1.0 / big, 0), dtype, dtype != torch.float32)


def test_rows_of_no_request_are_left_alone():
    gen = torch.Generator(device=DEV)
    gen.manual_seed(6)
    kv, sc, table = make_cache(gen, [60, 90], 16, 2, 64)
    for n_q in ([1, 1], [40, 50]):
        T = sum(n_q) + 5
        q = torch.randn(T, 4, 64, device=DEV)
        out = torch.full((T, 4, 64), 7.0, device=DEV)
        attend(q, kv, sc, table, [0, n_q[0], sum(n_q)], [60, 90], out=out)
        assert (out[sum(n_q):] == 7).all() and not (out[: sum(n_q)] == 7).any()


def test_bounds_that_are_loose_or_low():
    """max_q above the real one changes nothing but the division of work; max_kv below a real length costs time only."""
    for n_q in (1, 60):
        for bounds in ({"max_q": 300, "max_kv": 9000}, {"max_kv": 40}, {"max_kv": 0}):
            run_case(torch.float32, 16, 4, 2, 64, [700, 30], [n_q, 1], **bounds)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(7)
    kv, sc, table = make_cache(gen, [64], 16, 1, 64)
    q = torch.randn(50, 4, 64, device=DEV)
    whole, _ = attend(q, kv, sc, table, [0, 50], [64])
    out = torch.full_like(q, 7.0)
    attend(q, kv, sc, table, [0, 50], [64], out=out, max_q=3)  # only the first three are computed
    d = (out[:3] - whole[:3]).abs().max()
    assert d < 1e-4 and (out[3:] == 7).all()


def test_many_requests_and_no_requests():
    run_case(torch.bfloat16, 16, 4, 2, 64, [(i * 7) % 90 for i in range(600)], [1] * 600)
    kv, sc = kv8().allocate(1, 16, 2, 64)
    e = torch.zeros(0, 4, 64, device=DEV)
    o, lse = attend(e, kv, sc, torch.zeros(0, 1, dtype=torch.int32, device=DEV), [0], [], max_q=0, max_kv=0)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_long_history_in_spans():
    run_case(torch.bfloat16, 64, 28, 4, 128, [40000, 9], [1, 1])
    run_case(torch.float32, 16, 14, 2, 64, [9000], [1], window=7000)


def test_a_cache_beyond_32_bit_offsets():
    """Pages whose bytes lie past 2^31 and 2^32."""
    page, kvh, hd = 128, 8, 128
    n_pages = (9 << 30) // 2 // (2 * kvh * page * hd)      # 4.5 GB of codes
    kv = torch.zeros(n_pages, 2, kvh, page, hd, dtype=torch.int8, device=DEV)
    sc = torch.zeros(n_pages, 2, kvh, device=DEV)
    pages = [n_pages - 1, 1, n_pages // 2 + 3]
    n = 300
    k, v = torch.randn(n, kvh, hd, device=DEV), torch.randn(n, kvh, hd, device=DEV)
    slot = torch.tensor([pages[p // page] * page + p % page for p in range(n)], dtype=torch.int32, device=DEV)
    kv8().append(kv, sc, k, v, slot)
    rk, _ = kv8().read(kv, sc, slot)
    assert (rk - k).abs().max() <= float(sc.max())
    table = torch.tensor([pages], dtype=torch.int32, device=DEV)
    for n_q in (1, 200):
        q = torch.randn(n_q, 16, hd, device=DEV)
        o, lse = attend(q, kv, sc, table, [0, n_q], [n])
        close(o, lse, ref_attention(q, kv, sc, table, [0, n_q], [n], hd ** -0.5, 0), torch.float32, False)


def test_on_a_stream_of_its_own():
    gen = torch.Generator(device=DEV)
    gen.manual_seed(8)
    kv, sc, table = make_cache(gen, [700, 90], 16, 2, 64)
    q = torch.randn(2, 14, 64, device=DEV)
    want, want_lse = attend(q, kv, sc, table, [0, 1, 2], [700, 90])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, got_lse = attend(q, kv, sc, table, [0, 1, 2], [700, 90])
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)


@pytest.mark.parametrize("n_q", [1, 100])
def test_the_same_bits_every_time_and_in_a_graph(n_q):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(9)
    kv, sc, table = make_cache(gen, [3000, 500], 16, 4, 128)
    q = torch.randn(2 * n_q, 28, 128, device=DEV).to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    qs, kl = i32([0, n_q, 2 * n_q]), i32([3000, 500])
    call = lambda: kv8().attention(q, kv, sc, table, qs, kl, n_q, 3000)
    want = call()
    for _ in range(3):
        assert torch.equal(call(), want)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        got = call()
    q.mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, call()) and not torch.equal(got, want)


# ---------------------------------------------------------------------------------------------- a step, and refusals

def test_plan_append_attention_over_several_steps():
    """Requests that start, grow, are cut back and end over shared pages: after every step each request's output is the
    attention over its own rows as the cache holds them."""
    rng = np.random.default_rng(11)
    page, kvh, H, hd, R, cols = 16, 2, 4, 64, 5, 12
    n_pages = 30
    kv, sc = kv8().allocate(n_pages, page, kvh, hd)
    ring, state = kv8().free_pool(n_pages)
    table = torch.full((R, cols), -1, dtype=torch.int32, device=DEV)
    cached = [0] * R
    rows = [[] for _ in range(R)]
    for step in range(12):
        total = []
        for r in range(R):
            kind = rng.integers(0, 6)
            total.append(0 if kind == 0 else cached[r] // 2 if kind == 1 else min(90, cached[r] + int(rng.choice([1, 1, 2, 40]))))
        tokens = sum(max(0, t - c) for c, t in zip(cached, total))
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        p = kv8().plan(i32(cached), i32(total), table, ring, state, page, tokens)
        assert p.status.tolist() == [0, 0]
        state = p.free_state
        k, v = torch.randn(2, tokens, kvh, hd, device=DEV).unbind(0)
        q = torch.randn(tokens, H, hd, device=DEV)
        kv8().append(kv, sc, k, v, p.slot)
        n_q = [max(0, t - c) for c, t in zip(cached, total)]
        at = 0
        for r in range(R):
            rows[r] = rows[r][: total[r]] + [k[at + i] for i in range(n_q[r])]
            at += n_q[r]
        cached = total
        if tokens == 0:
            continue
        o, lse = kv8().attention(q, kv, sc, table, p.q_start, p.kv_len, max(n_q), max(total), return_lse=True)
        q_start = [0] + np.cumsum(n_q).tolist()
        close(o, lse, ref_attention(q, kv, sc, table, q_start, total, hd ** -0.5, 0), torch.float32, False)
        for r in range(R):  # the rows are the ones that were appended, within their steps
            if total[r]:
                pos = torch.arange(total[r], device=DEV)
                slot = (table[r, (pos // page)] * page + pos % page).int()
                rk, _ = kv8().read(kv, sc, slot)
                steps = sc[table[r, (pos // page)].long(), 0][..., None]
                assert ((rk - torch.stack(rows[r])).abs() <= 2.501 * steps).all()
    live = sum(-(-c // page) for c in cached)
    head, tail = state.tolist()
    held = {int(x) for r in range(R) for x in table[r, : -(-cached[r] // page)].tolist()}
    free = {int(ring[i % n_pages]) for i in range(head, tail)}
    assert tail - head == n_pages - live and held | free == set(range(n_pages)) and not held & free


def test_refusals_of_the_python_calls():
    from e2e_browser_voice_agent_b200._lib import H2CError
    m = kv8()
    kv, sc = m.allocate(4, 16, 2, 64)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 4, 64, device=DEV)
    table = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    ok = lambda **kw: m.attention(**{**dict(q=q, kv=kv, kv_scale=sc, block_table=table, q_start=i32(0, 1), kv_len=i32(1),
                                            max_q=1, max_kv=1), **kw})
    ok()
    for kw in (dict(q=q.double()), dict(kv=kv.float()), dict(kv_len=torch.tensor([1], device=DEV))):
        with pytest.raises(TypeError):
            ok(**kw)
    for kw in (dict(q=q[:, :, :32]), dict(q=q.cpu()), dict(q_start=i32(0)), dict(block_table=table[0]), dict(kv_scale=sc[:2]),
               dict(out=torch.zeros(2, 4, 64, device=DEV)), dict(q=torch.zeros(1, 4, 64, 2, device=DEV)[..., 0])):
        with pytest.raises(ValueError):
            ok(**kw)
    for kw in (dict(q=torch.zeros(1, 3, 64, device=DEV)), dict(max_q=-1), dict(window=-1)):
        with pytest.raises(H2CError):
            ok(**kw)
    with pytest.raises(H2CError):  # a page size and a head dimension that the kernels do not have
        m.read(torch.zeros(4, 2, 2, 8, 64, dtype=torch.int8, device=DEV), sc, i32(0))
    with pytest.raises(H2CError):
        m.read(torch.zeros(4, 2, 2, 16, 80, dtype=torch.int8, device=DEV), sc, i32(0))
    with pytest.raises(ValueError):
        m.append(kv, sc, q[:, :2], q[:, :2], i32())
    with pytest.raises(ValueError):
        m.append(kv, sc, q[:, :2], q[:, :2].half(), i32(0))
    ring, state = m.free_pool(4)
    with pytest.raises(ValueError):
        m.plan(i32(0), i32(1), table[:, 0], ring, state, 16, 1)
    with pytest.raises(TypeError):
        m.plan(i32(0), i32(1), table, ring, state.int(), 16, 1)
    p = m.plan(i32(0), i32(1), table, ring, state, 16, 1)
    with pytest.raises(H2CError):  # the new ring state over the old one
        m.plan(i32(1), i32(2), table, ring, p.free_state, 16, 1, out=p)
    with pytest.raises(H2CError):
        m.plan(i32(0), i32(1), table, ring, state, 24, 1)
