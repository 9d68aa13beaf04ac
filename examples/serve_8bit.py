"""Serving many sessions with 8-bit weights and an 8-bit paged KV cache: the operators of kv8, int8, rope and logits together.

A Qwen2-shaped model of synth.CONFIGS with seeded weights: every projection is int8.matmul (weights quantized once), int8.norm adds
the residual stream up and makes the codes of its norm that the next product takes, rope.rotate turns queries and keys where they lie, K
and V go through kv8.append into pages that kv8.plan hands out from the sessions' lengths, and kv8.attention serves prompts and single
tokens of one step together. With a system prompt, all sessions lie behind one session that holds it, and kv8.prefix_attention reads it
once for all of them. logits.adjust penalizes what a session said already, and masks the tokens that may come. The gate is plain torch.

  python examples/serve_8bit.py [--model qwen2-0.5b] [--layers 4] [--sessions 8] [--steps 32] [--system 200] [--repetition 1.1]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from e2e_browser_voice_agent_b200 import int8, kv8, logits, rope, synth  # noqa: E402


class Server:
    """step({session: new token ids}) runs one step of the listed sessions and returns each one's logits after its last
    token; cut(session, n) keeps a session's first n tokens; end(session) frees it. share(ids), before the first step, makes ids the
    beginning of every session: they are held once, by one more session that the others lie behind."""

    def __init__(self, cfg, layers, sessions, pages, page_size=16, ctx=2048, dtype=torch.bfloat16, seed=0):
        self.cfg, self.layers, self.page, self.dtype = cfg, layers, page_size, dtype
        self.heads, self.kvh = cfg["heads"], cfg["kv_heads"]
        self.hd = cfg["dim"] // self.heads
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)

        def weight(n, k):  # as a checkpoint's rows, quantized once
            return int8.quantize(torch.randn(n, k, generator=gen, device="cuda") * k ** -0.5)

        d, f, kv = cfg["dim"], cfg["ffn"], self.kvh * self.hd
        self.embed = torch.randn(cfg["vocab"], d, generator=gen, device="cuda").to(dtype)
        self.head = weight(cfg["vocab"], d)
        self.w = [{"qkv": weight(d + 2 * kv, d), "bias": 0.02 * torch.randn(d + 2 * kv, generator=gen, device="cuda"),
                   "o": weight(d, d), "gate_up": weight(2 * f, d), "down": weight(d, f)} for _ in range(layers)]
        # one cache and pool per layer share the same tables: a page number is valid in each
        self.cache = [kv8.allocate(pages, page_size, self.kvh, self.hd) for _ in range(layers)]
        self.free, self.free_state = kv8.free_pool(pages)
        self.table = torch.full((sessions, ctx // page_size), -1, dtype=torch.int32, device="cuda")
        self.kv_len = torch.zeros(sessions, dtype=torch.int32, device="cuda")
        self.length = [0] * sessions  # the same on the host, which knows what it sends
        self.norms = [torch.ones(d, device="cuda") for _ in range(2 * layers + 1)]
        self.frequency = rope.frequencies(self.hd, cfg["rope_theta"])
        self.prefix = None  # (table, length, group) of the shared beginning, and its length here

    def _plan(self, total, tokens):
        """Pages and slots for the step that takes the sessions to these lengths."""
        p = kv8.plan(self.kv_len, torch.tensor(total, dtype=torch.int32, device="cuda"), self.table, self.free,
                     self.free_state, self.page, tokens)
        code, missing = p.status.tolist()  # (the one place where the host waits for the step's plan)
        if code == 1:
            raise RuntimeError(f"out of pages: {missing} missing")
        if code:
            raise RuntimeError(f"lengths {total} do not fit tables of {self.table.shape[1] * self.page} positions")
        self.kv_len, self.free_state, self.length = p.kv_len, p.free_state, total
        return p

    def cut(self, session, n):
        self._plan([min(n, x) if s == session else x for s, x in enumerate(self.length)], 0)

    def end(self, session):
        self.cut(session, 0)

    def share(self, ids):
        """The sessions' common beginning: a session of its own in the last row of the tables."""
        if any(self.length) or self.prefix:
            raise RuntimeError("the shared beginning comes before the first step")
        n, page = len(self.length), self.page
        self.table = torch.cat([self.table, torch.full_like(self.table[:1], -1)])
        self.kv_len = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
        self.length = [0] * (n + 1)
        self.step({n: ids})
        used = -(-len(ids) // page)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        self.prefix = (self.table[n:, :used].contiguous(), i32([len(ids)]), i32([0, n]))

    def _norm(self, x, i, **kw):
        n = int8.norm(x, self.norms[i], self.cfg["eps"], **kw)
        return (n.codes, {"x_scale": n.scale, "k": self.cfg["dim"], "out_dtype": self.dtype})

    def _attention(self, q, codes, scales, p, new, total):
        if self.prefix is None:
            return kv8.attention(q, codes, scales, self.table, p.q_start, p.kv_len, max(new), max(total), out=q)
        table, length, group = self.prefix
        return kv8.prefix_attention(q, codes, scales, table, length, group, self.table, p.q_start, p.kv_len, max(new),
                                    max(total[:-1]), self.length[-1], out=q)

    def step(self, fed):
        new = [len(fed.get(s, ())) for s in range(len(self.length))]
        tokens = sum(new)
        total = [a + b for a, b in zip(self.length, new)]
        p = self._plan(total, tokens)
        ids = torch.tensor([t for s in range(len(new)) for t in fed.get(s, ())], device="cuda")
        position = p.position if self.prefix is None else p.position + self.prefix[1]
        x, more = self.embed[ids], None  # the residual stream, and what the next norm adds to it
        d, kv = self.cfg["dim"], self.kvh * self.hd
        for i, (w, (codes, scales)) in enumerate(zip(self.w, self.cache)):
            xq, how = self._norm(x, 2 * i) if more is None else self._norm(more, 2 * i, residual=x, out=x)
            qkv = int8.matmul(xq, *w["qkv"], bias=w["bias"], **how)
            q, k, v = (qkv[:, a:b].view(tokens, -1, self.hd) for a, b in ((0, d), (d, d + kv), (d + kv, d + 2 * kv)))
            rope.rotate(q, position, self.frequency, k=k, out=q, k_out=k)
            kv8.append(codes, scales, k, v, p.slot)
            self._attention(q, codes, scales, p, new, total)
            o = int8.matmul(qkv[:, :d], *w["o"])
            xq, how = self._norm(o, 2 * i + 1, residual=x, out=x)
            gate, up = int8.matmul(xq, *w["gate_up"], **how).chunk(2, dim=-1)
            more = int8.matmul(torch.nn.functional.silu(gate) * up, *w["down"])
        last = [e - 1 for e in torch.tensor(new).cumsum(0).tolist()]
        live = [s for s in range(len(new)) if new[s]]
        rows = [last[s] for s in live]
        xq, how = self._norm(more[rows], -1, residual=x[rows])
        out = int8.matmul(xq, *self.head, **{**how, "out_dtype": torch.float32})
        return dict(zip(live, out))


def choose(rows, said, repetition=1.0, allowed=None):
    """The next token of each row of logits, of which said lists what was said before: the most likely one after a repetition
    penalty, among the allowed ones (a mask of the vocabulary, or None)."""
    columns = max(len(s) for s in said)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    tokens = i32([s + [-1] * (columns - len(s)) for s in said])
    bits = None
    if allowed is not None:
        on = torch.nn.functional.pad(allowed, (0, -len(allowed) % 32)).view(-1, 32).long()
        words = (on << torch.arange(32, device="cuda")).sum(-1)
        bits = torch.where(words >= 2**31, words - 2**32, words).int().expand(len(rows), -1)
    logits.adjust(rows, tokens=tokens, length=i32([len(s) for s in said]),
                  repetition=torch.full((len(rows),), repetition, device="cuda"), allowed=bits, out=rows)
    return rows.argmax(-1).tolist()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--model", default="qwen2-0.5b", choices=sorted(synth.CONFIGS))
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--sessions", type=int, default=8)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--system", type=int, default=0, help="tokens of a system prompt that all sessions share")
    ap.add_argument("--repetition", type=float, default=1.1, help="penalty for tokens that a session said already")
    a = ap.parse_args()
    cfg = synth.CONFIGS[a.model]
    server = Server(cfg, a.layers, a.sessions, pages=a.sessions * 64 + a.system // 16 + 1)
    if a.system:
        server.share(synth.prompt_ids(cfg["vocab"], a.system, seed=1000).tolist())
    feed = {s: synth.prompt_ids(cfg["vocab"], 20 + 37 * s, seed=s).tolist() for s in range(a.sessions)}
    out = {s: [] for s in feed}
    said = {s: list(ids) for s, ids in feed.items()}
    for i in range(a.steps):
        if i == 1:
            torch.cuda.synchronize()
            t0 = time.perf_counter()
        rows = server.step(feed)
        picked = choose(torch.stack(list(rows.values())), [said[s] for s in rows], a.repetition)
        feed = {s: [t] for s, t in zip(rows, picked)}
        for s, (t,) in feed.items():
            out[s].append(t)
            said[s].append(t)
        if i == a.steps // 2:  # one session ends in the middle; its pages serve the others
            server.end(0)
            feed.pop(0, None)
    torch.cuda.synchronize()
    for s in sorted(out):
        print(f"session {s}: {server.length[s]} tokens cached, {len(out[s])} generated: {out[s][:8]} ...")
    print(f"{a.layers} layers: {(time.perf_counter() - t0) / max(1, a.steps - 1) * 1e3:.2f} ms per step of up to {a.sessions} sessions")


if __name__ == "__main__":
    main()
