"""Serving many sessions with 8-bit weights and an 8-bit paged KV cache: the operators of kv8 and int8 together.

A Qwen2-shaped model of synth.CONFIGS with seeded weights: every projection is int8.matmul (weights quantized once, tokens on
the way), K and V go through kv8.append into pages that kv8.plan hands out from the sessions' lengths, and kv8.attention
serves prompts and single tokens of one step together. Norms, RoPE and the gate are plain torch.

  python examples/serve_8bit.py [--model qwen2-0.5b] [--layers 4] [--sessions 8] [--steps 32]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from e2e_browser_voice_agent_b200 import int8, kv8, synth  # noqa: E402


class Server:
    """step({session: new token ids}) runs one step of the listed sessions and returns each one's logits after its last
    token; cut(session, n) keeps a session's first n tokens; end(session) frees it."""

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
        inv = cfg["rope_theta"] ** (-torch.arange(0, self.hd, 2, device="cuda", dtype=torch.float64) / self.hd)
        angle = torch.arange(ctx, device="cuda", dtype=torch.float64)[:, None] * inv
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

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

    def _norm(self, x):
        return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + self.cfg["eps"])).to(self.dtype)

    def _rope(self, x, position):
        a, b = x.float().chunk(2, dim=-1)
        c, s = self.cos[position][:, None], self.sin[position][:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1).to(self.dtype)

    def step(self, fed):
        new = [len(fed.get(s, ())) for s in range(len(self.length))]
        tokens = sum(new)
        total = [a + b for a, b in zip(self.length, new)]
        p = self._plan(total, tokens)
        ids = torch.tensor([t for s in range(len(new)) for t in fed.get(s, ())], device="cuda")
        position = p.position.long()
        x = self.embed[ids]
        d, kv = self.cfg["dim"], self.kvh * self.hd
        for w, (codes, scales) in zip(self.w, self.cache):
            qkv = int8.matmul(self._norm(x), *w["qkv"], bias=w["bias"])
            q = self._rope(qkv[:, :d].view(tokens, self.heads, self.hd), position)
            k = self._rope(qkv[:, d:d + kv].view(tokens, self.kvh, self.hd), position)
            kv8.append(codes, scales, k, qkv[:, d + kv:].view(tokens, self.kvh, self.hd), p.slot)
            att = kv8.attention(q, codes, scales, self.table, p.q_start, p.kv_len, max(new), max(total))
            x = x + int8.matmul(att.view(tokens, d), *w["o"])
            gate, up = int8.matmul(self._norm(x), *w["gate_up"]).chunk(2, dim=-1)
            x = x + int8.matmul(torch.nn.functional.silu(gate) * up, *w["down"])
        last = [e - 1 for e in torch.tensor(new).cumsum(0).tolist()]
        live = [s for s in range(len(new)) if new[s]]
        logits = int8.matmul(self._norm(x[[last[s] for s in live]]), *self.head, out_dtype=torch.float32)
        return dict(zip(live, logits))


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--model", default="qwen2-0.5b", choices=sorted(synth.CONFIGS))
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--sessions", type=int, default=8)
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    cfg = synth.CONFIGS[a.model]
    server = Server(cfg, a.layers, a.sessions, pages=a.sessions * 64)
    feed = {s: synth.prompt_ids(cfg["vocab"], 20 + 37 * s, seed=s).tolist() for s in range(a.sessions)}
    out = {s: [] for s in feed}
    for i in range(a.steps):
        if i == 1:
            torch.cuda.synchronize()
            t0 = time.perf_counter()
        logits = server.step(feed)
        feed = {s: [int(t)] for s, t in zip(logits, torch.stack(list(logits.values())).argmax(-1).tolist())}
        for s, (t,) in feed.items():
            out[s].append(t)
        if i == a.steps // 2:  # one session ends in the middle; its pages serve the others
            server.end(0)
            feed.pop(0, None)
    torch.cuda.synchronize()
    for s in sorted(out):
        print(f"session {s}: {server.length[s]} tokens cached, {len(out[s])} generated: {out[s][:8]} ...")
    print(f"{a.layers} layers: {(time.perf_counter() - t0) / max(1, a.steps - 1) * 1e3:.2f} ms per step of up to {a.sessions} sessions")


if __name__ == "__main__":
    main()
