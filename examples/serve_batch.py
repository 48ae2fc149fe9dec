"""Serving several requests at once from one paged, 8-bit KV cache.

    python examples/serve_batch.py [--requests N] [--tokens N] [--cache q8_0|f16]

A small decoder with synthetic Q4_K weights (random, seeded) answers prompts of
different lengths: the prompts of newly admitted requests run packed through
the layers (kv_append, paged_attention_prefill), then every running request
takes one token per step (kv_append, paged_attention_decode), drawn with its
own temperature / top-k / top-p / min-p (sample).  Pages are taken from a
shared pool as sequences grow and go back when a request ends, so the next one
waiting can start.
"""
from __future__ import annotations

import argparse
import os
import sys
from dataclasses import dataclass, field

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import guanaco_b200 as gb  # noqa: E402


@dataclass
class Request:
    prompt: list
    n_new: int
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0
    tokens: list = field(default_factory=list)    # drawn so far
    pages: list = field(default_factory=list)


class Decoder:
    """Weights and the layers' arithmetic for packed rows of any number of sequences."""

    def __init__(self, hidden=512, heads=8, kv_heads=2, layers=2, ff=1024, vocab=1000, max_seq=4096, seed=1,
                 eps=1e-6):
        self.hidden, self.heads, self.kv, self.hd = hidden, heads, kv_heads, hidden // heads
        self.ff, self.vocab, self.eps, self.max_seq = ff, vocab, eps, max_seq
        self.width = (heads + 2 * kv_heads) * self.hd   # q, k, v of one projection
        mats = [("qkv", self.width, hidden), ("o", hidden, heads * self.hd), ("gate", ff, hidden), ("up", ff, hidden),
                ("down", hidden, ff)]
        self.layers, stream = [], 0

        def matrix(rows, cols):
            nonlocal stream
            stream += 1
            w = torch.zeros(gb.matrix_bytes(gb.DT_Q4_K, rows, cols) + 16, dtype=torch.uint8, device="cuda")
            gb.synth_blocks(gb.DT_Q4_K, w, rows * cols // 256, seed, stream)
            return w, rows, cols

        for _ in range(layers):
            self.layers.append({n: matrix(r, c) for n, r, c in mats})
        self.head = matrix(vocab, hidden)
        self.embedding = torch.empty(vocab * hidden, device="cuda")
        gb.synth_normal(self.embedding, vocab * hidden, seed, 0)
        self.embedding = self.embedding.view(vocab, hidden)
        self.rope = torch.empty(max_seq * self.hd, device="cuda")
        gb.rope_table(self.rope, max_seq, self.hd)

    def _gemm(self, w, x, out=None, residual=None):
        mat, rows, cols = w
        y = torch.empty(x.shape[0], rows, device="cuda") if out is None else out
        gb.gemm(gb.DT_Q4_K, mat, x, y, rows, cols, x.shape[0], R=residual)
        return y

    def _norm(self, x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.eps)

    def forward(self, tokens, caches, batch, ws, rows):
        """tokens: packed int64 ids of the batch; rows: whose logits to return."""
        x = self.embedding[tokens].contiguous()
        qd, kvd = self.heads * self.hd, self.kv * self.hd
        q = torch.empty(len(tokens), qd, device="cuda")
        attn = torch.empty_like(q)
        attend = gb.paged_attention_prefill if batch.cu_seqlens else gb.paged_attention_decode
        for w, cache in zip(self.layers, caches):
            qkv = self._gemm(w["qkv"], self._norm(x))
            gb.kv_append(cache, batch, qkv[:, qd: qd + kvd], qkv[:, qd + kvd:], q=qkv[:, :qd], q_out=q,
                         rope_cs=self.rope)
            attend(cache, batch, q, attn, ws)
            self._gemm(w["o"], attn, out=x, residual=x)
            xn = self._norm(x)
            gate, up = self._gemm(w["gate"], xn), self._gemm(w["up"], xn)
            gb.silu_mul(gate, up, gate.numel())
            self._gemm(w["down"], gate, out=x, residual=x)
        return self._gemm(self.head, self._norm(x[rows].contiguous()))


class Server:
    """Admits requests while pages last; one step() is a packed prefill of the
    newly admitted or a token for everyone running."""

    def __init__(self, model, n_pages=64, page_size=16, cache_type=gb.DT_Q8_0, max_running=16):
        self.m, self.page, self.max_running = model, page_size, max_running
        self.free = list(range(n_pages))[::-1]
        nbytes = n_pages * gb.kv_page_bytes(cache_type, model.kv, model.hd, page_size)
        self.caches = [gb.KVCache(cache_type, model.kv, model.hd, page_size, n_pages,
                                  torch.zeros(nbytes, dtype=torch.uint8, device="cuda"),
                                  torch.zeros(nbytes, dtype=torch.uint8, device="cuda")) for _ in model.layers]
        self.ws = torch.zeros(gb.paged_workspace_bytes(model.heads, model.kv, model.hd, max_running), dtype=torch.uint8,
                              device="cuda")
        self.waiting, self.running = [], []

    def submit(self, request):
        if not request.prompt or request.n_new < 1:
            raise ValueError("a request has a prompt and asks for tokens")
        if -(-(len(request.prompt) + request.n_new) // self.page) > len(self.free) + sum(
                len(r.pages) for r in self.running) or len(request.prompt) + request.n_new > self.m.max_seq:
            raise ValueError("request longer than the cache")
        self.waiting.append(request)

    def _run(self, reqs, tokens, q_lens):
        """Forward over the packed tokens, one drawn token for each request."""
        i32 = dict(dtype=torch.int32, device="cuda")
        lens = [len(r.prompt) + len(r.tokens) for r in reqs]
        table = torch.zeros(len(reqs), max(len(r.pages) for r in reqs), dtype=torch.int32)
        for i, r in enumerate(reqs):
            table[i, : len(r.pages)] = torch.tensor(r.pages, dtype=torch.int32)
        ends = torch.tensor(q_lens).cumsum(0)
        cu = None if max(q_lens) == 1 else torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(**i32)
        batch = gb.KVBatch(len(reqs), len(tokens), torch.tensor(lens, **i32), table.cuda(), cu)
        logits = self.m.forward(torch.tensor(tokens, device="cuda"), self.caches, batch, self.ws, (ends - 1).cuda())
        out = torch.empty(len(reqs), **i32)
        col = lambda name, dt: torch.tensor([getattr(r, name) for r in reqs], dtype=dt, device="cuda")  # noqa: E731
        # each request's own random stream, so that its answer does not depend on the batch
        u = torch.tensor([torch.rand(1, generator=torch.Generator().manual_seed(r.seed * 65537 + len(r.tokens))).item()
                          for r in reqs], device="cuda")
        gb.sample(logits, out, u, temperature=col("temperature", torch.float32), top_k=col("top_k", torch.int32),
                  top_p=col("top_p", torch.float32), min_p=col("min_p", torch.float32))
        for r, token in zip(reqs, out.tolist()):
            r.tokens.append(token)
        return logits

    def step(self):
        """Returns the requests that ended."""
        new = []
        while self.waiting and len(self.running) + len(new) < self.max_running:
            need = -(-(len(self.waiting[0].prompt) + self.waiting[0].n_new) // self.page)
            if need > len(self.free):
                break
            r = self.waiting.pop(0)
            r.pages = [self.free.pop() for _ in range(need)]
            new.append(r)
        if new:
            self._run(new, [t for r in new for t in r.prompt], [len(r.prompt) for r in new])
            self.running += new
        elif self.running:
            self._run(self.running, [r.tokens[-1] for r in self.running], [1] * len(self.running))
        done = [r for r in self.running if len(r.tokens) >= r.n_new]
        for r in done:
            self.free += r.pages
            r.pages = []
            self.running.remove(r)
        return done

    def run(self):
        while self.waiting or self.running:
            self.step()
        err = gb.paged_error(clear=True)
        if err:
            raise gb.GBError("paged kernels", err)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=24)
    ap.add_argument("--cache", choices=["q8_0", "f16"], default="q8_0")
    args = ap.parse_args()
    model = Decoder()
    server = Server(model, cache_type=gb.DT_Q8_0 if args.cache == "q8_0" else gb.DT_F16)
    g = torch.Generator().manual_seed(0)
    requests = []
    for i in range(args.requests):
        n = int(torch.randint(1, 200, (1,), generator=g))
        prompt = torch.randint(0, model.vocab, (n,), generator=g).tolist()
        settings = [dict(), dict(temperature=0.8, top_k=40), dict(temperature=1.0, top_p=0.9),
                    dict(temperature=0.7, top_p=0.95, min_p=0.05)][i % 4]
        requests.append(Request(prompt, args.tokens, seed=i, **settings))
        server.submit(requests[-1])
    server.run()
    for i, r in enumerate(requests):
        print(f"request {i}: {len(r.prompt)} prompt tokens ->", *r.tokens)


if __name__ == "__main__":
    main()
