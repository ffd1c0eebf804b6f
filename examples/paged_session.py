"""A small serving loop over the paged key/value cache: prompts of different
lengths are prefilled in chunks, decode steps append to the pages, attend with a
window and sinks or over everything while the attention weights are added up, and
when the caches pass their budget the least attended positions are evicted in
place and their pages go back to the pool.

    python examples/paged_session.py [--steps 24] [--window 0] [--sinks 4] [--budget 96]

Random weights of a small model; needs a B200 and torch for device memory."""
from __future__ import annotations

import argparse
import os
import sys
from types import SimpleNamespace

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "project-obsidian_b200"))
import obsmoe  # noqa: E402

H, INTER, EXPERTS, TOP_K, VOCAB = 2048, 256, 16, 4, 4096
HEADS, KV_HEADS, HEAD_DIM, PAGE = 16, 2, 128, 16


def quantised(rng, rows, cols):
    """A random MLX 4-bit group-64 matrix: codes, scales, biases (bf16 bits)."""
    w = rng.integers(0, 1 << 32, (rows, cols // 8), dtype=np.uint32)
    s = (rng.uniform(0.5, 1.0, (rows, cols // 64)) / (4 * np.sqrt(cols))).astype(np.float32)
    to_bf16 = lambda a: (a.view(np.uint32) >> 16).astype(np.uint16)  # noqa: E731
    return w, to_bf16(s), to_bf16((-7.5 * s).astype(np.float32))


def make_model(n_layers, max_tokens, max_seq, n_seqs, seed=0):
    """A context with every layer's experts, attention and the model's ends.  Its n_seqs sequences live in the
    session's pages: no dense caches.  max_seq: RoPE's positions, which go on after an eviction."""
    rng = np.random.default_rng(seed)
    ctx = obsmoe.MoeContext(obsmoe.MoeShape(H, INTER, EXPERTS, TOP_K, n_layers=n_layers, max_tokens=max_tokens))
    ctx.attn_init(HEADS, KV_HEADS, HEAD_DIM, max_seq, n_seqs=0)
    ones = np.full(H, 0x3F80, np.uint16)
    for layer in range(n_layers):
        ctx.synth_layer(layer, seed)
        w = {"in_norm": ones, "q_norm": ones[:HEAD_DIM], "k_norm": ones[:HEAD_DIM]}
        for name, rows, cols in (("q", HEADS * HEAD_DIM, H), ("k", KV_HEADS * HEAD_DIM, H), ("v", KV_HEADS * HEAD_DIM, H),
                                 ("o", H, HEADS * HEAD_DIM)):
            w[name + "_w"], w[name + "_s"], w[name + "_b"] = quantised(rng, rows, cols)
        ctx.load_attn(layer, SimpleNamespace(**w))
    ew, es, eb = quantised(rng, VOCAB, H)
    lw, ls, lb = quantised(rng, VOCAB, H)
    ctx.load_head(VOCAB, SimpleNamespace(embed_w=ew, embed_s=es, embed_b=eb, lm_w=lw, lm_s=ls, lm_b=lb, norm_w=ones))
    return ctx


class Session:
    """The pages of n_seqs sequences in every layer, and the model's steps over them."""

    def __init__(self, torch, ctx, n_layers, n_seqs, max_len, window=0, sinks=0, weights=False):
        self.torch, self.ctx, self.layers, self.n = torch, ctx, n_layers, n_seqs
        self.window, self.sinks = window, sinks
        per = -(-max_len // PAGE)
        ctx.paged_init(HEADS, KV_HEADS, HEAD_DIM, PAGE, max_seqs=n_seqs, max_kv_len=per * PAGE, weights=weights)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.free = list(range(n_seqs * per))  # one list: every layer's pool has the same pages in use
        self.table = torch.full((n_seqs, per), -1, **i32)
        self.len = torch.zeros(n_seqs, **i32)       # positions held
        self.pos = [0] * n_seqs                     # tokens seen (RoPE's positions)
        self.held = [0] * n_seqs                    # positions held, on the host
        self.pages = [0] * n_seqs
        self.kv = []
        for _ in range(n_layers):
            k, v = (torch.zeros((n_seqs * per, PAGE, KV_HEADS, HEAD_DIM), dtype=torch.bfloat16, device="cuda") for _ in "kv")
            self.kv.append(obsmoe.PagedKV(k, v, self.table, self.len))
        self.w = [torch.zeros((n_seqs, KV_HEADS, per * PAGE), device="cuda") if weights else None for _ in range(n_layers)]

    def grow(self, counts):
        """Room for counts[s] more positions of each sequence; the new tokens' (seq, pos, slot)."""
        seq, pos, slot = [], [], []
        for s, c in enumerate(counts):
            while self.pages[s] * PAGE < self.held[s] + c:
                self.table[s, self.pages[s]] = self.free.pop()
                self.pages[s] += 1
            seq += [s] * c
            pos += range(self.pos[s], self.pos[s] + c)
            slot += range(self.held[s], self.held[s] + c)
            self.pos[s] += c
            self.held[s] += c
        t = self.torch
        self.len.copy_(t.tensor(self.held, dtype=t.int32))
        return (t.tensor(a, dtype=t.int32, device="cuda") for a in (seq, pos, slot))

    def forward(self, tokens, counts, q_start=None):
        """One step of the model over counts[s] new tokens of each sequence (q_start None: one each, a decode
        step); the residual stream after the last layer."""
        t, T = self.torch, len(tokens)
        seq, pos, slot = self.grow(counts)
        x, y = (t.empty((T, H), dtype=t.bfloat16, device="cuda") for _ in "xy")
        self.ctx.embed(t.tensor(tokens, dtype=t.int32, device="cuda"), T, x)
        for layer in range(self.layers):
            self.ctx.paged_attn_forward(layer, self.kv[layer], x, y, T, seq, pos, slot, q_start, window=self.window,
                                        n_sink=self.sinks, weights=None if q_start is not None else self.w[layer])
            self.ctx.moe_stack_forward(layer, 1, y, T)
            x, y = y, x
        return x

    def next_tokens(self, x):
        ids = self.torch.empty(len(x), dtype=self.torch.int32, device="cuda")
        self.ctx.lm_head(x.contiguous(), len(x), ids)
        return ids.tolist()

    def prefill(self, prompts, chunk):
        """The prompts in chunks of at most `chunk` tokens a step; each prompt's next token."""
        t, done, last = self.torch, [0] * self.n, [None] * self.n
        while any(d < len(p) for d, p in zip(done, prompts)):
            counts, room = [], chunk
            for d, p in zip(done, prompts):
                counts.append(min(len(p) - d, room))
                room -= counts[-1]
            start = np.concatenate([[0], np.cumsum(counts)])
            tokens = [tok for p, d, c in zip(prompts, done, counts) for tok in p[d:d + c]]
            x = self.forward(tokens, counts, t.tensor(start, dtype=t.int32, device="cuda"))
            for s, c in enumerate(counts):
                done[s] += c
                if c and done[s] == len(prompts[s]):
                    last[s] = x[start[s + 1] - 1:start[s + 1]]
        return self.next_tokens(t.cat(last))

    def evict(self, budget, recent):
        """Every layer's caches to at most `budget` positions, in place; pages past them are free again."""
        t = self.torch
        kept = t.empty((self.n, KV_HEADS, budget), dtype=t.int32, device="cuda")
        new_len = t.empty_like(self.len)
        for layer in range(self.layers):
            self.ctx.paged_evict(self.kv[layer], self.kv[layer], self.w[layer], self.w[layer], budget, n_sink=self.sinks,
                                 n_recent=recent, kept=kept, new_len=new_len)
        self.len.copy_(new_len)
        self.held = new_len.tolist()
        for s in range(self.n):
            while (self.pages[s] - 1) * PAGE >= self.held[s]:
                self.pages[s] -= 1
                self.free.append(int(self.table[s, self.pages[s]]))
                self.table[s, self.pages[s]] = -1


def run(steps=24, window=0, sinks=4, budget=96, n_layers=2, lens=(150, 33, 77), chunk=64, seed=0, log=print):
    import torch

    rng = np.random.default_rng(seed)
    prompts = [rng.integers(0, VOCAB, n).tolist() for n in lens]
    max_len = max(lens) + steps
    ctx = make_model(n_layers, chunk, max_len, len(lens), seed)
    s = Session(torch, ctx, n_layers, len(lens), max_len, window, sinks, weights=budget > 0)
    tokens = s.prefill(prompts, chunk)
    out = [[t] for t in tokens]
    for step in range(1, steps):
        tokens = s.next_tokens(s.forward(tokens, [1] * len(lens)))
        for o, t in zip(out, tokens):
            o.append(t)
        if budget and step % 8 == 0 and max(s.held) > budget:
            before = len(s.free)
            s.evict(budget, budget // 4)
            log(f"step {step}: evicted to {s.held} positions, {len(s.free) - before} pages free again")
    ctx.check_device()
    for i, o in enumerate(out):
        log(f"sequence {i}: {lens[i]} prompt tokens, then {o}")
    held = list(s.held)
    ctx.close()
    return out, held


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("steps", 24), ("window", 0), ("sinks", 4), ("budget", 96)):
        ap.add_argument(f"--{name}", type=int, default=default)
    run(**vars(ap.parse_args()))
