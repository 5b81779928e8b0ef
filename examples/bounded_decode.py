"""Decoding in bounded memory: one attention layer over an 8-bit KV cache that is cut back to a budget as it grows.

A batch of sequences is decoded greedily by a one-layer model with random weights (embedding, q/k/v/o projections of the
1B Granite's heads, an untied head).  Each step appends the new tokens' K and V to the cache, attends over it while the
weights that each slot receives accumulate, and, once the longest sequence reaches `limit` slots, evicts every sequence to
`budget` slots: the latest `recent` and the heaviest of the others.  Memory is that of two caches of `limit` slots (eviction
writes from one to the other) however long the sequences get.

    python examples/bounded_decode.py --tokens 300 --limit 256 --budget 128
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lastro-rust_b200"))
import lastro_b200 as LB  # noqa: E402


class Pages:
    """One cache's buffers: every sequence has `slots` slots in pages of its own."""

    def __init__(self, ctx, fmt, n_seqs, kv_heads, head_dim, slots):
        per = -(-slots // LB.KV8_PAGE)
        total, blocks = n_seqs * per, LB.KV8_PAGE // LB.KV8_BLOCK
        self.k, self.v = torch.empty((2, total, kv_heads, LB.KV8_PAGE, head_dim), dtype=torch.uint8, device="cuda").unbind()
        self.k_scale, self.v_scale = torch.empty((2, total, kv_heads, blocks), device="cuda").unbind()
        self.table = torch.arange(total, dtype=torch.int32, device="cuda").view(n_seqs, per)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.cache = LB.Kv8Cache(ctx, fmt, n_seqs, kv_heads, head_dim, total, per, self.k, self.v, self.k_scale,
                                 self.v_scale, self.table, self.status)


class BoundedCache:
    """Two sets of pages, of which one is in use: eviction writes the kept rows to the other."""

    def __init__(self, ctx, fmt, n_seqs, heads, kv_heads, head_dim, limit, budget, recent, max_new=1):
        self.n, self.heads, self.kv, self.limit, self.budget, self.recent = n_seqs, heads, kv_heads, limit, budget, recent
        self.slots = -(-limit // LB.KV8_PAGE) * LB.KV8_PAGE
        self.pages = [Pages(ctx, fmt, n_seqs, kv_heads, head_dim, limit) for _ in range(2)]
        self.mass = [torch.zeros((n_seqs, kv_heads, self.slots), device="cuda") for _ in range(2)]
        self.lens = [torch.zeros(n_seqs, dtype=torch.int32, device="cuda") for _ in range(2)]
        self.kept = torch.empty((n_seqs, kv_heads, budget), dtype=torch.int32, device="cuda")
        self.bytes = self.pages[0].cache.attend_workspace(heads, max_new, True)
        self.work = torch.empty(self.bytes, dtype=torch.uint8, device="cuda")
        self.max_new, self.longest, self.evictions = max_new, 0, 0

    def step(self, q, k, v, off, scale):
        """The new rows of every sequence (off: their offsets): into the cache, then attention over it."""
        if self.longest + self.max_new > self.limit:
            self._evict()
        pages, mass = self.pages[0], self.mass[0]
        pages.cache.append(self.lens[0], off, self.max_new, LB.rows_of(k), LB.rows_of(v), self.lens[1], mass, self.slots)
        self.lens.reverse()
        self.longest += self.max_new
        out = torch.empty_like(q)
        pages.cache.attend(self.lens[0], off, self.max_new, self.heads, LB.rows_of(q), scale, LB.rows_of(out), self.work,
                           self.bytes, mass_in=mass, mass_out=mass, mass_stride=self.slots)
        return out

    def _evict(self):
        self.pages[0].cache.evict(self.pages[1].cache, self.lens[0], self.budget, self.recent, self.mass[0], self.slots,
                                  self.kept, self.lens[1], self.mass[1], self.slots)
        for pair in (self.pages, self.mass, self.lens):
            pair.reverse()
        self.longest, self.evictions = self.budget, self.evictions + 1


def decode(n_seqs=4, tokens=300, limit=256, budget=128, recent=32, fmt="e4m3", seed=0):
    """Greedy ids [n_seqs, tokens] and the cache."""
    cfg = LB.configs.GRANITE_1B
    heads, kv, d, vocab = cfg["heads"], cfg["kv_heads"], cfg["head_dim"], 2048
    hidden = heads * d
    gen = torch.Generator("cuda").manual_seed(seed)

    def weight(*shape):
        return (torch.randn(shape, generator=gen, device="cuda") * shape[-1] ** -0.5).bfloat16()

    embed, head, wqkv, wo = weight(vocab, hidden) * 32, weight(vocab, hidden), weight((heads + 2 * kv) * d, hidden), weight(hidden, heads * d)
    ctx = LB.Context(0, torch.cuda.current_stream().cuda_stream or LB.LEGACY_STREAM)
    cache = BoundedCache(ctx, fmt, n_seqs, heads, kv, d, limit, budget, recent)
    off = torch.arange(n_seqs + 1, dtype=torch.int32, device="cuda")
    token = torch.arange(n_seqs, device="cuda") * 7 % vocab
    ids = []
    for _ in range(tokens):
        x = embed[token]
        qkv = (x @ wqkv.T).view(n_seqs, heads + 2 * kv, d)
        att = cache.step(qkv[:, :heads].contiguous(), qkv[:, heads:heads + kv], qkv[:, heads + kv:], off, d ** -0.5)
        token = ((x + att.reshape(n_seqs, -1) @ wo.T) @ head.T).argmax(-1)
        ids.append(token)
    out = torch.stack(ids, 1).cpu()
    if cache.pages[0].status.item() or cache.pages[1].status.item():
        raise RuntimeError("the cache's kernels met a page, length or offset they could not use")
    return out, cache


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--sequences", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=300)
    ap.add_argument("--limit", type=int, default=256)
    ap.add_argument("--budget", type=int, default=128)
    ap.add_argument("--recent", type=int, default=32)
    ap.add_argument("--format", choices=sorted(LB.KV8_FORMATS), default="e4m3")
    a = ap.parse_args()
    if not (0 <= a.recent <= a.budget < a.limit and a.budget > 0):
        ap.error("0 <= recent <= budget, 0 < budget < limit")
    ids, cache = decode(a.sequences, a.tokens, a.limit, a.budget, a.recent, a.format)
    for b in range(a.sequences):
        print(f"sequence {b}: {ids[b, :12].tolist()} ...")
    print(f"{a.tokens} tokens a sequence in {cache.slots} slots, {cache.evictions} evictions to {a.budget}")


if __name__ == "__main__":
    main()
