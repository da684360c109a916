"""Serving one attention layer with the MXFP4 key/value cache.

A batch of prompts of different lengths goes through the layer at once, then
every sequence grows by a token a step. The projections are MXFP8 products
(ops.mxfp8_gemm), keys and values go into the cache as they come (append), the
rows attend to it (attention), and what each token is given is added up
(attention_weights). Once the sequences have grown by `slack` tokens past `keep`, the
cache is thinned: the latest `recent` tokens and those with the most weight move to
fresh pages (evict) and the old pages are free again.

append() quantises by its default rule here; scale_rule=GA_MX_SCALE_OCP loses less
(values 0.12 of their root mean square instead of 0.20).

    python examples/mx4_cache_serving.py --seqs 16 --prompt 2000 --steps 300

The host knows every length (a sequence of more than `keep` tokens has `keep` of them
after an eviction), so none has to come back from the GPU.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from gcnasm_amd import mx4_cache, ops  # noqa: E402


class Pages:
    """Which pages of the cache are in use, and the table of the sequences' pages."""

    def __init__(self, num_pages, seqs, per_seq, page_size, device):
        self.free = list(range(num_pages))
        self.page_size, self.per_seq, self.device = page_size, per_seq, device
        self.held = [[] for _ in range(seqs)]
        self.table = torch.full((seqs, per_seq), -1, dtype=torch.int32, device=device)

    def grow(self, lens):
        """Pages for so many tokens of each sequence."""
        rows, cols, ids = [], [], []
        for b, n in enumerate(lens):
            while len(self.held[b]) * self.page_size < n:
                rows.append(b)
                cols.append(len(self.held[b]))
                ids.append(self.free.pop())
                self.held[b].append(ids[-1])
        if ids:
            self.table[rows, cols] = torch.tensor(ids, dtype=torch.int32, device=self.device)

    def slots(self, first, lens):
        """Slots of tokens first[b] .. lens[b] - 1 of the sequences, one after the other."""
        s = [self.held[b][t // self.page_size] * self.page_size + t % self.page_size
             for b in range(len(lens)) for t in range(first[b], lens[b])]
        return torch.tensor(s, dtype=torch.int64, device=self.device)

    def fresh(self, lens):
        """Other pages for so many tokens; the old ones are free for the next call."""
        other = Pages(0, len(self.held), self.per_seq, self.page_size, self.device)
        other.free = self.free
        other.grow(lens)
        for held in self.held:
            self.free.extend(held)
        return other


class Layer:
    def __init__(self, hidden, heads, kv_heads, head_dim, device, seed=0):
        g = torch.Generator(device).manual_seed(seed)
        self.heads, self.kv_heads, self.dim = heads, kv_heads, head_dim

        def weight(n, k):
            w = torch.randn((n, k), generator=g, device=device) * k ** -0.5
            return ops.prepare_mx_b(w.bfloat16())

        self.qkv = weight((heads + 2 * kv_heads) * head_dim, hidden)
        self.out = weight(hidden, heads * head_dim)

    def project(self, x):
        y = ops.mxfp8_gemm(ops.prepare_mx_a(x), self.qkv)[0]
        y = y[:x.shape[0]].view(x.shape[0], -1, self.dim)
        return y.split([self.heads, self.kv_heads, self.kv_heads], 1)

    def finish(self, out):
        y = ops.mxfp8_gemm(ops.prepare_mx_a(out.flatten(1)), self.out)[0]
        return y[:out.shape[0]]


class Server:
    """The layer, its cache and its sequences."""

    def __init__(self, layer, seqs, keep, recent, slack, prompt, page_size=64, device="cuda"):
        self.layer, self.keep, self.recent, self.device = layer, keep, recent, device
        self.limit = keep + slack
        self.most = max(prompt, self.limit)
        per_seq = (self.most + page_size - 1) // page_size
        kept = (keep + page_size - 1) // page_size  # the fresh pages of an eviction
        num_pages = seqs * (per_seq + kept)
        self.cache = mx4_cache.new_cache(num_pages, layer.kv_heads, layer.dim, page_size, device)
        self.pages = Pages(num_pages, seqs, per_seq, page_size, device)
        self.lens = [0] * seqs
        self.weights = torch.zeros((seqs, layer.kv_heads, self.most), device=device)
        self.evictions = 0

    def step(self, x, new):
        """x [sum of new, hidden] bfloat16, new[b] rows of each sequence -> the layer's output."""
        first = self.lens
        self.lens = [n + m for n, m in zip(first, new)]
        self.pages.grow(self.lens)
        lens = torch.tensor(self.lens, dtype=torch.int32, device=self.device)
        starts = None
        if max(new) > 1 or min(new) < 1:
            starts = torch.tensor([0] + new, device=self.device).cumsum(0).int()
        q, k, v = self.layer.project(x)
        mx4_cache.append(self.cache, k, v, self.pages.slots(first, self.lens))
        rows = dict(q_starts=starts, max_q=max(new), max_len=max(self.lens))
        out, lse = mx4_cache.attention(q, self.cache, self.pages.table, lens, **rows)
        mx4_cache.attention_weights(q, self.cache, self.pages.table, lens, lse, self.weights,
                                    out=self.weights, **rows)
        if max(self.lens) >= self.limit:
            self.evict(lens)
        return self.layer.finish(out)

    def evict(self, lens):
        left = [min(n, self.keep) for n in self.lens]
        old, self.pages = self.pages, self.pages.fresh(left)
        weights = torch.empty_like(self.weights)
        mx4_cache.evict(self.cache, old.table, lens, self.weights, self.keep, self.recent,
                        self.pages.table, self.layer.dim, new_weights=weights)
        self.lens, self.weights = left, weights
        self.evictions += 1


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--seqs", type=int, default=16)
    p.add_argument("--prompt", type=int, default=2000, help="longest prompt; the others from half")
    p.add_argument("--steps", type=int, default=300)
    p.add_argument("--keep", type=int, default=1024)
    p.add_argument("--recent", type=int, default=256)
    p.add_argument("--slack", type=int, default=128)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--heads", type=int, default=32)
    p.add_argument("--kv-heads", type=int, default=8)
    p.add_argument("--head-dim", type=int, default=128)
    a = p.parse_args(argv)
    device = torch.device("cuda")
    layer = Layer(a.hidden, a.heads, a.kv_heads, a.head_dim, device)
    server = Server(layer, a.seqs, a.keep, a.recent, a.slack, a.prompt, device=device)
    g = torch.Generator(device).manual_seed(1)
    new = [a.prompt - b * (a.prompt // 2) // max(a.seqs, 1) for b in range(a.seqs)]
    x = torch.randn((sum(new), a.hidden), generator=g, device=device).bfloat16()
    y = server.step(x, new)
    torch.cuda.synchronize()
    x = torch.randn((a.seqs, a.hidden), generator=g, device=device).bfloat16()
    begin = time.perf_counter()
    for _ in range(a.steps):
        y = server.step(x, [1] * a.seqs)
    torch.cuda.synchronize()
    ms = (time.perf_counter() - begin) * 1e3 / max(a.steps, 1)
    size = 2 * layer.kv_heads * layer.dim
    print("%d sequences, prompts of up to %d tokens, %d steps: %.3f ms a step, %d evictions" %
          (a.seqs, a.prompt, a.steps, ms, server.evictions))
    print("a token takes %d bytes of cache, %d in bfloat16; now %d to %d tokens a sequence" %
          (size * 17 // 32, 2 * size, min(server.lens), max(server.lens)))
    return server, y


if __name__ == "__main__":
    main()
