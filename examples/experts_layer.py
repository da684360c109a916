"""Serving a layer of experts in FP8 block scale.

Each token's logits choose `top` of the experts (experts.route: a sigmoid of each with a
bias for balance, or a softmax; groups of experts), the pairs of tokens and experts are put in
the order of the experts (arrange), and the layer's two products run over each
expert's rows (product), the gated activation between them (activate), the weighted sum
behind them (combine). Weights are quantised once, activations as they come. Nothing comes
back to the host: a step of the same number of tokens can be captured into a graph.

With --shards N the experts lie on N processes; this one computes the part of shard
--shard, and the parts add up to the layer (over one process each by all_reduce).

    python examples/experts_layer.py --tokens 64 --experts 128 --top 8 --graph
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from gcnasm_amd import experts, ops  # noqa: E402


class Layer:
    """Experts first .. first + held - 1 of a layer of `count`."""

    def __init__(self, hidden, inner, count, top, device, first=0, held=None, groups=1,
                 top_groups=1, scores="sigmoid", seed=0):
        self.top, self.first = top, first
        self.held = count - first if held is None else held
        self.choice = dict(scores=scores, groups=groups, top_groups=top_groups,
                           group_rank=2 if groups > 1 else 1)
        g = torch.Generator(device).manual_seed(seed)
        self.gate = torch.randn((count, hidden), generator=g, device=device) * hidden ** -0.5
        self.bias = 0.01 * torch.randn(count, generator=g, device=device)
        w1, w2 = [], []
        for e in range(count):  # every process draws them all, and keeps its own
            up = torch.randn((2 * inner, hidden), generator=g, device=device) * hidden ** -0.5
            down = torch.randn((hidden, inner), generator=g, device=device) * inner ** -0.5
            if first <= e < first + self.held:
                w1.append(ops.quant_fp8_128x128(up))
                w2.append(ops.quant_fp8_128x128(down))
        self.w1, self.s1 = (torch.stack(t) for t in zip(*w1))
        self.w2, self.s2 = (torch.stack(t) for t in zip(*w2))

    def route(self, x):
        bias = self.bias if self.choice["scores"] == "sigmoid" else None
        return experts.route(x.float() @ self.gate.t(), self.top, bias=bias, **self.choice)

    def __call__(self, x):
        """x [tokens, hidden] bfloat16 -> what this process's experts add to the layer."""
        ids, weights = self.route(x)
        starts, tokens, place = experts.arrange(ids, self.held, self.first)
        q, s = ops.quant_fp8_1x128(x)
        h = experts.product(q, s, self.w1, self.s1, starts, rows=tokens)
        q, s = experts.activate(h, starts)
        return experts.combine(experts.product(q, s, self.w2, self.s2, starts), place, weights)


class Graph:
    """A layer's step for a fixed number of tokens, captured once."""

    def __init__(self, layer, tokens, hidden, device):
        self.x = torch.zeros((tokens, hidden), dtype=torch.bfloat16, device=device)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(self.x)
        torch.cuda.current_stream().wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.y = layer(self.x)

    def __call__(self, x):
        self.x.copy_(x)
        self.graph.replay()
        return self.y


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--tokens", type=int, default=64)
    p.add_argument("--hidden", type=int, default=4096)
    p.add_argument("--inner", type=int, default=1024)
    p.add_argument("--experts", type=int, default=128)
    p.add_argument("--top", type=int, default=8)
    p.add_argument("--groups", type=int, default=1)
    p.add_argument("--top-groups", type=int, default=1)
    p.add_argument("--scores", choices=("sigmoid", "softmax"), default="sigmoid")
    p.add_argument("--shards", type=int, default=1)
    p.add_argument("--shard", type=int, default=0)
    p.add_argument("--steps", type=int, default=100)
    p.add_argument("--graph", action="store_true", help="capture the step into a graph")
    a = p.parse_args(argv)
    if not 1 <= a.shards <= a.experts or not 0 <= a.shard < a.shards:
        p.error("--shard must be 0 .. shards - 1, --shards 1 .. experts")
    device = torch.device("cuda")
    first = a.shard * a.experts // a.shards
    held = (a.shard + 1) * a.experts // a.shards - first
    layer = Layer(a.hidden, a.inner, a.experts, a.top, device, first, held, a.groups,
                  a.top_groups, a.scores)
    step = Graph(layer, a.tokens, a.hidden, device) if a.graph else layer
    g = torch.Generator(device).manual_seed(1)
    xs = [torch.randn((a.tokens, a.hidden), generator=g, device=device).bfloat16()
          for _ in range(3)]
    y = step(xs[0])
    torch.cuda.synchronize()
    begin = time.perf_counter()
    for i in range(a.steps):
        y = step(xs[i % 3])
    torch.cuda.synchronize()
    us = (time.perf_counter() - begin) * 1e6 / max(a.steps, 1)
    print("%d tokens, %d of %d experts (%d here), %d x %d: %.1f us a step" %
          (a.tokens, a.top, a.experts, held, a.hidden, a.inner, us))
    return layer, y


if __name__ == "__main__":
    main()
