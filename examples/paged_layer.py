"""One decoder layer's attention over a paged cache, as a server with continuous batching runs it: packed q, k, v and output
projections, and between them the cache.

    python examples/paged_layer.py [--steps 64]

Requests arrive one after another; a step takes one new token of every request that is generating and a chunk of the prompt
of one that is not.  The layer's input is random (there is no model here); what the steps return is compared with the same
attention over each whole request at once, and the time of a decode step is printed.
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import lloom_amd as L  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, PAGE = 2048, 16, 4, 128, 16


class Layer:
    """The attention of a layer: weights in Q4_K, keys and values in `pages` pages."""

    def __init__(self, pages, seed=0, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)

        def packed(n, k):
            w = torch.randn(n, k, device=device, generator=gen) / math.sqrt(k)
            return L.QMatMul.from_qtensor(L.QTensor.quantize(w, L.GgmlDType.Q4K))

        self.q, self.o = packed(HEADS * DIM, HIDDEN), packed(HIDDEN, HEADS * DIM)
        self.k, self.v = packed(KV_HEADS * DIM, HIDDEN), packed(KV_HEADS * DIM, HIDDEN)
        self.cache = L.PagedCache(pages, PAGE, KV_HEADS, DIM, device)

    def __call__(self, x, plan, max_new):
        n = x.shape[0]
        self.cache.append(self.k.forward(x).view(n, KV_HEADS, DIM), self.v.forward(x).view(n, KV_HEADS, DIM), plan.slots)
        y = self.cache.attention(self.q.forward(x).view(n, HEADS, DIM), plan, max_new=max_new)
        return self.o.forward(y.view(n, HEADS * DIM))


class Server:
    """The host's part of continuous batching: each request's length and pages, and what a step takes of it."""

    def __init__(self, layer, pages, requests, most, chunk, device="cuda"):
        self.layer, self.chunk, self.dev = layer, chunk, device
        self.free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(device, torch.int32)
        self.tables = torch.zeros(requests, -(-most // PAGE), dtype=torch.int32, device=device)
        self.done = [0] * requests

    def _ints(self, v):
        return torch.tensor(v, dtype=torch.int32, device=self.dev)

    def step(self, new, x):
        """new[b] tokens of request b, their rows of x side by side."""
        plan = L.paged_plan(self._ints(self.done), self._ints(new), x.shape[0], self.tables, self.free, PAGE)
        taken = sum(-(-(d + n) // PAGE) - -(-d // PAGE) for d, n in zip(self.done, new))
        self.free = self.free[taken:]
        self.done = [d + n for d, n in zip(self.done, new)]
        return self.layer(x, plan, max(new))

    def take(self, prompts):
        """What the next step takes: one token of each finished prompt, a chunk of the first that is not."""
        new, read = [0] * len(prompts), False
        for b, (d, p) in enumerate(zip(self.done, prompts)):
            if d >= p:
                new[b] = 1
            elif not read:
                new[b], read = min(self.chunk, p - d), True
        return new


def whole(layer, x):
    """The layer over one whole request, with plain products in f32 over the packed projections' outputs."""
    n = x.shape[0]
    q = layer.q.forward(x).view(n, HEADS, DIM)
    k, v = (m.forward(x).view(n, KV_HEADS, DIM).half().float() for m in (layer.k, layer.v))
    y = torch.empty(n, HEADS, DIM, device=x.device)
    later = torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1)
    for h in range(HEADS):
        j = h // (HEADS // KV_HEADS)
        z = torch.mm(q[:, h], k[:, j].t().contiguous()) / math.sqrt(DIM)
        y[:, h] = torch.mm(torch.softmax(z.masked_fill(later, -math.inf), 1), v[:, j])
    return layer.o.forward(y.view(n, -1))


def run(prompts=(300, 37, 700, 1), steps=24, chunk=256, seed=0, device="cuda"):
    """Largest difference of the steps' outputs from `whole`'s, relative to the outputs' size; and the microseconds of a
    decode step (all prompts read)."""
    gen = torch.Generator(device=device).manual_seed(seed)
    most = max(prompts) + 2 * steps
    pages = len(prompts) * -(-most // PAGE)
    layer = Layer(pages, seed, device)
    server = Server(layer, pages, len(prompts), most, chunk, device)
    inputs, outputs = [[] for _ in prompts], [[] for _ in prompts]
    times = []
    for _ in range(steps):
        new = server.take(prompts)
        x = torch.randn(sum(new), HIDDEN, device=device, generator=gen)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        y = server.step(new, x)
        end.record()
        times.append((max(new), start, end))
        for b, (xs, ys) in enumerate(zip(x.split(new), y.split(new))):
            inputs[b].append(xs)
            outputs[b].append(ys)
    L.paged_check()
    worst = 0.0
    for xs, ys in zip(inputs, outputs):
        want = whole(layer, torch.cat(xs))
        worst = max(worst, ((torch.cat(ys) - want).norm() / want.norm()).item())
    decode = sorted(a.elapsed_time(b) * 1e3 for n, a, b in times if n == 1)
    return worst, decode[len(decode) // 2] if decode else None


if __name__ == "__main__":
    p = argparse.ArgumentParser()
    p.add_argument("--steps", type=int, default=64)
    worst, us = run(steps=p.parse_args().steps)
    print(f"relative difference from whole requests {worst:.1e}; a decode step of the layer {us:.0f} us")
