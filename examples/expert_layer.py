"""A layer of routed experts with 8-bit floating-point weights, as a server runs it: router, gate and up, silu(gate) * up, down,
and the sum of each token's experts.

    python examples/expert_layer.py [--steps 20]

The weights are random (there is no model here), brought into 8 bits from f32; what a step returns is compared with the layer in
plain f32 products over the weights as they were, and the time of a step is printed.
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import lloom_amd as L  # noqa: E402

HIDDEN, INNER, EXPERTS, TOPK = 2048, 768, 32, 4


class Experts:
    def __init__(self, seed=0, device="cuda"):
        gen = torch.Generator(device=device).manual_seed(seed)

        def random(*shape):
            return torch.randn(*shape, device=device, generator=gen) / math.sqrt(shape[-1])

        self.router = random(EXPERTS, HIDDEN)
        self.up32, self.down32 = random(EXPERTS, 2 * INNER, HIDDEN), random(EXPERTS, HIDDEN, INNER)
        self.up, self.down = L.fp8_quantize_weight(self.up32), L.fp8_quantize_weight(self.down32)

    def route(self, x):
        """Each token's experts and their weights."""
        p, ids = torch.softmax(x.float() @ self.router.t(), 1).topk(TOPK, 1)
        return ids.int(), p / p.sum(1, keepdim=True)

    def __call__(self, x):
        ids, p = self.route(x)
        plan = L.expert_plan(ids, EXPERTS)
        h = L.fp8_grouped_matmul(x, *self.up, plan.starts, gather=plan.tokens)
        q, s = L.fp8_silu_mul(h[:, :INNER], h[:, INNER:])
        y = L.fp8_grouped_matmul(q, *self.down, plan.starts, x_scales=s, scatter=plan.planes, out_dtype=x.dtype)
        return (y.view(-1, TOPK, HIDDEN) * p[..., None].to(x.dtype)).sum(1)

    def plain(self, x):
        """The layer in f32, one expert after another, over the weights before they were brought into 8 bits."""
        ids, p = self.route(x)
        y = torch.zeros(x.shape[0], HIDDEN, device=x.device)
        for e in range(EXPERTS):
            token, slot = torch.nonzero(ids == e, as_tuple=True)
            if not len(token):
                continue
            h = x[token].float() @ self.up32[e].t()
            a = torch.nn.functional.silu(h[:, :INNER]) * h[:, INNER:]
            y.index_add_(0, token, (a @ self.down32[e].t()) * p[token, slot, None])
        return y


def run(tokens=(1, 16, 256), steps=20, dtype=torch.bfloat16, seed=0, device="cuda"):
    """Largest difference from `plain`, relative to the outputs' size, and the microseconds of the last size's step."""
    layer, gen = Experts(seed, device), torch.Generator(device=device).manual_seed(seed + 1)
    worst, us = 0.0, 0.0
    for n in tokens:
        x = torch.randn(n, HIDDEN, device=device, generator=gen).to(dtype)
        y, want = layer(x).float(), layer.plain(x)
        worst = max(worst, ((y - want).norm() / want.norm()).item())
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        for _ in range(steps):
            layer(x)
        end.record()
        end.synchronize()
        us = start.elapsed_time(end) / steps * 1e3
        print(f"{n:5d} tokens: {us:8.1f} us a step, {worst:.4f} off")
    L.paged_check()
    return worst, us


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=20)
    run(steps=ap.parse_args().steps)
