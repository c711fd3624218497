"""A layer of experts as a decoder serves and trains it: gated experts over a prefill and then token by token, in bf16 and
with 8-bit weights behind the norm that quantizes for them, and a training step of the layer.

    python examples/expert_decoder.py            # on an MI355X
    python examples/expert_decoder.py --tokens 4096 --hidden 4096 --inner 2048 --experts 64 --chosen 8

A block is

    norm    -- hk.ops.block_norm: the residual add and the norm, its output as 8-bit rows for the 8-bit form
    route   -- the router's product (hk.ops.matmul, or hk.ops.scaled_mm on the 8-bit rows) and hk.ops.experts.route
    experts -- hk.ops.experts.gemm(silu_mul=True) on rows gathered by token, hk.ops.experts.gemm
    combine -- hk.ops.experts.combine: the experts' rows back to their tokens

of which the last three are hk.ops.experts.mlp. The stream is checked against the same arithmetic in fp32 torch.
"""

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "hk-dsl_amd"))

import hk  # noqa: E402

experts, fp8, block_norm = hk.ops.experts, hk.ops.fp8, hk.ops.block_norm


class Decoder:
    """`layers` blocks of gated experts; with `wide` False their weights in 8 bits, quantized once as they are loaded."""

    def __init__(self, hidden, inner, count, chosen, layers, wide=True, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def r(*size, std=1.0, mean=0.0):
            return (torch.randn(*size, generator=g, device=device) * std + mean).bfloat16()

        self.chosen, self.wide = chosen, wide
        self.blocks = []
        for _ in range(layers):
            up, down = r(count, 2 * inner, hidden, std=hidden ** -0.5), r(count, hidden, inner, std=inner ** -0.5)
            b = dict(norm=r(hidden, std=0.1, mean=1), router=r(count, hidden, std=hidden ** -0.5), up=up, down=down)
            if not wide:
                (b["up"], su), (b["down"], sd), (b["router"], sr) = fp8.quant(up), fp8.quant(down), fp8.quant(b["router"])
                b["scales"] = dict(gate_up_scale=su.squeeze(2), down_scale=sd.squeeze(2))
                b["router_scale"] = sr
            self.blocks.append(b)

    def __call__(self, x, kept=None):
        """x (tokens, hidden) bf16 -> the stream after the last block, bf16. kept: takes each block's router logits."""
        branch = torch.zeros_like(x)
        for b in self.blocks:
            x, y = block_norm(branch, x, pre=b["norm"], quant=None if self.wide else "fp8")
            if self.wide:
                logits = hk.ops.matmul(y, b["router"])
                branch = experts.mlp(y, logits, self.chosen, b["up"], b["down"])
            else:
                logits = hk.ops.scaled_mm(y[0], b["router"], y[1], b["router_scale"])
                branch = experts.mlp(y, logits, self.chosen, b["up"], b["down"], **b["scales"])
            if kept is not None:
                kept.append(logits)
        return x + branch

    def plain(self, x, kept):
        """The same in fp32 torch, every expert for every token, on the weights' own values; kept: the router's logits."""
        h = x.float()
        for b, logits in zip(self.blocks, kept):
            y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * b["norm"].float()
            weights, picked, _ = experts.route(logits, self.chosen)
            up, down = b["up"].float(), b["down"].float()
            if not self.wide:
                up, down = (w * s.unsqueeze(2) for w, s in zip((up, down), b["scales"].values()))
            for e in range(up.shape[0]):
                gate, lin = (y @ up[e].t()).chunk(2, dim=1)
                share = torch.where(picked == e, weights, 0.0).sum(1, keepdim=True)
                h = h + share * ((torch.nn.functional.silu(gate) * lin) @ down[e].t())
        return h


def train_step(tokens, hidden, inner, count, chosen, device="cuda", seed=1):
    """One step's gradients of a layer's weights, its router and its input, by name."""
    g = torch.Generator(device=device).manual_seed(seed)

    def r(*size, std=1.0):
        return (torch.randn(*size, generator=g, device=device) * std).bfloat16().requires_grad_()

    leaf = dict(x=r(tokens, hidden), router=r(count, hidden, std=hidden ** -0.5),
                up=r(count, 2 * inner, hidden, std=hidden ** -0.5), down=r(count, hidden, inner, std=inner ** -0.5))
    logits = leaf["x"] @ leaf["router"].t()
    y = experts.mlp(leaf["x"], logits, chosen, leaf["up"], leaf["down"])
    target = torch.randn(tokens, hidden, generator=g, device=device)
    (y.float() - target).square().mean().backward()
    return {n: t.grad for n, t in leaf.items()}


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, v in (("tokens", 1024), ("hidden", 1024), ("inner", 768), ("experts", 16), ("chosen", 4), ("layers", 2), ("steps", 32)):
        p.add_argument(f"--{name}", type=int, default=v)
    a = p.parse_args(argv)
    x = torch.randn(a.tokens, a.hidden, device="cuda").bfloat16()
    offs, same = [], []
    for wide in (True, False):
        model = Decoder(a.hidden, a.inner, a.experts, a.chosen, a.layers, wide)
        kept = []
        y = model(x, kept)
        ref = model.plain(x, kept)
        offs.append(((y.float() - ref).norm() / ref.norm()).item())
        token = x[-1:].clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):  # a graph captures the calls of a step as they are
            model(token)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = model(token)
        torch.cuda.current_stream().wait_stream(stream)
        graph.replay()
        same.append(torch.equal(out, model(token)))
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(a.steps):
            graph.replay()
        torch.cuda.synchronize()
        us = (time.perf_counter() - start) / a.steps * 1e6
        print(f"{'bf16' if wide else '8-bit'} weights: prefill of {a.tokens} tokens {offs[-1]:.4f} of the fp32 stream's norm away; "
              f"decode of one token {us:.1f} us a step of {a.layers} layers, the graph's step is the eager one: {same[-1]}")
    grads = train_step(a.tokens, a.hidden, a.inner, a.experts, a.chosen)
    print("training step, gradients' norms " + ", ".join(f"{n} {t.float().norm().item():.3g}" for n, t in grads.items()))
    return offs, same, grads


if __name__ == "__main__":
    main()
