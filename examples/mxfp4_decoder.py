"""The MXFP4 path as a decoder serves it: a stack of gated MLP blocks with 4-bit weights, over a prefill
and then token by token, and what stands between two blocks in training.

    python examples/mxfp4_decoder.py            # on an MI355X
    python examples/mxfp4_decoder.py --tokens 4096 --hidden 4096 --inner 14336 --layers 4

A block is three calls that hand each other their operands as the kernels take them:

    gate_up -- hk.ops.mxfp4.gemm(silu_mul=True) on the normed stream, which the norm before it stored as MXFP8
    down    -- hk.ops.mxfp4.linear, its activation quantized on the way
    between -- hk.ops.block_norm: the norm of the branch, the gated residual add, the next block's norm

The stream is checked against the same arithmetic in fp32 torch on the weights' and activations' own values.
"""

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "hk-dsl_amd"))

import hk  # noqa: E402

mxfp4, mxfp8, block_norm = hk.ops.mxfp4, hk.ops.mxfp8, hk.ops.block_norm


class Decoder:
    """`layers` gated MLP blocks; weights quantized once, as they are loaded."""

    def __init__(self, hidden, inner, layers, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def r(*size, std=1.0, mean=0.0):
            return torch.randn(*size, generator=g, device=device) * std + mean

        self.hidden = hidden
        self.blocks = [dict(gate_up=mxfp4.quant(r(2 * inner, hidden, std=hidden ** -0.5)),
                            down=mxfp4.quant(r(hidden, inner, std=inner ** -0.5)),
                            post=r(hidden, std=0.1, mean=1).bfloat16(), pre=r(hidden, std=0.1, mean=1).bfloat16(),
                            gate=r(hidden, std=0.1, mean=0.5).bfloat16())
                       for _ in range(layers)]
        self.first = r(hidden, std=0.1, mean=1).bfloat16()

    def __call__(self, x):
        """x (tokens, hidden) bf16 -> the normed stream after the last block, bf16."""
        h, (y, s) = block_norm(torch.zeros_like(x), x, pre=self.first, quant="mxfp8")
        for i, b in enumerate(self.blocks):
            a = mxfp4.gemm(y, b["gate_up"][0], s, b["gate_up"][1], silu_mul=True)
            branch = mxfp4.linear(a, *b["down"])
            last = i + 1 == len(self.blocks)
            h, y = block_norm(branch, h, post=b["post"], pre=b["pre"], gate=b["gate"],
                              quant=None if last else "mxfp8")
            if not last:
                y, s = y
        return y

    def plain(self, x):
        """The same in fp32 torch: weights and activations as the numbers their codes stand for."""
        def norm(v, w):
            return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w.float()

        def q8(v):  # to MXFP8 and back
            return mxfp8.dequant(*mxfp8.quant(v.bfloat16().contiguous()), dtype=torch.float32)

        h = x.float()
        y = norm(h, self.first)
        for b in self.blocks:
            z = q8(y) @ mxfp4.dequant(*b["gate_up"], dtype=torch.float32).t()
            g, u = z.chunk(2, dim=1)
            branch = q8(torch.nn.functional.silu(g) * u) @ mxfp4.dequant(*b["down"], dtype=torch.float32).t()
            h = h + b["gate"].float() * norm(branch, b["post"])
            y = norm(h, b["pre"])
        return y


def train_between(tokens, hidden, steps=8, rate=4.0, device="cuda", seed=1):
    """What stands between two blocks fitted to a target by its norms' weights and its gate (plain gradient
    descent): (the loss at each step, the last step's gradients by name)."""
    g = torch.Generator(device=device).manual_seed(seed)
    x, residual, target = (torch.randn(2, tokens, hidden, generator=g, device=device).bfloat16() for _ in range(3))
    target = (target * 0.1 + 0.8 * residual + 0.6 * x).float()
    x.requires_grad_()
    w = {n: torch.full((hidden,), v, device=device, requires_grad=True) for n, v in (("post", 1.0), ("pre", 1.0), ("gate", 0.1))}
    losses = []
    for _ in range(steps):
        for t in (x, *w.values()):
            t.grad = None
        _, y = block_norm(x, residual, **w)
        loss = (y.float() - target).square().mean()
        loss.backward()
        losses.append(loss.item())
        with torch.no_grad():
            for t in w.values():
                t -= rate * t.grad * hidden / 16
    return losses, {n: t.grad for n, t in (("x", x), *w.items())}


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, v in (("tokens", 1024), ("hidden", 2048), ("inner", 5632), ("layers", 2), ("steps", 32)):
        p.add_argument(f"--{name}", type=int, default=v)
    a = p.parse_args(argv)
    model = Decoder(a.hidden, a.inner, a.layers)
    x = torch.randn(a.tokens, a.hidden, device="cuda").bfloat16()

    y, ref = model(x), model.plain(x)
    off = ((y.float() - ref).norm() / ref.norm()).item()
    print(f"prefill of {a.tokens} tokens: {off:.4f} of the fp32 stream's norm away")

    token = x[-1:].clone()
    model(token)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):  # a graph captures the calls of a step as they are
        model(token)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = model(token)
    torch.cuda.current_stream().wait_stream(stream)
    graph.replay()
    same = torch.equal(out, model(token))
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(a.steps):
        graph.replay()
    torch.cuda.synchronize()
    us = (time.perf_counter() - start) / a.steps * 1e6
    print(f"decode of one token: {us:.1f} us a step of {a.layers} layers; the graph's step is the eager one: {same}")

    losses, grads = train_between(a.tokens, a.hidden)
    print(f"training, loss {losses[0]:.4f} to {losses[-1]:.4f} in {len(losses)} steps; gradients' norms "
          + ", ".join(f"{n} {t.float().norm().item():.3g}" for n, t in grads.items()))
    return off, same


if __name__ == "__main__":
    main()
