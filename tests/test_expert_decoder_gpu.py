"""examples/expert_decoder.py on the GPU.

The stream's tolerance. bf16: a block rounds its normed input, the gated product, each expert's row, their sum and the
stream to bf16, 2^-8 of a value at most each, some 2^-9.8 rms and independent: five of them 0.0025 a block, 0.01 with a
margin. 8 bits: the normed input and the gated product are rounded to e4m3, 2^-4 at most and some 2^-5.5 rms each: 0.031
of a branch, which is no larger than the stream, 0.05 for two blocks."""

import importlib.util
from pathlib import Path

import pytest
import torch

from oracle import experts_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

PATH = Path(__file__).resolve().parents[1] / "examples" / "expert_decoder.py"
SPEC = importlib.util.spec_from_file_location("expert_decoder", PATH)
decoder = importlib.util.module_from_spec(SPEC)
SPEC.loader.exec_module(decoder)


@pytest.mark.parametrize("wide,limit", [(True, 0.01), (False, 0.05)], ids=["bf16", "fp8"])
@pytest.mark.parametrize("tokens", [1, 19, 300])
def test_the_stream_is_fp32s(tokens, wide, limit):
    model = decoder.Decoder(256, 160, 12, 3, 2, wide)
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x = torch.randn(tokens, 256, generator=g, device=DEV).bfloat16()
    kept = []
    y = model(x, kept)
    ref = model.plain(x, kept)
    assert y.shape == ref.shape and y.dtype == torch.bfloat16
    assert float((y.float() - ref).norm() / ref.norm()) < limit


def test_the_example_runs(capsys):
    offs, same, grads = decoder.main(["--tokens", "64", "--hidden", "256", "--inner", "96", "--experts", "8", "--chosen", "2", "--steps", "3"])
    assert offs[0] < 0.01 and offs[1] < 0.05 and all(same)
    assert "training step" in capsys.readouterr().out
    assert set(grads) == {"x", "router", "up", "down"}
    assert all(t.isfinite().all() and t.abs().max() > 0 for t in grads.values())


def test_the_training_steps_gradients():
    """Against the same step in float64: a 2-norm of six bf16 roundings, 2^-8 each at most (the router's logits are the
    bf16 product's, as in the step)."""
    tokens, hidden, inner, count, chosen = 60, 64, 48, 6, 2
    grads = decoder.train_step(tokens, hidden, inner, count, chosen)
    g = torch.Generator(device=DEV).manual_seed(1)

    def r(*size, std=1.0):
        return (torch.randn(*size, generator=g, device=DEV) * std).bfloat16().cpu().double().requires_grad_()

    leaf = dict(x=r(tokens, hidden), router=r(count, hidden, std=hidden ** -0.5),
                up=r(count, 2 * inner, hidden, std=hidden ** -0.5), down=r(count, hidden, inner, std=inner ** -0.5))
    target = torch.randn(tokens, hidden, generator=g, device=DEV).cpu().double()
    exact = leaf["x"] @ leaf["router"].t()
    rounded = (leaf["x"].detach().bfloat16().to(DEV) @ leaf["router"].detach().bfloat16().to(DEV).t()).cpu().double()
    logits = exact + (rounded - exact).detach()
    _, picked, offsets, rows, slots = O.route(logits.detach(), chosen)
    weights = torch.softmax(torch.gather(logits, 1, picked), 1)
    a, _ = O.gemm(leaf["x"], leaf["up"], offsets, rows, silu_mul=True)
    y = O.combine(O.gemm(a, leaf["down"], offsets)[0], slots, weights)
    (y - target).square().mean().backward()
    for n, t in leaf.items():
        assert float((grads[n].cpu().double() - t.grad).norm() / t.grad.norm()) < 6 * 2.0 ** -8, n
