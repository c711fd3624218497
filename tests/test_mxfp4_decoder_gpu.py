"""examples/mxfp4_decoder.py, and operands past 32-bit offsets, on the GPU.

The stream's tolerance: an activation rounded to e4m3 is 2^-4 of it off at most, some 2^-5.5 rms, and where
the kernel's value and fp32's fall on two sides of a step the two differ by a whole step; that happens to the
share of values that a bf16 rounding (2^-9 at most) moves over a step (2^-3 to 2^-4), some 1/40, at 2^-3.5 each:
0.014 rms a quantization. Two a layer, with the gates of 0.5 between: 0.03 for two layers, 0.05 with a margin."""

import importlib.util
from pathlib import Path

import pytest
import torch

import hk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

PATH = Path(__file__).resolve().parents[1] / "examples" / "mxfp4_decoder.py"
SPEC = importlib.util.spec_from_file_location("mxfp4_decoder", PATH)
decoder = importlib.util.module_from_spec(SPEC)
SPEC.loader.exec_module(decoder)


@pytest.mark.parametrize("tokens", [1, 19, 200])
def test_the_stream_is_fp32s(tokens):
    model = decoder.Decoder(512, 1376, 2)
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x = torch.randn(tokens, 512, generator=g, device=DEV).bfloat16()
    y, ref = model(x), model.plain(x)
    assert y.shape == ref.shape and y.dtype == torch.bfloat16
    assert float((y.float() - ref).norm() / ref.norm()) < 0.05


def test_the_example_runs(capsys):
    off, same = decoder.main(["--tokens", "64", "--hidden", "256", "--inner", "704", "--steps", "3"])
    assert off < 0.05 and same
    assert "training" in capsys.readouterr().out


def test_training_what_stands_between_lowers_its_loss():
    """(The gradients themselves are held against the formula's in test_block_norm_gpu.py.)"""
    losses, grads = decoder.train_between(50, 192)
    assert losses[-1] < 0.8 * losses[0], losses
    assert set(grads) == {"x", "post", "pre", "gate"} and all(t.isfinite().all() for t in grads.values())


# ------------------------------------------------------------------ past 32 bits


def _free(need):
    if torch.cuda.mem_get_info()[0] < need * 2 ** 30:
        pytest.skip(f"needs {need} GiB")


def test_block_norm_past_32_bits():
    """Rows that start past 2^32 bytes, forward and backward, are what they are in a call of their own."""
    _free(60)
    rows, d = 300000, 8192
    x = torch.empty(rows, d, dtype=torch.bfloat16, device=DEV)
    x.copy_(torch.randn(1, d, device=DEV)).mul_(torch.linspace(0.5, 2, rows, device=DEV).bfloat16()[:, None])
    w = torch.linspace(0.9, 1.1, d, device=DEV).bfloat16()
    gate = torch.linspace(0, 1, rows, device=DEV).bfloat16()[:, None]
    h, y = hk.ops.block_norm(x, x, post=w, pre=w, gate=gate)
    for at in (0, rows // 2, rows - 40):
        p = slice(at, at + 40)
        h1, y1 = hk.ops.block_norm(x[p].clone(), x[p].clone(), post=w, pre=w, gate=gate[p].clone())
        assert torch.equal(h[p], h1) and torch.equal(y[p], y1)
    del h, y
    a = x.detach().requires_grad_()
    h, y = hk.ops.block_norm(a, x, post=w, pre=w, gate=gate)
    dx, = torch.autograd.grad(y, a, x)
    for at in (0, rows - 40):
        p = slice(at, at + 40)
        a1 = x[p].clone().requires_grad_()
        h1, y1 = hk.ops.block_norm(a1, x[p].clone(), post=w, pre=w, gate=gate[p].clone())
        assert torch.equal(dx[p], torch.autograd.grad(y1, a1, x[p].clone())[0])


def test_quant_and_dequant_past_32_bits():
    _free(40)
    m, k = 300000, 8192
    x = torch.empty(m, k, dtype=torch.bfloat16, device=DEV)
    x.copy_(torch.randn(1, k, device=DEV)).mul_(torch.linspace(0.5, 2, m, device=DEV).bfloat16()[:, None])
    q, s = hk.ops.mxfp4.quant(x)
    back = hk.ops.mxfp4.dequant(q, s)
    for at in (0, m // 2, m - 40):
        p = slice(at, at + 40)
        q1, s1 = hk.ops.mxfp4.quant(x[p].clone())
        assert torch.equal(q[p], q1) and torch.equal(s[p], s1)
        assert torch.equal(back[p], hk.ops.mxfp4.dequant(q1, s1))


@pytest.mark.parametrize("wide", [False, True], ids=["a4", "a8"])
def test_gemm_with_a_c_past_32_bits(wide):
    _free(20)
    m, n, k = 100000, 24000, 64
    g = torch.Generator(device=DEV).manual_seed(5)
    a = torch.randint(0, 256, (m, k // 2), generator=g, device=DEV, dtype=torch.uint8) if not wide else torch.randn(
        m, k, generator=g, device=DEV).to(torch.float8_e4m3fn)
    b = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    sa = torch.randint(120, 134, (m, 2), generator=g, device=DEV, dtype=torch.uint8)
    sb = torch.randint(120, 134, (n, 2), generator=g, device=DEV, dtype=torch.uint8)
    c = hk.ops.mxfp4.gemm(a, b, sa, sb)
    step = hk.ops.mxfp8.dequant if wide else hk.ops.mxfp4.dequant
    bv = hk.ops.mxfp4.dequant(b, sb, dtype=torch.float32)
    for at in (0, m // 2, m - 300):  # (64 products of few bits: fp32 sums them within 2^-17 of their magnitudes)
        p = slice(at, at + 300)
        av = step(a[p].clone(), sa[p].clone(), dtype=torch.float32)
        ref = av.double() @ bv.double().t()
        tol = 2.0 ** -8 * ref.abs() + 2.0 ** -11 * (av.abs().double() @ bv.abs().double().t())
        assert ((c[p].double() - ref).abs() <= tol).all()
