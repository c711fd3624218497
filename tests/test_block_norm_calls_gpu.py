"""hk.ops.block_norm on the GPU by the way it is called -- many gates, kept layouts, factors of the norms --
against the float64 oracle, with the tolerances of test_block_norm_gpu.py."""

import pytest
import torch

import hk
import test_block_norm_gpu as T
from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("gate_dtype", [BF16, F32])
@pytest.mark.parametrize("shape,one", [((70000, 2, 64), False), ((66000, 3, 37), False), ((70000, 2, 40), True),
                                       ((2100, 5, 1032), False), ((4099, 2, 130), True)])
def test_gradients_of_more_gates_than_workers(shape, one, gate_dtype):
    """A gate shared by a few rows (by the heads of a token, say), a value a column or one for all."""
    print(f"case gates {shape} one={one} {gate_dtype}", flush=True)
    a = T._inputs(shape, (BF16, F32, F32), "sequence", 21, gate_dtype)
    if one:
        a["gate"] = a["gate"][..., :1].clone()
    T._check_grads(a, 22, **T.SCALES)


@pytest.mark.parametrize("exponent", [0, -70, 40])
@pytest.mark.parametrize("d", [64, 333, 1000, 4096, 16384])
def test_a_norms_factor_is_rounded_once(d, exponent):
    """Rows of small whole numbers (times 2^exponent: squares that are subnormal, or large), whose sums of
    squares fp32 holds exactly in any order: 1 / sqrt(sum / d) of 64 bits to half a step of fp32, and 2^-20
    of one."""
    from hk.ops import norm

    g = torch.Generator().manual_seed(d)
    rows = 2000
    x = torch.randint(-9, 10, (rows, d), generator=g).float()
    x *= (torch.arange(rows) % 3 + 1)[:, None]  # (27^2 16384 < 2^24)
    x[:, 0] = 1 + torch.arange(rows) % 7        # (no row of zeros)
    exact = (x.double().square().sum(-1) / d).rsqrt() * 2.0 ** -exponent
    x = torch.ldexp(x, torch.tensor(exponent)).to(DEV)
    step = torch.exp2(torch.floor(torch.log2(exact)) - 23)
    w, zero = torch.ones(d, device=DEV), torch.zeros_like(x)
    # after the block (a backward pass is to follow, so the factors are kept; D to 8192 there), and before
    # the next: with no norm after the block h is x
    for post, pre, at in ((w, None, 0), (None, w, 1)):
        (_, _, rstd), *_ = norm._forward(x, zero, post, pre, None, (1.0, 1.0, 0.0), None, True)
        off = (rstd[:, at].cpu().double() - exact).abs() / step
        assert (off <= 0.5 + 2.0 ** -20).all(), f"{float(off.max()):.4f} of a step"


def test_a_norm_of_zeros_without_eps_is_nan_and_of_infinity_zero():
    x = torch.zeros(3, 64, device=DEV)
    x[1], x[2] = 1e30, 1.0  # (squares past fp32)
    h, _ = hk.ops.block_norm(x, torch.zeros_like(x), post=torch.ones(64, device=DEV), eps=0.0)
    assert torch.isnan(h[0]).all() and (h[1] == 0).all() and (h[2] == 1).all()


@pytest.mark.parametrize("rows,d", [(400, 64), (4096, 200), (999, 1111), (16384, 40)])
def test_sums_over_workers_lose_nothing(rows, d):
    """A channel gate's gradient sums dh x over the rows: 2^24 from one row, 1 from each after the second,
    which an fp32 sum of the workers' would drop one by one. The whole is rounded once."""
    x = torch.ones(rows, d, device=DEV)
    x[0], x[1] = 2.0 ** 12, 0.0
    gate = torch.ones(d, device=DEV, requires_grad=True)
    h, _ = hk.ops.block_norm(x, torch.zeros_like(x), gate=gate)
    grad, = torch.autograd.grad(h, gate, x)
    per = -(-rows // min(2048, (rows + 1) // 2))
    if per <= 2:  # (a worker's own sum is of fp32)
        assert (grad == torch.tensor(2.0 ** 24 + rows - 2, dtype=torch.float64).float().item()).all()
    else:         # (those of the first worker's rows alone)
        assert ((grad.double() - 2.0 ** 24 - rows + 2).abs() <= per).all()
