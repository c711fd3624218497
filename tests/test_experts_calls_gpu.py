"""Calls of hk.ops.experts on the GPU beside those of test_experts_gpu.py, with its tolerances: a bf16 result is within
half a step (2^-8 of it) of an fp32 sum, which is within 2^-23 a term of the terms' magnitudes."""

import pytest
import torch

from hk.ops import experts
from test_experts_gpu import BF16, DEV, _plan, kernel  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _hand_the_memory_back():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("t,e,k,n,d,dead", [(9, 4, 2, 40, 24, 1), (150, 6, 4, 136, 200, 9), (700, 8, 8, 128, 64, 33),
                                            (3000, 4, 4, 264, 520, 0), (600, 2, 2, 2824, 264, 5)])
def test_a_gathered_rows_gradient_is_rounded_once(t, e, k, n, d, dead, kernel):  # noqa: F811
    """Experts that nearly cancel: a token's rows are large, their sum is not, and what each row lost would show."""
    plan, (offsets, rows, slots) = _plan(t, e, k, seed=t, dead=dead)
    g = torch.Generator().manual_seed(n)
    x = torch.randn(t, d, generator=g).to(BF16)
    sign = 1.0 - 2.0 * (torch.arange(e) % 2).reshape(e, 1, 1)
    w = (sign * torch.randn(1, n, d, generator=g) + 0.01 * torch.randn(e, n, d, generator=g)).to(BF16)
    v = torch.randn(t, n, generator=g).to(BF16)
    dy = torch.where((rows >= 0).unsqueeze(1), v[rows.clamp(min=0)], torch.zeros((), dtype=BF16))
    leaf = x.to(DEV).requires_grad_()
    y = experts.gemm(leaf, w.to(DEV), plan, gather=True)
    (dx,) = torch.autograd.grad(y, leaf, dy.to(DEV))
    assert dx.dtype == BF16 and dx.shape == x.shape
    ref, mag = torch.zeros(t, d, dtype=torch.float64, device=DEV), torch.zeros(t, d, dtype=torch.float64, device=DEV)
    off, wd, dyd = offsets.tolist(), w.to(DEV).double(), dy.to(DEV).double()
    for i in range(e):
        a, to = dyd[off[i]:off[i + 1]], rows[off[i]:off[i + 1]].to(DEV)
        ref.index_add_(0, to, a @ wd[i])
        mag.index_add_(0, to, a.abs() @ wd[i].abs())
    # (the sums of a row, and then of k rows; the one rounding)
    err = (n + 2 + k) * 2.0 ** -23 * mag
    assert ((dx.double() - ref).abs() <= err + 2.0 ** -8 * (ref.abs() + err)).all()


def test_the_routers_gradient_past_a_launch():
    """More tokens than one launch takes: those at the seams have the gradients that they have by themselves."""
    t, e = (1 << 26) + 5, 2
    g = torch.Generator(device=DEV).manual_seed(3)
    block = torch.randn(1 << 16, e, generator=g, device=DEV).to(BF16)
    logits = torch.empty(t, e, dtype=BF16, device=DEV)
    dw = torch.empty(t, 1, device=DEV)
    for at in range(0, t, 1 << 16):
        n = min(1 << 16, t - at)
        logits[at:at + n] = block[:n]
        dw[at:at + n] = block[:n, :1].float() + at / t
    logits.requires_grad_()
    (got,) = torch.autograd.grad(experts.route(logits, 1, renormalize=False)[0], logits, dw)
    for at in (0, (1 << 25) - 7, (1 << 26) - 7, t - 11):
        part = logits.detach()[at:at + 11].clone().requires_grad_()
        (want,) = torch.autograd.grad(experts.route(part, 1, renormalize=False)[0], part, dw[at:at + 11].clone())
        assert torch.equal(got[at:at + 11], want) and want.any()


def test_a_gathered_gradient_past_a_launch():
    """More tokens than one launch of their rows' sum takes."""
    t, d = (1 << 24) + 9, 8
    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.zeros(t, d, dtype=BF16, device=DEV, requires_grad=True)
    w = torch.randint(-3, 4, (2, 8, d), generator=g, device=DEV).to(BF16)
    half = t // 2
    offsets = torch.tensor([0, half, t], dtype=torch.int32, device=DEV)
    rows = torch.arange(t - 1, -1, -1, dtype=torch.int32, device=DEV)  # token t - 1 first
    plan = experts.Plan(offsets, rows, rows.reshape(t, 1))
    dy = torch.zeros(t, 8, dtype=BF16, device=DEV)
    dy[:, 0] = (torch.arange(t, device=DEV) % 61).to(BF16)
    (dx,) = torch.autograd.grad(experts.gemm(x, w, plan, gather=True), x, dy)
    # (small whole numbers: exact)
    for at in (0, t - half - 5, (1 << 23) - 5, (1 << 24) - 6, t - 10):
        row = rows[at:at + 10].long()
        want = dy[row, :1].float() * w[(row >= half).long(), 0].float()
        assert torch.equal(dx[at:at + 10].float(), want) and want.any()


def test_a_gathered_gradient_of_rows_past_4_gib(kernel):  # noqa: F811
    """The rows' fp32 gradient is 5.4 GB; small whole numbers, so that it is exact."""
    t, e, k, d = 66_001, 3, 5, 4096
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.zeros(t, d, dtype=BF16, device=DEV, requires_grad=True)
    w = torch.randint(-2, 3, (e, 8, d), generator=g, device=DEV).to(BF16)
    slots = torch.randperm(t * k, generator=g, device=DEV).int().reshape(t, k)
    rows = torch.empty(t * k, dtype=torch.int32, device=DEV)
    rows[slots.flatten().long()] = torch.arange(t, dtype=torch.int32, device=DEV).repeat_interleave(k)
    offsets = torch.tensor([0, 1001, 200_003, t * k], dtype=torch.int32, device=DEV)
    dy = torch.randint(-1, 2, (t * k, 8), generator=g, device=DEV).to(BF16)
    (dx,) = torch.autograd.grad(experts.gemm(x, w, experts.Plan(offsets, rows, slots), gather=True), x, dy)
    for at in (0, t // 2, t - 300):
        s = slots[at:at + 300].long()
        of = torch.bucketize(s, offsets[1:].long(), right=True)
        want = (dy[s].float().unsqueeze(3) * w[of].float()).sum((1, 2))
        assert torch.equal(dx[at:at + 300].float(), want) and want.any()


def _ints(*shape, seed):
    """-2 .. 2: sums are exact in any order."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = torch.empty(shape, dtype=BF16, device=DEV)
    flat, step = out.view(-1), 999_983 * 16
    block = torch.randint(-2, 3, (step,), generator=g, device=DEV, dtype=torch.int8)
    for at in range(0, flat.numel(), step):
        flat[at:at + step] = block[:min(step, flat.numel() - at)]
    return out


@pytest.mark.parametrize("silu_mul", [False, True], ids=["plain", "paired"])
def test_rows_gathered_from_just_under_4_gib(silu_mul, kernel):  # noqa: F811
    """The largest x that a call gathers from: its last rows among them, and the gradients."""
    t, k, n, r = 524_284, 4096, 72, 3001
    x, w = _ints(t, k, seed=1), _ints(3, 2 * n if silu_mul else n, k, seed=2) * 2.0 ** -7
    g = torch.Generator(device=DEV).manual_seed(3)
    rows = torch.randperm(t, generator=g, device=DEV)[:r].int()
    rows[:4] = torch.tensor([t - 1, 0, t - 2, t // 2], device=DEV)
    rows[4:] = torch.where((rows[4:] >= t - 2) | (rows[4:] == 0) | (rows[4:] == t // 2), -1, rows[4:])
    plan = experts.Plan(torch.tensor([0, 5, 1400, r - 9], dtype=torch.int32, device=DEV), rows)
    own = x[rows.clamp(min=0).long()] * (rows >= 0).unsqueeze(1)
    own[r - 9:] = 0
    y = experts.gemm(x, w, plan, gather=True, silu_mul=silu_mul)
    assert torch.equal(y, experts.gemm(own, w, plan._replace(rows=None), silu_mul=silu_mul)) and y[:4].any(1).all()
    slots = torch.full((t, 1), -1, dtype=torch.int32, device=DEV)
    live = torch.arange(r, device=DEV, dtype=torch.int32)[rows >= 0]
    slots[rows[live.long()].long(), 0] = live
    dy = _ints(r, n, seed=4)
    leaf, one = x.requires_grad_(), own.requires_grad_()
    w.requires_grad_()
    dx, dw = torch.autograd.grad(experts.gemm(leaf, w, plan._replace(slots=slots), gather=True, silu_mul=silu_mul), (leaf, w), dy)
    d1, w1 = torch.autograd.grad(experts.gemm(one, w, plan._replace(rows=None), silu_mul=silu_mul), (one, w), dy)
    assert torch.equal(dw, w1) and dw.any()
    assert torch.equal(dx[rows[live.long()].long()], d1[live.long()]) and d1[:4].any(1).all()
    dx[rows[live.long()].long()] = 0
    assert not dx.any()


@pytest.mark.parametrize("silu_mul", [False, True], ids=["plain", "paired"])
def test_an_experts_weight_of_just_under_4_gib(silu_mul, kernel):  # noqa: F811
    """The largest w[e] that a call takes: columns at its ends and in the middle are what they are by themselves."""
    n, k, r = 262_128, 8192, 300
    w, x = _ints(1, n, k, seed=1) * 2.0 ** -7, _ints(r, k, seed=2)
    plan = experts.Plan(torch.tensor([0, r - 4], dtype=torch.int32, device=DEV))
    y = experts.gemm(x, w, plan, silu_mul=silu_mul)
    half = n // 2
    for at in (0, half // 2 + 8, half - 40):
        if silu_mul:
            part = torch.cat((w[:, at:at + 40], w[:, half + at:half + at + 40]), 1)
        else:
            at = 2 * at if at != half - 40 else n - 40
            part = w[:, at:at + 40].contiguous()
        assert torch.equal(y[:, at:at + 40], experts.gemm(x, part, plan, silu_mul=silu_mul)) and y[0, at:at + 40].any()
    assert not y[r - 4:].any()
