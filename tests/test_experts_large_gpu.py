"""Layers of experts whose operands pass 4 GiB, or whose rows pass a launch, on the GPU: rows at the ends and in the middle
are what they are in a call of their own. The operands are small integers: sums are exact in any order, on any kernel."""

import pytest
import torch

from hk.ops import experts, fp8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn
KERNELS = pytest.mark.parametrize("kernel", [0, 1, 2, 3, 4, 6], ids=["auto", "tile16", "tile64", "tile128", "quad", "skinny"])


@pytest.fixture(autouse=True)
def _hand_the_memory_back():
    yield
    torch.cuda.empty_cache()


def _free(need):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < need * 2 ** 30:
        pytest.skip(f"needs {need} GiB")


def _on(kernel, monkeypatch):
    real = experts._run

    def run(g, device, need=None):
        g.kernel = kernel
        real(g, device)

    monkeypatch.setattr(experts, "_run", run)


def _ints(*shape, seed):
    """-2 .. 2, a block of 2^20 values over and over (a prime's rows apart)."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    block = torch.randint(-2, 3, (1 << 20,), generator=g, device=DEV).to(torch.int8)
    n = 1
    for s in shape:
        n *= s
    out = torch.empty(n, dtype=BF16, device=DEV)
    step = 999983
    for at in range(0, n, step * 64):
        m = min(step * 64, n - at)
        out[at:at + m] = block[:step].repeat(64)[:m]
    return out.view(shape)


def _ends(n, width=40):
    return [slice(0, width), slice(n // 2, n // 2 + width), slice(n - width, n)]


def _offsets(*at):
    return torch.tensor(at, dtype=torch.int32, device=DEV)


@KERNELS
def test_rows_past_4_gib(kernel, monkeypatch):
    """x, C and z each past 4 GiB; gathered; their gradients."""
    _on(kernel, monkeypatch)
    _free(60)
    r, k, n = 530_001, 4104, 24
    x, w = _ints(r, k, seed=1), _ints(3, n, k, seed=2)
    cut = (0, 1000, r // 2 + 11, r - 7)
    plan = experts.Plan(_offsets(*cut))

    def part(p):  # the plan of rows p alone
        return experts.Plan(_offsets(*(min(max(c - p.start, 0), p.stop - p.start) for c in cut)))

    y = experts.gemm(x, w, plan)
    for p in _ends(r):
        assert torch.equal(y[p], experts.gemm(x[p].clone(), w, part(p))) and y[p][:20].any()
    del x, y
    a, wide = _ints(r, 16, seed=3), _ints(3, k, 16, seed=4)
    y = experts.gemm(a, wide, plan)
    for p in _ends(r):
        assert torch.equal(y[p], experts.gemm(a[p].clone(), wide, part(p))) and y[p][:20].any()
    rows = torch.arange(r, device=DEV, dtype=torch.int32) % 997
    got = experts.gemm(a[:997].clone(), wide, plan._replace(rows=rows), gather=True)
    for p in _ends(r):
        assert torch.equal(got[p], experts.gemm(a[:997][rows[p].long()], wide, part(p)))
    del got
    # dx (R, 16) of dy past 4 GiB, and dw over its rows
    leaf, weights = a.requires_grad_(), wide.requires_grad_()
    dx, dw = torch.autograd.grad(experts.gemm(leaf, weights, plan), (leaf, weights), y)
    assert torch.isfinite(dw.float()).all()
    for p in _ends(r):
        one = a.detach()[p].clone().requires_grad_()
        (d1,) = torch.autograd.grad(experts.gemm(one, wide.detach(), part(p)), one, y[p].clone())
        assert torch.equal(dx[p], d1) and d1[:20].any() and not dx[-7:].any()


@KERNELS
def test_gate_and_up_rows_past_4_gib(kernel, monkeypatch):
    """z (R, 2 N) kept for the backward pass."""
    _on(kernel, monkeypatch)
    _free(60)
    r, k, n = 4_100_003, 16, 264
    x, w = _ints(r, k, seed=1), _ints(2, 2 * n, k, seed=2) * 0.125
    cut = (0, 5000, r - 3)
    plan = experts.Plan(_offsets(*cut))
    leaf = x.requires_grad_()
    y = experts.gemm(leaf, w, plan, silu_mul=True)
    (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    for p in _ends(r):
        e, live = int(p.start >= cut[1]), min(p.stop, cut[2]) - p.start
        part = x.detach()[p].clone().requires_grad_()
        y1 = experts.gemm(part, w[e:e + 1].clone(), experts.Plan(_offsets(0, live)), silu_mul=True)
        assert torch.equal(y[p], y1) and y1[:20].any()
        (d1,) = torch.autograd.grad(y1, part, torch.ones_like(y1))
        # (each rounded by 2^-8 at most; fp32 sums of 528 terms in another order, dz up to 8.8 and w 0.25: 528 x 2^-23 x 528 x 2.2)
        assert ((dx[p].float() - d1.float()).abs() <= 2.0 ** -7 * d1.float().abs() + 0.073).all()


@KERNELS
def test_weights_past_4_gib(kernel, monkeypatch):
    """All experts' w and dw."""
    _on(kernel, monkeypatch)
    _free(60)
    e, n, k, each = 70, 4104, 8200, 3
    w = _ints(e, n, k, seed=2)
    x = _ints(each * e, k, seed=1).requires_grad_()
    plan = experts.Plan(torch.arange(e + 1, dtype=torch.int32, device=DEV) * each)
    w.requires_grad_()
    y = experts.gemm(x, w, plan)
    dy = _ints(each * e, n, seed=5)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for i in (0, e // 2, e - 1):
        p = slice(each * i, each * i + each)
        a, b = x.detach()[p].clone().requires_grad_(), w.detach()[i:i + 1].clone().requires_grad_()
        y1 = experts.gemm(a, b, experts.Plan(_offsets(0, each)))
        assert torch.equal(y[p], y1) and y1.any()
        dx1, dw1 = torch.autograd.grad(y1, (a, b), dy[p].clone())
        assert torch.equal(dx[p], dx1) and torch.equal(dw[i], dw1[0]) and dw1.any()


def test_8_bit_rows_past_4_gib():
    _free(60)
    r, k, n = 530_001, 8208, 40
    x = torch.empty(r, k, dtype=E4M3, device=DEV)
    block = _ints(4096, k, seed=1).to(E4M3)
    for at in range(0, r, 4096):
        x[at:at + 4096] = block[:min(4096, r - at)]
    w = _ints(2, n, k, seed=2).to(E4M3)
    sa = (torch.arange(r, device=DEV) % 5 + 1).float()
    sb = torch.ones(2, n, device=DEV)
    y = experts.gemm(x, w, experts.Plan(_offsets(0, 77, r)), scale_a=sa, scale_b=sb)
    for p in _ends(r):
        e = int(p.start >= 77)
        y1 = experts.gemm(x[p].clone(), w[e:e + 1].clone(), experts.Plan(_offsets(0, 40)), scale_a=sa[p].clone(), scale_b=sb[:1])
        assert torch.equal(y[p], y1) and y1.any()


def test_combination_past_4_gib():
    _free(60)
    t, k, d = 300_011, 4, 2048
    y = _ints(t * k, d, seed=1).requires_grad_()
    slots = torch.randperm(t * k, device=DEV, dtype=torch.int32).view(t, k)
    weights = ((torch.arange(t * k, device=DEV) % 3 + 1).float().view(t, k)).requires_grad_()
    out = experts.combine(y, experts.Plan(None, None, slots), weights)
    dy, dw = torch.autograd.grad(out, (y, weights), out.detach())
    for p in _ends(t):
        at = slots[p].long()
        want = (y.detach()[at].float() * weights.detach()[p].unsqueeze(2)).sum(1)
        assert torch.equal(out[p].float(), want)
        assert torch.equal(dy[at].float(), weights.detach()[p].unsqueeze(2) * want.unsqueeze(1))
        dots = (y.detach()[at].float() * want.unsqueeze(1)).sum(2)
        assert torch.equal(dw[p], dots)


@pytest.mark.parametrize("m,k", [((1 << 24) + 5, 16), (530_001, 8200)])
def test_rows_to_8_bits_past_a_launch_and_4_gib(m, k):
    _free(60)
    x = _ints(m, k, seed=1) * 0.75
    q, s = fp8.quant(x)
    for p in _ends(m):
        q1, s1 = fp8.quant(x[p].clone())
        assert torch.equal(q[p].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[p], s1) and q1.float().any()


def test_router_of_many_tokens():
    """5 million tokens: logits past 4 GiB."""
    _free(60)
    t, e, k = 5_000_011, 256, 4
    logits = torch.empty(t, e, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    block = torch.randn(9973, e, generator=g, device=DEV)
    for at in range(0, t, 9973):
        logits[at:at + 9973] = block[:min(9973, t - at)]
    weights, chosen, plan = experts.route(logits, k)
    for p in _ends(t):
        w1, c1, _ = experts.route(logits[p].clone(), k)
        assert torch.equal(weights[p], w1) and torch.equal(chosen[p], c1)
    token = torch.arange(t, device=DEV, dtype=torch.int32).repeat_interleave(k)
    flat = chosen.flatten()
    order = torch.sort(flat, stable=True)
    assert torch.equal(plan.rows, token[order.indices])
    assert torch.equal(plan.slots.flatten()[order.indices], torch.arange(t * k, device=DEV, dtype=torch.int32))
    assert torch.equal(plan.offsets[1:].long(), torch.bincount(flat, minlength=e).cumsum(0))
