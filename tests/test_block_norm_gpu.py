"""hk.ops.block_norm on the GPU against the float64 oracle (oracle/mxfp4_oracle.py): both outputs over
types, gates and sizes (odd ones, one row, one column), the quantized output, the gradients against
float64 autograd and against differences, and the calls that are refused.

Tolerances. A stored value is one rounding of its type (2^-9 of it for bf16, 2^-12 for fp16, with a factor
2) from an fp32 result whose own error is some 2^-20 of the terms it is made of; terms are bounded by the
largest of a row (an output) or by the sum of magnitudes (a gradient summed over rows)."""

import pytest
import torch

import hk
from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROUND = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -22}
LEAST = {BF16: 0.0, F16: 2.0 ** -24, F32: 0.0}  # (fp16's subnormal step)
FP32_TERMS = 2.0 ** -18

TYPES = [(BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16), (F32, F32, F32)]
GATES = ["none", "channel", "sequence", "token", "one", "full"]


def _gate(kind, shape, g, dtype):
    b, s, d = shape
    size = {"none": None, "channel": (d,), "sequence": (b, 1, d), "token": (b, s, 1), "one": (1,),
            "full": (b, s, d)}[kind]
    return None if size is None else (torch.randn(size, generator=g) * 0.5 + 0.5).to(dtype)


def _inputs(shape, types, gate, seed, gate_dtype=None):
    g = torch.Generator().manual_seed(seed)
    xt, rt, wt = types
    d = shape[-1]
    x = torch.randn(shape, generator=g).to(xt)
    r = (torch.randn(shape, generator=g) * 2).to(rt)
    w1 = (torch.randn(d, generator=g) * 0.3 + 1).to(wt)
    w2 = (torch.randn(d, generator=g) * 0.3 + 1).to(wt)
    return dict(x=x, residual=r, post=w1, pre=w2, gate=_gate(gate, shape, g, gate_dtype or xt))


SCALES = dict(branch_scale=0.7, residual_scale=1.3)


def _on(args):
    return {n: (t.to(DEV) if torch.is_tensor(t) else t) for n, t in args.items()}


def _near(got, ref, dtype, terms):
    tol = ROUND[dtype] * ref.abs() + LEAST[dtype] + FP32_TERMS * terms
    off = (got.cpu().double() - ref).abs()
    assert got.dtype == dtype and got.shape == ref.shape
    over = ref.abs() > torch.finfo(dtype).max  # (a sum past fp16's range is its infinity)
    assert (got.cpu()[over] == torch.sign(ref[over]) * float("inf")).all()
    off = torch.where(over, torch.zeros_like(off), off)
    assert (off <= tol).all(), f"{float((off / (tol + 1e-300)).max()):.3g} times the tolerance"


def _rowmax(t):
    return t.abs().amax(-1, keepdim=True)


SHAPES = [(1, 1, 1), (1, 1, 8), (2, 3, 40), (1, 5, 64), (3, 1, 500), (2, 2, 512), (1, 3, 520), (2, 7, 1000),
          (1, 2, 1024), (2, 2, 1111), (1, 3, 2048), (2, 5, 4096), (1, 2, 5001), (1, 3, 8192)]


@pytest.mark.parametrize("types", TYPES, ids=["bf16", "bf16r32", "fp16", "fp16r32", "fp32"])
@pytest.mark.parametrize("shape", SHAPES + [(1, 2, 9000), (1, 1, 12345), (1, 2, 16384)])
def test_forward(shape, types):
    gate = GATES[sum(shape) % len(GATES)]
    print(f"case norm {shape} {types} {gate}", flush=True)
    a = _inputs(shape, types, gate, sum(shape))
    h, y = hk.ops.block_norm(**_on(a), **SCALES)
    rh, ry = O.block_norm(**a, **SCALES)
    terms = a["residual"].double().abs() + _rowmax(rh)
    _near(h, rh, types[1], terms)
    _near(y, ry, types[0], _rowmax(ry))


@pytest.mark.parametrize("gate_dtype", [BF16, F32])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("d", [96, 333, 2048])
def test_forward_gates(d, gate, gate_dtype):
    a = _inputs((3, 5, d), (BF16, F32, BF16), gate, d, gate_dtype)
    h, y = hk.ops.block_norm(**_on(a), **SCALES)
    rh, ry = O.block_norm(**a, **SCALES)
    _near(h, rh, F32, a["residual"].double().abs() + _rowmax(rh))
    _near(y, ry, BF16, _rowmax(ry))


@pytest.mark.parametrize("post,pre", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("d", [77, 512, 4096])
def test_without_a_norm(d, post, pre):
    a = _inputs((2, 3, d), (BF16, BF16, BF16), "channel", d)
    if not post:
        a["post"] = None
    if not pre:
        a["pre"] = None
    h, y = hk.ops.block_norm(**_on(a), eps=1e-5)
    rh, ry = O.block_norm(**a, eps=1e-5)
    _near(h, rh, BF16, a["residual"].double().abs() + _rowmax(rh))
    if pre:
        _near(y, ry, BF16, _rowmax(ry))
    else:
        assert y is None


def test_weights_of_two_types():
    a = _inputs((2, 3, 256), (BF16, BF16, BF16), "none", 1)
    a["pre"] = a["pre"].float()
    h, y = hk.ops.block_norm(**_on(a))
    rh, ry = O.block_norm(**a)
    _near(h, rh, BF16, a["residual"].double().abs() + _rowmax(rh))
    _near(y, ry, BF16, _rowmax(ry))


def test_rows_that_are_zero_or_not_finite():
    a = _inputs((1, 6, 640), (F32, F32, F32), "none", 2)
    a["x"][0, 1] = 0.0
    a["residual"][0, 2] = 0.0
    a["x"][0, 2] = 0.0
    a["x"][0, 3, 5] = float("nan")
    a["residual"][0, 4, 9] = float("inf")
    h, y = (t.cpu() for t in hk.ops.block_norm(**_on(a)))
    rh, ry = O.block_norm(**a)
    rows = torch.tensor([0, 1, 2, 5])
    _near(h[0, rows], rh[0, rows], F32, a["residual"][0, rows].double().abs() + _rowmax(rh[0, rows]))
    _near(y[0, rows], ry[0, rows], F32, _rowmax(ry[0, rows]))
    assert not y[0, 2].any()
    assert torch.isnan(h[0, 3]).all() and torch.isnan(y[0, 3]).all()
    assert torch.isinf(h[0, 4, 9]) and torch.isfinite(h[0, 4]).sum() == 639
    assert torch.isnan(y[0, 4, 9]) and (y[0, 4, :9] == 0).all()


@pytest.mark.parametrize("d", [264, 1111])
def test_strides(d):
    """Rows of a wider tensor, a transposed batch, rows that start at odd elements."""
    g = torch.Generator().manual_seed(d)
    wide = torch.randn(7, 2 * d + 16, generator=g).to(BF16)
    res = torch.randn(d, 7, generator=g).to(BF16)
    a = dict(x=wide[:, 8:8 + d], residual=res.t(), post=torch.randn(d + 1, generator=g).to(BF16)[1:],
             pre=torch.randn(2 * d, generator=g).to(BF16)[::2], gate=wide[:, d + 9:d + 10])
    dev = _on(dict(w=wide, r=res))
    h, y = hk.ops.block_norm(dev["w"][:, 8:8 + d], dev["r"].t(), post=a["post"].to(DEV), pre=a["pre"].to(DEV),
                             gate=dev["w"][:, d + 9:d + 10])
    rh, ry = O.block_norm(**a)
    _near(h, rh, BF16, a["residual"].double().abs() + _rowmax(rh))
    _near(y, ry, BF16, _rowmax(ry))


@pytest.mark.parametrize("quant", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("shape,types", [((1, 1, 32), 0), ((3, 5, 96), 1), ((2, 2, 512), 2), ((4, 33, 1056), 3),
                                         ((1, 3, 4096), 4), ((2, 16, 4096), 0), ((1, 2, 16384), 1)])
def test_quantized(shape, types, quant):
    """y's numbers are the quantization of an fp32 y: a value that fp32's error moves over a rounding
    boundary is a step off, so each is within half a step of the exact y, and that error."""
    a = _inputs(shape, TYPES[types], GATES[sum(shape) % 6], 3)
    h, (q, s) = hk.ops.block_norm(**_on(a), **SCALES, quant=quant)
    rh, ry = O.block_norm(**a, **SCALES)
    d = shape[-1]
    ry = ry.reshape(-1, d)
    assert q.shape[:-1] == s.shape[:-1] == shape[:-1]
    q, s = q.flatten(0, -2), s.flatten(0, -2)
    v = O.values(q.cpu(), s.cpu())
    _near(h, rh, TYPES[types][1], a["residual"].double().abs() + _rowmax(rh))
    assert s.shape == (ry.shape[0], d // 32)
    scale = torch.exp2(s.cpu().double() - 127).repeat_interleave(32, 1)
    top = 448.0 if quant == "mxfp8" else 6.0
    near = torch.ldexp(torch.ones(()), torch.frexp(ry.abs() / scale)[1] - 1).double()  # 2^floor(log2)
    step = (near.clamp(min=2.0 ** -6) * 2.0 ** -3 if quant == "mxfp8" else near.clamp(min=1.0) * 0.5) * scale
    assert ((v - ry).abs() <= 0.5 * step + FP32_TERMS * _rowmax(ry)).all()
    amax = ry.abs().reshape(-1, d // 32, 32).amax(-1)
    block = torch.exp2(s.cpu().double() - 127)
    assert (amax <= top * block * (1 + 1e-5)).all() and (amax > top / 2 * block * (1 - 1e-5)).all()
    if quant == "mxfp8":
        assert torch.equal(hk.ops.mxfp8.dequant(q, s, F32).cpu().double(), v)
        assert (v != O.quant8(ry)).double().mean() < 1e-3


def _grads(a, dh, dy, **kw):
    names = [n for n, t in a.items() if t is not None]
    leaf = {n: a[n].clone().requires_grad_() for n in names}
    h, y = (O.block_norm if kw.pop("exact") else hk.ops.block_norm)(
        **{n: leaf.get(n) for n in a}, **kw)
    outs, grads = ([h], [dh]) if y is None else ([h, y], [dh, dy])
    return dict(zip(names, torch.autograd.grad(outs, [leaf[n] for n in names], grads)))


def _check_grads(a, seed, **kw):
    """Each gradient against float64 autograd, its terms' magnitudes from the formula."""
    g = torch.Generator().manual_seed(seed)
    dh = torch.randn(a["x"].shape, generator=g).to(a["residual"].dtype)
    dy = torch.randn(a["x"].shape, generator=g).to(a["x"].dtype)
    double = {n: (t.double() if t is not None else None) for n, t in a.items()}
    want = _grads(double, dh.double(), dy.double(), exact=True, **kw)
    got = _grads(_on(a), dh.to(DEV), dy.to(DEV), exact=False, **kw)
    x = double["x"]
    big = _rowmax(want["residual"]) + _rowmax(dh.double()) + 1e-3
    xh = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) if a["post"] is not None else x
    u = xh if a["post"] is None else xh * double["post"]
    gate = double["gate"] if a["gate"] is not None else torch.ones(())
    terms = {"residual": 2 * big, "x": _rowmax(want["x"]) + big * gate.abs() / (
        torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) if a["post"] is not None else 1)}
    flat = tuple(range(x.dim() - 1))
    if "post" in want:
        terms["post"] = (big * gate.abs() * xh.abs()).sum(flat)
    if "pre" in want:
        h, y = O.block_norm(**double, **kw)
        hh = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6)
        terms["pre"] = (dy.double().abs() * (hh.abs() + _rowmax(hh))).sum(flat)
    if "gate" in want:
        terms["gate"] = (big * u.abs()).sum_to_size(a["gate"].shape)
    for n in want:
        try:
            _near(got[n], want[n], a[n].dtype, 2 * terms[n])
        except AssertionError as e:
            raise AssertionError(f"d{n}: {e}") from None


@pytest.mark.parametrize("types", TYPES, ids=["bf16", "bf16r32", "fp16", "fp16r32", "fp32"])
@pytest.mark.parametrize("shape", SHAPES + [(2, 300, 264), (3, 333, 1111), (2, 700, 64), (1, 1000, 130)])
def test_gradients(shape, types):
    gate = GATES[(sum(shape) + len(str(types))) % len(GATES)]
    print(f"case grad {shape} {types} {gate}", flush=True)
    _check_grads(_inputs(shape, types, gate, sum(shape)), sum(shape), **SCALES)


@pytest.mark.parametrize("gate_dtype", [BF16, F32])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("shape", [(3, 40, 96), (2, 9, 333), (3, 200, 1536), (700, 2, 64), (1500, 1, 40)])
def test_gradients_of_gates(shape, gate, gate_dtype):
    print(f"case grad gate {shape} {gate} {gate_dtype}", flush=True)
    _check_grads(_inputs(shape, (BF16, F32, F32), gate, 5, gate_dtype), 6, **SCALES)


@pytest.mark.parametrize("post,pre", [(False, True), (True, False), (False, False)])
@pytest.mark.parametrize("d", [77, 512, 4096])
def test_gradients_without_a_norm(d, post, pre):
    a = _inputs((2, 3, d), (F32, F32, F32), "channel", d)
    if not post:
        a["post"] = None
    if not pre:
        a["pre"] = None
    _check_grads(a, d, **SCALES)


@pytest.mark.parametrize("shape,gate", [((2, 3, 96), "sequence"), ((1, 4, 130), "token"), ((2, 2, 1032), "channel")])
def test_gradients_against_differences(shape, gate):
    """Central differences of the float64 oracle along random directions."""
    a = _inputs(shape, (F32, F32, F32), gate, 8)
    g = torch.Generator().manual_seed(9)
    dh, dy = torch.randn(shape, generator=g), torch.randn(shape, generator=g)
    got = _grads(_on(a), dh.to(DEV), dy.to(DEV), exact=False, **SCALES)

    def loss(v):
        h, y = O.block_norm(**v, **SCALES)
        return float((h * dh.double()).sum() + (y * dy.double()).sum())

    for n in a:
        way = torch.randn(a[n].shape, generator=g).double()
        eps = 1e-6
        lo, hi = ({**{k: t.double() for k, t in a.items()}, n: a[n].double() + f * eps * way} for f in (-1, 1))
        slope = (loss(hi) - loss(lo)) / (2 * eps)
        mine = float((got[n].cpu().double() * way).sum())
        size = float((got[n].cpu().double() * way).abs().sum())
        assert abs(mine - slope) <= 1e-5 * size + 1e-4, n


def test_gradients_of_one_output_and_of_some_inputs():
    a = _on(_inputs((2, 5, 520), (BF16, F32, BF16), "sequence", 11))
    for use in ("h", "y"):
        leaf = {n: t.clone().requires_grad_(n in ("x", "gate")) for n, t in a.items()}
        h, y = hk.ops.block_norm(**leaf)
        (h if use == "h" else y).float().square().sum().backward()
        ref = {n: t.cpu().double().requires_grad_(n in ("x", "gate")) for n, t in a.items()}
        rh, ry = O.block_norm(**ref)
        (rh if use == "h" else ry).square().sum().backward()
        for n in ("x", "gate"):
            off = (leaf[n].grad.cpu().double() - ref[n].grad).norm() / ref[n].grad.norm()
            assert off < 2.0 ** -7, (use, n)
        assert leaf["residual"].grad is None and leaf["post"].grad is None


def test_gradients_are_the_same_every_time():
    a = _on(_inputs((3, 333, 520), (BF16, BF16, F32), "sequence", 12))
    dh = torch.randn(3, 333, 520, device=DEV).to(BF16)
    first = _grads(a, dh, dh, exact=False)
    for _ in range(3):
        again = _grads(a, dh, dh, exact=False)
        assert all(torch.equal(first[n], again[n]) for n in first)


def test_in_a_graph():
    a = _on(_inputs((2, 64, 1024), (BF16, F32, BF16), "sequence", 13))
    leaf = {n: t.clone().requires_grad_() for n, t in a.items()}
    dh, dy = torch.randn_like(a["residual"]), torch.randn_like(a["x"])

    def step():
        h, y = hk.ops.block_norm(**leaf)
        return (h, y, *torch.autograd.grad((h, y), list(leaf.values()), (dh, dy)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(w, o) for w, o in zip(want, got))
        eager = step()
        assert torch.equal(eager[2], want[2])


def test_of_nothing():
    x = torch.empty(0, 64, dtype=BF16, device=DEV, requires_grad=True)
    w = torch.ones(64, dtype=BF16, device=DEV, requires_grad=True)
    h, y = hk.ops.block_norm(x, x.detach(), post=w, pre=w)
    assert h.shape == y.shape == (0, 64)
    (h.sum() + y.sum()).backward()
    assert x.grad.shape == (0, 64) and not w.grad.any()


def test_refusals():
    x = torch.zeros(2, 3, 64, dtype=BF16, device=DEV)
    w = torch.ones(64, dtype=BF16, device=DEV)
    f = hk.ops.block_norm
    with pytest.raises(TypeError):
        f(x, x.half(), pre=w)
    with pytest.raises(TypeError):
        f(x.int(), x.int())
    with pytest.raises(TypeError):
        f(x, x, pre=w.half())
    with pytest.raises(ValueError):
        f(x, x[:1], pre=w)
    with pytest.raises(ValueError):
        f(x, x, pre=w[:32])
    with pytest.raises(ValueError):
        f(x, x, pre=w, gate=torch.ones(2, 3, 32, dtype=BF16, device=DEV))
    with pytest.raises(ValueError):
        f(x, x, pre=w, gate=torch.ones(1, 3, 64, dtype=BF16, device=DEV))
    with pytest.raises(ValueError):
        f(x, x, pre=w.cpu())
    with pytest.raises(ValueError):
        f(x.cpu(), x.cpu())
    with pytest.raises(ValueError):
        f(x, x, pre=w, quant="int8")
    with pytest.raises(ValueError):
        f(x, x, quant="mxfp8")
    with pytest.raises(ValueError):
        f(x[..., :40], x[..., :40], pre=w[:40], quant="mxfp4")
    with pytest.raises(ValueError):
        f(x.clone().requires_grad_(), x, pre=w, quant="mxfp8")
    big = torch.zeros(1, 16385, device=DEV)
    with pytest.raises(ValueError):
        f(big, big)
    with pytest.raises(ValueError):
        f(big[:, :8193].clone().requires_grad_(), big[:, :8193])
