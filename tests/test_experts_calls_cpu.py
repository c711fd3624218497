"""Derivatives that hk.ops.experts, hk.ops.fp8 and hk.ops.block_norm do not take are refused, not dropped (no GPU: the
library is a stub that launches nothing)."""

import ctypes
import types

import pytest
import torch
import torch.autograd.forward_ad as ad

import hk  # noqa: F401
from hk import _native as nat
from hk.ops import block_norm, experts, fp8, norm

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU."""

    is_cuda = True

    def get_device(self):
        return 0


def _t(*size, dtype=BF16):
    return torch.zeros(size, dtype=dtype).as_subclass(OnGpu)


PLAN = experts.Plan(_t(5, dtype=torch.int32), _t(24, dtype=torch.int32), _t(12, 2, dtype=torch.int32))


@pytest.fixture
def stub(monkeypatch):
    class Lib:
        def __getattr__(self, name):
            return lambda *a: 0

    monkeypatch.setattr(nat, "lib", lambda: Lib())
    monkeypatch.setattr(nat, "stream_of", lambda device: 0)
    monkeypatch.setattr(nat, "current", lambda device: nat._HERE)
    monkeypatch.setattr(nat, "empty", lambda like, shape, dtype: _t(*shape, dtype=dtype))
    for module, stores in ((experts, ("_GEMM", "_COMBINE", "_ROUTE")), (fp8, ("_QUANT",)), (norm, ("_PLANS",))):
        for name in stores:
            monkeypatch.setattr(module, name, {})


def _calls():
    """(what is called, its arguments, the names of those that may carry a derivative)."""
    gemm = dict(x=_t(24, 32), w=_t(4, 40, 32), bias=_t(4, 40))
    wide = dict(x=_t(24, 32).to(E4M3), w=_t(4, 40, 32).to(E4M3), scale_a=_t(24, dtype=F32), scale_b=_t(4, 40, dtype=F32))
    rows = dict(y=_t(24, 32), weights=_t(12, 2, dtype=F32))
    norms = dict(x=_t(6, 64), residual=_t(6, 64), pre=_t(64), post=_t(64), gate=_t(6, 64))
    return [
        ("gemm", lambda x, w, **kw: experts.gemm(x, w, PLAN, **kw), gemm, ("x", "w", "bias")),
        ("gemm", lambda x, w, **kw: experts.gemm(x, w, PLAN, **kw), wide, ("scale_a", "scale_b")),
        ("combine", lambda y, weights: experts.combine(y, PLAN, weights), rows, ("y", "weights")),
        ("route", lambda logits: experts.route(logits, 2), dict(logits=_t(12, 4, dtype=F32)), ("logits",)),
        ("fp8.quant", fp8.quant, dict(x=_t(6, 64)), ("x",)),
        ("block_norm", block_norm, norms, tuple(norms)),
        ("block_norm", lambda **kw: block_norm(**kw, quant="fp8"), norms, tuple(norms)),
        ("block_norm", lambda **kw: block_norm(**kw, quant="mxfp8"), norms, tuple(norms)),
    ]


@pytest.mark.parametrize("at", range(8))
@pytest.mark.parametrize("known", [False, True])
def test_a_forward_mode_derivative_is_refused(stub, at, known):
    call, run, given, names = _calls()[at]
    for name in names:
        if known:
            run(**given)  # (a call of known layout checks too)
        with ad.dual_level():
            run(**given)  # (a level alone is none's business)
            dual = dict(given, **{name: ad.make_dual(given[name], torch.ones_like(given[name]))})
            with pytest.raises(ValueError, match=f"{call}: no forward-mode"):
                run(**dual)


def test_a_forward_mode_derivative_beside_gradients_is_refused(stub):
    w = _t(4, 40, 32).requires_grad_()
    with ad.dual_level(), pytest.raises(ValueError, match="gemm: no forward-mode"):
        experts.gemm(ad.make_dual(_t(24, 32), _t(24, 32)), w, PLAN)


@pytest.mark.parametrize("name", ["scale_a", "scale_b"])
@pytest.mark.parametrize("known", [False, True])
def test_a_gradient_of_a_scale_is_refused(stub, name, known):
    _, run, given, _ = _calls()[1]
    if known:
        run(**given)
    wants = dict(given, **{name: given[name].clone().requires_grad_()})
    with pytest.raises(ValueError, match="quantized"):
        run(**wants)
    with torch.no_grad():
        run(**wants)


def test_a_gradient_of_a_layers_scales_is_refused(stub):
    x, up, down = _t(12, 32), _t(4, 64, 32).to(E4M3), _t(4, 32, 32).to(E4M3)
    scales = dict(gate_up_scale=_t(4, 64, dtype=F32), down_scale=_t(4, 32, dtype=F32))
    for name in scales:
        wants = dict(scales, **{name: scales[name].clone().requires_grad_()})
        with pytest.raises(ValueError, match="quantized"):
            experts.mlp(x, _t(12, 4, dtype=F32), 2, up, down, **wants)


@pytest.mark.parametrize("quant", [None, "fp8"])
def test_block_norm_is_launched_on_its_tensors_device(stub, monkeypatch, quant):
    """The stream alone does not say which: device 0's default stream and device 1's are both 0."""
    inside, at = [], []

    class Current:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            inside.append(self.device)

        def __exit__(self, *a):
            inside.pop()

    class Lib:
        def __getattr__(self, name):
            return lambda *a: at.append((name, list(inside))) or 0

    monkeypatch.setattr(nat, "lib", lambda: Lib())
    monkeypatch.setattr(nat, "current", Current)
    x, pre = _t(6, 64), _t(64)
    for _ in range(2):  # (and of known layout)
        block_norm(x, x, pre=pre, quant=quant)
    want = [("hkx_block_norm", [x.device])] * 2
    if quant is None:
        leaf = x.clone().requires_grad_()
        h, y = block_norm(leaf, x, pre=pre)
        torch.autograd.grad((h, y), leaf, (x, x))
        want += [("hkx_block_norm", [x.device]), ("hkx_block_norm_backward", [x.device])]
    assert [(n, d) for n, d in at if not n.endswith("workspace")] == want


def test_tokens_whose_plan_has_no_rows_have_a_gradient_of_zeros(stub, monkeypatch):
    """Every choice dropped: no rows, and slots of -1. Nothing is launched (the library refuses a null address)."""

    class Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} of no rows")

    monkeypatch.setattr(nat, "lib", lambda: Lib())
    x, w = _t(12, 32).requires_grad_(), _t(4, 40, 32).requires_grad_()
    slots = torch.full((12, 2), -1, dtype=torch.int32).as_subclass(OnGpu)
    y = experts.gemm(x, w, experts.Plan(PLAN.offsets, _t(0, dtype=torch.int32), slots), gather=True)
    assert y.shape == (0, 40)
    dx, dw = torch.autograd.grad(y, (x, w), _t(0, 40))
    assert dx.shape == (12, 32) and dw.shape == (4, 40, 32) and not dx.any() and not dw.any()


def test_rows_whose_tiles_an_int_does_not_count_are_refused():
    """A group of rows is counted in tiles of up to 256: rows + 255 is an int too."""
    L, at = nat.lib(), 1 << 20
    most = 2 ** 31 - 1 - 255
    for op, sizes in ((experts.NT, dict(k=8)), (experts.NN, dict(k=8)), (experts.TN, dict(m=8))):
        g = nat.HkxExpertsGemmArgs()
        g.size, g.op, g.ab_dtype, g.experts, g.n, g.kernel = ctypes.sizeof(g), op, nat.BF16, 2, 8, 4
        g.a = g.b = g.c = g.offsets = at
        g.lda = g.ldb = g.ldc = 8
        g.b_expert = g.c_expert = 64
        for name, v in sizes.items():
            setattr(g, name, v)
        for rows in (most + 1, 2 ** 31 - 1):
            g.rows = rows
            assert L.hkx_experts_gemm(ctypes.byref(g), None) == nat.ERR_SHAPE and "rows" in nat.last_error()
    for rows in (most + 1, 2 ** 31 - 1):
        assert L.hkx_experts_bias_grad(at, 8, at, at, nat.BF16, 2, rows, 8, None) == nat.ERR_SHAPE


def test_the_rows_gradients_refusals():
    L, at = nat.lib(), 1 << 20
    for rc, code in [
        (L.hkx_experts_gather_grad(None, 8, at, at, 8, 4, 2, 8, 8, None), nat.ERR_ARG),
        (L.hkx_experts_gather_grad(at, 8, None, at, 8, 4, 2, 8, 8, None), nat.ERR_ARG),
        (L.hkx_experts_gather_grad(at, 8, at, None, 8, 4, 2, 8, 8, None), nat.ERR_ARG),
        (L.hkx_experts_gather_grad(at, 7, at, at, 8, 4, 2, 8, 8, None), nat.ERR_SHAPE),
        (L.hkx_experts_gather_grad(at, 8, at, at, 7, 4, 2, 8, 8, None), nat.ERR_SHAPE),
        (L.hkx_experts_gather_grad(at, 8, at, at, 8, 4, 0, 8, 8, None), nat.ERR_SHAPE),
        (L.hkx_experts_gather_grad(at, 8, at, at, 8, 4, 2, -1, 8, None), nat.ERR_SHAPE),
        (L.hkx_experts_gather_grad(at + 2, 8, at, at, 8, 4, 2, 8, 8, None), nat.ERR_SHAPE),
        (L.hkx_experts_gather_grad(at, 8, at, at + 1, 8, 4, 2, 8, 8, None), nat.ERR_SHAPE),
        (L.hkx_experts_gather_grad(at, 8, at, at, 8, 0, 2, 8, 8, None), nat.OK),
    ]:
        assert rc == code, nat.last_error()


@pytest.mark.parametrize("kw,code,match", [
    (dict(op=experts.NT), nat.ERR_DTYPE, "fp32 where"), (dict(op=experts.TN, m=8, c_expert=64), nat.ERR_DTYPE, "fp32 where"),
    (dict(c_dtype=nat.FP16), nat.ERR_DTYPE, "fp32 where"), (dict(c=(1 << 20) + 8), nat.ERR_SHAPE, "an fp32 C's 16"),
    (dict(ldc=10), nat.ERR_SHAPE, "an fp32 C's 16"), (dict(ldc=1 << 22), nat.ERR_SHAPE, "4 GiB")])
def test_an_fp32_product_is_the_rows_gradient_alone(kw, code, match):
    at = 1 << 20
    g = nat.HkxExpertsGemmArgs()
    g.size, g.op, g.ab_dtype, g.c_dtype = ctypes.sizeof(g), experts.NN, nat.BF16, nat.FP32
    g.experts, g.rows, g.n, g.k = 2, 24, 8, 8
    g.a = g.b = g.c = g.offsets = at
    g.lda = g.ldb = g.ldc = 8
    g.b_expert = 64
    for name, v in kw.items():
        setattr(g, name, v)
    assert nat.lib().hkx_experts_gemm(ctypes.byref(g), None) == code and match in nat.last_error()


def test_only_a_gathered_rows_product_is_fp32(monkeypatch, stub):
    seen = []

    class Lib:
        def __getattr__(self, name):
            def call(*a):
                if name == "hkx_experts_gemm":
                    seen.append((a[0]._obj.op, a[0]._obj.c_dtype))
                return 0
            return call

    monkeypatch.setattr(nat, "lib", lambda: Lib())
    w = _t(4, 40, 32).requires_grad_()
    for gather, x in ((False, _t(24, 32)), (True, _t(12, 32))):
        x.requires_grad_()
        torch.autograd.grad(experts.gemm(x, w, PLAN, gather=gather), (x, w), _t(24, 40))
    bf16 = nat.BF16
    assert seen == [(experts.NT, bf16), (experts.NN, bf16), (experts.TN, bf16),
                    (experts.NT, bf16), (experts.NN, nat.FP32), (experts.TN, bf16)]
