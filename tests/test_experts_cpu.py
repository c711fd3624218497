"""hk.ops.experts and hk.ops.fp8 without a GPU: the oracle against torch, what the calls refuse, what they pass to the
library, and the C calls' own refusals (nothing is launched)."""

import ctypes
import functools
import math
import shutil
import subprocess
import tempfile
from pathlib import Path
import math
import types

import pytest
import torch

import hk  # noqa: F401
from hk import _native as nat
from hk.ops import experts, fp8
from oracle import experts_oracle as O

BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
AT = 1 << 20


class OnGpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU."""

    is_cuda = True

    def get_device(self):
        return 0


def _t(*size, dtype=BF16):
    return torch.zeros(size, dtype=dtype).as_subclass(OnGpu)


def _plan(e=4, r=24, t=12, k=2):
    return experts.Plan(_t(e + 1, dtype=torch.int32), _t(r, dtype=torch.int32), _t(t, k, dtype=torch.int32))


# ------------------------------------------------------------------ the oracle


def test_the_oracles_router_is_a_stable_sort():
    g = torch.Generator().manual_seed(0)
    logits = (torch.randn(50, 12, generator=g) * 2).round()
    weights, chosen, offsets, rows, slots = O.route(logits, 4)
    top = torch.sort(logits, dim=1, descending=True, stable=True)
    assert torch.equal(chosen, top.indices[:, :4])
    torch.testing.assert_close(weights, torch.softmax(top.values[:, :4].double(), 1))
    all_weights = O.route(logits, 4, renormalize=False)[0]
    torch.testing.assert_close(all_weights, torch.gather(torch.softmax(logits.double(), 1), 1, chosen))
    assert offsets[-1] == 200 and (offsets[1:] >= offsets[:-1]).all()
    assert torch.equal(rows[slots], torch.arange(50).unsqueeze(1).expand(50, 4))
    of = torch.bucketize(slots, offsets[1:], right=True)
    assert torch.equal(of, chosen)


def test_the_oracles_router_with_missing_experts():
    logits = torch.tensor([[0.0, -math.inf, 1.0], [-math.inf] * 3, [math.nan, 2.0, 5.0]])
    weights, chosen, offsets, rows, slots = O.route(logits, 2)
    assert chosen.tolist() == [[2, 0], [-1, -1], [0, 2]] and slots.tolist() == [[2, 0], [-1, -1], [1, 3]]
    assert offsets.tolist() == [0, 2, 2, 4] and rows.tolist() == [0, 2, 0, 2, -1, -1]
    assert not weights[1].any() and torch.isnan(weights[2]).all()


def test_the_oracles_rows_of_8_bits():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 96, generator=g)
    x[3] = 0
    v, s = O.quant8(x)
    assert torch.equal(v.float(), (x / s.float()).to(E4M3).float()) and s[3] == 1
    x[5, 7] = math.inf
    assert torch.isnan(O.quant8(x)[1][5])


# ------------------------------------------------------------------ refusals


def _refused(error, match, call, *args, **kw):
    with pytest.raises(error, match=match):
        call(*args, **kw)


def test_gemm_refuses():
    x, w, plan = _t(24, 32), _t(4, 40, 32), _plan()
    for error, match, args, kw in [
        (TypeError, "both bf16 or both", (x.float(), w, plan), {}),
        (TypeError, "both bf16 or both", (x, w.to(E4M3), plan), {}),
        (ValueError, "K\\)", (_t(24, 24), w, plan), {}),
        (ValueError, "K\\)", (x, _t(40, 32), plan), {}),
        (ValueError, "multiple of 8", (x, _t(4, 36, 32), plan), {}),
        (ValueError, "multiple of 8", (_t(24, 36), _t(4, 40, 36), plan), {}),
        (ValueError, "gate rows", (x, _t(4, 41, 32), plan), dict(silu_mul=True)),
        (ValueError, "multiple of 8", (x, _t(4, 40, 32), plan), dict(silu_mul=True)),
        (ValueError, "experts", (x, _t(1025, 8, 32), plan), {}),
        (ValueError, "plan.offsets", (x, _t(5, 40, 32), plan), {}),
        (ValueError, "plan.offsets", (x, w, experts.Plan(None)), {}),
        (TypeError, "int32", (x, w, plan._replace(offsets=plan.offsets.long())), {}),
        (TypeError, "int32", (x, w, plan._replace(rows=plan.rows.long())), dict(gather=True)),
        (ValueError, "gather takes", (x, w, experts.Plan(plan.offsets)), dict(gather=True)),
        (ValueError, "from none", (_t(0, 32), w, plan), dict(gather=True)),
        (ValueError, "gather=True", (_t(12, 32), w, plan), {}),
        (ValueError, "bias", (x, w, plan), dict(bias=_t(4, 41))),
        (ValueError, "bias", (x, w, plan), dict(bias=_t(4, 40, dtype=torch.int32))),
        (ValueError, "scales go", (x, w, plan), dict(scale_a=_t(1, dtype=F32))),
        (TypeError, "scale_a", (x.to(E4M3), w.to(E4M3), plan), {}),
        (TypeError, "scale_b", (x.to(E4M3), w.to(E4M3), plan), dict(scale_a=_t(1, dtype=F32), scale_b=_t(4, 40))),
        (ValueError, "scale_a", (x.to(E4M3), w.to(E4M3), plan), dict(scale_a=_t(23, dtype=F32), scale_b=_t(4, dtype=F32))),
        (ValueError, "scale_b", (x.to(E4M3), w.to(E4M3), plan), dict(scale_a=_t(24, dtype=F32), scale_b=_t(40, dtype=F32))),
        (ValueError, "out is", (x, w, plan), dict(out=_t(24, 41))),
        (ValueError, "out is", (x, w, plan), dict(out=_t(40, 24).t())),
        (ValueError, "out is", (x, w, plan), dict(out=_t(24, 40, dtype=F32))),
        (ValueError, "on a GPU", (torch.zeros(24, 32, dtype=BF16), w, plan), {}),
        (ValueError, "not on", (x, torch.zeros(4, 40, 32, dtype=BF16, device="meta"), plan), {}),
    ]:
        _refused(error, match, experts.gemm, *args, **kw)


def test_gemm_with_gradients_refuses():
    x, w, plan = _t(24, 32), _t(4, 40, 32), _plan()
    w.requires_grad_()
    _refused(ValueError, "out=", experts.gemm, x, w, plan, out=_t(24, 40))
    _refused(ValueError, "quantized", experts.gemm, x.to(E4M3), w, plan)
    x = _t(12, 32).requires_grad_()
    _refused(ValueError, "slots", experts.gemm, x, w, plan._replace(slots=None), gather=True)
    _refused(ValueError, "slots", experts.gemm, x, w, plan._replace(slots=_t(11, 2, dtype=torch.int32)), gather=True)


def test_combine_and_route_refuse():
    y, plan = _t(24, 32), _plan()
    for error, match, args in [
        (TypeError, "bf16, fp16 or fp32", (y.to(E4M3), plan)), (TypeError, "bf16, fp16 or fp32", (_t(24), plan)),
        (ValueError, "slots", (_t(23, 32), plan)), (ValueError, "slots", (y, plan._replace(slots=None))),
        (TypeError, "int32", (y, plan._replace(slots=plan.slots.long()))),
        (ValueError, "weights", (y, plan, _t(12, 2))), (ValueError, "weights", (y, plan, _t(12, 3, dtype=F32))),
        (ValueError, "on a GPU", (torch.zeros(24, 32), plan)),
    ]:
        _refused(error, match, experts.combine, *args)
    for error, match, args in [
        (TypeError, "T, E", (_t(4, 3, 8), 2)), (TypeError, "T, E", (_t(4, 8, dtype=torch.int32), 2)),
        (ValueError, "k=0", (_t(4, 8), 0)), (ValueError, "k=9", (_t(4, 8), 9)), (ValueError, "k=65", (_t(4, 80), 65)),
        (ValueError, "1025", (_t(4, 1025), 2)), (ValueError, "on a GPU", (torch.zeros(4, 8), 2)),
    ]:
        _refused(error, match, experts.route, *args)


def test_fp8_quant_refuses():
    _refused(TypeError, "bf16, fp16 or fp32", fp8.quant, _t(4, 16, dtype=torch.int32))
    _refused(ValueError, "K=0", fp8.quant, _t(4, 0))
    _refused(ValueError, "on a GPU", fp8.quant, torch.zeros(4, 16))
    _refused(ValueError, "gradient", fp8.quant, _t(4, 16, dtype=F32).requires_grad_())
    _refused(ValueError, "out is", fp8.quant, _t(4, 16), out=(_t(4, 16, dtype=E4M3), _t(4, dtype=F32)))


def test_mlp_refuses_a_mixed_call():
    x, up, down = _t(12, 32), _t(4, 80, 32), _t(4, 32, 40)
    logits = _t(12, 4, dtype=F32)
    _refused(TypeError, "scales", experts.mlp, (x, _t(12, 1, dtype=F32)), logits, 2, up, down)
    _refused(TypeError, "scales", experts.mlp, x, logits, 2, up, down, gate_up_scale=_t(4, 80, dtype=F32))
    _refused(ValueError, "a row a token", experts.mlp, x[:11], logits, 2, up, down)


# ------------------------------------------------------------------ what a call passes on


@pytest.fixture
def launches(monkeypatch):
    real, seen = nat.lib(), []

    def product(ref, _stream):
        seen.append(nat.HkxExpertsGemmArgs.from_buffer_copy(ref._obj))
        return nat.OK

    monkeypatch.setattr(nat, "lib", lambda: types.SimpleNamespace(
        hkx_experts_gemm=product, hkx_experts_gemm_workspace=real.hkx_experts_gemm_workspace))
    monkeypatch.setattr(nat, "stream_of", lambda device: 0)
    monkeypatch.setattr(nat, "current", lambda device: nat._HERE)
    monkeypatch.setattr(nat, "workspace", lambda device, need: types.SimpleNamespace(data_ptr=lambda: AT))
    monkeypatch.setattr(experts, "_GEMM", {})
    return seen


def test_a_call_of_known_layout_passes_the_same_arguments(launches):
    plan = _plan()
    x, w, bias = _t(12, 32), _t(4, 80, 32), _t(4, 80)
    for _ in range(2):
        experts.gemm(x, w, plan, gather=True, silu_mul=True, bias=bias)
    first, again = launches
    assert len(experts._GEMM) == 1
    for name, _ in nat.HkxExpertsGemmArgs._fields_:
        if name != "c":
            assert getattr(first, name) == getattr(again, name), name
    assert (first.n, first.k, first.rows, first.a_rows, first.experts, first.silu_mul) == (40, 32, 24, 12, 4, 1)
    assert first.index == plan.rows.data_ptr() and first.zero_rest == 1
    experts.gemm(x, w, plan._replace(rows=_t(48, dtype=torch.int32)), gather=True, silu_mul=True, bias=bias)
    assert launches[-1].rows == 48
    experts.gemm(x, w, plan, gather=True, silu_mul=True, bias=bias, out=_t(24, 40))
    assert launches[-1].zero_rest == 0


def test_strides_and_the_workspace(launches):
    big = _t(6, 4096, 4096)
    x = _t(8192, 4096)
    plan = experts.Plan(_t(4, dtype=torch.int32))
    experts.gemm(x, big[::2, 8:2056], plan)
    g = launches[-1]
    assert (g.ldb, g.b_expert, g.lda, g.ldc) == (4096, 2 * 4096 * 4096, 4096, 2048)
    assert g.ws == AT and g.ws_bytes == nat.lib().hkx_experts_gemm_workspace(ctypes.byref(g)) > 0


# ------------------------------------------------------------------ the C calls


def _args(**kw):
    g = nat.HkxExpertsGemmArgs()
    g.size, g.op, g.ab_dtype, g.experts, g.rows, g.n, g.k = ctypes.sizeof(g), experts.NT, nat.BF16, 4, 24, 40, 32
    g.a = g.b = g.c = g.offsets = AT
    g.lda = g.ldb = 32
    g.ldc, g.b_expert = 40, 40 * 32
    for name, v in kw.items():
        setattr(g, name, v)
    return g


FP8 = dict(ab_dtype=nat.FP8E4M3, sa=AT, sb=AT)
TNS = dict(op=experts.TN, m=16, n=40, lda=16, ldb=40, ldc=40, c_expert=16 * 40)


@pytest.mark.parametrize("kw,code,match", [
    (dict(size=8), nat.ERR_ARG, "bytes"), (dict(op=3), nat.ERR_ARG, "op 3"), (dict(ab_dtype=nat.FP32), nat.ERR_DTYPE, "bf16 or e4m3"),
    (dict(a=None), nat.ERR_ARG, "null"), (dict(offsets=None), nat.ERR_ARG, "null"), (dict(FP8, sb=None), nat.ERR_ARG, "null"),
    (dict(FP8, op=experts.NN), nat.ERR_DTYPE, "gradient"), (dict(experts=0), nat.ERR_SHAPE, "experts=0"),
    (dict(experts=1025), nat.ERR_SHAPE, "1024"), (dict(rows=-1), nat.ERR_SHAPE, "rows=-1"), (dict(k=0), nat.ERR_SHAPE, "k=0"),
    (dict(n=36), nat.ERR_SHAPE, "multiples of 8"), (dict(k=28), nat.ERR_SHAPE, "multiples of 8"),
    (dict(FP8, k=24), nat.ERR_SHAPE, "multiples of 8"), (dict(TNS, m=12), nat.ERR_SHAPE, "multiples of 8"),
    (dict(op=experts.NN, silu_mul=1, ldb=40), nat.ERR_ARG, "go with NT"), (dict(TNS, bias=AT), nat.ERR_ARG, "go with NT"),
    (dict(TNS, index=AT), nat.ERR_ARG, "go with NT"), (dict(z=AT, ldz=80), nat.ERR_ARG, "silu_mul"),
    (dict(bias=AT, bias_ld=40, bias_dtype=nat.INT8), nat.ERR_DTYPE, "bias"), (dict(index=AT), nat.ERR_SHAPE, "index into 0"),
    (dict(lda=24), nat.ERR_SHAPE, "row strides"), (dict(ldc=32), nat.ERR_SHAPE, "row strides"),
    (dict(bias=AT, bias_ld=32), nat.ERR_SHAPE, "row strides"), (dict(silu_mul=1, z=AT, ldz=72), nat.ERR_SHAPE, "row strides"),
    (dict(lda=36), nat.ERR_SHAPE, "16-byte"), (dict(a=AT + 8), nat.ERR_SHAPE, "16-byte"), (dict(b_expert=1284), nat.ERR_SHAPE, "16-byte"),
    (dict(c=AT + 4), nat.ERR_SHAPE, "8-byte"), (dict(ldc=42), nat.ERR_SHAPE, "8-byte"),
    (dict(bias=AT + 8, bias_ld=40), nat.ERR_SHAPE, "bias"), (dict(FP8, sb=AT + 4, sb_col=1, sb_ld=40), nat.ERR_SHAPE, "scales"),
    (dict(ldb=1 << 27), nat.ERR_SHAPE, "4 GiB"), (dict(index=AT, a_rows=1 << 30, lda=32), nat.ERR_SHAPE, "4 GiB"),
    (dict(kernel=7), nat.ERR_ARG, "kernel 7"), (dict(kernel=4, c=AT + 8), nat.ERR_SHAPE, "16-byte aligned rows"),
    (dict(kernel=4, k=4096, lda=4096, ldb=4096, b_expert=4096 * 40), nat.ERR_WORKSPACE, "workspace"),
])
def test_the_products_refusals(kw, code, match):
    L = nat.lib()
    g = _args(**kw)
    assert L.hkx_experts_gemm(ctypes.byref(g), None) == code
    assert match in nat.last_error()
    if code != nat.ERR_WORKSPACE:
        assert L.hkx_experts_gemm_workspace(ctypes.byref(g)) == 0


def test_calls_of_no_rows_launch_nothing():
    L = nat.lib()
    assert L.hkx_experts_gemm(ctypes.byref(_args(rows=0)), None) == nat.OK
    assert L.hkx_experts_combine(AT, 8, 0, AT, None, AT, 8, 0, 2, 0, 8, None) == nat.OK
    assert L.hkx_fp8_quant(AT, 16, 0, AT, 16, AT, 0, 16, None) == nat.OK
    assert L.hkx_experts_gather(AT, 16, AT, AT, 16, 0, 4, 16, None) == nat.OK
    assert L.hkx_experts_silu_grad(AT, 32, AT, 16, AT, 32, AT, 4, 0, 16, None) == nat.OK


def test_the_routers_refusals():
    L = nat.lib()

    def call(**kw):
        g = nat.HkxExpertsRouteArgs()
        g.size, g.dtype, g.t, g.e, g.k, g.ld = ctypes.sizeof(g), nat.FP32, 12, 8, 2, 8
        g.logits = g.weights = g.chosen = g.offsets = g.rows = g.slots = AT
        for name, v in kw.items():
            setattr(g, name, v)
        return L.hkx_experts_route(ctypes.byref(g), None), nat.last_error(), L.hkx_experts_route_workspace(ctypes.byref(g))

    for kw, code, match in [(dict(size=4), nat.ERR_ARG, "bytes"), (dict(slots=None), nat.ERR_ARG, "null"),
                            (dict(dtype=nat.INT8), nat.ERR_DTYPE, "logits"), (dict(t=0), nat.ERR_SHAPE, "t=0"),
                            (dict(e=1025, ld=1025), nat.ERR_SHAPE, "e=1025"), (dict(k=9), nat.ERR_SHAPE, "k=9"),
                            (dict(e=80, ld=80, k=65), nat.ERR_SHAPE, "k=65"), (dict(ld=7), nat.ERR_SHAPE, "t=12"),
                            (dict(t=1 << 30, k=2), nat.ERR_SHAPE, "t="), (dict(t=65), nat.ERR_WORKSPACE, "workspace")]:
        rc, msg, need = call(**kw)
        assert rc == code and match in msg, kw
        assert (need > 0) == (code == nat.ERR_WORKSPACE or kw.get("t", 0) > 64)
    assert L.hkx_experts_route_backward(AT, 8, nat.FP32, AT, AT, None, AT, 8, 12, 8, 2, 1, None) == nat.ERR_ARG
    assert L.hkx_experts_route_backward(AT, 8, nat.INT8, AT, AT, AT, AT, 8, 12, 8, 2, 1, None) == nat.ERR_DTYPE
    assert L.hkx_experts_route_backward(AT, 7, nat.FP32, AT, AT, AT, AT, 8, 12, 8, 2, 1, None) == nat.ERR_SHAPE


def test_the_other_calls_refusals():
    L = nat.lib()
    for rc, code in [
        (L.hkx_experts_combine(None, 8, 0, AT, None, AT, 8, 4, 2, 8, 8, None), nat.ERR_ARG),
        (L.hkx_experts_combine(AT, 8, nat.INT8, AT, None, AT, 8, 4, 2, 8, 8, None), nat.ERR_DTYPE),
        (L.hkx_experts_combine(AT, 7, 0, AT, None, AT, 8, 4, 2, 8, 8, None), nat.ERR_SHAPE),
        (L.hkx_experts_combine(AT, 8, 0, AT, None, AT, 8, 1 << 24, 2, 8, 8, None), nat.ERR_SHAPE),
        (L.hkx_experts_combine_backward(None, 8, AT, 8, 0, AT, None, AT, 8, AT, AT, 4, 2, 8, 8, None), nat.ERR_ARG),
        (L.hkx_experts_combine_backward(AT, 8, AT, 8, 0, AT, None, AT, 8, AT, None, 4, 2, 8, 8, None), nat.ERR_ARG),
        (L.hkx_experts_combine_backward(AT, 8, AT, 8, 0, AT, None, None, 8, None, AT, 4, 2, 8, 8, None), nat.ERR_ARG),
        (L.hkx_experts_combine_backward(AT, 8, AT, 8, 0, AT, None, AT, 8, AT, AT + 2, 4, 2, 8, 8, None), nat.ERR_SHAPE),
        (L.hkx_experts_combine_backward(AT, 8, AT, 8, 0, AT, None, AT, 8, AT, AT, 4, 2, 9, 8, None), nat.ERR_SHAPE),
        (L.hkx_fp8_quant(AT, 16, nat.INT8, AT, 16, AT, 4, 16, None), nat.ERR_DTYPE),
        (L.hkx_fp8_quant(AT, 8, 0, AT, 16, AT, 4, 16, None), nat.ERR_SHAPE),
        (L.hkx_fp8_quant(AT + 1, 16, 0, AT, 16, AT, 4, 16, None), nat.ERR_SHAPE),
        (L.hkx_experts_gather(AT, 12, AT, AT, 16, 4, 4, 12, None), nat.ERR_SHAPE),
        (L.hkx_experts_silu_grad(AT, 31, AT, 16, AT, 32, AT, 4, 4, 16, None), nat.ERR_SHAPE),
        (L.hkx_experts_bias_grad(AT, 16, AT, AT, nat.INT8, 4, 4, 16, None), nat.ERR_DTYPE),
        (L.hkx_experts_bias_grad(AT, 16, AT, AT, nat.BF16, 0, 4, 16, None), nat.ERR_SHAPE),
    ]:
        assert rc == code, nat.last_error()


# ------------------------------------------------------------------ the choice between the kernels

SHIM = """
#include "hkx_group_rules.hpp"
extern "C" int pick(int op, int fp8, int experts, int rows, int m, int n, int k, int quad, int cus) {
  return hkx::group_pick({op, fp8 != 0, experts, rows, m, n, k}, quad != 0, cus);
}
extern "C" double cost(int op, int fp8, int experts, int rows, int m, int n, int k, int kernel, int cus) {
  return hkx::group_cost({op, fp8 != 0, experts, rows, m, n, k}, kernel, cus);
}
"""


@functools.lru_cache(maxsize=None)
def _rules():
    cxx = shutil.which("g++") or shutil.which("c++") or "/opt/rocm/bin/amdclang++"
    csrc = Path(__file__).resolve().parents[1] / "hk-dsl_amd" / "csrc"
    with tempfile.TemporaryDirectory() as d:
        src, so = Path(d) / "shim.cpp", Path(d) / "shim.so"
        src.write_text(SHIM)
        subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{csrc}", str(src), "-o", str(so)], check=True)
        lib = ctypes.CDLL(str(so))
        lib.cost.restype = ctypes.c_double
        return lib


def test_a_pick_is_one_that_the_product_has():
    for op in range(3):
        for fp8 in (0, 1) if op == 0 else (0,):
            for e in (1, 2, 8, 64, 1024):
                for rows in (0, 1, 7, 500, 16384, 2 ** 31 - 1):
                    for n in (8, 2048, 2 ** 31 - 8):
                        for k in (16, 4096, 2 ** 31 - 16):
                            for quad in (0, 1):
                                got = _rules().pick(op, fp8, e, rows, 4096, n, k, quad, 256)
                                assert (3 if op == 2 else 1) <= got <= (6 if op == 0 else 4) and (quad or got != 4)
                                kernels = range(3 if op == 2 else 1, 7 if op == 0 else 5)
                                costs = [_rules().cost(op, fp8, e, rows, 4096, n, k, j, 256) for j in kernels]
                                assert all(math.isfinite(c) and c > 0 for c in costs)


@pytest.mark.parametrize("op,fp8,e,rows,m,n,k,kernels", [
    (0, 0, 64, 8, 0, 2048, 2048, (5,)), (0, 0, 64, 512, 0, 8192, 512, (1, 2)), (0, 1, 64, 16376, 0, 2048, 4096, (4,)),
    (0, 0, 8, 8192, 0, 14336, 4096, (4,)), (1, 0, 8, 8192, 0, 2048, 8192, (4,)), (2, 0, 8, 8192, 8192, 2048, 0, (4,)),
    (2, 0, 5, 666, 904, 1112, 0, (3,)), (1, 0, 3, 90, 0, 512, 512, (1,))])
def test_picks(op, fp8, e, rows, m, n, k, kernels):
    """What measured fastest of all kernels at shapes far apart."""
    assert _rules().pick(op, fp8, e, rows, m, n, k, 1, 256) in kernels
