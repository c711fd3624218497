"""The MXFP4 path without a GPU: the float64 oracle against the definitions it stands for, what the C
calls refuse before any launch, and the product's choice between its kernels
(csrc/hkx_mx4_rules.hpp, for a GPU of 256 CUs)."""

import ctypes
import functools
import math
import shutil
import subprocess
import tempfile
from pathlib import Path

import pytest
import torch

from hk import _native as nat
from oracle import mxfp4_oracle as O

CSRC = Path(__file__).resolve().parents[1] / "hk-dsl_amd" / "csrc"

# ------------------------------------------------------------------ the oracle


@pytest.mark.parametrize("exponent", [-140, -126, -20, 0, 15, 100, 127])
def test_quant_by_its_definition(exponent):
    """2^e the least power of two (from 2^-127) with 6 2^e >= the block's largest magnitude, and every
    code's value as near to x 2^-e as any of the eight; the value given back within half a step."""
    g = torch.Generator().manual_seed(exponent + 200)
    x = torch.ldexp(torch.randn(9, 96, generator=g, dtype=torch.float64), torch.tensor(exponent)).float()
    x = torch.where(torch.isfinite(x), x, torch.ones(()))
    x[3, 32:64] = 0
    x[5, :32] = torch.ldexp(torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] * 4), torch.tensor(exponent))
    codes, s = O.quant(x)
    bad = ~torch.isfinite(x.reshape(9, 3, 32)).all(-1)  # (6 2^127 is infinity)
    assert (s[bad] == 255).all() and (s[~bad] < 255).all() and bool(bad.any()) == (exponent == 127)
    x, s = torch.where(bad.repeat_interleave(32, 1), torch.zeros(()), x), torch.where(bad, torch.zeros_like(s), s)
    v = x.double().reshape(9, 3, 32)
    e = s.int() - 127
    amax = v.abs().amax(-1)
    assert (torch.ldexp(torch.full_like(amax, 6.0), e) >= amax).all()
    less = torch.ldexp(torch.full_like(amax, 6.0), e - 1) < amax
    assert (less | (e == -127)).all()
    t = torch.ldexp(v, -e.unsqueeze(-1)).reshape(9, 96)
    got = O.FP4[(codes & 7).long()]
    near = (t.abs().unsqueeze(-1) - O.FP4).abs().amin(-1)
    assert torch.equal((t.abs() - got).abs(), near)
    # ties go to the even code: 0.25 -> 0, 0.75 -> 1, 1.25 -> 1, 1.75 -> 2, 2.5 -> 2, 3.5 -> 4, 5 -> 4
    if exponent in (-126, -20, 0, 15, 100):
        assert (codes[5, :8] & 7).tolist() == [7, 0, 2, 2, 4, 4, 6, 6]
    back = O.values(O.pack(codes), s)
    assert ((back - x.double()).abs() <= torch.ldexp(torch.ones(9, 96, dtype=torch.float64), e.repeat_interleave(32, 1))).all()


def test_quant_of_infinity_and_nan_is_a_nan_block():
    x = torch.ones(1, 96)
    x[0, 5], x[0, 40] = float("inf"), float("nan")
    codes, s = O.quant(x)
    assert s.tolist()[0][:2] == [255, 255] and s[0, 2] == 125 and (codes[0, :64] == 0).all()
    back = O.values(O.pack(codes), s)
    assert back[0, :64].isnan().all() and (back[0, 64:] == 1).all()


def test_gemm_by_a_loop():
    g = torch.Generator().manual_seed(0)
    a, b = (torch.randint(0, 256, (n, 32), generator=g).to(torch.uint8) for n in (3, 4))
    sa, sb = (torch.randint(120, 134, (n, 2), generator=g).to(torch.uint8) for n in (3, 4))
    av, bv = O.values(a, sa), O.values(b, sb)
    z = [[sum(float(av[i, k]) * float(bv[j, k]) for k in range(64)) for j in range(4)] for i in range(3)]
    got, err = O.gemm(a, b, sa, sb)
    assert torch.allclose(got, torch.tensor(z, dtype=torch.float64), rtol=1e-12) and (err > 0).all()
    got, _ = O.gemm(a, b, sa, sb, silu_mul=True)

    def silu(v):
        return v / (1 + math.exp(-v)) if v > 0 else v * math.exp(v) / (1 + math.exp(v))

    want = [[silu(r[j]) * r[j + 2] for j in range(2)] for r in z]
    assert torch.allclose(got, torch.tensor(want, dtype=torch.float64), rtol=1e-10)


@pytest.mark.parametrize("gate", [None, (5,), (2, 1, 5), (2, 3, 1), (2, 3, 5)])
@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False)])
def test_block_norm_gradients_are_the_differences(gate, post, pre):
    g = torch.Generator().manual_seed(7)

    def r(*size):
        return torch.randn(*size, generator=g, dtype=torch.float64).requires_grad_()

    args = [r(2, 3, 5), r(2, 3, 5), r(5) if post else None, r(5) if pre else None, r(*gate) if gate else None]

    def f(x, residual, *w):
        w = iter(w)
        h, y = O.block_norm(x, residual, *(None if a is None else next(w) for a in args[2:]),
                            branch_scale=0.7, residual_scale=1.3)
        return (h,) if y is None else (h, y)

    assert torch.autograd.gradcheck(f, [a for a in args if a is not None], atol=1e-7, rtol=1e-5)


# ------------------------------------------------------------------ refusals of the C calls

AT = 1 << 20  # an address that is never read: every call here ends before a launch


def _gemm_args(**over):
    g = nat.HkxMx4GemmArgs()
    g.size = ctypes.sizeof(g)
    g.a_dtype = nat.FP8E4M3
    g.a = g.b = g.sa = g.sb = g.c = AT
    g.m, g.n, g.k = 64, 256, 256
    g.lda, g.ldb, g.sa_ld, g.sb_ld, g.ldc = 256, 128, 8, 8, 256
    for name, v in over.items():
        setattr(g, name, v)
    return g


@pytest.mark.parametrize("over,code,says", [
    (dict(size=8), nat.ERR_ARG, "args of 8 bytes"),
    (dict(a=None), nat.ERR_ARG, "null pointer"), (dict(sb=None), nat.ERR_ARG, "null pointer"),
    (dict(c=None), nat.ERR_ARG, "null pointer"),
    (dict(a_dtype=nat.BF16), nat.ERR_DTYPE, "packed 4-bit or e4m3"),
    (dict(bias=AT, bias_dtype=nat.INT8), nat.ERR_DTYPE, "bias"),
    (dict(bias=AT + 2, bias_dtype=nat.BF16), nat.ERR_SHAPE, "bias needs 16-byte"),
    (dict(m=0), nat.ERR_SHAPE, "M=0"), (dict(n=-1), nat.ERR_SHAPE, "N=-1"),
    (dict(k=48), nat.ERR_SHAPE, "multiple of 32"),
    (dict(lda=128), nat.ERR_SHAPE, "row strides"), (dict(ldb=64), nat.ERR_SHAPE, "row strides"),
    (dict(sa_ld=4), nat.ERR_SHAPE, "row strides"), (dict(ldc=255), nat.ERR_SHAPE, "row strides"),
    (dict(a=AT + 8), nat.ERR_SHAPE, "16-byte aligned"), (dict(ldb=136), nat.ERR_SHAPE, "16-byte aligned"),
    (dict(lda=1 << 28), nat.ERR_SHAPE, "4 GiB"), (dict(sb_ld=1 << 28), nat.ERR_SHAPE, "4 GiB"),
    (dict(kernel=9), nat.ERR_ARG, "kernel 9"), (dict(kernel=nat.MX4_TILE64, splits=-1), nat.ERR_ARG, "splits -1"),
    (dict(silu_mul=1, n=2 ** 31 - 1, ldc=2 ** 31), nat.ERR_SHAPE, "N="),
    (dict(kernel=nat.MX4_QUAD, m=300, k=1024, lda=1024, ldb=512, sa_ld=32, sb_ld=32), nat.ERR_WORKSPACE, "workspace"),
    (dict(kernel=nat.MX4_TILE64, splits=2, k=1024, lda=1024, ldb=512, sa_ld=32, sb_ld=32, ws=AT + 4, ws_bytes=1 << 30),
     nat.ERR_WORKSPACE, "workspace"),
])
def test_gemm_refusals(over, code, says):
    got = nat.lib().hkx_mx4_gemm(ctypes.byref(_gemm_args(**over)), None)
    assert got == code and says in nat.last_error(), (got, nat.last_error())


def test_null_arguments():
    L = nat.lib()
    for f in (L.hkx_mx4_gemm, L.hkx_block_norm, L.hkx_block_norm_backward):
        assert f(None, None) == nat.ERR_ARG and "null" in nat.last_error()
    assert L.hkx_mx4_gemm_workspace(None) == 0 and L.hkx_block_norm_backward_workspace(None) == 0


@pytest.mark.parametrize("call,args,code,says", [
    ("quant", (None, 64, nat.BF16, AT, 32, AT, 2, 4, 64), nat.ERR_ARG, "null"),
    ("quant", (AT, 64, nat.INT8, AT, 32, AT, 2, 4, 64), nat.ERR_DTYPE, "bf16, fp16 or fp32"),
    ("quant", (AT, 64, nat.BF16, AT, 32, AT, 2, 4, 40), nat.ERR_SHAPE, "multiple of 32"),
    ("quant", (AT, 32, nat.BF16, AT, 32, AT, 2, 4, 64), nat.ERR_SHAPE, "row strides"),
    ("quant", (AT + 2, 64, nat.BF16, AT, 32, AT, 2, 4, 64), nat.ERR_SHAPE, "aligned"),
    ("quant", (AT, 64, nat.BF16, AT, 32, AT, 2, -1, 64), nat.ERR_SHAPE, "M=-1"),
    ("dequant", (AT, 32, nat.FP4E2M1, None, 2, AT, 64, nat.FP32, 4, 64), nat.ERR_ARG, "null"),
    ("dequant", (AT, 32, nat.BF16, AT, 2, AT, 64, nat.FP32, 4, 64), nat.ERR_DTYPE, "packed 4-bit or e4m3"),
    ("dequant", (AT, 32, nat.FP4E2M1, AT, 2, AT, 64, nat.INT8, 4, 64), nat.ERR_DTYPE, "bf16, fp16 or fp32"),
    ("dequant", (AT, 32, nat.FP8E4M3, AT, 2, AT, 64, nat.FP32, 4, 64), nat.ERR_SHAPE, "row strides"),
    ("dequant", (AT + 2, 32, nat.FP4E2M1, AT, 2, AT, 64, nat.FP32, 4, 64), nat.ERR_SHAPE, "aligned"),
])
def test_quant_refusals(call, args, code, says):
    f = nat.lib().hkx_mx4_quant if call == "quant" else nat.lib().hkx_mx_dequant
    got = f(*args, None)
    assert got == code and says in nat.last_error(), (got, nat.last_error())


def _norm_args(**over):
    g = nat.HkxBlockNormArgs()
    g.size = ctypes.sizeof(g)
    g.rows, g.d = 6, 64
    g.x = g.residual = g.post = g.pre = g.h = g.y = g.rstd = AT
    g.ldx = g.ldr = g.ldh = g.ldy = 64
    g.branch_scale = g.residual_scale = 1.0
    for name, v in over.items():
        setattr(g, name, v)
    return g


@pytest.mark.parametrize("over,code,says", [
    (dict(size=8), nat.ERR_ARG, "args of 8 bytes"), (dict(x=None), nat.ERR_ARG, "null"),
    (dict(h=None), nat.ERR_ARG, "null"), (dict(y=None), nat.ERR_ARG, "null"),
    (dict(d=0), nat.ERR_SHAPE, "d=0"), (dict(rows=-1), nat.ERR_SHAPE, "rows=-1"),
    (dict(d=16385, ldx=16385, ldr=16385, ldh=16385, ldy=16385), nat.ERR_SHAPE, "at most 16384"),
    (dict(r_dtype=nat.FP16), nat.ERR_DTYPE, "residual"), (dict(w_dtype=nat.FP16), nat.ERR_DTYPE, "weights"),
    (dict(gate=AT, gate_rows=1, gate_dtype=nat.FP16), nat.ERR_DTYPE, "gate"),
    (dict(gate=AT, gate_rows=4), nat.ERR_SHAPE, "gates of 4"), (dict(gate=AT), nat.ERR_SHAPE, "gates of 0"),
    (dict(ldx=63), nat.ERR_SHAPE, "row strides"), (dict(ldy=63), nat.ERR_SHAPE, "row strides"),
    (dict(quant=3), nat.ERR_ARG, "quant=3"), (dict(quant=1), nat.ERR_ARG, "scales"),
    (dict(quant=1, y_scales=AT, ldys=1), nat.ERR_SHAPE, "row strides"),
    (dict(quant=2, y_scales=AT, ldys=2, d=48), nat.ERR_SHAPE, "multiple of 32"),
    (dict(quant=2, y_scales=AT, ldys=2, x=AT + 4), nat.ERR_SHAPE, "16-byte aligned"),
])
def test_block_norm_refusals(over, code, says):
    got = nat.lib().hkx_block_norm(ctypes.byref(_norm_args(**over)), None)
    assert got == code and says in nat.last_error(), (got, nat.last_error())


@pytest.mark.parametrize("f,over,code,says", [
    ({}, dict(size=8), nat.ERR_ARG, "args of 8 bytes"), (dict(residual=None), {}, nat.ERR_ARG, "null"),
    (dict(rstd=None), {}, nat.ERR_ARG, "null"), ({}, dict(dx=None), nat.ERR_ARG, "null"),
    (dict(d=8193, ldx=8193, ldr=8193), {}, nat.ERR_SHAPE, "at most 8192"),
    ({}, dict(lddh=63), nat.ERR_SHAPE, "row strides"), (dict(rows=0), {}, nat.ERR_SHAPE, "no rows"),
    ({}, dict(dpost=AT), nat.ERR_WORKSPACE, "workspace"),
    (dict(gate=AT, gate_rows=1, gate_col=1, gate_dtype=nat.INT8), {}, nat.ERR_DTYPE, "gate"),
])
def test_block_norm_backward_refusals(f, over, code, says):
    q = nat.HkxBlockNormGradArgs()
    q.size = ctypes.sizeof(q)
    q.f = _norm_args(**f)
    q.dh = q.dy = q.dx = q.dresidual = AT
    q.lddh = q.lddy = q.lddx = q.lddr = 64 if q.f.d == 64 else q.f.d
    for name, v in over.items():
        setattr(q, name, v)
    got = nat.lib().hkx_block_norm_backward(ctypes.byref(q), None)
    assert got == code and says in nat.last_error(), (got, nat.last_error())


# ------------------------------------------------------------------ the choice between the kernels

SHIM = """
#include "hkx_mx4_rules.hpp"
extern "C" int plan(int m, int n, int k, int a8, int pair, int quad, int vec, int cus, int* out) {
  const hkx::Mx4Plan p = hkx::mx4_plan(m, n, k, a8, pair, quad, vec, cus);
  out[0] = p.splits;
  return p.kernel;
}
extern "C" int splits(int kernel, int units, int s) { return hkx::mx4_splits(kernel, units, s); }
extern "C" int per(int kernel, int units, int s) { return hkx::mx4_split_units(kernel, units, s); }
"""


@functools.lru_cache(maxsize=None)
def _rules():
    cxx = shutil.which("g++") or shutil.which("c++") or "/opt/rocm/bin/amdclang++"
    with tempfile.TemporaryDirectory() as d:
        src, so = Path(d) / "shim.cpp", Path(d) / "shim.so"
        src.write_text(SHIM)
        subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(src), "-o", str(so)],
                       check=True)
        return ctypes.CDLL(str(so))


def _plan(m, n, k, a8=False, pair=False, quad=True, vec=True, cus=256):
    out = ctypes.c_int()
    return _rules().plan(m, n, k, a8, pair, quad, vec, cus, ctypes.byref(out)), out.value


def test_splits_cover_k_and_none_is_empty():
    for kernel in (nat.MX4_TILE64, nat.MX4_TILE128, nat.MX4_QUAD):
        for units in range(1, 130):
            for s in range(1, 9):
                n, per = _rules().splits(kernel, units, s), _rules().per(kernel, units, s)
                assert 1 <= n <= s and (n - 1) * per < units <= n * per


def test_a_plan_is_one_that_its_kernel_takes():
    for m in (1, 16, 17, 33, 64, 65, 128, 129, 500, 512, 513, 4096):
        for n in (1, 100, 4096, 28672):
            for k in (32, 992, 4096, 4128, 8192, 14336):
                for a8 in (False, True):
                    for pair in (False, True):
                        for quad in (False, True):
                            kernel, splits = _plan(m, n, k, a8, pair, quad)
                            assert kernel in (nat.MX4_TILE64, nat.MX4_TILE128, nat.MX4_QUAD, nat.MX4_SKINNY)
                            assert quad or kernel != nat.MX4_QUAD
                            units = -(-k // 256)
                            assert splits == 1 if kernel == nat.MX4_SKINNY else (
                                1 <= splits <= units and _rules().splits(kernel, units, splits) == splits)


def test_the_decode_kernel_where_it_was_measured_faster():
    """us of the decode kernel and the best other plan, cold weights: 37 x 1001 x 2976 fp8 7.1, 11.3; 128 x
    4096 x 4096 fp8 10.4, 14.3; 256 x 1024 x 4096 fp4 6.2, 11.3; 128 x 1024 x 8192 fp4 10.9, 12.2; 48 x 4096
    x 8192 fp4 11.2, 14.8."""
    for m, n, k, a8 in ((1, 28672, 4096, True), (16, 28672, 4096, False), (32, 16384, 4096, True), (37, 1001, 2976, True),
                        (128, 4096, 4096, True), (256, 1024, 4096, False), (384, 512, 4096, True), (512, 1024, 4096, False),
                        (128, 1024, 8192, False), (48, 4096, 8192, False), (8, 8192, 14336, True)):
        assert _plan(m, n, k, a8) == (nat.MX4_SKINNY, 1), (m, n, k, a8)
    for m, n, k, a8 in ((32, 28672, 4096, True), (64, 28672, 4096, False), (192, 4096, 4096, True), (384, 2048, 4096, True),
                        (384, 1024, 8192, False), (128, 1024, 8192, True), (48, 4096, 8192, True), (24, 8192, 8192, False),
                        (640, 256, 1024, False)):
        assert _plan(m, n, k, a8)[0] != nat.MX4_SKINNY, (m, n, k, a8)


def test_the_workspace_is_the_plans():
    """None for the decode kernel and whole tiles, a split's fp32 shares, and the quadrant kernel's packed scales."""
    L = nat.lib()
    for m, n, k, a8, pair in ((16, 4096, 4096, True, False), (300, 1024, 4096, False, False), (777, 4096, 12288, False, False),
                              (4096, 12288, 4096, False, False), (2048, 4096, 4096, True, True), (130, 520, 8192, True, False)):
        g = _gemm_args(a_dtype=nat.FP8E4M3 if a8 else nat.FP4E2M1, m=m, n=n, k=k, lda=k if a8 else k // 2, ldb=k // 2,
                       sa_ld=k // 32, sb_ld=k // 32, ldc=n, silu_mul=int(pair))
        kernel, splits = _plan(m, n, k, a8, pair)
        want = (splits * m * n * 4 * (2 if pair else 1) + 15) // 16 * 16 if splits > 1 else 0
        if kernel == nat.MX4_QUAD:
            chunks = -(-k // 512)
            want += (-(-m // 256) + -(-n // (128 if pair else 256))) * chunks * 4096
        assert L.hkx_mx4_gemm_workspace(ctypes.byref(g)) == want, (m, n, k, kernel, splits)
