"""What hk.ops.mxfp4.gemm passes to the library, without a GPU: its tensors stand on the CPU and say
they are on one, and the launch is recorded instead of made."""

import ctypes
import types

import pytest
import torch

from hk import _native as nat
from hk.ops import mxfp4

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class OnGpu(torch.Tensor):
    is_cuda = True

    def get_device(self):
        return 0


def _empty(*size, dtype=torch.uint8):
    return torch.empty(size, dtype=dtype).as_subclass(OnGpu)


@pytest.fixture
def launches(monkeypatch):
    """The arguments of each product that would have been launched, as the library's own struct."""
    real, seen = nat.lib(), []

    def product(ref, _stream):
        seen.append(nat.HkxMx4GemmArgs.from_buffer_copy(ref._obj))
        return nat.OK

    monkeypatch.setattr(nat, "lib", lambda: types.SimpleNamespace(
        hkx_mx4_gemm=product, hkx_mx4_gemm_workspace=real.hkx_mx4_gemm_workspace))
    monkeypatch.setattr(nat, "stream_of", lambda device: 0)
    monkeypatch.setattr(nat, "workspace", lambda device, need: types.SimpleNamespace(data_ptr=lambda: 1 << 20))
    monkeypatch.setattr(mxfp4, "_GEMM", {})
    return seen


def _operands(m, n, k, wide, pair):
    rows = 2 * n if pair else n
    a = _empty(m, k, dtype=torch.float8_e4m3fn) if wide else _empty(m, k // 2)
    return a, _empty(rows, k // 2), _empty(m, k // 32), _empty(rows, k // 32)


def _asked(args):
    """The bytes that the library wants for exactly this launch."""
    return nat.lib().hkx_mx4_gemm_workspace(ctypes.byref(args))


@pytest.mark.parametrize("bias", [None, BF16, F16, F32])
@pytest.mark.parametrize("pair", [False, True], ids=["plain", "paired"])
@pytest.mark.parametrize("wide", [False, True], ids=["a4", "a8"])
@pytest.mark.parametrize("m,n,k", [(129, 8219, 20480), (458, 4131, 15360), (532, 3743, 16384), (136, 11029, 13312),
                                   (300, 1001, 4096), (1024, 4096, 4096), (2048, 12288, 4096), (4096, 513, 2048)])
def test_the_workspace_is_what_the_launch_needs(launches, m, n, k, wide, pair, bias):
    """Also where the plan would go by the bias: odd columns, a paired product, 16-bit bias."""
    a, b, sa, sb = _operands(m, n, k, wide, pair)
    bias = None if bias is None else _empty(b.shape[0], dtype=bias)
    for _ in range(2):  # the first call of the layout, and one that knows it
        mxfp4.gemm(a, b, sa, sb, bias=bias, silu_mul=pair)
    assert [_asked(g) for g in launches] == [g.ws_bytes for g in launches], (m, n, k)


@pytest.mark.parametrize("m,n,k", [(1024, 12288, 4096), (2048, 12288, 4096), (4096, 12288, 4096)])
def test_an_out_leaves_the_layouts_template_alone(launches, m, n, k):
    """C 8 bytes off 16 takes another plan than a new C: neither's workspace is the other's."""
    a, b, sa, sb = _operands(m, n, k, False, False)
    off = _empty(m * n + 4, dtype=BF16)[4:].view(m, n)
    assert off.data_ptr() % 16 == 8 and off.is_contiguous()
    for out in (off, None, None, off, None):
        mxfp4.gemm(a, b, sa, sb, out=out)
    assert [_asked(g) for g in launches] == [g.ws_bytes for g in launches]
    assert launches[0].ws_bytes != launches[1].ws_bytes == launches[2].ws_bytes == launches[4].ws_bytes
    assert launches[0].c % 16 == 8 and launches[1].c % 16 == 0


@pytest.mark.parametrize("args,code,says", [
    ((None, 64, 1 << 20, 64, 1 << 20, 2, 4, 64), nat.ERR_ARG, "null"),
    ((1 << 20, 64, 1 << 20, 64, 1 << 20, 2, 4, 40), nat.ERR_SHAPE, "multiple of 32"),
    ((1 << 20, 64, 1 << 20, 32, 1 << 20, 2, 4, 64), nat.ERR_SHAPE, "row strides"),
    (((1 << 20) + 2, 64, 1 << 20, 64, 1 << 20, 2, 4, 64), nat.ERR_SHAPE, "aligned"),
])
def test_both_mxfp8_quantizations_refuse_the_same(args, code, says):
    for f in (nat.lib().hkx_mx_quant, nat.lib().hkx_mx_quant_nan):
        assert f(*args, None) == code and says in nat.last_error(), nat.last_error()


def test_a_gradient_is_refused_and_not_dropped(launches):
    a, b, sa, sb = _operands(64, 128, 256, False, False)
    x = _empty(64, 256, dtype=BF16).requires_grad_()
    bias = _empty(128, dtype=F32).requires_grad_()
    for name, f in (("quant", lambda: mxfp4.quant(x)), ("linear", lambda: mxfp4.linear(x, b, sb)),
                    ("linear", lambda: mxfp4.linear(x, b, sb, act="mxfp4")),
                    ("linear", lambda: mxfp4.linear(x.detach(), b, sb, bias=bias)),
                    ("gemm", lambda: mxfp4.gemm(a, b, sa, sb, bias=bias)),
                    ("gemm", lambda: mxfp4.gemm(x.detach().to(torch.float8_e4m3fn).requires_grad_(), b, sa, sb))):
        with pytest.raises(ValueError, match=f"mxfp4.{name}: no gradient"):
            f()
    assert not launches
    with torch.no_grad():
        mxfp4.gemm(a, b, sa, sb, bias=bias)
    with torch.inference_mode():
        mxfp4.gemm(a, b, sa, sb, bias=bias)
    mxfp4.gemm(a, b, sa, sb, bias=bias.detach())
    assert len(launches) == 3


@pytest.mark.parametrize("rows", [2 ** 31, 2 ** 32 + 16])
def test_sizes_past_32_bits_are_refused_and_not_cut_short(launches, rows):
    """(A row that stands for all of them: nothing of that size is made.)"""
    from hk.ops import block_norm, mxfp8

    def wide(n, dtype=torch.uint8):
        return torch.empty(1, n, dtype=dtype).expand(rows, n).as_subclass(OnGpu)

    a, b, sa, sb = wide(16), _empty(8, 16), wide(1), _empty(8, 1)
    x = wide(32, BF16)
    for f in (lambda: mxfp4.quant(x), lambda: mxfp8.quant(x), lambda: mxfp4.linear(x, b, sb),
              lambda: mxfp4.linear(x, b, sb, act="mxfp4"), lambda: mxfp4.gemm(a, b, sa, sb),
              lambda: mxfp4.gemm(b, a, sb, sa), lambda: mxfp4.dequant(a, sa),
              lambda: mxfp8.dequant(wide(32, torch.float8_e4m3fn), sa), lambda: block_norm(x, x)):
        with pytest.raises(ValueError, match=f"={rows}, at most 2"):
            f()
    assert not launches


#: Calls of hk.ops.mxfp4.gemm whose plan is each kernel: (M, N, K, 8-bit A, paired) and (kernel, splits).
PLANS = [((40, 512, 2048, True, False), (nat.MX4_SKINNY, 1)), ((300, 200, 2048, False, True), (nat.MX4_SKINNY, 1)),
         ((640, 512, 1024, False, False), (nat.MX4_TILE64, 1)), ((600, 1024, 4096, True, False), (nat.MX4_TILE64, 2)),
         ((1024, 2048, 2080, False, True), (nat.MX4_TILE128, 1)), ((520, 1024, 8192, False, False), (nat.MX4_TILE128, 4)),
         ((2300, 6144, 1056, False, False), (nat.MX4_QUAD, 1)), ((1100, 4099, 12320, False, False), (nat.MX4_QUAD, 2)),
         ((777, 8192, 1056, False, True), (nat.MX4_QUAD, 1)), ((1100, 2051, 12320, False, True), (nat.MX4_QUAD, 2)),
         ((2300, 6152, 1056, True, False), (nat.MX4_QUAD, 1)), ((2300, 1024, 12320, True, False), (nat.MX4_QUAD, 4)),
         ((777, 8192, 1056, True, True), (nat.MX4_QUAD, 1)), ((1100, 2051, 12320, True, True), (nat.MX4_QUAD, 2))]


def test_the_plans_of_the_calls_that_the_gpu_tests_make():
    import test_mx4_cpu as R

    got = [(call, R._plan(*call[:3], call[3], call[4], vec=call[1] % 8 == 0)) for call, _ in PLANS]
    assert got == PLANS
