"""MXFP4 on gfx950: 4-bit weights with an E8M0 scale a row and 32 columns.

    q, s = hk.ops.mxfp4.quant(w)                    # bf16, fp16 or fp32 rows, once a weight
    y = hk.ops.mxfp4.linear(x, q, s, bias=b)        # x quantized to MXFP8, then the product
    y = hk.ops.mxfp4.gemm(a, q, sa, s)              # operands quantized already
    y = hk.ops.mxfp4.gemm(a, q, sa, s, silu_mul=True)  # q: gate rows, then up rows

The OCP MX layout: two e2m1 codes a byte, the even column in the low bits (uint8, or torch's
float4_e2m1fn_x2), and one E8M0 byte (2^(s - 127); 255 is NaN) a row and 32 columns. Scales whose rows
start at multiples of 4 bytes are read in place (`quant` makes such rows at any K); others are copied
every call, so a weight's scales are best laid out once by `scale_rows`.
"""

from __future__ import annotations

import ctypes

from .. import _native as nat
from .mxfp8 import _dequant, _on
from .mxfp8 import quant as _quant8


def _packed(t, call, name):
    """`t` as bytes of packed codes."""
    import torch  # noqa: PLC0415

    if t.dtype == torch.uint8:
        return t
    if t.dtype == getattr(torch, "float4_e2m1fn_x2", None):
        return t.view(torch.uint8)
    raise TypeError(f"{call}: {name} holds packed 4-bit codes (uint8 or float4_e2m1fn_x2), got {t.dtype}")


def scale_rows(s):
    """E8M0 scales (rows, K/32) with rows that start at multiples of 4 bytes: `s` itself where it has
    them, else a copy."""
    if s.stride(1) == 1 and s.stride(0) % 4 == 0 and s.data_ptr() % 4 == 0:
        return s
    rows, k32 = s.shape
    out = s.new_empty((rows, (k32 + 3) // 4 * 4))[:, :k32]
    out.copy_(s)
    return out


def _scales(s, rows, k, name):
    import torch  # noqa: PLC0415

    if s.dtype != torch.uint8 and s.dtype != torch.float8_e8m0fnu:
        raise TypeError(f"mxfp4.gemm: {name} holds E8M0 bytes (uint8), got {s.dtype}")
    if s.shape != (rows, k // 32):
        raise ValueError(f"mxfp4.gemm: {name} is {tuple(s.shape)}, expected ({rows}, {k // 32})")
    if s.dtype != torch.uint8:
        s = s.view(torch.uint8)
    return scale_rows(s)


def _rows16(t):
    """`t` with rows the kernels read in place: unit stride along K, 16-byte aligned."""
    st = t.stride()
    if st[1] == 1 and st[0] % 16 == 0 and t.data_ptr() % 16 == 0 and (st[0] >= t.shape[1]):
        return t
    return t.clone(memory_format=_contiguous())


def _contiguous():
    import torch  # noqa: PLC0415

    return torch.contiguous_format


def quant(x, out=None):
    """(q, s) for x (M, K) bf16, fp16 or fp32, K a multiple of 32: q uint8 (M, K/2) of packed codes, s
    uint8 (M, K/32). A block's scale is 2^ceil(log2(amax / 6)) (nothing is clamped), its codes x over
    that rounded to the nearest, ties to even; a block with an infinity or a NaN is NaN (scale 255).
    `out`: (q, s) to write into."""
    import torch  # noqa: PLC0415

    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32) or x.dim() != 2:
        raise TypeError(f"mxfp4.quant: x is bf16, fp16 or fp32 (M, K), got {x.dtype} {tuple(x.shape)}")
    m, k = x.shape
    if k % 32 or k == 0:
        raise ValueError(f"mxfp4.quant: K={k}, a multiple of 32")
    if not x.is_cuda:
        raise ValueError(f"mxfp4.quant: x is on a GPU, got {x.device}")
    per = 16 // x.element_size()
    if x.stride(1) != 1 or x.stride(0) % per or x.stride(0) < k or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    if out is not None:
        q, s = out
        q = _packed(q, "mxfp4.quant", "out")
        if (tuple(q.shape) != (m, k // 2) or tuple(s.shape) != (m, k // 32) or s.dtype != torch.uint8
                or q.stride(1) != 1 or s.stride(1) != 1 or q.stride(0) % 4 or q.data_ptr() % 4
                or q.stride(0) < k // 2 or s.stride(0) < k // 32):
            raise ValueError(f"mxfp4.quant: out is uint8 ({m}, {k // 2}) with 4-byte aligned rows and "
                             f"uint8 ({m}, {k // 32})")
        _on(x.device, "mxfp4.quant", q=q, s=s)
    else:
        q = nat.empty(x, (m, k // 2), torch.uint8)
        s = nat.empty(x, (m, (k // 32 + 3) // 4 * 4), torch.uint8)
        if k % 128:
            s = s[:, :k // 32]
    if m == 0:
        return q, s
    nat.check(nat.lib().hkx_mx4_quant(x.data_ptr(), x.stride(0), nat.dtype_code(x.dtype),
                                      q.data_ptr(), q.stride(0), s.data_ptr(), s.stride(0), m, k,
                                      nat.stream_of(x.device)))
    return q, s


def dequant(q, s, dtype=None):
    """The numbers that (q, s) stand for, (M, K) bf16 or `dtype` (fp16, fp32), rounded once."""
    if q.dim() != 2:
        raise ValueError(f"mxfp4.dequant: q is (M, K/2), got {tuple(q.shape)}")
    q = _packed(q, "mxfp4.dequant", "q")
    return _dequant("mxfp4.dequant", q, s, dtype, nat.FP4E2M1, 2 * q.shape[1])


def gemm(a, b, sa, sb, *, bias=None, silu_mul=False, out=None):
    """bf16 (M, N) = (sa . a)(sb . b)^T (+ bias): a (M, K/2) packed codes or (M, K) float8_e4m3fn, b
    (N, K/2) packed codes, sa and sb their E8M0 scales (rows, K/32), bias (N,) bf16, fp16 or fp32. With
    silu_mul, b (2N, K/2) holds gate rows, then up rows: silu(z[:, :N]) * z[:, N:] of z (M, 2N) with its
    bias. Any M and N, K a multiple of 32; sums in fp32, rounded once."""
    import torch  # noqa: PLC0415

    if a.dim() != 2 or b.dim() != 2:
        raise ValueError(f"mxfp4.gemm: a and b are matrices, got {tuple(a.shape)} and {tuple(b.shape)}")
    b = _packed(b, "mxfp4.gemm", "b")
    wide = a.dtype == torch.float8_e4m3fn
    if not wide:
        a = _packed(a, "mxfp4.gemm", "a")
    m, k = a.shape
    rows, kb = b.shape
    if not wide:
        k *= 2
    if k != 2 * kb or k % 32 or k == 0:
        raise ValueError(f"mxfp4.gemm: K is {k} in a and {2 * kb} in b, the same multiple of 32")
    n = rows
    if silu_mul:
        if rows % 2:
            raise ValueError(f"mxfp4.gemm: silu_mul takes gate rows, then as many up rows: b has {rows}")
        n = rows // 2
    d = a.get_device()
    if d < 0 or b.get_device() != d:
        raise ValueError("mxfp4.gemm: a and b are on one GPU")
    if sa.get_device() != d or sb.get_device() != d:
        _on(a.device, "mxfp4.gemm", sa=sa, sb=sb)
    sa, sb = _scales(sa, m, k, "sa"), _scales(sb, rows, k, "sb")
    if bias is not None:
        if bias.dtype not in (torch.bfloat16, torch.float16, torch.float32) or bias.shape != (rows,):
            raise ValueError(f"mxfp4.gemm: bias is bf16, fp16 or fp32 ({rows},), got {bias.dtype} "
                             f"{tuple(bias.shape)}")
        _on(a.device, "mxfp4.gemm", bias=bias)
        bias = bias.contiguous()
    if out is None:
        out = nat.empty(a, (m, n), torch.bfloat16)
    else:
        if out.dtype != torch.bfloat16 or tuple(out.shape) != (m, n) or out.stride(1) != 1 or out.stride(0) < n:
            raise ValueError(f"mxfp4.gemm: out is bf16 ({m}, {n}) with unit column stride")
        _on(a.device, "mxfp4.gemm", out=out)
    if m == 0 or n == 0:
        return out
    a, b = _rows16(a), _rows16(b)
    g = nat.HkxMx4GemmArgs()
    g.size = ctypes.sizeof(g)
    g.a_dtype = nat.FP8E4M3 if wide else nat.FP4E2M1
    g.a, g.b, g.sa, g.sb, g.c = a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), out.data_ptr()
    g.lda, g.ldb, g.sa_ld, g.sb_ld, g.ldc = a.stride(0), b.stride(0), sa.stride(0), sb.stride(0), out.stride(0)
    g.m, g.n, g.k, g.silu_mul = m, n, k, 1 if silu_mul else 0
    if bias is not None:
        g.bias, g.bias_dtype = bias.data_ptr(), nat.dtype_code(bias.dtype)
    L = nat.lib()
    need = L.hkx_mx4_gemm_workspace(ctypes.byref(g))
    if need:
        ws = nat.workspace(a.device, need)
        g.ws, g.ws_bytes = ws.data_ptr(), need
    nat.check(L.hkx_mx4_gemm(ctypes.byref(g), nat.stream_of(a.device)))
    return out


def linear(x, w, ws, *, bias=None, silu_mul=False, act="mxfp8"):
    """x (M, K) @ (ws . w)^T, w packed codes (N, K/2) with scales ws: the activation quantized to
    `act` ("mxfp8": bf16 x; "mxfp4": bf16, fp16 or fp32), then `gemm`."""
    if act not in ("mxfp8", "mxfp4"):
        raise ValueError(f"mxfp4.linear: act is 'mxfp8' or 'mxfp4', got {act!r}")
    xq, xs = _quant8(x) if act == "mxfp8" else quant(x)
    return gemm(xq, w, xs, ws, bias=bias, silu_mul=silu_mul)


__all__ = ["quant", "dequant", "gemm", "linear", "scale_rows"]
