"""MXFP4 on gfx950: 4-bit weights with an E8M0 scale a row and 32 columns.

    q, s = hk.ops.mxfp4.quant(w)                    # bf16, fp16 or fp32 rows, once a weight
    y = hk.ops.mxfp4.linear(x, q, s, bias=b)        # x quantized to MXFP8, then the product
    y = hk.ops.mxfp4.gemm(a, q, sa, s)              # operands quantized already
    y = hk.ops.mxfp4.gemm(a, q, sa, s, silu_mul=True)  # q: gate rows, then up rows

The OCP MX layout: two e2m1 codes a byte, the even column in the low bits (uint8, or torch's
float4_e2m1fn_x2), and one E8M0 byte (2^(s - 127); 255 is NaN) a row and 32 columns.

There is no gradient through quantized values: an activation or a bias that requires one is refused where
gradients are taken.

A call's checks and layout are kept by the shapes, strides and types they depend on, as a template of
the library's arguments; a call of known layout fills in its addresses.
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


def _no_gradient(call):
    """For a call of which a tensor requires a gradient: there is none through quantized values."""
    import torch  # noqa: PLC0415

    if torch.is_grad_enabled():
        raise ValueError(f"{call}: no gradient through quantized values (detach, or torch.no_grad())")


def _e8m0(s, shape, name):
    import torch  # noqa: PLC0415

    if s.dtype == torch.float8_e8m0fnu:
        s = s.view(torch.uint8)
    if s.dtype != torch.uint8:
        raise TypeError(f"mxfp4.gemm: {name} holds E8M0 bytes (uint8), got {s.dtype}")
    if tuple(s.shape) != shape:
        raise ValueError(f"mxfp4.gemm: {name} is {tuple(s.shape)}, expected {shape}")
    return s


def _scale_rows(s):
    """`s` with unit stride along K (the kernels read rows at any alignment)."""
    return s if s.stride(1) == 1 and (s.shape[0] < 2 or s.stride(0) >= s.shape[1]) else s.contiguous()


def _rows16(t):
    """`t` with rows the kernels read in place: unit stride along K, 16-byte aligned."""
    rows, st = t.shape[0], t.stride()
    if t.data_ptr() % 16 == 0 and st[1] == 1 and (rows < 2 or (st[0] % 16 == 0 and st[0] >= t.shape[1])):
        return t
    out = t.new_empty(t.shape)
    out.copy_(t)
    return out


def _ld(t, least):
    """A matrix's row stride (a single row's is anything)."""
    return t.stride(0) if t.shape[0] > 1 else least


#: What quant knows of a layout of x: (rows, K, x's type code, x's row stride, the scales' row stride, the
#: shapes of q and s, s's strides).
_QUANT: dict = {}


def _padded(lead, n):
    """(shape, strides) of scales (*lead, n) with rows of whole dwords."""
    strides, step = [1], (n + 3) // 4 * 4
    for size in reversed(lead):
        strides.insert(0, step)
        step *= size
    return (*lead, n), tuple(strides)


def quant(x, out=None):
    """(q, s) for x (..., K) bf16, fp16 or fp32, K a multiple of 32: q uint8 (..., K/2) of packed codes, s
    uint8 (..., K/32). A block's scale is 2^ceil(log2(amax / 6)) (nothing is clamped), its codes x over
    that rounded to the nearest, ties to even; a block with an infinity or a NaN is NaN (scale 255).
    `out`: (q, s) to write into (also as float4_e2m1fn_x2 and float8_e8m0fnu); their bytes are the result."""
    if x.requires_grad:
        _no_gradient("mxfp4.quant")
    key = (x.shape, x.stride(), x.dtype)
    plan = _QUANT.get(key)
    if plan is None or out is not None or x.data_ptr() & 15 or x.get_device() < 0:
        return _quant(x, out, key)
    import torch  # noqa: PLC0415

    m, k, code, ldx, lds, q_shape, s_shape, s_strides = plan
    if type(x) is torch.Tensor:
        q = x.new_empty(q_shape, dtype=torch.uint8)
        s = x.new_empty_strided(s_shape, s_strides, dtype=torch.uint8)
    else:
        q = nat.empty(x, q_shape, torch.uint8)
        s = torch.empty_strided(s_shape, s_strides, dtype=torch.uint8, device=x.device)
    nat.check(nat.lib().hkx_mx4_quant(x.data_ptr(), ldx, code, q.data_ptr(), k >> 1, s.data_ptr(), lds,
                                      m, k, nat.stream_of(x.device)))
    return q, s


def _quant(x, out, key):
    import torch  # noqa: PLC0415

    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32) or x.dim() < 1:
        raise TypeError(f"mxfp4.quant: x is bf16, fp16 or fp32 (..., K), got {x.dtype} {tuple(x.shape)}")
    lead, k = tuple(x.shape[:-1]), x.shape[-1]
    if k % 32 or k == 0:
        raise ValueError(f"mxfp4.quant: K={k}, a multiple of 32")
    if not x.is_cuda:
        raise ValueError(f"mxfp4.quant: x is on a GPU, got {x.device}")
    m, given = x.numel() // k, x
    nat.int32("mxfp4.quant", M=m, K=k)
    if x.dim() != 2:
        x = x.reshape(m, k)
    per, ldx = 16 // x.element_size(), _ld(x, k)
    q_shape, (s_shape, s_strides) = (*lead, k // 2), _padded(lead, k // 32)
    lds = (k // 32 + 3) // 4 * 4
    if x.stride(1) != 1 or ldx % per or ldx < k or x.data_ptr() % 16:
        x, ldx = x.clone(memory_format=torch.contiguous_format), k
    elif m and x.data_ptr() == given.data_ptr():
        nat.remember(_QUANT, key, (m, k, nat.dtype_code(x.dtype), ldx, lds, q_shape, s_shape, s_strides), 4096)
    if out is not None:
        q, s = out
        q = _packed(q, "mxfp4.quant", "out")
        if s.dtype == torch.float8_e8m0fnu:
            s = s.view(torch.uint8)
        _on(x.device, "mxfp4.quant", q=q, s=s)
        ok = tuple(q.shape) == q_shape and tuple(s.shape) == s_shape and s.dtype == torch.uint8
        if ok:
            try:
                q2, s2 = q.view(m, k // 2), s.view(m, k // 32)
            except RuntimeError:  # leading sizes that are no rows of one stride
                ok = False
            else:
                ldq, lds = _ld(q2, k // 2), _ld(s2, k // 32)
                ok = not (q2.stride(1) != 1 or s2.stride(1) != 1 or ldq % 4 or q.data_ptr() % 4
                          or ldq < k // 2 or lds < k // 32)
        if not ok:
            raise ValueError(f"mxfp4.quant: out is uint8 {q_shape} with 4-byte aligned rows and uint8 {s_shape}")
    else:
        ldq = k // 2
        q = nat.empty(x, q_shape, torch.uint8)
        s = torch.empty_strided(s_shape, s_strides, dtype=torch.uint8, device=x.device)
    if m:
        nat.check(nat.lib().hkx_mx4_quant(x.data_ptr(), ldx, nat.dtype_code(x.dtype), q.data_ptr(), ldq,
                                          s.data_ptr(), lds, m, k, nat.stream_of(x.device)))
    return q, s


def dequant(q, s, dtype=None):
    """The numbers that (q, s) stand for, (..., K) bf16 or `dtype` (fp16, fp32), rounded once: q (...,
    K/2) packed codes with E8M0 scales s (..., K/32). A block of scale 255 is NaN."""
    return _dequant("mxfp4.dequant", _packed(q, "mxfp4.dequant", "q"), s, dtype, nat.FP4E2M1, 2)


#: Layouts of gemm's operands: (arguments filled in but for their addresses, workspace bytes, C's shape).
_GEMM: dict = {}


def gemm(a, b, sa, sb, *, bias=None, silu_mul=False, out=None):
    """bf16 (..., N) = (sa . a)(sb . b)^T (+ bias): a (..., K/2) packed codes or (..., K)
    float8_e4m3fn, b (N, K/2) packed codes, sa and sb their E8M0 scales (..., K/32), bias (N,) bf16, fp16
    or fp32. With silu_mul, b (2N, K/2) holds gate rows, then up rows: silu(z[..., :N]) * z[..., N:] of z
    (..., 2N) with its bias. Any sizes, K a multiple of 32; sums in fp32, rounded once."""
    if a.requires_grad or (bias is not None and bias.requires_grad):
        _no_gradient("mxfp4.gemm")
    key = (a.shape, a.stride(), a.dtype, b.shape, b.stride(), b.dtype, sa.shape, sa.stride(), sa.dtype,
           sb.shape, sb.stride(), sb.dtype, bias is None or (bias.shape, bias.stride(), bias.dtype), silu_mul)
    plan = _GEMM.get(key)
    if plan is None or out is not None:
        return _gemm(a, b, sa, sb, bias, silu_mul, out, key if out is None else None)
    args, need, shape = plan
    pa, pb, ps, pt = a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr()
    d = a.get_device()
    if ((pa | pb) & 15 or d < 0 or b.get_device() != d or sa.get_device() != d
            or sb.get_device() != d
            or (bias is not None and (bias.get_device() != d or bias.data_ptr() & 15))):
        return _gemm(a, b, sa, sb, bias, silu_mul, out, None)
    g = nat.HkxMx4GemmArgs.from_buffer_copy(args)
    return _launch(g, need, a, pa, pb, ps, pt, bias, nat.empty(a, shape, _bf16()))


_BF16: list = []


def _bf16():
    if not _BF16:
        import torch  # noqa: PLC0415

        _BF16.append(torch.bfloat16)
    return _BF16[0]


def _launch(g, need, a, pa, pb, ps, pt, bias, out):
    g.a, g.b, g.sa, g.sb, g.c = pa, pb, ps, pt, out.data_ptr()
    if bias is not None:
        g.bias = bias.data_ptr()
    if need:
        ws = nat.workspace(a.device, need)
        g.ws, g.ws_bytes = ws.data_ptr(), need
    nat.check(nat.lib().hkx_mx4_gemm(ctypes.byref(g), nat.stream_of(a.device)))
    return out


def _gemm(a, b, sa, sb, bias, silu_mul, out, key):
    import torch  # noqa: PLC0415

    if a.dim() < 1 or b.dim() != 2:
        raise ValueError(f"mxfp4.gemm: a (..., K) and b a matrix, got {tuple(a.shape)} and {tuple(b.shape)}")
    given = (a, b, sa, sb, bias)
    b = _packed(b, "mxfp4.gemm", "b")
    wide = a.dtype == torch.float8_e4m3fn
    if not wide:
        a = _packed(a, "mxfp4.gemm", "a")
    lead, rows = tuple(a.shape[:-1]), b.shape[0]
    k = a.shape[-1] if wide else 2 * a.shape[-1]
    if k != 2 * b.shape[1] or k % 32 or k == 0:
        raise ValueError(f"mxfp4.gemm: K is {k} in a and {2 * b.shape[1]} in b, the same multiple of 32")
    n = rows
    if silu_mul:
        if rows % 2:
            raise ValueError(f"mxfp4.gemm: silu_mul takes gate rows, then as many up rows: b has {rows}")
        n = rows // 2
    if not a.is_cuda or b.device != a.device:
        raise ValueError("mxfp4.gemm: a and b are on one GPU")
    m = a.numel() // a.shape[-1]
    nat.int32("mxfp4.gemm", M=m, N=rows, K=k)
    _on(a.device, "mxfp4.gemm", sa=sa, sb=sb, bias=bias, out=out)
    sa = _e8m0(sa, (*lead, k // 32), "sa")
    sb = _e8m0(sb, (rows, k // 32), "sb")
    if bias is not None and (bias.dtype not in (torch.bfloat16, torch.float16, torch.float32)
                             or bias.shape != (rows,)):
        raise ValueError(f"mxfp4.gemm: bias is bf16, fp16 or fp32 ({rows},), got {bias.dtype} "
                         f"{tuple(bias.shape)}")
    if out is None:
        out = nat.empty(a, (*lead, n), torch.bfloat16)
    elif out.dtype != torch.bfloat16 or tuple(out.shape) != (*lead, n):
        raise ValueError(f"mxfp4.gemm: out is bf16 {(*lead, n)}, got {out.dtype} {tuple(out.shape)}")
    if m == 0 or n == 0:
        return out
    a, sa = a.reshape(m, a.shape[-1]), sa.reshape(m, k // 32)
    c = out if out.dim() == 2 else out.view(m, n)
    if c.stride(1) != 1 or (m > 1 and c.stride(0) < n):
        raise ValueError("mxfp4.gemm: out has unit column stride and rows that do not overlap")
    a, b, sa, sb = _rows16(a), _rows16(b), _scale_rows(sa), _scale_rows(sb)
    if bias is not None:
        bias = bias.contiguous()
        if bias.data_ptr() % 16:
            bias = bias.clone()
    g = nat.HkxMx4GemmArgs()
    g.size = ctypes.sizeof(g)
    g.a_dtype = nat.FP8E4M3 if wide else nat.FP4E2M1
    g.lda, g.ldb = _ld(a, a.shape[1]), _ld(b, k // 2)
    up4 = (k // 32 + 3) // 4 * 4
    g.sa_ld, g.sb_ld, g.ldc = _ld(sa, up4), _ld(sb, up4), _ld(c, n)
    g.c = c.data_ptr()
    g.m, g.n, g.k, g.silu_mul = m, n, k, 1 if silu_mul else 0
    if bias is not None:
        g.bias, g.bias_dtype = bias.data_ptr(), nat.dtype_code(bias.dtype)
    need = nat.lib().hkx_mx4_gemm_workspace(ctypes.byref(g))
    # (a template only where every operand was read where it is and C is new: the plan and its workspace
    # go by C's alignment, which a given one has of its own)
    if key is not None and all(
            x is None or x.data_ptr() == y.data_ptr() for x, y in zip((a, b, sa, sb, bias), given)):
        nat.remember(_GEMM, key, (bytes(g), need, (*lead, n)), 4096)
    _launch(g, need, a, a.data_ptr(), b.data_ptr(), sa.data_ptr(), sb.data_ptr(), bias, c)
    return out


def linear(x, w, ws, *, bias=None, silu_mul=False, act="mxfp8"):
    """x (..., K) @ (ws . w)^T, w packed codes (N, K/2) with scales ws: the activation quantized to
    `act` ("mxfp8": bf16 x; "mxfp4": bf16, fp16 or fp32), then `gemm`. A row of x with an infinity or a
    NaN gives a row of NaN."""
    if act not in ("mxfp8", "mxfp4"):
        raise ValueError(f"mxfp4.linear: act is 'mxfp8' or 'mxfp4', got {act!r}")
    if x.requires_grad or (bias is not None and bias.requires_grad):
        _no_gradient("mxfp4.linear")
    if act == "mxfp4":
        xq, xs = quant(x)
        return gemm(xq, w, xs, ws, bias=bias, silu_mul=silu_mul)
    lead = None
    if x.dim() != 2:
        if x.dim() < 1:
            raise ValueError("mxfp4.linear: x is (..., K), got a single value")
        lead, k = x.shape[:-1], x.shape[-1]
        x = x.reshape(lead.numel(), k)
    xq, xs = _quant8(x, nan_blocks=True)
    y = gemm(xq, w, xs, ws, bias=bias, silu_mul=silu_mul)
    return y if lead is None else y.view(*lead, y.shape[1])


__all__ = ["quant", "dequant", "gemm", "linear"]
