"""Rows in 8 bits under one fp32 scale each: the operands of hk.ops.scaled_mm and hk.ops.experts.gemm.

    q, s = hk.ops.fp8.quant(x)                  # x (..., K) bf16, fp16 or fp32
    y = hk.ops.scaled_mm(q, w8, s, sw)          # x (M, K)

s = max |x| / 448 of a row (rounded once, at least 2^-126; 1 for a row of zeros) and q = x / s, the fp32
quotient rounded to float8_e4m3fn, ties to even. A row with an infinity or a NaN has s = NaN: what it is
multiplied with is NaN. hk.ops.block_norm(quant="fp8") does the same with its y.
"""

from __future__ import annotations

from .. import _native as nat
from .mxfp8 import _on


#: Layouts of x: (rows, K, its type code, its row stride, the shapes and types of q and s).
_QUANT: dict = {}


def quant(x, out=None):
    """(q, s) of x (..., K), any K: q float8_e4m3fn (..., K), s fp32 (..., 1). `out`: (q, s) to write
    into, contiguous. There is no gradient through quantized values."""
    nat.no_tangents("fp8.quant", x)
    known = None
    if out is None and not x.requires_grad:
        key = (x.shape, x.stride(), x.dtype)
        known = _QUANT.get(key)
    if known is None or x.get_device() < 0:
        return _quant(x, out)
    m, k, code, ldx, q_shape, q_type, s_shape, s_type = known
    device = x.device
    q, s = nat.empty(x, q_shape, q_type), nat.empty(x, s_shape, s_type)
    with nat.current(device):
        nat.check(nat.lib().hkx_fp8_quant(x.data_ptr(), ldx, code, q.data_ptr(), k, s.data_ptr(), m, k,
                                          nat.stream_of(device)))
    return q, s


def _quant(x, out):
    import torch  # noqa: PLC0415

    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("fp8.quant: no gradient through quantized values (detach, or torch.no_grad())")
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32) or x.dim() < 1:
        raise TypeError(f"fp8.quant: x is bf16, fp16 or fp32 (..., K), got {x.dtype} {tuple(x.shape)}")
    k = x.shape[-1]
    if k == 0:
        raise ValueError("fp8.quant: K=0")
    if not x.is_cuda:
        raise ValueError(f"fp8.quant: x is on a GPU, got {x.device}")
    shape = x.shape
    m = x.numel() // k
    if (m | k) >> 31:
        nat.int32("fp8.quant", M=m, K=k)
    if out is not None:
        q, s = out
        _on(x.device, "fp8.quant", q=q, s=s)
        if (q.dtype != torch.float8_e4m3fn or s.dtype != torch.float32 or q.shape != shape
                or s.shape != (*shape[:-1], 1) or not q.is_contiguous() or not s.is_contiguous()):
            raise ValueError(f"fp8.quant: out is contiguous float8_e4m3fn {tuple(shape)} and fp32 "
                             f"{(*shape[:-1], 1)}")
    else:
        q, s = nat.empty(x, shape, torch.float8_e4m3fn), nat.empty(x, (*shape[:-1], 1), torch.float32)
    if m == 0:
        return q, s
    given = x
    if x.dim() != 2:
        x = x.reshape(m, k)
    ldx = x.stride(0) if m > 1 else k
    if x.stride(1) != 1 or ldx < k:
        x, ldx = x.clone(memory_format=torch.contiguous_format), k
    elif out is None and x.data_ptr() == given.data_ptr():
        nat.remember(_QUANT, (given.shape, given.stride(), given.dtype),
                     (m, k, nat.dtype_code(x.dtype), ldx, q.shape, q.dtype, s.shape, s.dtype), 4096)
    with nat.current(x.device):
        nat.check(nat.lib().hkx_fp8_quant(x.data_ptr(), ldx, nat.dtype_code(x.dtype), q.data_ptr(), k, s.data_ptr(),
                                          m, k, nat.stream_of(x.device)))
    return q, s


__all__ = ["quant"]
