"""What stands between two blocks of a decoder layer, in one pass: the norm after a block, its gated and
scaled residual add, and the norm before the next.

    h, y = hk.ops.block_norm(x, residual, post=w1, pre=w2, gate=g)

    u = x / rms(x) * post                                     (u = x without post)
    h = residual_scale * residual + branch_scale * gate * u
    y = h / rms(h) * pre                                      (y is None without pre)

with rms(v) = sqrt(mean(v^2) + eps) over the last dimension. x (..., D) is bf16, fp16 or fp32 and y the
same; the residual stream and h have x's type or are fp32; post and pre (D,) and the gate have x's type
or are fp32. The gate is broadcast over x: (D,), (B, 1, D), (B, S, 1), (B, S, D) and the like -- its
leading sizes are x's, then ones. Sums and both norms are fp32; h is rounded only as it is stored.
D up to 16384 (8192 where gradients are taken).

quant="mxfp8" or "mxfp4" gives y as (q, s), an MX product's operand (hk.ops.mxfp8.gemm, hk.ops.mxfp4.gemm)
without another pass: x is then 2-dimensional or y's rows are x's leading dimensions flattened, and D a
multiple of 32.

Differentiable in x, residual, post, pre and gate (not through a quantized y): one backward pass over the
same bytes, with the gradients of post, pre and a broadcast gate summed in fp32 in a fixed order.
"""

from __future__ import annotations

import ctypes

from .. import _native as nat

QUANT = {None: 0, "mxfp8": 1, "mxfp4": 2}


def _rows(t, d):
    """`t` (..., D) as rows with unit stride: a view where it has one."""
    t = t.reshape(-1, d) if t.dim() != 2 else t
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t


def _ld(t, d):
    """The row stride of a single row is anything."""
    return t.stride(0) if t.shape[0] > 1 else d


def _gate_shape(gate, x):
    """(rows that share a row of the gate, whether it has a value a column)."""
    lead, gl = tuple(x.shape[:-1]), tuple(gate.shape)
    if len(gl) > x.dim():
        raise ValueError(f"block_norm: gate {gl} does not broadcast to x {tuple(x.shape)}")
    gl = (1,) * (x.dim() - len(gl)) + gl
    d = x.shape[-1]
    if gl[-1] not in (1, d):
        raise ValueError(f"block_norm: gate {tuple(gate.shape)} does not broadcast to x {tuple(x.shape)}")
    i = 0
    while i < len(lead) and gl[i] == lead[i]:
        i += 1
    shared = 1
    for a, b in zip(lead[i:], gl[i:-1]):
        if b != 1:
            raise ValueError(f"block_norm: the gate's leading sizes are x's, then ones: got "
                             f"{tuple(gate.shape)} for x {tuple(x.shape)}")
        shared *= a
    return shared, int(gl[-1] == d)


def _args(x, residual, post, pre, gate, branch_scale, residual_scale, eps):
    """The call's arguments, and what keeps their memory alive."""
    d = x.shape[-1]
    xr, rr = _rows(x, d), _rows(residual, d)
    keep = [xr, rr]
    g = nat.HkxBlockNormArgs()
    g.size = ctypes.sizeof(g)
    g.x_dtype, g.r_dtype = nat.dtype_code(x.dtype), nat.dtype_code(residual.dtype)
    g.rows, g.d = xr.shape[0], d
    g.branch_scale, g.residual_scale, g.eps = branch_scale, residual_scale, eps
    g.x, g.residual, g.ldx, g.ldr = xr.data_ptr(), rr.data_ptr(), _ld(xr, d), _ld(rr, d)
    if post is not None and pre is not None and post.dtype != pre.dtype:
        post, pre = post.float(), pre.float()
    for name, w in (("post", post), ("pre", pre)):
        if w is not None:
            w = w.contiguous()
            keep.append(w)
            g.w_dtype = nat.dtype_code(w.dtype)
            setattr(g, name, w.data_ptr())
    if gate is not None:
        gate = gate.contiguous()
        keep.append(gate)
        g.gate, g.gate_dtype = gate.data_ptr(), nat.dtype_code(gate.dtype)
        g.gate_rows, g.gate_col = _gate_shape(gate, x)
    return g, keep


def _forward(x, residual, post, pre, gate, branch_scale, residual_scale, eps, quant, keep_rstd):
    import torch  # noqa: PLC0415

    d = x.shape[-1]
    g, keep = _args(x, residual, post, pre, gate, branch_scale, residual_scale, eps)
    h = nat.empty(residual, residual.shape, residual.dtype)
    rows = g.rows
    y = scales = rstd = None
    g.h, g.ldh = h.data_ptr(), d
    if pre is not None:
        g.quant = QUANT[quant]
        if quant is None:
            y = nat.empty(x, x.shape, x.dtype)
            g.ldy = d
        else:
            y = (nat.empty(x, (rows, d), torch.float8_e4m3fn) if quant == "mxfp8"
                 else nat.empty(x, (rows, d // 2), torch.uint8))
            scales = nat.empty(x, (rows, (d // 32 + 3) // 4 * 4), torch.uint8)
            g.y_scales, g.ldys, g.ldy = scales.data_ptr(), scales.stride(0), y.stride(0)
            if d % 128:
                scales = scales[:, :d // 32]
        g.y = y.data_ptr()
    if keep_rstd:
        rstd = nat.empty(x, (rows, 2), torch.float32)
        g.rstd = rstd.data_ptr()
    if rows:
        nat.check(nat.lib().hkx_block_norm(ctypes.byref(g), nat.stream_of(x.device)))
    return h, (y if quant is None else (y, scales)), rstd


_FUNCTION: list = []


def _function():
    """The autograd function, made at the first call that takes gradients."""
    if _FUNCTION:
        return _FUNCTION[0]
    import torch  # noqa: PLC0415

    class BlockNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, residual, post, pre, gate, scales):
            h, y, rstd = _forward(x, residual, post, pre, gate, *scales, None, True)
            ctx.save_for_backward(x, residual, post, pre, gate, rstd)
            ctx.scales = scales
            ctx.set_materialize_grads(False)
            return h, y

        @staticmethod
        @torch.autograd.function.once_differentiable
        def backward(ctx, dh, dy):
            x, residual, post, pre, gate, rstd = ctx.saved_tensors
            need = ctx.needs_input_grad
            return (*_backward(x, residual, post, pre, gate, rstd, dh, dy, ctx.scales, need), None)

    _FUNCTION.append(BlockNorm)
    return BlockNorm


def _backward(x, residual, post, pre, gate, rstd, dh, dy, scales, need):
    import torch  # noqa: PLC0415

    d = x.shape[-1]
    if dh is None and dy is None:
        return (None,) * 5
    q = nat.HkxBlockNormGradArgs()
    q.size = ctypes.sizeof(q)
    q.f, keep = _args(x, residual, post, pre, gate, *scales)
    q.f.rstd = rstd.data_ptr()
    for name, t in (("dh", dh), ("dy", dy)):
        if t is not None:
            t = _rows(t, d)
            keep.append(t)
            setattr(q, name, t.data_ptr())
            setattr(q, "ld" + name, _ld(t, d))
    dx, dr = nat.empty(x, x.shape, x.dtype), nat.empty(residual, residual.shape, residual.dtype)
    q.dx, q.dresidual, q.lddx, q.lddr = dx.data_ptr(), dr.data_ptr(), d, d
    wt = None if post is None else post.dtype
    if post is not None and pre is not None and pre.dtype != wt:
        wt = torch.float32  # mixed types go to the kernels as fp32
    wt = pre.dtype if wt is None and pre is not None else wt
    dpost = nat.empty(x, (d,), wt) if post is not None and need[2] else None
    dpre = nat.empty(x, (d,), wt) if pre is not None and need[3] else None
    dgate = nat.empty(x, gate.shape, gate.dtype) if gate is not None and need[4] else None
    for name, t in (("dpost", dpost), ("dpre", dpre), ("dgate", dgate)):
        if t is not None:
            setattr(q, name, t.data_ptr())
    if q.f.rows == 0:
        for t in (dpost, dpre, dgate):
            if t is not None:
                t.zero_()
    else:
        L = nat.lib()
        nws = L.hkx_block_norm_backward_workspace(ctypes.byref(q))
        if nws:
            ws = nat.workspace(x.device, nws)
            q.ws, q.ws_bytes = ws.data_ptr(), nws
        nat.check(L.hkx_block_norm_backward(ctypes.byref(q), nat.stream_of(x.device)))
    if dpost is not None and dpost.dtype != post.dtype:
        dpost = dpost.to(post.dtype)
    if dpre is not None and dpre.dtype != pre.dtype:
        dpre = dpre.to(pre.dtype)
    return dx, dr, dpost, dpre, dgate


def block_norm(x, residual, *, post=None, pre=None, gate=None, branch_scale=1.0, residual_scale=1.0,
               eps=1e-6, quant=None):
    """(h, y): see the module's docstring."""
    import torch  # noqa: PLC0415

    floats = (torch.bfloat16, torch.float16, torch.float32)
    if x.dtype not in floats or residual.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"block_norm: x is bf16, fp16 or fp32 and the residual the same or fp32, got "
                        f"{x.dtype} and {residual.dtype}")
    if x.dim() < 1 or x.shape != residual.shape or x.shape[-1] == 0:
        raise ValueError(f"block_norm: x and the residual are (..., D) alike, got {tuple(x.shape)} and "
                         f"{tuple(residual.shape)}")
    if not x.is_cuda:
        raise ValueError(f"block_norm: x is on a GPU, got {x.device}")
    d = x.shape[-1]
    for name, t in (("residual", residual), ("post", post), ("pre", pre), ("gate", gate)):
        if t is None:
            continue
        if t.device != x.device:
            raise ValueError(f"block_norm: {name} is on {t.device}, not on {x.device}")
        if name == "residual":
            continue
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"block_norm: {name} has x's type or is fp32, got {t.dtype} for {x.dtype}")
        if name != "gate" and t.shape != (d,):
            raise ValueError(f"block_norm: {name} is ({d},), got {tuple(t.shape)}")
    if gate is not None:
        _gate_shape(gate, x)
    if quant not in QUANT:
        raise ValueError(f"block_norm: quant is None, 'mxfp8' or 'mxfp4', got {quant!r}")
    if quant is not None and (pre is None or d % 32):
        raise ValueError(f"block_norm: a quantized y needs pre and D={d} a multiple of 32")
    limit = 16384
    grad = torch.is_grad_enabled() and any(
        t is not None and t.requires_grad for t in (x, residual, post, pre, gate))
    if grad:
        if quant is not None:
            raise ValueError("block_norm: no gradient through a quantized y")
        limit = 8192
    if d > limit:
        raise ValueError(f"block_norm: D={d}, at most {limit}{' where gradients are taken' if grad else ''}")
    scales = (float(branch_scale), float(residual_scale), float(eps))
    if quant is not None:  # (rows of 16-byte pieces)
        x, residual, post, pre, gate = (
            t if t is None or (t.data_ptr() % 16 == 0 and t.is_contiguous()) else t.clone(
                memory_format=torch.contiguous_format) for t in (x, residual, post, pre, gate))
    if grad:
        return _function().apply(x, residual, post, pre, gate, scales)
    h, y, _ = _forward(x, residual, post, pre, gate, *scales, quant, False)
    return h, y


__all__ = ["block_norm"]
