"""What stands between two blocks of a decoder layer, in one pass: the norm after a block, its gated and
scaled residual add, and the norm before the next.

    h, y = hk.ops.block_norm(x, residual, post=w1, pre=w2, gate=g)

    u = x / rms(x) * post                                     (u = x without post)
    h = residual_scale * residual + branch_scale * gate * u
    y = h / rms(h) * pre                                      (y is None without pre)

with rms(v) = sqrt(mean(v^2) + eps) over the last dimension. x (..., D) is bf16, fp16 or fp32 and y the
same; the residual stream and h have x's type or are fp32; post and pre (D,) and the gate have x's type
or are fp32. The gate is broadcast over x: (D,), (B, 1, D), (B, S, 1), (B, S, D) and the like -- its
leading sizes are x's, then ones. A row's sums are fp32, the norms' factors made in 64 bits and rounded once;
h is rounded only as it is stored.
D up to 16384 (8192 where gradients are taken).

quant="mxfp8" or "mxfp4" gives y as (q, s), the operand of an MX product (hk.ops.mxfp4.gemm), without
another pass: q (..., D) float8_e4m3fn, or (..., D/2) packed codes, and s (..., D/32); D a multiple of 32.
quant="fp8" gives the operands of hk.ops.scaled_mm and hk.ops.experts.gemm: q (..., D) float8_e4m3fn and
s (..., 1) fp32, as hk.ops.fp8.quant makes them of the fp32 y; any D.

Differentiable in x, residual, post, pre and gate (not through a quantized y, nor in forward mode): one backward pass over the
same bytes, with the gradients of post, pre and a broadcast gate summed in a fixed order, a run of rows in
fp32 and the runs in 64 bits.

A call's checks and layout are kept by the shapes, strides and types they depend on, as a template of
the library's arguments; a call of known layout fills in its addresses.
"""

from __future__ import annotations

import ctypes

from .. import _native as nat

QUANT = {None: 0, "mxfp8": 1, "mxfp4": 2, "fp8": 4}


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


#: Layouts of a call: (arguments filled in but for their addresses, the shapes of the outputs).
_PLANS: dict = {}


def _forward(x, residual, post, pre, gate, scales, quant, keep_rstd):
    """(h, y, the norms' factors): a checked call."""
    import torch  # noqa: PLC0415

    d = x.shape[-1]
    g, keep = _args(x, residual, post, pre, gate, *scales)
    g.ldh = d
    y_shape = y_type = s_shape = s_stride = None
    if pre is not None:
        g.quant = QUANT[quant]
        y_shape, y_type = tuple(x.shape), x.dtype
        if quant is not None:
            y_type = torch.uint8 if quant == "mxfp4" else torch.float8_e4m3fn
            y_shape = (*x.shape[:-1], d // 2 if quant == "mxfp4" else d)
        if quant == "fp8":
            s_shape = (*x.shape[:-1], 1)
        elif quant is not None:
            s_shape = (*x.shape[:-1], d // 32)
            s_stride, step = [1], (d // 32 + 3) // 4 * 4
            for n in reversed(s_shape[:-1]):
                s_stride.insert(0, step)
                step *= n
            g.ldys = (d // 32 + 3) // 4 * 4
        g.ldy = y_shape[-1]
    plan = (g.rows, y_shape, y_type, s_shape, s_stride)
    out = _run(g, plan, x, residual, keep_rstd)
    return out, bytes(g), plan, keep


def _run(g, plan, x, residual, keep_rstd):
    """Outputs for arguments whose inputs are in place, and the launch."""
    rows, y_shape, y_type, s_shape, s_stride = plan
    h = nat.empty(residual, residual.shape, residual.dtype)
    g.h = h.data_ptr()
    y = rstd = None
    if y_shape is not None:
        y = nat.empty(x, y_shape, y_type)
        g.y = y.data_ptr()
        if s_shape is not None:
            import torch  # noqa: PLC0415

            if s_stride is None:
                s = nat.empty(x, s_shape, torch.float32)
            else:
                s = torch.empty_strided(s_shape, s_stride, dtype=torch.uint8, device=x.device)
            g.y_scales = s.data_ptr()
            y = (y, s)
    if keep_rstd:
        import torch  # noqa: PLC0415

        rstd = nat.empty(x, (rows, 2), torch.float32)
        g.rstd = rstd.data_ptr()
    if rows:
        with nat.current(x.device):
            nat.check(nat.lib().hkx_block_norm(ctypes.byref(g), nat.stream_of(x.device)))
    return h, y, rstd


_FUNCTION: list = []


def _function():
    """The autograd function, made at the first call that takes gradients."""
    if _FUNCTION:
        return _FUNCTION[0]
    import torch  # noqa: PLC0415

    class BlockNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, residual, post, pre, gate, scales):
            h, y, rstd = _call(x, residual, post, pre, gate, scales, None, True)
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


#: Layouts of a backward call: (arguments filled in but for their addresses, workspace bytes, the
#: types of dpost and dpre as the kernels write them).
_GRAD_PLANS: dict = {}


def _backward(x, residual, post, pre, gate, rstd, dh, dy, scales, need):
    """The gradients of (x, residual, post, pre, gate); post, pre and gate's None where not needed."""
    if dh is None and dy is None:
        return (None,) * 5
    key = (_layout(x), _layout(residual), _layout(post), _layout(pre), _layout(gate), _layout(dh),
           _layout(dy), scales, need)
    plan, keep = _GRAD_PLANS.get(key), None
    if plan is None:
        plan, keep = _grad_plan(x, residual, post, pre, gate, dh, dy, scales, need)
        if keep is None:
            nat.remember(_GRAD_PLANS, key, plan, 4096)
    args, nws, tpost, tpre = plan
    q = nat.HkxBlockNormGradArgs.from_buffer_copy(args)
    f = q.f
    f.x, f.residual, f.post, f.pre, f.gate, q.dh, q.dy = keep[0] if keep is not None else [
        None if t is None else t.data_ptr() for t in (x, residual, post, pre, gate, dh, dy)]
    f.rstd = rstd.data_ptr()
    dx, dr = nat.empty(x, x.shape, x.dtype), nat.empty(residual, residual.shape, residual.dtype)
    q.dx, q.dresidual = dx.data_ptr(), dr.data_ptr()
    dpost = dpre = dgate = None
    if post is not None and need[2]:
        dpost = nat.empty(x, post.shape, tpost)
        q.dpost = dpost.data_ptr()
    if pre is not None and need[3]:
        dpre = nat.empty(x, pre.shape, tpre)
        q.dpre = dpre.data_ptr()
    if gate is not None and need[4]:
        dgate = nat.empty(x, gate.shape, gate.dtype)
        q.dgate = dgate.data_ptr()
    if f.rows == 0:
        for t in (dpost, dpre, dgate):
            if t is not None:
                t.zero_()
    else:
        if nws:
            ws = nat.workspace(x.device, nws)
            q.ws, q.ws_bytes = ws.data_ptr(), nws
        with nat.current(x.device):
            nat.check(nat.lib().hkx_block_norm_backward(ctypes.byref(q), nat.stream_of(x.device)))
    if dpost is not None and tpost != post.dtype:
        dpost = dpost.to(post.dtype)
    if dpre is not None and tpre != pre.dtype:
        dpre = dpre.to(pre.dtype)
    return dx, dr, dpost, dpre, dgate


def _grad_plan(x, residual, post, pre, gate, dh, dy, scales, need):
    """(the plan, None), or with (the operands' addresses, what holds them) where one had to be copied."""
    import torch  # noqa: PLC0415

    d = x.shape[-1]
    q = nat.HkxBlockNormGradArgs()
    q.size = ctypes.sizeof(q)
    q.f, keep = _args(x, residual, post, pre, gate, *scales)
    ptr = [q.f.x, q.f.residual, q.f.post, q.f.pre, q.f.gate]
    for name, t in (("dh", dh), ("dy", dy)):
        if t is not None:
            t = _rows(t, d)
            keep.append(t)
            setattr(q, name, t.data_ptr())
            setattr(q, "ld" + name, _ld(t, d))
        ptr.append(None if t is None else t.data_ptr())
    q.lddx = q.lddr = d
    tpost, tpre = (None if w is None else w.dtype for w in (post, pre))
    if tpost != tpre and tpost is not None and tpre is not None:
        tpost = tpre = torch.float32  # (weights of two types go to the kernels as fp32)
    # which sums are wanted, for the workspace's size: any address that is not null
    q.dpost = 16 if post is not None and need[2] else None
    q.dpre = 16 if pre is not None and need[3] else None
    q.dgate = 16 if gate is not None and need[4] else None
    q.dx = q.dresidual = 16
    nws = nat.lib().hkx_block_norm_backward_workspace(ctypes.byref(q))
    q.dpost = q.dpre = q.dgate = q.dx = q.dresidual = None
    plan = (bytes(q), nws, tpost, tpre)
    mine = [None if t is None else t.data_ptr() for t in (x, residual, post, pre, gate, dh, dy)]
    return plan, None if [p or None for p in ptr] == [p or None for p in mine] else (ptr, keep)


def _layout(t):
    return None if t is None else (t.shape, t.stride(), t.dtype)


def _call(x, residual, post, pre, gate, scales, quant, grad):
    key = (_layout(x), _layout(residual), _layout(post), _layout(pre), _layout(gate), scales, quant, grad)
    plan = _PLANS.get(key)
    d = x.get_device()
    ptr = [None if t is None else t.data_ptr() for t in (x, residual, post, pre, gate)]
    if plan is None or d < 0 or any(t is not None and t.get_device() != d for t in (residual, post, pre, gate)) or (
            quant is not None and any(p and p & 15 for p in ptr)):
        x, residual, post, pre, gate = _checked(x, residual, post, pre, gate, quant, grad)
        out, args, plan, keep = _forward(x, residual, post, pre, gate, scales, quant, grad)
        # (a template only where every operand was read where it is)
        if all(a is None or a == b.data_ptr() for a, b in zip(ptr, (x, residual, post, pre, gate))) and all(
                t is None or t.data_ptr() in ptr for t in keep):
            nat.remember(_PLANS, key, (args, plan), 4096)
        return out
    args, plan = plan
    g = nat.HkxBlockNormArgs.from_buffer_copy(args)
    g.x, g.residual, g.post, g.pre, g.gate = ptr
    return _run(g, plan, x, residual, grad)


def block_norm(x, residual, *, post=None, pre=None, gate=None, branch_scale=1.0, residual_scale=1.0,
               eps=1e-6, quant=None):
    """(h, y): see the module's docstring."""
    import torch  # noqa: PLC0415

    nat.no_tangents("block_norm", x, residual, post, pre, gate)
    scales = (float(branch_scale), float(residual_scale), float(eps))
    if torch.is_grad_enabled() and (x.requires_grad or residual.requires_grad or any(
            t is not None and t.requires_grad for t in (post, pre, gate))):
        if quant is not None:
            raise ValueError("block_norm: no gradient through a quantized y")
        return _function().apply(x, residual, post, pre, gate, scales)
    return _call(x, residual, post, pre, gate, scales, quant, False)[:2]


def _checked(x, residual, post, pre, gate, quant, grad):
    """The operands, refused where the kernels do not take them (copied where a quantized y needs
    them aligned)."""
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
    nat.int32("block_norm", rows=x.numel() // d)
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
        raise ValueError(f"block_norm: quant is None, 'mxfp8', 'mxfp4' or 'fp8', got {quant!r}")
    if quant is not None and (pre is None or (d % 32 and quant != "fp8")):
        raise ValueError(f"block_norm: a quantized y needs pre and D={d} a multiple of 32")
    limit = 8192 if grad else 16384
    if d > limit:
        raise ValueError(f"block_norm: D={d}, at most {limit}{' where gradients are taken' if grad else ''}")
    if quant is None:
        return x, residual, post, pre, gate
    return tuple(t if t is None or (t.data_ptr() % 16 == 0 and t.is_contiguous())
                 else t.clone(memory_format=torch.contiguous_format) for t in (x, residual, post, pre, gate))


__all__ = ["block_norm"]
