"""A layer of experts on gfx950: the router, the products of each expert's rows with its weight, and the way back
to the tokens; forward and backward.

    weights, chosen, plan = experts.route(logits, k)                     # (T, E) -> (T, k)
    a = experts.gemm(x, gate_up, plan, gather=True, silu_mul=True)       # x (T, K) -> (T k, I), rows by expert
    y = experts.gemm(a, down, plan)                                      # (T k, D)
    out = experts.combine(y, plan, weights)                              # (T, D)

or all of it as `experts.mlp(x, logits, k, gate_up, down)`. T tokens have k experts each: R = T k rows, in the order of
(expert, token). How many each expert has is known to the GPU alone: nothing here waits for the GPU, and every
call can be captured in a graph after a first call. (A captured backward pass: while an eager graph of the same leaves is
alive, torch's engine joins that one's stream to the captured one, which ends the process; drop its results first.)

A `Plan` is three int32 tensors on the GPU: offsets (E + 1), of expert e the rows offsets[e] .. offsets[e + 1], from
0; rows (R), the token of each row, -1 behind the last; slots (T, k), the row of each choice, -1 for one that has no
expert. To drop a choice, set its slot to -1 (its row is then computed, and passes no gradient). A token whose logits are
all -inf (padding) has no rows, and its output is zero. Plans from elsewhere may leave out `rows` where no call gathers,
and `slots` where none combines or has a gathered gradient. Offsets out of order or past the rows are clamped and an index
out of range stands for a row of zeros: nothing is read or written outside the tensors.

Derivatives are the backward pass's, of bf16 products: a forward-mode one, a second one, and one through 8-bit operands or
their scales are refused.

The rows behind the last expert's are zeros in a new output and stay as they were in one that is passed in.

A call's checks and layout are kept by the shapes, strides and types they depend on, as a template of the library's
arguments; a call of known layout fills in its addresses.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

from .. import _native as nat
from . import fp8
from .mxfp8 import _on

MAX_EXPERTS, MAX_CHOSEN = 1024, 64
NT, NN, TN = range(3)  # the library's products (include/hkx.h)

_TORCH: list = []


def _torch():
    """torch, looked up once (an import statement costs a call 0.3 us)."""
    if not _TORCH:
        import torch  # noqa: PLC0415

        _TORCH.append(torch)
    return _TORCH[0]


class Plan(NamedTuple):
    """The order of rows by expert (the module's docstring)."""

    offsets: object
    rows: object = None
    slots: object = None


def _int32(call, device, **tensors):
    import torch  # noqa: PLC0415

    for name, t in tensors.items():
        if t is None:
            continue
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise TypeError(f"{call}: plan.{name} is contiguous int32, got {t.dtype} {tuple(t.shape)}")
        if t.device != device:
            raise ValueError(f"{call}: plan.{name} is on {t.device}, not on {device}")


def _ld(t, least):
    """A matrix's row stride (a single row's is anything)."""
    return t.stride(0) if t.shape[0] > 1 else least


def _rows16(t):
    """`t` (rows, columns) with rows the kernels read in place: unit stride, 16-byte aligned."""
    per = 16 // t.element_size()
    if t.data_ptr() % 16 == 0 and t.stride(1) == 1 and (t.shape[0] < 2 or (
            t.stride(0) % per == 0 and t.stride(0) >= t.shape[1])):
        return t
    out = t.new_empty(t.shape)
    out.copy_(t)
    return out


def _experts16(w):
    """`w` (E, rows, columns) likewise."""
    per = 16 // w.element_size()
    if (w.data_ptr() % 16 == 0 and w.stride(2) == 1 and (w.shape[1] < 2 or (
            w.stride(1) % per == 0 and w.stride(1) >= w.shape[2])) and (w.shape[0] < 2 or w.stride(0) % per == 0)):
        return w
    out = w.new_empty(w.shape)
    out.copy_(w)
    return out


def _grad(*tensors):
    for t in tensors:
        if t is not None and t.requires_grad:
            return _torch().is_grad_enabled()
    return False


def _elsewhere(d, *tensors):
    """Whether a tensor is not on GPU d (a device's number; below 0: none)."""
    if d < 0:
        return True
    for t in tensors:
        if t is not None and t.get_device() != d:
            return True
    return False


# ---------------------------------------------------------------- the products


#: Layouts of gemm's operands: (arguments filled in but for their addresses, C's shape, the workspace's bytes).
_GEMM: dict = {}


def _layout(t):
    return None if t is None else (t.shape, t.stride(), t.dtype)


def gemm(x, w, plan, *, gather=False, bias=None, silu_mul=False, scale_a=None, scale_b=None, out=None):
    """bf16 (R, N): row r is x[r] (gather: x[plan.rows[r]]) times its expert's w[e] (N, K) transposed (+ bias[e]).

    * x (R, K), or with `gather` (T, K), and w (E, N, K): bf16, or float8_e4m3fn with fp32 scales: scale_a one a row of
      x ((rows,) or (rows, 1)) or one for all, scale_b one a row of w ((E, N)) or an expert ((E,) or (E, 1));
    * bias (E, N) bf16, fp16 or fp32;
    * silu_mul: w[e] (and scale_b, bias) holds N gate rows, then N up rows: silu(z[:, :N]) * z[:, N:] of z (R, 2N);
    * out: bf16 (R, N) to write into (no gradient), columns next to each other.

    K and N multiples of 8, an 8-bit K of 16; E up to 1024, R up to 2^31 - 256; an expert's w, and an x that is gathered,
    under 4 GiB.
    Sums are fp32, rounded once. Differentiable in x, w and bias (bf16): with silu_mul z is kept in bf16 for the backward
    pass and its gradient, which the other products read, rounded to bf16; a gathered x's gradient adds a token's rows,
    which stay fp32 till then, in order of its choices. No atomics: the same bits every time."""
    nat.no_tangents("experts.gemm", x, w, bias, scale_a, scale_b)
    if _grad(x, w, bias, scale_a, scale_b):
        return _gemm_grad(x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out)
    return _gemm(x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out, None)


def _gemm(x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out, z):
    index = plan.rows if gather else None
    key = (_layout(x), _layout(w), _layout(plan.offsets), _layout(plan.rows), _layout(bias), silu_mul, gather,
           _layout(scale_a), _layout(scale_b), z is None)
    known = _GEMM.get(key) if out is None else None
    d = x.get_device()
    offsets = plan.offsets
    if known is None or _elsewhere(d, x, w, offsets, index, bias, scale_a, scale_b):
        return _gemm_checked(x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out, z, key)
    pa, pb = x.data_ptr(), w.data_ptr()
    bits = pa | pb
    g = nat.HkxExpertsGemmArgs.from_buffer_copy(known[0])
    g.a, g.b, g.offsets = pa, pb, offsets.data_ptr()
    if index is not None:
        g.index = index.data_ptr()
    if bias is not None:
        at = bias.data_ptr()
        g.bias = at
        bits |= at
    if scale_a is not None:
        at = scale_b.data_ptr()
        g.sa, g.sb = scale_a.data_ptr(), at
        bits |= at
    if bits & 15:
        return _gemm_checked(x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out, z, key)
    return _launch(g, x, nat.empty(x, known[1], _torch().bfloat16), z, known[2])


def _launch(g, x, out, z, need=None):
    g.c = out.data_ptr()
    if z is not None:
        g.z, g.ldz = z.data_ptr(), _ld(z, z.shape[1])
    _run(g, x.device, need)
    return out


def _run(g, device, need=None):
    """The launch; need: the workspace's bytes, where they are known."""
    with nat.current(device):
        if need is None:
            need = nat.lib().hkx_experts_gemm_workspace(ctypes.byref(g))
        if need:
            ws = nat.workspace(device, need)
            g.ws, g.ws_bytes = ws.data_ptr(), need
        nat.check(nat.lib().hkx_experts_gemm(ctypes.byref(g), nat.stream_of(device)))


def _check(call, x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out):
    """(R, N) of a call, refused where the kernels do not take it."""
    import torch  # noqa: PLC0415

    wide = x.dtype == torch.float8_e4m3fn
    if x.dtype not in (torch.bfloat16, torch.float8_e4m3fn) or w.dtype != x.dtype:
        raise TypeError(f"{call}: x and w are both bf16 or both float8_e4m3fn, got {x.dtype} and {w.dtype}")
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2]:
        raise ValueError(f"{call}: x (rows, K) and w (E, N, K), got {tuple(x.shape)} and {tuple(w.shape)}")
    e, n, k = w.shape
    if silu_mul:
        if n % 2:
            raise ValueError(f"{call}: silu_mul takes gate rows, then as many up rows: w has {n}")
        n //= 2
    step = 16 if wide else 8
    if n % 8 or n == 0 or k % step or k == 0:
        raise ValueError(f"{call}: N={n} a multiple of 8 and K={k} of {step}")
    if not 1 <= e <= MAX_EXPERTS:
        raise ValueError(f"{call}: {e} experts, 1 to {MAX_EXPERTS}")
    if not x.is_cuda:
        raise ValueError(f"{call}: x is on a GPU, got {x.device}")
    if plan.offsets is None or plan.offsets.shape != (e + 1,):
        raise ValueError(f"{call}: plan.offsets is ({e + 1},)")
    _on(x.device, call, w=w, bias=bias, scale_a=scale_a, scale_b=scale_b, out=out)
    _int32(call, x.device, offsets=plan.offsets, rows=plan.rows if gather else None)
    r = x.shape[0]
    if gather:
        if plan.rows is None or plan.rows.dim() != 1:
            raise ValueError(f"{call}: gather takes the plan's rows")
        r = plan.rows.shape[0]
        if r and not x.shape[0]:
            raise ValueError(f"{call}: {r} rows gathered from none")
    elif plan.rows is not None and plan.rows.numel() != r:
        raise ValueError(f"{call}: x has {r} rows and the plan {plan.rows.numel()} (gather=True for x by token)")
    nat.int32(call, rows=max(r, x.shape[0]), N=w.shape[1], K=k)
    if bias is not None and (bias.shape != w.shape[:2] or bias.dtype not in (
            torch.bfloat16, torch.float16, torch.float32)):
        raise ValueError(f"{call}: bias is bf16, fp16 or fp32 {tuple(w.shape[:2])}, got {bias.dtype} "
                         f"{tuple(bias.shape)}")
    if wide:
        for name, s in (("scale_a", scale_a), ("scale_b", scale_b)):
            if s is None or s.dtype != torch.float32:
                raise TypeError(f"{call}: float8_e4m3fn operands take {name} in fp32")
        if scale_a.numel() != 1 and tuple(scale_a.shape) not in ((x.shape[0],), (x.shape[0], 1)):
            raise ValueError(f"{call}: scale_a is one value or ({x.shape[0]},), got {tuple(scale_a.shape)}")
        if tuple(scale_b.shape) not in (tuple(w.shape[:2]), (e,), (e, 1)):
            raise ValueError(f"{call}: scale_b is {tuple(w.shape[:2])} or ({e},), got {tuple(scale_b.shape)}")
    elif scale_a is not None or scale_b is not None:
        raise ValueError(f"{call}: scales go with float8_e4m3fn operands")
    if out is not None and (out.dtype != torch.bfloat16 or tuple(out.shape) != (r, n) or out.stride(1) != 1
                            or (r > 1 and (out.stride(0) < n or out.stride(0) % 4)) or out.data_ptr() % 8):
        raise ValueError(f"{call}: out is bf16 ({r}, {n}) with unit column stride and 8-byte aligned rows")
    return r, n


def _gemm_checked(x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out, z, key):
    import torch  # noqa: PLC0415

    r, n = _check("experts.gemm", x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out)
    given = (x, w, bias, scale_a, scale_b)
    new = out is None
    if new:
        out = nat.empty(x, (r, n), torch.bfloat16)
    if r == 0:
        return out
    x, w = _rows16(x), _experts16(w)
    if bias is not None and (bias.data_ptr() % 16 or bias.stride(1) != 1 or (
            bias.shape[0] > 1 and (bias.stride(0) % 4 or bias.stride(0) < bias.shape[1]))):
        bias = bias.clone(memory_format=torch.contiguous_format)
    if scale_a is not None:
        scale_a = scale_a.contiguous()
        scale_b = scale_b.contiguous()
        if scale_b.data_ptr() % 16:
            scale_b = scale_b.clone()
    g = nat.HkxExpertsGemmArgs()
    g.size, g.op, g.ab_dtype = ctypes.sizeof(g), NT, nat.dtype_code(x.dtype)
    g.experts, g.rows, g.a_rows, g.n, g.k = w.shape[0], r, x.shape[0], n, w.shape[2]
    g.silu_mul, g.zero_rest = int(bool(silu_mul)), int(new)
    g.lda, g.ldb, g.ldc = _ld(x, x.shape[1]), w.stride(1) if w.shape[1] > 1 else w.shape[2], _ld(out, n)
    g.b_expert = w.stride(0) if w.shape[0] > 1 else 0
    g.a, g.b, g.offsets = x.data_ptr(), w.data_ptr(), plan.offsets.data_ptr()
    if gather:
        g.index = plan.rows.data_ptr()
    if bias is not None:
        g.bias, g.bias_dtype, g.bias_ld = bias.data_ptr(), nat.dtype_code(bias.dtype), _ld(bias, bias.shape[1])
    if scale_a is not None:
        g.sa, g.sa_ld, g.sb = scale_a.data_ptr(), int(scale_a.numel() > 1), scale_b.data_ptr()
        g.sb_col = int(scale_b.dim() == 2 and scale_b.shape[1] == w.shape[1] and w.shape[1] > 1)
        g.sb_ld = w.shape[1] if g.sb_col else 1
    # (a template only where every operand was read where it is, and C is new)
    known = bytes(g) if new and all(a is None or a.data_ptr() == b.data_ptr() for a, b in zip(
        given, (x, w, bias, scale_a, scale_b))) else None
    g.c = out.data_ptr()
    if z is not None:
        g.z, g.ldz = z.data_ptr(), _ld(z, z.shape[1])
    with nat.current(x.device):
        need = nat.lib().hkx_experts_gemm_workspace(ctypes.byref(g))
    if known is not None:
        nat.remember(_GEMM, key, (known, (r, n), need), 4096)
    return _launch(g, x, out, z, need)


def _product(op, a, b, plan, out):
    """A gradient's product into `out`: NN dx (R, K) = dz (R, N) . w (E, N, K), bf16 or fp32, TN dw (E, N, K) = dz^T x."""
    g = nat.HkxExpertsGemmArgs()
    g.size, g.op, g.ab_dtype = ctypes.sizeof(g), op, nat.BF16
    g.c_dtype = nat.dtype_code(out.dtype)
    g.experts, g.rows, g.n, g.zero_rest = plan.offsets.shape[0] - 1, a.shape[0], out.shape[-1], 1
    g.a, g.b, g.c, g.offsets = a.data_ptr(), b.data_ptr(), out.data_ptr(), plan.offsets.data_ptr()
    g.lda = _ld(a, a.shape[1])
    if op == NN:
        g.k, g.ldb, g.b_expert = b.shape[1], b.stride(1) if b.shape[1] > 1 else b.shape[2], b.stride(0)
        g.ldc = _ld(out, out.shape[1])
    else:
        g.m, g.ldb, g.ldc, g.c_expert = a.shape[1], _ld(b, b.shape[1]), out.stride(1), out.stride(0)
    _run(g, a.device)
    return out


def _gemm_grad(x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out):
    import torch  # noqa: PLC0415

    if out is not None:
        raise ValueError("experts.gemm: no gradient through out=")
    if x.dtype == torch.float8_e4m3fn or scale_a is not None or scale_b is not None:
        raise ValueError("experts.gemm: no gradient through quantized values (detach, or torch.no_grad())")
    if x.dim() != 2 or w.dim() != 3:
        _check("experts.gemm", x, w, plan, gather, bias, silu_mul, scale_a, scale_b, out)
    if gather and x.requires_grad:
        if plan.slots is None or plan.slots.dim() != 2 or plan.slots.shape[0] != x.shape[0]:
            raise ValueError("experts.gemm: a gathered x's gradient takes the plan's slots (T, k)")
        _int32("experts.gemm", x.device, slots=plan.slots)
    return _functions()[0].apply(x, w, bias, plan, gather, silu_mul)


def _gemm_backward(x, w, bias, z, plan, gather, need, dy):
    """(dx, dw, dbias). Rounded to bf16 on the way: dz, as the products read bf16, and z, kept in bf16 (fp32 would double
    its write and its read, for an error of the size of dz's). A gathered row's gradient stays fp32 until its token's rows
    are added, which may cancel."""
    import torch  # noqa: PLC0415

    r, e = dy.shape[0], w.shape[0]
    rows16 = _rows16(dy)
    L, dev = nat.lib(), x.device
    dz = rows16
    if z is not None:
        dz = nat.empty(x, z.shape, torch.bfloat16)
        if r:
            with nat.current(dev):
                nat.check(L.hkx_experts_silu_grad(z.data_ptr(), z.shape[1], rows16.data_ptr(),
                                                  _ld(rows16, rows16.shape[1]), dz.data_ptr(), dz.shape[1],
                                                  plan.offsets.data_ptr(), e, r, rows16.shape[1], nat.stream_of(dev)))
    dx = dw = db = None
    if need[0]:
        dx = nat.empty(x, (r, w.shape[2]), torch.float32 if gather else torch.bfloat16)
        if r:
            _product(NN, dz, _experts16(w), plan, dx)
        if gather:
            dx = _gather_backward(x, dx, plan.slots)
    if need[1]:
        dw = nat.empty(x, w.shape, torch.bfloat16)
        xr = _rows16(x)
        if gather and r:
            sorted_x = nat.empty(x, (r, x.shape[1]), torch.bfloat16)
            with nat.current(dev):
                nat.check(L.hkx_experts_gather(xr.data_ptr(), _ld(xr, xr.shape[1]), plan.rows.data_ptr(),
                                               sorted_x.data_ptr(), xr.shape[1], r, xr.shape[0], xr.shape[1],
                                               nat.stream_of(dev)))
            xr = sorted_x
        if r:
            _product(TN, dz, xr, plan, dw)
        else:
            dw.zero_()
    if need[2]:
        db = nat.empty(x, bias.shape, bias.dtype)
        if r:
            with nat.current(dev):
                nat.check(L.hkx_experts_bias_grad(dz.data_ptr(), _ld(dz, dz.shape[1]), plan.offsets.data_ptr(),
                                                  db.data_ptr(), nat.dtype_code(bias.dtype), e, r, dz.shape[1],
                                                  nat.stream_of(dev)))
        else:
            db.zero_()
    return dx, dw, db


def _gather_backward(x, dr, slots):
    """bf16 (T, K) from the rows' dr (R, K) fp32."""
    t, k = slots.shape
    dx = nat.empty(x, (t, dr.shape[1]), x.dtype)
    if t == 0 or k == 0 or dr.shape[0] == 0:
        return dx.zero_()
    with nat.current(x.device):
        nat.check(nat.lib().hkx_experts_gather_grad(dr.data_ptr(), dr.shape[1], slots.data_ptr(), dx.data_ptr(), dr.shape[1],
                                                    t, k, dr.shape[0], dr.shape[1], nat.stream_of(x.device)))
    return dx


# ---------------------------------------------------------------- the way back


def combine(y, plan, weights=None):
    """(T, D): out[t] = sum over j of weights[t, j] * y[plan.slots[t, j]], y (R, D) bf16, fp16 or fp32 and weights
    (T, k) fp32 (None: ones), in fp32 and in order of j, rounded once to y's type. A choice without a row (slot -1)
    adds nothing. Differentiable in y and weights (a row that no choice has gets zeros)."""
    nat.no_tangents("experts.combine", y, weights)
    slots = plan.slots
    key = (_layout(y), _layout(slots), _layout(weights))
    if key not in _COMBINE or _elsewhere(y.get_device(), y, slots, weights):
        _check_combine(y, plan, weights)
        nat.remember(_COMBINE, key, True, 4096)
    if _grad(y, weights):
        return _functions()[1].apply(y, weights, slots)
    return _combine(y, slots, weights)


#: Layouts of combine's operands that were checked.
_COMBINE: dict = {}


def _check_combine(y, plan, weights):
    import torch  # noqa: PLC0415

    if y.dtype not in (torch.bfloat16, torch.float16, torch.float32) or y.dim() != 2 or y.shape[1] == 0:
        raise TypeError(f"experts.combine: y is bf16, fp16 or fp32 (R, D), got {y.dtype} {tuple(y.shape)}")
    slots = plan.slots
    if slots is None or slots.dim() != 2 or slots.numel() != y.shape[0]:
        raise ValueError(f"experts.combine: plan.slots is (T, k) with T k = {y.shape[0]}, y's rows")
    if not y.is_cuda:
        raise ValueError(f"experts.combine: y is on a GPU, got {y.device}")
    _int32("experts.combine", y.device, slots=slots)
    _on(y.device, "experts.combine", weights=weights)
    if weights is not None and (weights.dtype != torch.float32 or weights.shape != slots.shape):
        raise ValueError(f"experts.combine: weights are fp32 {tuple(slots.shape)}, got {weights.dtype} "
                         f"{tuple(weights.shape)}")
    nat.int32("experts.combine", rows=y.shape[0], D=y.shape[1])


def _unit(t):
    """`t` (rows, columns) with columns next to each other and rows apart."""
    return t if t.stride(1) == 1 and (t.shape[0] < 2 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _combine(y, slots, weights):
    t, k = slots.shape
    out = nat.empty(y, (t, y.shape[1]), y.dtype)
    if t == 0 or k == 0:
        return out.zero_()
    y = _unit(y)
    if weights is not None:
        weights = weights.contiguous()
    with nat.current(y.device):
        nat.check(nat.lib().hkx_experts_combine(
            y.data_ptr(), _ld(y, y.shape[1]), nat.dtype_code(y.dtype), slots.data_ptr(),
            None if weights is None else weights.data_ptr(), out.data_ptr(), y.shape[1], t, k, y.shape[0], y.shape[1],
            nat.stream_of(y.device)))
    return out


def _combine_backward(y, weights, slots, need, dout):
    import torch  # noqa: PLC0415

    t, k = slots.shape
    dw = nat.empty(y, (t, k), torch.float32) if need[1] else None
    dy = nat.empty(y, y.shape, y.dtype) if need[0] else None
    if t == 0 or k == 0:
        return dy, dw
    y, dout = _unit(y), _unit(dout)
    w = None if weights is None else weights.contiguous()
    with nat.current(y.device):
        ws = nat.workspace(y.device, 8 * t * k) if need[0] else None
        nat.check(nat.lib().hkx_experts_combine_backward(
            y.data_ptr(), _ld(y, y.shape[1]), dout.data_ptr(), _ld(dout, dout.shape[1]), nat.dtype_code(y.dtype),
            slots.data_ptr(), None if w is None else w.data_ptr(), None if dy is None else dy.data_ptr(), y.shape[1],
            None if dw is None else dw.data_ptr(), None if ws is None else ws.data_ptr(), t, k, y.shape[0], y.shape[1],
            nat.stream_of(y.device)))
    return dy, dw


# ---------------------------------------------------------------- the router


def route(logits, k, *, renormalize=True):
    """(weights, chosen, plan) of the k largest of each row of logits (T, E), bf16, fp16 or fp32: chosen (T, k) int32 in
    falling order, a tie to the lower expert, and weights (T, k) fp32, the softmax over the chosen's logits, or
    without `renormalize` over all E. An expert of logit -inf is not chosen: -1, weight 0, no row. NaN counts as the
    largest and makes its token's weights NaN. E up to 1024, k up to 64. The weights are differentiable in the
    logits."""
    nat.no_tangents("experts.route", logits)
    weights, chosen, offsets, rows, slots = _route(logits, k, renormalize)
    if _grad(logits):
        weights = _functions()[2].apply(logits, weights, chosen, bool(renormalize))
    return weights, chosen, Plan(offsets, rows, slots)


#: Layouts of route's logits: (arguments filled in but for their addresses, the workspace's bytes).
_ROUTE: dict = {}


def _check_route(logits, k):
    import torch  # noqa: PLC0415

    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32) or logits.dim() != 2:
        raise TypeError(f"experts.route: logits are bf16, fp16 or fp32 (T, E), got {logits.dtype} "
                        f"{tuple(logits.shape)}")
    t, e = logits.shape
    if not 1 <= e <= MAX_EXPERTS or not 1 <= k <= min(e, MAX_CHOSEN):
        raise ValueError(f"experts.route: {e} experts (1 to {MAX_EXPERTS}), k={k} (1 to {MAX_CHOSEN} and E)")
    if not logits.is_cuda:
        raise ValueError(f"experts.route: logits are on a GPU, got {logits.device}")
    nat.int32("experts.route", rows=t * k)


def _route(logits, k, renormalize):
    torch = _torch()
    key = (logits.shape, logits.stride(), logits.dtype, k, renormalize)
    known = _ROUTE.get(key)
    device = logits.device
    if known is None or logits.get_device() < 0:
        _check_route(logits, k)
        t, e = logits.shape
        if t == 0:
            known = None
        else:
            given, logits = logits, _unit(logits)
            g = nat.HkxExpertsRouteArgs()
            g.size, g.dtype, g.t, g.e, g.k = ctypes.sizeof(g), nat.dtype_code(logits.dtype), t, e, k
            g.renormalize, g.ld = int(bool(renormalize)), _ld(logits, e)
            known = (bytes(g), nat.lib().hkx_experts_route_workspace(ctypes.byref(g)))
            if logits is given:
                nat.remember(_ROUTE, key, known, 4096)
    t, e = logits.shape
    empty, int32 = nat.empty, torch.int32
    weights = empty(logits, (t, k), torch.float32)
    chosen, slots = empty(logits, (t, k), int32), empty(logits, (t, k), int32)
    offsets, rows = empty(logits, (e + 1,), int32), empty(logits, (t * k,), int32)
    if known is None:
        return weights, chosen, offsets.zero_(), rows, slots
    g = nat.HkxExpertsRouteArgs.from_buffer_copy(known[0])
    g.logits, g.weights, g.chosen = logits.data_ptr(), weights.data_ptr(), chosen.data_ptr()
    g.offsets, g.rows, g.slots = offsets.data_ptr(), rows.data_ptr(), slots.data_ptr()
    with nat.current(device):
        if known[1]:
            ws = nat.workspace(device, known[1])
            g.ws, g.ws_bytes = ws.data_ptr(), known[1]
        nat.check(nat.lib().hkx_experts_route(ctypes.byref(g), nat.stream_of(device)))
    return weights, chosen, offsets, rows, slots


def _route_backward(logits, weights, chosen, renormalize, dw):
    t, e = logits.shape
    dl = nat.empty(logits, (t, e), logits.dtype)
    if t == 0:
        return dl
    logits, dw = _unit(logits), dw.contiguous()
    with nat.current(logits.device):
        nat.check(nat.lib().hkx_experts_route_backward(
            logits.data_ptr(), _ld(logits, e), nat.dtype_code(logits.dtype), weights.data_ptr(), chosen.data_ptr(),
            dw.data_ptr(), dl.data_ptr(), e, t, e, weights.shape[1], int(renormalize), nat.stream_of(logits.device)))
    return dl


# ---------------------------------------------------------------- gradients


_FUNCTIONS: list = []


def _functions():
    """The autograd functions of gemm, combine and route, made at the first call that takes gradients."""
    if _FUNCTIONS:
        return _FUNCTIONS
    import torch  # noqa: PLC0415

    once = torch.autograd.function.once_differentiable

    class ExpertsGemm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w, bias, plan, gather, silu_mul):
            z = None
            if silu_mul:
                r = plan.rows.shape[0] if gather and plan.rows is not None else x.shape[0]
                z = nat.empty(x, (r, w.shape[1]), torch.bfloat16)
            y = _gemm(x, w, plan, gather, bias, silu_mul, None, None, None, z)
            ctx.save_for_backward(x, w, bias, z, *plan)
            ctx.gather = gather
            return y

        @staticmethod
        @once
        def backward(ctx, dy):
            x, w, bias, z, *plan = ctx.saved_tensors
            return (*_gemm_backward(x, w, bias, z, Plan(*plan), ctx.gather, ctx.needs_input_grad, dy),
                    None, None, None)

    class ExpertsCombine(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y, weights, slots):
            ctx.save_for_backward(y, weights, slots)
            return _combine(y, slots, weights)

        @staticmethod
        @once
        def backward(ctx, dout):
            y, weights, slots = ctx.saved_tensors
            return (*_combine_backward(y, weights, slots, ctx.needs_input_grad, dout), None)

    class ExpertsRoute(torch.autograd.Function):
        @staticmethod
        def forward(ctx, logits, weights, chosen, renormalize):  # (of weights made already)
            ctx.save_for_backward(logits, weights, chosen)
            ctx.renormalize = renormalize
            return weights.detach()

        @staticmethod
        @once
        def backward(ctx, dw):
            logits, weights, chosen = ctx.saved_tensors
            return _route_backward(logits, weights, chosen, ctx.renormalize, dw), None, None, None

    _FUNCTIONS[:] = [ExpertsGemm, ExpertsCombine, ExpertsRoute]
    return _FUNCTIONS


# ---------------------------------------------------------------- the layer


def mlp(x, logits, k, gate_up, down, *, gate_up_scale=None, down_scale=None, renormalize=True):
    """bf16 (T, D): each token's k experts' gated MLPs, weighted by its router's logits (T, E). x (T, K) bf16, gate_up
    (E, 2 I, K) and down (E, D, I) bf16; differentiable in x, logits and both. Or gate_up and down float8_e4m3fn with
    the scales of their rows ((E, 2 I) and (E, D)), and x bf16 or quantized already, (q, s) as
    hk.ops.block_norm(quant="fp8") gives it: each product's rows are quantized by hk.ops.fp8.quant."""
    if (gate_up_scale is None) != (down_scale is None) or (isinstance(x, tuple) and down_scale is None):
        raise TypeError("experts.mlp: 8-bit weights come with both scales, a quantized x with 8-bit weights")
    rows = x[0] if isinstance(x, tuple) else x
    if rows.shape[:1] != logits.shape[:1]:
        raise ValueError(f"experts.mlp: x has {tuple(rows.shape)}, logits {tuple(logits.shape)}: a row a token")
    weights, _, plan = route(logits, k, renormalize=renormalize)
    if gate_up_scale is None and down_scale is None:
        a = gemm(x, gate_up, plan, gather=True, silu_mul=True)
        return combine(gemm(a, down, plan), plan, weights)
    q, s = x if isinstance(x, tuple) else fp8.quant(x)
    a = gemm(q, gate_up, plan, gather=True, silu_mul=True, scale_a=s, scale_b=gate_up_scale)
    q, s = fp8.quant(a)
    return combine(gemm(q, down, plan, scale_a=s, scale_b=down_scale), plan, weights)


__all__ = ["Plan", "route", "gemm", "combine", "mlp"]
