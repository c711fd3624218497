"""The MXFP4 path in 64 bits on the CPU: what hk.ops.mxfp4, hk.ops.mxfp8.dequant and
hk.ops.block_norm compute, written from their definitions."""

import torch

FP4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def fp4_codes(v):
    """e2m1 codes of float64 v, |v| <= 6: the nearest value, a tie to the even code."""
    dist = (v.abs().unsqueeze(-1) - FP4).abs()
    best = dist.min(-1, keepdim=True).values
    near = dist == best  # one value, or two neighbours at a tie
    even = near & (torch.arange(8) % 2 == 0)
    pick = torch.where(near.sum(-1, keepdim=True) > 1, even, near)
    return pick.to(torch.uint8).argmax(-1).to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)


def quant(x):
    """(codes (M, K) uint8, scale bytes (M, K/32)) of x (M, K)."""
    m, k = x.shape
    v = x.double().reshape(m, k // 32, 32)
    bad = ~torch.isfinite(v).all(-1)
    v = torch.where(bad.unsqueeze(-1), torch.zeros_like(v), v)
    amax = v.abs().amax(-1)
    f, ex = torch.frexp(amax)  # amax = f 2^ex, f in [0.5, 1): amax / 6 = (f / 0.75) 2^(ex - 3)
    e = ex - 3 + (f > 0.75).to(ex.dtype)
    e = torch.where(amax == 0, torch.full_like(e, -127), e.clamp(min=-127))
    codes = fp4_codes(torch.ldexp(v, -e.unsqueeze(-1)))
    codes = torch.where(bad.unsqueeze(-1), torch.zeros_like(codes), codes)
    return codes.reshape(m, k), torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def pack(codes):
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(q):
    out = torch.empty(q.shape[0], 2 * q.shape[1], dtype=torch.uint8)
    out[:, 0::2], out[:, 1::2] = q & 15, q >> 4
    return out


def values(q, s):
    """The float64 numbers of packed codes (uint8) or e4m3 q with E8M0 bytes s."""
    if q.dtype == torch.uint8:
        c = unpack(q)
        v = FP4[(c & 7).long()] * torch.where(c > 7, -1.0, 1.0).double()
    else:
        v = q.double()
    scale = torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s.int() - 127)
    scale = torch.where(s == 255, torch.full_like(scale, float("nan")), scale)
    return v * scale.repeat_interleave(32, dim=1)


def gemm(a, b, sa, sb, bias=None, silu_mul=False):
    """(C, a bound of |kernel - C|) in float64.

    The bound: C's rounding to bf16 (2^-9 of it; twice that here), fp32 sums over K products in any
    order (K 2^-24 of the sum of their magnitudes) and the scaled MFMA's alignment of the products of
    one instruction (under 2^-12 of that sum); through silu(g) u by its derivatives, |silu'| < 1.1, with
    2^-18 for its exponential and reciprocal."""
    av, bv = values(a, sa), values(b, sb)
    z = av @ bv.t()
    k = av.shape[1]
    err = (2.0 ** -12 + k * 2.0 ** -24) * (av.abs() @ bv.abs().t()) + 1e-30
    if bias is not None:
        z = z + bias.double()
        err = err + 2.0 ** -23 * z.abs()
    if silu_mul:
        n = z.shape[1] // 2
        g, u = z[:, :n], z[:, n:]
        eg, eu = err[:, :n], err[:, n:]
        act = g * torch.sigmoid(g)
        z = act * u
        err = 1.1 * eg * (u.abs() + eu) + act.abs() * eu + 2.0 ** -18 * z.abs()
    return z, err + 2.0 ** -8 * z.abs()


def block_norm(x, residual, post=None, pre=None, gate=None, branch_scale=1.0, residual_scale=1.0,
               eps=1e-6):
    """(h, y) in float64, differentiable."""
    def norm(v):
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)

    x, residual = x.double(), residual.double()
    u = x if post is None else norm(x) * post.double()
    if gate is not None:
        u = u * gate.double()
    h = residual_scale * residual + branch_scale * u
    return h, None if pre is None else norm(h) * pre.double()


def quant8(y):
    """MXFP8's numbers of float64 y (..., D), D a multiple of 32: e4m3 under 2^ceil(log2(amax / 448))."""
    v = y.reshape(-1, 32)
    f, ex = torch.frexp(v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -126))
    e = ex - 9 + (f > 0.875).to(ex.dtype)
    return torch.ldexp(torch.ldexp(v, -e).float().to(torch.float8_e4m3fn).double(), e).reshape(y.shape)
