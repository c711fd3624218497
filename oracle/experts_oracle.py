"""A layer of experts in 64 bits on the CPU: what hk.ops.experts and hk.ops.fp8 compute, written from their
definitions, a token and an expert at a time."""

import math

import torch


def route(logits, k, renormalize=True):
    """(weights float64 (T, k), chosen, offsets, rows, slots) of logits (T, E)."""
    t, e = logits.shape
    weights = torch.zeros(t, k, dtype=torch.float64)
    chosen = torch.full((t, k), -1, dtype=torch.int64)
    taken = [[] for _ in range(e)]
    for i, row in enumerate(logits.double().tolist()):
        order = sorted(range(e), key=lambda j: (-math.inf if math.isnan(row[j]) else -row[j], j))
        # (NaN above an infinity)
        order.sort(key=lambda j: not math.isnan(row[j]))
        picked = [j for j in order[:k] if row[j] != -math.inf]
        over = picked if renormalize else [j for j in range(e) if row[j] != -math.inf]
        if picked:
            v = torch.tensor([row[j] for j in over], dtype=torch.float64)
            top = row[picked[0]]
            total = torch.exp(v - top).sum()
            for n, j in enumerate(picked):
                chosen[i, n] = j
                weights[i, n] = math.nan if math.isnan(row[j] - top) else math.exp(row[j] - top)
                taken[j].append((i, n))
            weights[i, : len(picked)] /= total
    offsets, rows, slots = [0], [], torch.full((t, k), -1, dtype=torch.int64)
    for j in range(e):
        for i, n in taken[j]:
            slots[i, n] = len(rows)
            rows.append(i)
        offsets.append(len(rows))
    rows += [-1] * (t * k - len(rows))
    return weights, chosen, torch.tensor(offsets), torch.tensor(rows), slots


def gemm(x, w, offsets, rows=None, bias=None, silu_mul=False):
    """(y, z): the products in float64, in x's and w's own precision if it is wider; rows behind the last are 0."""
    off = offsets.tolist()
    r = x.shape[0] if rows is None else rows.numel()
    parts = []
    for e, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        xe = x[lo:hi] if rows is None else x[rows[lo:hi].long()]
        z = xe.double() @ w[e].double().t()
        parts.append(z if bias is None else z + bias[e].double())
    z = torch.cat([*parts, torch.zeros(r - off[-1], w.shape[1], dtype=torch.float64, device=w.device)])
    if not silu_mul:
        return z, z
    n = w.shape[1] // 2
    return torch.nn.functional.silu(z[:, :n]) * z[:, n:], z


def combine(y, slots, weights=None):
    # (0 times them: a result without rows has their gradients too)
    out = torch.zeros(slots.shape[0], y.shape[1], dtype=torch.float64) + 0.0 * y.double().sum()
    if weights is not None:
        out = out + 0.0 * weights.double().sum()
    for j in range(slots.shape[1]):
        for i in range(slots.shape[0]):
            s = int(slots[i, j])
            if s >= 0:
                out[i] = out[i] + y[s].double() * (1.0 if weights is None else weights[i, j].double())
    return out


def quant8(x):
    """(the codes' values float64, s float64) of rows x (M, K) in 8 bits: the nearest e4m3 value of x / s, a tie to the
    even code, with s in fp32 and the quotient rounded to fp32 first, as defined."""
    x = x.float()
    top = x.abs().amax(1, keepdim=True)
    s = torch.where(top > 0, (top / 448).clamp(min=2.0 ** -126), torch.ones_like(top))
    s = torch.where(torch.isfinite(x).all(1, keepdim=True), s, torch.full_like(s, math.nan))
    q = (x / s).double()
    q = torch.where(torch.isnan(s), torch.zeros_like(q), q)
    e = torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return (torch.round(q / step) * step).clamp(-448, 448), s.double()
