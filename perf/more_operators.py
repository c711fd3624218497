"""A layer of experts' operators, as cases that can be timed and compared.

    route    hk.ops.experts.route: a token's experts, their weights and the order of rows by expert; its gradient
    gemm     hk.ops.experts.gemm: the product of each expert's rows with its weight, bf16 or fp8
    train    the same, forward and backward
    combine  hk.ops.experts.combine: the experts' rows back to their tokens, weighted; its gradient
    norm     hk.ops.block_norm: residual add and norm, y as fp8 rows with a scale each

Where `own` is false `run` is the operators' plain form in elementary torch operations: the experts' rows
are laid out in a padded batch, one product a batch, in fp32.
"""

import math
import sys
from pathlib import Path

import torch

own = False

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": BF16, "fp16": F16, "fp32": F32}
EPS = 1e-6


def listed():
    return [
        # a decode batch of 16 tokens routed: the smallest call, latency alone
        dict(name="route_decode_16", kind="route", t=16, e=64, k=8, dtype="fp32", norm=True, train=False, pad=0),
        # a training batch routed, with the logits' gradient; a padded tail has no experts
        dict(name="route_train_16384", kind="route", t=16384, e=128, k=8, dtype="bf16", norm=True, train=True,
             pad=500),
        # one token's gate and up projections: eight experts' weights are the time
        dict(name="gemm_decode_1", kind="gemm", t=1, e=64, k=8, n=2048, d=2048, dtype="bf16", gather=True,
             silu_mul=True, bias=False, quant=False, pad=0),
        # a decode batch of 64 through 8-bit down projections, the activations' rows quantized on the way
        dict(name="gemm_decode_64_fp8", kind="gemm", t=64, e=64, k=8, n=2048, d=1024, dtype="fp8", gather=False,
             silu_mul=False, bias=False, quant=True, pad=0),
        # a prefill chunk of odd length, some 256 rows an expert: 8-bit gate and up projections
        dict(name="gemm_chunk_2047_fp8", kind="gemm", t=2047, e=64, k=8, n=2048, d=4096, dtype="fp8", gather=True,
             silu_mul=True, bias=False, quant=False, pad=0),
        # a long prefill through few large experts: the largest product
        dict(name="gemm_prefill_4096", kind="gemm", t=4096, e=8, k=2, n=14336, d=4096, dtype="bf16", gather=True,
             silu_mul=True, bias=False, quant=False, pad=0),
        # a training step's gate and up projections, forward and backward
        dict(name="train_4096", kind="train", t=4096, e=8, k=2, n=8192, d=2048, gather=True, silu_mul=True,
             bias=False, pad=0),
        # odd sizes with a bias, sorted rows, a padded tail
        dict(name="train_odd_333", kind="train", t=333, e=5, k=2, n=904, d=1112, gather=False, silu_mul=False,
             bias=True, pad=30),
        # a decode batch's rows back to its tokens
        dict(name="combine_decode_16", kind="combine", t=16, e=64, k=8, d=2048, dtype="bf16", train=False, pad=0),
        # a training batch's, forward and backward
        dict(name="combine_train_8192", kind="combine", t=8192, e=64, k=4, d=4096, dtype="bf16", train=True, pad=100),
        # before the experts at a decode batch of 16
        dict(name="norm_decode_16", kind="norm", rows=16, d=4096, dtype="bf16", rdtype="bf16"),
        # before the experts over a prefill, with an fp32 residual stream
        dict(name="norm_prefill_8192", kind="norm", rows=8192, d=4096, dtype="bf16", rdtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["route", "gemm", "gemm", "train", "combine", "norm"])
    if kind == "norm":
        d = _log(rng, 64, 8192)
        dtype, rdtype = rng.choice([("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"), ("fp32", "fp32")])
        return dict(kind=kind, rows=_log(rng, 1, min(16384, (1 << 25) // d)), d=d, dtype=dtype, rdtype=rdtype)
    e = _log(rng, 2, 256)
    k = rng.randint(1, min(8, e))
    if kind == "route":
        t = _log(rng, 1, 16384)
        return dict(kind=kind, t=t, e=e, k=k, dtype=rng.choice(list(DTYPES)), norm=rng.random() < 0.7,
                    train=rng.random() < 0.5, pad=rng.choice([0, t // 10]))
    if kind == "combine":
        d = _log(rng, 64, 8192)
        t = _log(rng, 1, min(8192, (1 << 26) // (d * k)))
        return dict(kind=kind, t=t, e=e, k=k, d=d, dtype=rng.choice(list(DTYPES)), train=rng.random() < 0.5,
                    pad=rng.choice([0, t // 10]))
    dtype = "bf16" if kind == "train" else rng.choice(["bf16", "fp8"])
    n = 16 * _log(rng, 4, 512)
    d = (16 if dtype == "fp8" else 8) * _log(rng, 8, 256)
    # weights to 2^28 values (half as many in training), and products within the largest listed one's
    e = max(2, min(e, (1 << (27 if kind == "train" else 28)) // (n * d)))
    k = min(k, e)
    t = _log(rng, 1 if kind == "gemm" else 16, min(8192, (1 << 38) // (n * d * k) if kind == "gemm" else (1 << 36) // (n * d * k)))
    case = dict(kind=kind, t=t, e=e, k=k, n=n, d=d, gather=rng.random() < 0.5, silu_mul=rng.random() < 0.5,
                bias=rng.random() < 0.3, pad=rng.choice([0, t // 10]))
    if kind == "train":
        return case
    return dict(case, dtype=dtype, quant=dtype == "fp8" and rng.random() < 0.5)


# ------------------------------------------------------------------ the operators' plain forms


def _plain_route(logits, k, norm):
    """(weights, experts, offsets, rows, slots, the softmax)."""
    v = logits.float()
    t, e = v.shape
    top = torch.sort(v, dim=1, descending=True, stable=True)
    chosen, value = top.indices[:, :k], top.values[:, :k]
    live = value > -math.inf
    p = torch.exp(v - v.amax(1, keepdim=True).clamp(min=torch.finfo(F32).min))
    p = p / p.sum(1, keepdim=True).clamp(min=torch.finfo(F32).tiny)
    w = torch.gather(p, 1, chosen)
    if norm:
        # (of the chosen logits alone: the ratio of two small p would lose bits)
        w = torch.exp(value - value[:, :1].clamp(min=torch.finfo(F32).min))
        w = w / w.sum(1, keepdim=True).clamp(min=torch.finfo(F32).tiny)
    of = torch.where(live, chosen, e).flatten()
    order = torch.sort(of, stable=True)
    offsets = torch.cat((of.new_zeros(1), torch.bincount(of, minlength=e + 1)[:e].cumsum(0)))
    rows = torch.where(order.values < e, order.indices // k, -1)
    slots = torch.empty_like(of)
    slots[order.indices] = torch.arange(t * k, device=v.device)
    slots = torch.where(of < e, slots, -1).reshape(t, k)
    return w, torch.where(live, chosen, -1).int(), offsets.int(), rows.int(), slots.int(), p


def _plain_route_grad(w, experts, p, dw, norm):
    """The gradient of the logits from dw, that of the weights."""
    if norm:
        g, at = w * (dw - (w * dw).sum(1, keepdim=True)), experts
        return torch.zeros_like(p).scatter_add(1, at.long().clamp(min=0), torch.where(at >= 0, g, 0.0))
    live = torch.where(experts >= 0, dw, 0.0)
    g = torch.zeros_like(p).scatter_add(1, experts.long().clamp(min=0), live)
    return p * (g - (w * live).sum(1, keepdim=True))


def _padded(offsets, count):
    """Of each of `count` rows: whether it has an expert, its expert, its place among the expert's rows; and
    the largest expert's rows."""
    at = torch.arange(count, device=offsets.device)
    off = offsets.long()
    e = torch.bucketize(at, off[1:], right=True)
    live = e < off.numel() - 1
    e = torch.where(live, e, 0)
    return live, e, torch.where(live, at - off[e], 0), max(1, int((off[1:] - off[:-1]).max()))


def _batch(v, pad, experts):
    """Rows (R, D) as a batch (E, rows, D) with zeros behind an expert's last."""
    live, e, at, cap = pad
    out = v.new_zeros(experts, cap, v.shape[1])
    out[e[live], at[live]] = v[live]
    return out


def _unbatch(b, pad):
    live, e, at, _ = pad
    return torch.where(live.unsqueeze(1), b[e, at], 0.0)


def _plain_e4m3(v):
    """(values, scales) of fp32 rows in 8 bits: v / s to e4m3, s the largest of a row over 448."""
    s = v.abs().amax(-1, keepdim=True) / 448
    s = torch.where(s > 0, s, 1.0)
    return (v / s).clamp(-448, 448).to(E4M3).float(), s


def _plain_forward(st):
    """(z before silu_mul, the product's rows, the rows x in expert order, the padded layout)."""
    x, w, plan = st["x"].float(), st["w"].float(), st["plan"]
    if st["quant"]:
        q, s = _plain_e4m3(x)
        x = q * s
    elif st["scale_a"] is not None:
        x = x * st["scale_a"]
    if st["scale_b"] is not None:
        w = w * st["scale_b"].unsqueeze(2)
    if st["gather"]:
        x = x[plan[1].long().clamp(min=0)]
    pad = _padded(plan[0], plan[1].numel())
    z = torch.bmm(_batch(x, pad, w.shape[0]), w.transpose(1, 2).contiguous())
    if st["bias"] is not None:
        z = z + st["bias"].float().unsqueeze(1)
    z = _unbatch(z, pad)
    if not st["silu_mul"]:
        return z, z, x, pad
    g, u = z.chunk(2, dim=1)
    return z, g / (1.0 + torch.exp(-g)) * u, x, pad


def _plain_train(st):
    z, y, x, pad = _plain_forward(st)
    dz = st["dy"].float()
    if st["silu_mul"]:
        g, u = z.chunk(2, dim=1)
        s = 1.0 / (1.0 + torch.exp(-g))
        dz = torch.cat((dz * u * s * (1.0 + g * (1.0 - s)), dz * g * s), dim=1)
    w = st["w"].float()
    dzb = _batch(dz, pad, w.shape[0])
    dx = _unbatch(torch.bmm(dzb, w), pad)
    if st["gather"]:
        slots = st["plan"][2].long()
        dx = torch.where((slots >= 0).unsqueeze(2), dx[slots.clamp(min=0)], 0.0).sum(1)
    dw = torch.bmm(dzb.transpose(1, 2).contiguous(), _batch(x, pad, w.shape[0]))
    out = {"y": y.to(BF16), "dx": dx.to(BF16), "dw": dw.to(BF16)}
    if st["bias"] is not None:
        out["dbias"] = dzb.sum(1).to(BF16)
    return out


def _plain_combine(st):
    slots = st["plan"][2].long()
    live, at = slots >= 0, slots.clamp(min=0)
    y = st["y"].float()
    rows = torch.where(live.unsqueeze(2), y[at], 0.0)
    w = torch.where(live, st["weights"], 0.0)
    out = {"out": (w.unsqueeze(2) * rows).sum(1).to(st["y"].dtype)}
    if st["train"]:
        do = st["dout"].float()
        dy = torch.zeros_like(y)
        dy[slots[live]] = (w.unsqueeze(2) * do.unsqueeze(1))[live]
        out["dy"] = dy.to(st["y"].dtype)
        out["dweights"] = torch.where(live, (rows * do.unsqueeze(1)).sum(2), 0.0)
    return out


def _plain_norm(st):
    h = st["residual"].float() + st["x"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * st["pre"].float()
    q, s = _plain_e4m3(y)
    return {"h": h.to(st["residual"].dtype), "y": (q * s).to(BF16), "scale": s}


# ------------------------------------------------------------------ the cases


def _randn(gen, *shape, dtype=F32, std=1.0, mean=0.0):
    t = torch.randn(*shape, generator=gen, device="cuda")
    return (t * std + mean).to(dtype)


def _logits(gen, case):
    """Router logits with favoured experts (their loads are ragged); a padded tail is -inf."""
    v = _randn(gen, case["t"], case["e"]) + _randn(gen, case["e"], std=0.5)
    v[case["t"] - case["pad"]:] = -math.inf
    return v


def _e4m3_rows(x):
    s = x.abs().amax(-1, keepdim=True).clamp(min=1e-6) / 448
    return (x / s).clamp(-448, 448).to(E4M3), s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "norm":
        rows, d = case["rows"], case["d"]
        return dict(kind=kind, x=_randn(gen, rows, d, dtype=DTYPES[case["dtype"]]),
                    residual=_randn(gen, rows, d, dtype=DTYPES[case["rdtype"]], std=2.0),
                    pre=_randn(gen, d, dtype=DTYPES[case["dtype"]], std=0.1, mean=1.0))
    logits = _logits(gen, case)
    if kind == "route":
        return dict(kind=kind, logits=logits.to(DTYPES[case["dtype"]]), k=case["k"], norm=case["norm"],
                    dw=_randn(gen, case["t"], case["k"]) if case["train"] else None)
    weights, _, *plan = _plain_route(logits, case["k"], True)[:5]
    r = case["t"] * case["k"]
    if kind == "combine":
        dt = DTYPES[case["dtype"]]
        return dict(kind=kind, plan=plan, weights=weights, y=_randn(gen, r, case["d"], dtype=dt),
                    train=case["train"], dout=_randn(gen, case["t"], case["d"], dtype=dt) if case["train"] else None)
    n, d = case["n"], case["d"]
    wide = case.get("dtype") != "fp8"
    st = dict(kind=kind, plan=plan, gather=case["gather"], silu_mul=case["silu_mul"], quant=case.get("quant", False),
              scale_a=None, scale_b=None,
              bias=_randn(gen, case["e"], n, dtype=BF16, std=0.1) if case["bias"] else None)
    x = _randn(gen, case["t"] if case["gather"] else r, d)
    w = _randn(gen, case["e"], n, d, std=d ** -0.5)
    if wide:
        st["x"], st["w"] = x.to(BF16), w.to(BF16)
    else:
        st["w"], s = _e4m3_rows(w)
        st["scale_b"] = s.squeeze(2)
        if st["quant"]:
            st["x"] = x.to(BF16)
        else:
            st["x"], st["scale_a"] = _e4m3_rows(x)
    if kind == "train":
        st["dy"] = _randn(gen, r, n // 2 if case["silu_mul"] else n, dtype=BF16)
    return st


def _package():
    path = str(Path(__file__).resolve().parents[1] / "hk-dsl_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import hk  # noqa: PLC0415

    return hk.ops


def _own(st):
    ops = _package()
    experts, kind = ops.experts, st["kind"]
    if kind == "norm":
        h, (q, s) = ops.block_norm(st["x"], st["residual"], pre=st["pre"], eps=EPS, quant="fp8")
        return {"h": h, "y": (q.float() * s).to(BF16), "scale": s}
    if kind == "route":
        logits, dw = st["logits"], st["dw"]
        if dw is not None:
            logits = logits.detach().requires_grad_()
        weights, chosen, plan = experts.route(logits, st["k"], renormalize=st["norm"])
        out = {"weights": weights.detach(), "experts": chosen, "offsets": plan.offsets, "rows": plan.rows,
               "slots": plan.slots}
        if dw is not None:
            out["dlogits"] = torch.autograd.grad(weights, logits, dw)[0]
        return out
    plan = experts.Plan(*st["plan"])
    if kind == "combine":
        if not st["train"]:
            return {"out": experts.combine(st["y"], plan, st["weights"])}
        y, w = st["y"].detach().requires_grad_(), st["weights"].detach().requires_grad_()
        out = experts.combine(y, plan, w)
        dy, dw = torch.autograd.grad(out, (y, w), st["dout"])
        return {"out": out.detach(), "dy": dy, "dweights": dw}
    args = dict(gather=st["gather"], silu_mul=st["silu_mul"])
    if kind == "gemm":
        x, sa = ops.fp8.quant(st["x"]) if st["quant"] else (st["x"], st["scale_a"])
        return experts.gemm(x, st["w"], plan, bias=st["bias"], scale_a=sa, scale_b=st["scale_b"], **args)
    leaf = {n: st[n].detach().requires_grad_() for n in ("x", "w", "bias") if st[n] is not None}
    y = experts.gemm(leaf["x"], leaf["w"], plan, bias=leaf.get("bias"), **args)
    grads = torch.autograd.grad(y, list(leaf.values()), st["dy"])
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(leaf, grads)}}


def run(state):
    if own:
        return _own(state)
    kind = state["kind"]
    if kind == "route":
        weights, chosen, offsets, rows, slots, p = _plain_route(state["logits"], state["k"], state["norm"])
        out = {"weights": weights, "experts": chosen, "offsets": offsets, "rows": rows, "slots": slots}
        if state["dw"] is not None:
            g = _plain_route_grad(weights, chosen, p, state["dw"], state["norm"])
            out["dlogits"] = g.to(state["logits"].dtype)
        return out
    if kind == "gemm":
        return _plain_forward(state)[1].to(BF16)
    if kind == "train":
        return _plain_train(state)
    return _plain_combine(state) if kind == "combine" else _plain_norm(state)


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["d"]
        return {"bytes": n * (size[case["dtype"]] + 2 * size[case["rdtype"]] + 1) + 4 * case["rows"]
                + case["d"] * size[case["dtype"]], "flops": 8 * n}
    t, e, k = case["t"], case["e"], case["k"]
    r = t * k
    if kind == "route":
        n = t * e
        # the logits once; weights, experts, rows and slots; the logits' gradient from the weights'
        return {"bytes": n * size[case["dtype"]] * (2 if case["train"] else 1) + r * (20 if case["train"] else 16)
                + 4 * (e + 1), "flops": n * (k + 4)}
    if kind == "combine":
        b = size[case["dtype"]]
        n, m = r * case["d"], t * case["d"]
        if not case["train"]:
            return {"bytes": b * (n + m) + 8 * r, "flops": 2 * n}
        return {"bytes": b * (2 * n + 2 * m) + 12 * r, "flops": 5 * n}
    n, d = case["n"], case["d"]
    # the experts that some row goes to
    touched = e * (1 - (1 - k / e) ** t)
    b = 1 if case.get("dtype") == "fp8" else 2
    x = (t if case["gather"] else r) * d * (2 if case.get("quant") else b)
    w = touched * n * (d * b + (2 if case["bias"] else 0) + (4 if b == 1 else 0))
    y = 2 * r * (n // 2 if case["silu_mul"] else n)
    if kind == "gemm":
        return {"bytes": x + w + y + 4 * r, "flops": 2 * r * n * d}
    # both directions, each operand and gradient once
    return {"bytes": 2 * (x + w + y) + 8 * r, "flops": 6 * r * n * d}


# ------------------------------------------------------------------ in 64 bits


E4M3_GRID = tuple(m * 2.0 ** -9 for m in range(8)) + tuple(
    (8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8) if (8 + m) * 2.0 ** (e - 3) < 449)


def _exact_rows8(v):
    """(values, scales): the nearest of the grid, a tie to the even one."""
    s = v.abs().amax(-1, keepdim=True) / 448
    s = torch.where(s == 0, torch.ones_like(s), s)
    g = torch.tensor(E4M3_GRID, dtype=torch.float64, device=v.device)
    t = (v.abs() / s).clamp(max=448.0)
    hi = torch.searchsorted(g, t.contiguous()).clamp(1, len(E4M3_GRID) - 1)
    below, above = t - g[hi - 1], g[hi] - t
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return torch.where(up, g[hi], g[hi - 1]) * torch.sign(v), s


def _exact_route(st):
    l = st["logits"].double()
    if st["dw"] is not None:
        l.requires_grad_()
    t, e = l.shape
    k = st["k"]
    host = l.detach().cpu()
    # the largest k, a tie to the lower index: by (-logit, index)
    import numpy as np  # noqa: PLC0415

    v = host.numpy()
    order = np.lexsort((np.broadcast_to(np.arange(e), (t, e)), -v), axis=1)[:, :k]
    picked = np.take_along_axis(v, order, 1)
    chosen = np.where(np.isneginf(picked), -1, order)
    flat = chosen.reshape(-1)
    by = np.argsort(np.where(flat < 0, e, flat), kind="stable")
    live = int((flat >= 0).sum())
    rows = np.full(t * k, -1)
    rows[:live] = by[:live] // k
    slots = np.full(t * k, -1)
    slots[by[:live]] = np.arange(live)
    offsets = np.searchsorted(np.sort(flat[flat >= 0]), np.arange(e + 1))
    c = torch.from_numpy(chosen).to(l.device)
    dead = torch.isneginf(l).all(1, keepdim=True)
    p = torch.softmax(torch.where(dead, torch.zeros_like(l), l), dim=1)
    w = torch.where(c >= 0, torch.gather(p, 1, c.clamp(min=0)), torch.zeros((), dtype=torch.float64, device=l.device))
    if st["norm"]:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    out = {"weights": w.detach(), "experts": c, "offsets": torch.from_numpy(offsets).to(l.device),
           "rows": torch.from_numpy(rows).to(l.device), "slots": torch.from_numpy(slots).to(l.device).reshape(t, k)}
    if st["dw"] is not None:
        out["dlogits"] = torch.autograd.grad(w, l, st["dw"].double())[0]
    return out


def _exact_gemm(st):
    x, w = st["x"].double(), st["w"].double()
    if st["quant"]:
        q, s = _exact_rows8(x)
        x = q * s
    if st["scale_a"] is not None:
        x = x * st["scale_a"].double()
    if st["scale_b"] is not None:
        w = w * st["scale_b"].double()[:, :, None]
    names = {"x": x, "w": w}
    if st["bias"] is not None:
        names["bias"] = st["bias"].double()
    train = st["kind"] == "train"
    if train:
        for v in names.values():
            v.requires_grad_()
    off, rows = st["plan"][0].tolist(), st["plan"][1].long()
    parts = []
    for e, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        if lo == hi:
            continue
        xe = names["x"][rows[lo:hi]] if st["gather"] else names["x"][lo:hi]
        z = xe @ names["w"][e].t()
        if "bias" in names:
            z = z + names["bias"][e]
        if st["silu_mul"]:
            half = z.shape[1] // 2
            z = torch.sigmoid(z[:, :half]) * z[:, :half] * z[:, half:]
        parts.append(z)
    width = w.shape[1] // 2 if st["silu_mul"] else w.shape[1]
    parts.append(torch.zeros(rows.numel() - off[-1], width, dtype=torch.float64, device=w.device))
    y = torch.cat(parts)
    if not train:
        return y
    grads = torch.autograd.grad(y, list(names.values()), st["dy"].double())
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _exact_combine(st):
    slots = st["plan"][2].long()
    y, w = st["y"].double(), st["weights"].double()
    out = torch.zeros(slots.shape[0], y.shape[1], dtype=torch.float64, device=y.device)
    dy, dw = torch.zeros_like(y), torch.zeros_like(w)
    for j in range(slots.shape[1]):
        live = slots[:, j] >= 0
        at = slots[live, j]
        out[live] += w[live, j, None] * y[at]
        if st["train"]:
            do = st["dout"].double()[live]
            dy[at] = w[live, j, None] * do
            dw[live, j] = (do * y[at]).sum(1)
    return {"out": out, "dy": dy, "dweights": dw} if st["train"] else {"out": out}


def exact(case, seed):
    st = prepare(case, seed)
    if st["kind"] == "route":
        return _exact_route(st)
    if st["kind"] == "combine":
        return _exact_combine(st)
    if st["kind"] != "norm":
        return _exact_gemm(st)
    h = st["residual"].double() + st["x"].double()
    q, s = _exact_rows8(h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * st["pre"].double())
    return {"h": h, "y": q * s, "scale": s}
