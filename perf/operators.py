"""The MXFP4 linear path's operators, as cases that can be timed and compared.

    quant   hk.ops.mxfp4.quant: rows to 4-bit values and E8M0 scales, given back as numbers
    gemm    hk.ops.mxfp4.gemm: 4-bit weights, 4- or 8-bit activations, bias, silu(gate) * up
    norm    hk.ops.block_norm: post-norm, gated and scaled residual add, pre-norm
    train   the same, forward and backward

Where `own` is false `run` is the operators' plain form in elementary torch operations.
"""

import math
import sys
from pathlib import Path

import torch

own = False

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DTYPES = {"bf16": BF16, "fp16": F16, "fp32": F32}
EPS = 1e-6


def listed():
    return [
        # a decode batch's activations quantized: the smallest call, latency alone
        dict(name="quant_decode_16", kind="quant", m=16, k=4096, dtype="bf16"),
        # an fp32 master weight quantized once for serving
        dict(name="quant_weight_fp32", kind="quant", m=12288, k=4096, dtype="fp32"),
        # one token through an up projection with bias: the weight's bytes are the time
        dict(name="gemm_decode_1", kind="gemm", m=1, n=12288, k=4096, a="fp8", bias=True,
             silu_mul=False),
        # a decode batch of 16 through a merged gate and up projection
        dict(name="gemm_gate_up_decode_16", kind="gemm", m=16, n=24576, k=4096, a="fp8",
             bias=False, silu_mul=True),
        # a short ragged batch and odd sizes: K ends inside every tile, N too
        dict(name="gemm_ragged_37", kind="gemm", m=37, n=1001, k=2976, a="fp8", bias=True,
             silu_mul=False),
        # a prefill chunk of odd length through a down projection, both sides 4 bit
        dict(name="gemm_chunk_777", kind="gemm", m=777, n=4096, k=12288, a="fp4", bias=False,
             silu_mul=False),
        # a long prefill through the up projection, both sides 4 bit: the largest product
        dict(name="gemm_prefill_4096", kind="gemm", m=4096, n=12288, k=4096, a="fp4", bias=True,
             silu_mul=False),
        # a prefill chunk through the merged gate and up projection, 8-bit activations
        dict(name="gemm_gate_up_2048", kind="gemm", m=2048, n=24576, k=4096, a="fp8",
             bias=False, silu_mul=True),
        # between two blocks at a decode batch of 16, a layer scale as the gate
        dict(name="norm_decode_16", kind="norm", b=16, s=1, d=4096, dtype="bf16", rdtype="bf16",
             gate="channel", quant="none"),
        # the same over a prefill with an fp32 residual stream, y stored for an MX product
        dict(name="norm_prefill_mxfp8", kind="norm", b=2, s=2048, d=4096, dtype="bf16",
             rdtype="fp32", gate="none", quant="mxfp8"),
        # a training step's batch, forward and backward, a gate a sequence
        dict(name="train_4x2048", kind="train", b=4, s=2048, d=4096, dtype="bf16",
             rdtype="bf16", wdtype="fp32", gate="sequence"),
        # odd sizes in fp32, a gate a token
        dict(name="train_odd_fp32", kind="train", b=3, s=333, d=1111, dtype="fp32",
             rdtype="fp32", wdtype="fp32", gate="token"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "gemm", "gemm", "norm", "train"])
    if kind == "quant":
        k = 32 * _log(rng, 1, 448)
        return dict(kind=kind, m=_log(rng, 1, min(16384, (1 << 26) // k)), k=k,
                    dtype=rng.choice(list(DTYPES)))
    if kind == "gemm":
        silu_mul = rng.random() < 0.3
        n = _log(rng, 16, 24576)
        k = 32 * _log(rng, 1, 448)
        k = min(k, 32 * ((1 << 27) // (32 * n)))
        return dict(kind=kind, m=_log(rng, 1, 4096), n=n + (n % 2 if silu_mul else 0), k=k,
                    a=rng.choice(["fp4", "fp8"]), bias=rng.random() < 0.5, silu_mul=silu_mul)
    d = _log(rng, 64, 8192)
    tokens = _log(rng, 1 if kind == "norm" else 64, (1 << 25) // d if d > 4096 else 8192)
    b = rng.choice([1, 1, 2, 3, 4, 8])
    dtype, rdtype = rng.choice([("bf16", "bf16"), ("bf16", "fp32"), ("fp16", "fp16"),
                                ("fp16", "fp32"), ("fp32", "fp32")])
    case = dict(kind=kind, b=b, s=max(1, tokens // b), d=d, dtype=dtype, rdtype=rdtype,
                gate=rng.choice(["none", "channel", "sequence", "token", "full"]))
    if kind == "train":
        return dict(case, wdtype=rng.choice([dtype, "fp32"]))
    if rng.random() < 0.3:
        return dict(case, d=max(64, d // 32 * 32), quant="mxfp8")
    return dict(case, quant="none")


# ------------------------------------------------------------------ the operators' plain forms


def _plain_fp4(v):
    """|v| <= 6 to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6, ties to the even one's code."""
    t = v.abs()
    r = 0.5 * ((t > 0.25).float() + (t >= 0.75).float() + (t > 1.25).float()
               + (t >= 1.75).float())
    r = r + (t > 2.5).float() + (t >= 3.5).float() + 2.0 * (t > 5.0).float()
    return torch.copysign(r, v)


def _plain_quant4(x):
    """(values with their scale taken out, exponents) of x's blocks of 32, in fp32."""
    v = x.float().reshape(*x.shape[:-1], -1, 32)
    f, ex = torch.frexp(v.abs().amax(-1, keepdim=True))
    e = ex - 3 + (f > 0.75).int()
    e = torch.where(f == 0, torch.full_like(e, -127), e.clamp(min=-127))
    return _plain_fp4(torch.ldexp(torch.ldexp(v, -(e // 2)), -(e - e // 2))), e


def _scaled(v, e):
    """v 2^e in fp32 in two exact steps (2^e alone may leave fp32's normal range)."""
    return torch.ldexp(torch.ldexp(v, e // 2), e - e // 2).flatten(-2)


def _plain_quant8(y):
    """MXFP8's values of fp32 y, as numbers: e4m3 under e = ceil(log2(amax / 448))."""
    v = y.reshape(*y.shape[:-1], -1, 32)
    f, ex = torch.frexp(v.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -126))
    e = ex - 9 + (f > 0.875).int()
    q = torch.ldexp(torch.ldexp(v, -(e // 2)), -(e - e // 2)).clamp(-448, 448)
    return _scaled(q.to(torch.float8_e4m3fn).float(), e)


def _plain_operand(q, s):
    """Packed 4-bit or e4m3 rows and their E8M0 bytes, as fp32 numbers."""
    if q.dtype == torch.uint8:
        c = torch.stack((q & 15, q >> 4), -1).flatten(-2).to(torch.int32)
        mag = c & 7
        v = torch.where(mag < 2, 0.5 * mag.float(),
                        torch.ldexp(1.0 + 0.5 * (mag & 1).float(), (mag >> 1) - 1))
        v = torch.where(c > 7, -v, v)
    else:
        v = q.float()
    return _scaled(v.reshape(v.shape[0], -1, 32), s.int().unsqueeze(-1) - 127)


def _plain_gemm(st):
    z = _plain_operand(st["a"], st["sa"]) @ _plain_operand(st["w"], st["sw"]).t()
    if st["bias"] is not None:
        z = z + st["bias"].float()
    if st["silu_mul"]:
        g, u = z.chunk(2, dim=1)
        z = g / (1.0 + torch.exp(-g)) * u
    return z.to(BF16)


def _rms(v):
    r = torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)
    return v * r, r


def _plain_forward(st):
    xh, rx = _rms(st["x"].float())
    u = xh * st["post"].float()
    g = st["gate"].float() if st["gate"] is not None else 1.0
    h = st["residual_scale"] * st["residual"].float() + st["branch_scale"] * g * u
    hh, rh = _rms(h)
    return xh, rx, u, g, h, hh, rh, hh * st["pre"].float()


def _plain_norm(st):
    h, y = (t for i, t in enumerate(_plain_forward(st)) if i in (4, 7))
    y = _plain_quant8(y).to(BF16) if st["quant"] else y.to(st["x"].dtype)
    return {"h": h.to(st["residual"].dtype), "y": y}


def _plain_train(st):
    xh, rx, u, g, h, hh, rh, y = _plain_forward(st)
    dy = st["dy"].float()
    t = dy * st["pre"].float()
    dh = st["dh"].float() + rh * (t - hh * (t * hh).mean(-1, keepdim=True))
    du = st["branch_scale"] * g * dh
    t = du * st["post"].float()
    dx = rx * (t - xh * (t * xh).mean(-1, keepdim=True))
    out = {"h": h.to(st["residual"].dtype), "y": y.to(st["x"].dtype),
           "dx": dx.to(st["x"].dtype),
           "dresidual": (st["residual_scale"] * dh).to(st["residual"].dtype),
           "dpost": (du * xh).sum((0, 1)).to(st["post"].dtype),
           "dpre": (dy * hh).sum((0, 1)).to(st["pre"].dtype)}
    if st["gate"] is not None:
        dg = st["branch_scale"] * dh * u
        out["dgate"] = dg.sum_to_size(st["gate"].shape).to(st["gate"].dtype)
    return out


# ------------------------------------------------------------------ the cases


def _randn(gen, *shape, dtype=F32, std=1.0, mean=0.0):
    t = torch.randn(*shape, generator=gen, device="cuda")
    return (t * std + mean).to(dtype)


def _packed(x):
    """x's rows as packed 4-bit codes (the even column in the low bits) and E8M0 bytes."""
    v, e = _plain_quant4(x)
    a = v.flatten(-2).abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, 0.5 * a + 4)).to(torch.uint8)
    code = code + 8 * torch.signbit(v.flatten(-2)).to(torch.uint8)
    return code[:, ::2] + 16 * code[:, 1::2], (e.squeeze(-1) + 127).to(torch.uint8)


def _e4m3(x):
    """x's rows as e4m3 and E8M0 bytes."""
    v = x.reshape(x.shape[0], -1, 32)
    e = torch.ceil(torch.log2(v.abs().amax(-1, keepdim=True) / 448)).int()
    return (torch.ldexp(v, -e).clamp(-448, 448).flatten(1).to(torch.float8_e4m3fn),
            (e.squeeze(-1) + 127).to(torch.uint8))


def _package():
    if own:
        path = str(Path(__file__).resolve().parents[1] / "hk-dsl_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import hk  # noqa: F401, PLC0415


def prepare(case, seed):
    _package()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "quant":
        # rows of unit variance with a few large channels, as activations and weights have
        x = _randn(gen, case["m"], case["k"])
        x *= 1.0 + 9.0 * (torch.rand(case["k"], generator=gen, device="cuda") < 0.01)
        return dict(kind=kind, x=x.to(DTYPES[case["dtype"]]))
    if kind == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        x = _randn(gen, m, k)
        a, sa = _packed(x) if case["a"] == "fp4" else _e4m3(x)
        w, sw = _packed(_randn(gen, n, k, std=0.02))
        return dict(kind=kind, a=a, sa=sa, w=w, sw=sw, silu_mul=case["silu_mul"],
                    bias=_randn(gen, n, dtype=BF16, std=0.1) if case["bias"] else None)
    b, s, d = case["b"], case["s"], case["d"]
    dt, rdt = DTYPES[case["dtype"]], DTYPES[case["rdtype"]]
    wdt = DTYPES[case.get("wdtype", case["dtype"])]
    shape = {"none": None, "channel": (d,), "sequence": (b, 1, d), "token": (b, s, 1),
             "full": (b, s, d)}[case["gate"]]
    st = dict(kind=kind, x=_randn(gen, b, s, d, dtype=dt),
              residual=_randn(gen, b, s, d, dtype=rdt, std=2.0),
              post=_randn(gen, d, dtype=wdt, std=0.1, mean=1.0),
              pre=_randn(gen, d, dtype=wdt, std=0.1, mean=1.0),
              gate=None if shape is None else _randn(gen, *shape, dtype=dt, std=0.3, mean=0.5),
              branch_scale=0.5, residual_scale=0.9, quant=case.get("quant") == "mxfp8")
    if kind == "train":
        st["dh"] = _randn(gen, b, s, d, dtype=rdt)
        st["dy"] = _randn(gen, b, s, d, dtype=dt)
    return st


def _own(st):
    import hk  # noqa: PLC0415

    ops = hk.ops
    if st["kind"] == "quant":
        return ops.mxfp4.dequant(*ops.mxfp4.quant(st["x"]))
    if st["kind"] == "gemm":
        return ops.mxfp4.gemm(st["a"], st["w"], st["sa"], st["sw"], bias=st["bias"],
                              silu_mul=st["silu_mul"])
    args = dict(branch_scale=st["branch_scale"], residual_scale=st["residual_scale"], eps=EPS)
    if st["kind"] == "norm":
        h, y = ops.block_norm(st["x"], st["residual"], post=st["post"], pre=st["pre"],
                              gate=st["gate"], quant="mxfp8" if st["quant"] else None, **args)
        return {"h": h, "y": ops.mxfp8.dequant(*y) if st["quant"] else y}
    names = ["x", "residual", "post", "pre"] + (["gate"] if st["gate"] is not None else [])
    leaf = {n: st[n].detach().requires_grad_() for n in names}
    h, y = ops.block_norm(leaf["x"], leaf["residual"], post=leaf["post"], pre=leaf["pre"],
                          gate=leaf.get("gate"), **args)
    grads = torch.autograd.grad((h, y), list(leaf.values()), (st["dh"], st["dy"]))
    return {"h": h.detach(), "y": y.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def run(state):
    if own:
        return _own(state)
    kind = state["kind"]
    if kind == "quant":
        return _scaled(*_plain_quant4(state["x"])).to(BF16)
    if kind == "gemm":
        return _plain_gemm(state)
    return _plain_norm(state) if kind == "norm" else _plain_train(state)


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    kind = case["kind"]
    if kind == "quant":
        n = case["m"] * case["k"]
        return {"bytes": n * (size[case["dtype"]] + 2), "flops": 4 * n}
    if kind == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        wide = 0.5 if case["a"] == "fp4" else 1.0
        cols = n // 2 if case["silu_mul"] else n
        return {"bytes": m * k * (wide + 1 / 32) + n * k * (0.5 + 1 / 32) + 2 * m * cols
                + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    rows, d = case["b"] * case["s"], case["d"]
    e, r = size[case["dtype"]], size[case["rdtype"]]
    gate = {"none": 0, "channel": d, "sequence": case["b"] * d, "token": rows,
            "full": rows * d}[case["gate"]] * e
    w = 2 * d * size[case.get("wdtype", case["dtype"])]
    n = rows * d
    out = 2 if case.get("quant") == "mxfp8" else e
    forward = n * (e + 2 * r + out) + gate + w
    if kind == "norm":
        return {"bytes": forward, "flops": 12 * n}
    # x, residual, gate and weights once for both directions, and the gradients
    return {"bytes": forward + n * (2 * r + 2 * e) + gate + w, "flops": 40 * n}


# ------------------------------------------------------------------ in 64 bits


def _exact_round(v, grid):
    """v to the nearest of the sorted non-negative grid (even index at a tie), with its sign."""
    g = torch.tensor(grid, dtype=torch.float64, device=v.device)
    t = v.abs().contiguous()
    hi = torch.searchsorted(g, t).clamp(1, len(grid) - 1)
    below, above = t - g[hi - 1], g[hi] - t
    up = (above < below) | ((above == below) & (hi % 2 == 0))
    return torch.where(up, g[hi], g[hi - 1]) * torch.sign(v)


FP4_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
E4M3_GRID = tuple(m * 2.0 ** -9 for m in range(8)) + tuple(
    (8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8) if (8 + m) * 2.0 ** (e - 3) < 449)


def _exact_quant(x, grid, least):
    v = x.double().unflatten(-1, (-1, 32))
    amax = v.abs().amax(-1, keepdim=True).clamp(min=least)
    e = torch.floor(torch.log2(amax / grid[-1]))
    e = torch.where(torch.exp2(e) * grid[-1] < amax, e + 1, e).clamp(-127, 127)
    return (_exact_round(v / torch.exp2(e), grid) * torch.exp2(e)).flatten(-2)


def _exact_operand(q, s):
    if q.dtype == torch.uint8:
        table = torch.tensor(FP4_GRID + tuple(-v for v in FP4_GRID), dtype=torch.float64,
                             device=q.device)
        v = torch.empty(q.shape[0], 2 * q.shape[1], dtype=torch.float64, device=q.device)
        v[:, 0::2] = table[(q % 16).long()]
        v[:, 1::2] = table[(q // 16).long()]
    else:
        v = q.double()
    return v * torch.exp2(s.double() - 127).repeat_interleave(32, dim=1)


def exact(case, seed):
    st = prepare(case, seed)
    if st["kind"] == "quant":
        return _exact_quant(st["x"], FP4_GRID, 6.0 * 2.0 ** -127)
    if st["kind"] == "gemm":
        z = _exact_operand(st["a"], st["sa"]) @ _exact_operand(st["w"], st["sw"]).t().contiguous()
        if st["bias"] is not None:
            z += st["bias"].double()
        if st["silu_mul"]:
            half = z.shape[1] // 2
            z = torch.sigmoid(z[:, :half]) * z[:, :half] * z[:, half:]
        return z
    names = [n for n in ("x", "residual", "post", "pre", "gate") if st[n] is not None]
    v = {n: st[n].double().requires_grad_(st["kind"] == "train") for n in names}
    norm = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS)  # noqa: E731
    branch = norm(v["x"]) * v["post"] * st["branch_scale"]
    h = v["residual"] * st["residual_scale"] + (branch * v["gate"] if "gate" in v else branch)
    y = norm(h) * v["pre"]
    if st["kind"] == "norm":
        return {"h": h, "y": _exact_quant(y, E4M3_GRID, 2.0 ** -126) if st["quant"] else y}
    grads = torch.autograd.grad((h, y), [v[n] for n in names],
                                (st["dh"].double(), st["dy"].double()))
    return {"h": h.detach(), "y": y.detach(), **{"d" + n: g for n, g in zip(names, grads)}}
