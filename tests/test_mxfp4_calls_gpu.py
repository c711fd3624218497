"""Calls of hk.ops.mxfp4 on the GPU by the way they are made -- outputs given, kept layouts, bias and scale
forms on each kernel -- against the float64 oracle."""

import ctypes

import pytest
import torch

from hk import _native as nat
from hk.ops import mxfp4, mxfp8
from oracle import mxfp4_oracle as O
from test_mx4_calls_cpu import PLANS

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
KERNELS = [nat.MX4_TILE64, nat.MX4_TILE128, nat.MX4_QUAD, nat.MX4_SKINNY]


def _gen(*seed):
    return torch.Generator().manual_seed(hash(seed) % (1 << 31))


def _operand(rows, k, wide, g, spread=2):
    s = torch.randint(127 - spread, 128 + spread, (rows, k // 32), generator=g).to(torch.uint8)
    if wide:
        return torch.randn(rows, k, generator=g).to(torch.float8_e4m3fn), s
    return torch.randint(0, 256, (rows, k // 2), generator=g).to(torch.uint8), s


def _operands(m, n, k, wide, pair, *seed):
    g = _gen(m, n, k, *seed)
    a, sa = _operand(m, k, wide, g)
    b, sb = _operand(2 * n if pair else n, k, False, g)
    return g, a, b, sa, sb - (6 if pair else 0)


def _within(c, ref, err):
    bad = ~((c.cpu().double() - ref).abs() <= err)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("wide", [False, True], ids=["a4", "a8"])
@pytest.mark.parametrize("m,n,k", [(129, 1035, 8224), (300, 1001, 4096), (520, 999, 1056)])
def test_gemm_silu_mul_of_odd_columns_with_a_bias(m, n, k, wide, dtype):
    """2N bias values of which the up half starts at an odd element."""
    print(f"case {m}x{n}x{k} wide={wide} {dtype}", flush=True)
    g, a, b, sa, sb = _operands(m, n, k, wide, True)
    bias = torch.randn(2 * n, generator=g).to(dtype)
    ref, err = O.gemm(a, b, sa, sb, bias, True)
    dev = [t.to(DEV) for t in (a, b, sa, sb)]
    for _ in range(2):
        _within(mxfp4.gemm(*dev, bias=bias.to(DEV), silu_mul=True), ref, err)


@pytest.mark.parametrize("m,n,k", [(1024, 12288, 4096), (300, 264, 1056)])
def test_gemm_after_an_out_8_bytes_off(m, n, k):
    """A contiguous out that is not 16-byte aligned, then calls of the same layout without one."""
    print(f"case {m}x{n}x{k}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(n)
    a, b = (torch.randint(0, 256, (r, k // 2), generator=g, device=DEV, dtype=torch.uint8) for r in (m, n))
    sa, sb = (torch.randint(127, 129, (r, k // 32), generator=g, device=DEV, dtype=torch.uint8) for r in (m, n))
    out = torch.empty(m * n + 4, dtype=BF16, device=DEV)[4:].view(m, n)
    assert out.data_ptr() % 16 == 8
    given = mxfp4.gemm(a, b, sa, sb, out=out)
    first, again = mxfp4.gemm(a, b, sa, sb), mxfp4.gemm(a, b, sa, sb)
    assert given.data_ptr() == out.data_ptr()
    # (a product of codes is a multiple of 1/4 up to 36, of scales 1 to 4: sums of 4096 are exact in fp32)
    assert torch.equal(first, out) and torch.equal(first, again)
    p = slice(0, 40)
    ref, err = O.gemm(a[p].cpu(), b.cpu(), sa[p].cpu(), sb.cpu())
    _within(first[p], ref, err)


@pytest.mark.parametrize("shapes", [((512, 4096, 4096), (768, 2048, 8192)), ((1024, 1001, 2048), (300, 512, 8192))])
def test_threads_on_one_stream(shapes):
    """Calls of several launches (packed scales, a split's shares) by two threads at a time."""
    import threading

    g = torch.Generator(device=DEV).manual_seed(3)
    cases = []
    for m, n, k in shapes:
        a, b = (torch.randint(0, 256, (r, k // 2), generator=g, device=DEV, dtype=torch.uint8) for r in (m, n))
        sa, sb = (torch.randint(125, 130, (r, k // 32), generator=g, device=DEV, dtype=torch.uint8) for r in (m, n))
        cases.append((a, b, sa, sb))
    want = [mxfp4.gemm(*c) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        for _ in range(40):
            got[i].append(mxfp4.gemm(*cases[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 40 and all(torch.equal(want[i], c) for c in got[i])


@pytest.mark.parametrize("act", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("m", [5, 700])
def test_linear_of_a_row_that_is_not_finite_is_nan(m, act):
    """On either path of the activation, and the other rows as without it; block_norm's quantized y, which
    linear's activation stands for, is NaN there too."""
    g = _gen(m, 12)
    x = torch.randn(m, 512, generator=g).to(BF16)
    w, ws = mxfp4.quant((torch.randn(96, 512, generator=g) * 0.05).to(DEV))
    clean = mxfp4.linear(x.to(DEV), w, ws, act=act).cpu()
    bad = {0: float("nan"), 2: float("inf"), m - 1: float("-inf")}
    for row, v in bad.items():
        x[row, 37 * (row % 13)] = v
    y = mxfp4.linear(x.to(DEV), w, ws, act=act).cpu()
    rows = torch.tensor(sorted(bad))
    assert torch.isnan(y[rows]).all()
    rest = torch.tensor([r for r in range(m) if r not in bad])
    assert torch.equal(y[rest], clean[rest])
    if act == "mxfp8":
        q, s = mxfp8.quant(x.to(DEV), nan_blocks=True)
        block = torch.zeros(m, 16, dtype=torch.bool)
        for row in bad:
            block[row, 37 * (row % 13) // 32] = True
        assert torch.equal(s.cpu() == 255, block)
        assert not q.cpu().view(torch.uint8).view(m, 16, 32)[block].any()
        q0, s0 = mxfp8.quant(x.to(DEV))  # (the other blocks are that rule's, and it leaves no NaN)
        assert torch.equal(q.cpu().view(torch.uint8).view(m, 16, 32)[~block], q0.cpu().view(torch.uint8).view(m, 16, 32)[~block])
        assert torch.equal(s.cpu()[~block], s0.cpu()[~block]) and (s0 < 255).all()


@pytest.mark.parametrize("lead", [(), (1,), (30,), (2, 3, 5), (0,), (4, 0, 2)])
def test_quant_and_linear_of_any_leading_sizes(lead):
    g = _gen(len(lead), 13)
    rows = torch.Size(lead).numel()
    x = torch.randn(*lead, 416, generator=g).to(BF16).to(DEV)
    flat = x.reshape(rows, 416)
    w, ws = mxfp4.quant((torch.randn(24, 416, generator=g) * 0.05).to(DEV))
    bias = torch.randn(24, generator=g).to(BF16).to(DEV)
    q0, s0 = mxfp4.quant(flat)
    for _ in range(2):  # the first call of a layout, and one that knows it
        q, s = mxfp4.quant(x)
        assert q.shape == (*lead, 208) and s.shape == (*lead, 13)
        assert torch.equal(q.reshape(rows, 208), q0) and torch.equal(s.reshape(rows, 13), s0)
        for act in ("mxfp8", "mxfp4"):
            y = mxfp4.linear(x, w, ws, bias=bias, act=act)
            assert y.shape == (*lead, 24) and y.dtype == BF16
            assert torch.equal(y.reshape(rows, 24), mxfp4.linear(flat, w, ws, bias=bias, act=act))
    y = mxfp4.linear(x, w, ws, silu_mul=True)
    assert y.shape == (*lead, 12)
    out = (torch.empty(*lead, 208, dtype=torch.uint8, device=DEV), torch.empty(*lead, 13, dtype=torch.uint8, device=DEV))
    mxfp4.quant(x, out=out)
    assert torch.equal(out[0].reshape(rows, 208), q0) and torch.equal(out[1].reshape(rows, 13), s0)


def test_quant_of_leading_sizes_of_any_strides():
    x = torch.randn(6, 5, 96, generator=_gen(14)).to(BF16).to(DEV)
    q0, s0 = mxfp4.quant(x.reshape(30, 96))
    w, ws = mxfp4.quant(torch.randn(8, 96, generator=_gen(15)).to(DEV))
    for v in (x.transpose(0, 1), x[::2], x[:, 1:4], x[..., :64], x.new_empty(6, 5, 104)[..., 3:99].copy_(x)):
        flat = v.reshape(-1, v.shape[-1]).contiguous()
        for _ in range(2):
            q, s = mxfp4.quant(v)
            qf, sf = mxfp4.quant(flat)
            assert torch.equal(q.reshape(qf.shape), qf) and torch.equal(s.reshape(sf.shape), sf)
        k = v.shape[-1]
        for act in ("mxfp8", "mxfp4"):
            y = mxfp4.linear(v, w[:, :k // 2], ws[:, :k // 32], act=act)
            assert torch.equal(y.reshape(-1, 8), mxfp4.linear(flat, w[:, :k // 2].clone(), ws[:, :k // 32].clone(), act=act))
    wide = torch.zeros(5, 6, 64, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError):  # (rows of two strides)
        mxfp4.quant(x, out=(wide.transpose(0, 1)[..., :48], torch.empty(6, 5, 3, dtype=torch.uint8, device=DEV)))
    q, s = wide.view(6, 5, 64)[..., :48], torch.empty(6, 5, 3, dtype=torch.uint8, device=DEV)
    mxfp4.quant(x, out=(q, s))
    assert torch.equal(q.reshape(30, 48), q0) and torch.equal(s.reshape(30, 3), s0)
    with pytest.raises(TypeError):
        mxfp4.quant(x[0, 0, 0])
    with pytest.raises(ValueError):
        mxfp4.linear(x[0, 0, 0], w, ws)


@pytest.mark.parametrize("act", ["mxfp8", "mxfp4"])
def test_linear_of_no_rows(act):
    w, ws = mxfp4.quant(torch.randn(24, 416, generator=_gen(16)).to(DEV))
    x = torch.empty(0, 416, dtype=BF16, device=DEV)
    assert mxfp4.linear(x, w, ws, act=act).shape == (0, 24)
    q, s = mxfp8.quant(x)
    assert q.shape == (0, 416) and s.shape == (0, 13)


def test_scales_as_e8m0_wherever_they_are_taken():
    x = torch.randn(7, 96, generator=_gen(17)).to(BF16).to(DEV)
    e8m0, fp4 = torch.float8_e8m0fnu, torch.float4_e2m1fn_x2
    q, s = mxfp4.quant(x)
    assert torch.equal(mxfp4.dequant(q, s.view(e8m0)), mxfp4.dequant(q, s))
    assert torch.equal(mxfp4.dequant(q.view(fp4), s.view(e8m0), F32), mxfp4.dequant(q, s, F32))
    out = torch.zeros(7, 48, dtype=torch.uint8, device=DEV).view(fp4), torch.zeros(7, 3, dtype=torch.uint8, device=DEV).view(e8m0)
    got = mxfp4.quant(x, out=out)
    for o in (out, got):
        assert torch.equal(o[0].view(torch.uint8), q) and torch.equal(o[1].view(torch.uint8), s)
    q8, s8 = mxfp8.quant(x)
    assert torch.equal(mxfp8.dequant(q8, s8.view(e8m0)), mxfp8.dequant(q8, s8))
    with pytest.raises(ValueError):
        mxfp4.dequant(q, s.int())


@pytest.mark.parametrize("exponent", [-134, -126, -122, -119, -117, -100, 0, 110])
def test_the_activations_quantization_keeps_a_blocks_size(exponent):
    """linear's MXFP8 quantization: within half a step of e4m3 (2^-4 of
    the value, 2^-10 of the scale where it is subnormal) of x, down to the least scale's blocks, where x
    itself is subnormal."""
    x = torch.ldexp(torch.randn(9, 96, generator=_gen(exponent)), torch.tensor(exponent)).to(BF16)
    q, s = mxfp8.quant(x.to(DEV), nan_blocks=True)
    v = O.values(q.cpu(), s.cpu())
    scale = torch.ldexp(torch.ones(9, 3, dtype=torch.float64), s.cpu().int() - 127).repeat_interleave(32, 1)
    assert (s < 255).all() and ((v - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -10 * scale).all()
    top = x.double().abs().view(9, 3, 32).amax(-1)
    assert (448 * scale[:, ::32] >= top).all() and ((224 * scale[:, ::32] < top) | (s.cpu() == 0)).all()


@pytest.mark.parametrize("call,plan", PLANS)
def test_gemm_by_each_plan(call, plan):
    """hk.ops.mxfp4.gemm where its plan is each kernel (test_mx4_calls_cpu.py holds that it is), with a 16-bit
    bias; the layout's second call takes the kept template, on operands of other values."""
    print(f"case {call} {plan}", flush=True)
    m, n, k, wide, pair = call
    for seed, dtype in enumerate((BF16, BF16, F16)):
        g, a, b, sa, sb = _operands(m, n, k, wide, pair, seed)
        bias = torch.randn(b.shape[0], generator=g).to(dtype)
        c = mxfp4.gemm(*(t.to(DEV) for t in (a, b, sa, sb)), bias=bias.to(DEV), silu_mul=pair)
        rows = torch.cat([torch.arange(0, 70), torch.arange(m // 2, m // 2 + 40), torch.arange(m - 70, m)]) if m > 200 else torch.arange(m)
        _within(c[rows.to(DEV)], *O.gemm(a[rows], b, sa[rows], sb, bias, pair))


def _forced(kernel, splits, a, b, sa, sb, n, k, bias=None, pair=False):
    """A product on a kernel and split given, of operands as they stand (row strides, any scale address)."""
    m = a.shape[0]
    g = nat.HkxMx4GemmArgs()
    g.size = ctypes.sizeof(g)
    g.a_dtype = nat.FP8E4M3 if a.dtype == torch.float8_e4m3fn else nat.FP4E2M1
    out = torch.full((m + 1, n + 8), 7.0, dtype=BF16, device=DEV)
    g.a, g.b, g.sa, g.sb, g.c = (t.data_ptr() for t in (a, b, sa, sb, out))
    g.lda, g.ldb, g.sa_ld, g.sb_ld, g.ldc = (t.stride(0) for t in (a, b, sa, sb, out))
    g.m, g.n, g.k, g.silu_mul, g.kernel, g.splits = m, n, k, int(pair), kernel, splits
    if bias is not None:
        g.bias, g.bias_dtype = bias.data_ptr(), nat.dtype_code(bias.dtype)
    need = nat.lib().hkx_mx4_gemm_workspace(g)
    ws = torch.full((need // 4 + 4,), float("nan"), device=DEV)
    g.ws, g.ws_bytes = ws.data_ptr(), need
    nat.check(nat.lib().hkx_mx4_gemm(g, nat.stream_of(a.device)))
    torch.cuda.synchronize()
    assert (out[m] == 7.0).all() and (out[:, n:] == 7.0).all()  # (nothing stored past M and N)
    return out[:m, :n]


def _inside(t, width, fill, at=0, odd=0):
    """t's rows inside wider ones of `fill`, `at` bytes from an aligned address, `odd` bytes a row more."""
    rows, n = t.shape
    big = torch.full((rows * (width + odd) + at + 64,), fill, dtype=torch.uint8, device=DEV)
    v = big[at:at + rows * (width + odd)].view(rows, width + odd)[:, :n]
    v.copy_(t.view(torch.uint8).to(DEV))
    return v.view(t.dtype)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("wide", [False, True], ids=["a4", "a8"])
@pytest.mark.parametrize("m,n,k,splits,pair", [(70, 264, 352, 1, False), (300, 520, 1056, 3, False), (13, 40, 96, 1, True),
                                               (270, 264, 2208, 2, True), (300, 77, 4128, 1, False)])
def test_every_kernel_reads_nothing_past_k(m, n, k, splits, pair, wide, kernel):
    """Rows wider than K, NaN bytes and NaN scales past it, scale rows off a dword by their base and by their
    stride; then a row of NaNs on each side: its own outputs alone are NaN."""
    print(f"case past k {kernel} {m}x{n}x{k}/{splits} pair={pair} wide={wide}", flush=True)
    g, a, b, sa, sb = _operands(m, n, k, wide, pair, 31)
    rows = b.shape[0]
    bias = torch.randn(rows, generator=g).to(F16).to(DEV)
    ref, err = O.gemm(a, b, sa, sb, bias.cpu(), pair)
    up16 = lambda x: (x + 47) // 16 * 16  # noqa: E731
    at, odd = (1, 0) if m % 2 else (3, 1)
    va, vb = _inside(a, up16(a.shape[1]), 0x7f), _inside(b, up16(k // 2), 0x7f)
    vsa, vsb = _inside(sa, k // 32 + 4, 255, at, odd), _inside(sb, k // 32 + 4, 255, 4 - at, odd + 1)
    if kernel == nat.MX4_SKINNY:
        splits = 1
    c = _forced(kernel, splits, va, vb, vsa, vsb, n, k, bias, pair)
    _within(c, ref, err)
    row, col = m // 2, n // 3
    vsa[row] = 255
    if wide:
        va.view(torch.uint8)[row] = 0x7f
    vsb[col] = 255
    c = _forced(kernel, splits, va, vb, vsa, vsb, n, k, bias, pair).cpu().double()
    nan = torch.zeros(m, n, dtype=torch.bool)
    nan[row], nan[:, col] = True, True
    assert torch.equal(torch.isnan(c), nan)
    assert ((c - ref).abs() <= err)[~nan].all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("wide", [False, True], ids=["a4", "a8"])
def test_every_kernel_takes_extreme_scales_and_those_of_one_block(wide, kernel):
    """Scale bytes 0 and 254 on opposite sides (their product is taken before fp32), and one block of one row
    of each side scaled by 32, in every 32-K place of a unit."""
    m, n, k = 270, 264, 800
    g, a, b, sa, sb = _operands(m, n, k, wide, False, 32)
    dev = [a.to(DEV), b.to(DEV)]
    for lo, hi in ((0, 254), (254, 0)):
        ta, tb = torch.full_like(sa, lo), torch.full_like(sb, hi)
        _within(_forced(kernel, 1, *dev, ta.to(DEV), tb.to(DEV), n, k), *O.gemm(a, b, ta, tb))
    for block in range(0, 25, 3):
        ta, tb = sa.clone(), sb.clone()
        ta[(37 * block) % m, block] += 5
        tb[(53 * block) % n, 24 - block] += 5
        _within(_forced(kernel, 1, *dev, ta.to(DEV), tb.to(DEV), n, k), *O.gemm(a, b, ta, tb))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("m,n,splits,pair", [(300, 264, 1, False), (300, 264, 2, False), (300, 263, 1, False),
                                             (300, 136, 1, True), (300, 136, 2, True), (300, 135, 1, True)])
def test_every_kernel_takes_every_bias(m, n, splits, pair, kernel, dtype):
    """By its own epilogue and through shares: N a multiple of 8 or odd, where the up half's bias starts off
    a dword."""
    k = 1056
    g, a, b, sa, sb = _operands(m, n, k, False, pair, 33)
    bias = torch.randn(b.shape[0], generator=g).to(dtype)
    if kernel == nat.MX4_SKINNY:
        splits = 1
    c = _forced(kernel, splits, *(t.to(DEV) for t in (a, b, sa, sb)), n, k, bias.to(DEV), pair)
    _within(c, *O.gemm(a, b, sa, sb, bias, pair))
