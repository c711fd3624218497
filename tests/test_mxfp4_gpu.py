"""hk.ops.mxfp4 on the GPU against the float64 oracle (oracle/mxfp4_oracle.py): quantization and its
numbers bit for bit, the product within the oracle's bound, over the sizes, strides and values where
each could go wrong; and the calls that are refused."""

import pytest
import torch

import hk
from hk import _native as nat
from hk.ops import mxfp4, mxfp8
from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(*seed):
    return torch.Generator().manual_seed(hash(seed) % (1 << 31))


# ------------------------------------------------------------------ quantization


def _rows(m, k, dtype, g):
    """Rows with blocks of every magnitude: ties, zeros, subnormals, the largest values."""
    x = torch.randn(m, k, generator=g)
    x *= torch.exp2(torch.randint(-20, 14, (m, k // 32), generator=g)).repeat_interleave(32, 1).float()
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0, -2.5, -0.25, -5.0])
    x[0, :32] = grid[torch.arange(32) % 12]
    if m > 1:
        x[1, :32] = 0.0
        x[1, -32:] = grid[torch.arange(32) % 12] * 2.0 ** -14
    if m > 2:
        x[2, :32] = torch.finfo(dtype).smallest_normal * torch.linspace(-2, 2, 32)
        x[2, 3] = torch.finfo(dtype).max
    if m > 3:
        x[3, -32:] = torch.finfo(dtype).smallest_normal * torch.linspace(-1, 1, 32)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,k", [(1, 32), (2, 64), (5, 96), (16, 4096), (33, 2976), (1, 14336), (700, 160)])
def test_quant_is_the_oracles_bit_for_bit(m, k, dtype):
    print(f"case quant {m}x{k} {dtype}", flush=True)
    x = _rows(m, k, dtype, _gen(m, k))
    q, s = mxfp4.quant(x.to(DEV))
    codes, scales = O.quant(x)
    assert torch.equal(s.cpu(), scales)
    assert torch.equal(O.unpack(q.cpu()), codes)
    for out in (BF16, F16, F32):
        v = mxfp4.dequant(q, s, out).cpu()
        assert torch.equal(v, O.values(q.cpu(), s.cpu()).to(out)), out


def test_quant_of_blocks_that_are_not_finite():
    x = torch.randn(4, 128, generator=_gen(1))
    x[0, 5], x[1, 64], x[2, 127] = float("inf"), float("nan"), float("-inf")
    q, s = mxfp4.quant(x.to(DEV))
    assert torch.equal(s.cpu() == 255, torch.tensor([[1, 0, 0, 0], [0, 0, 1, 0], [0, 0, 0, 1], [0, 0, 0, 0]]).bool())
    v = mxfp4.dequant(q, s, F32).cpu()
    want = O.values(q.cpu(), s.cpu()).float()
    assert torch.equal(torch.isnan(v), torch.isnan(want)) and torch.isnan(v).sum() == 96
    assert torch.equal(v[3], want[3])


def test_quant_takes_strides_and_writes_into_out():
    big = torch.randn(40, 400, generator=_gen(2)).to(BF16).to(DEV)
    ref = O.quant(big[:, 8:264].cpu())
    for x in (big[:, 8:264], big[:, 8:264].t().contiguous().t()):
        q, s = mxfp4.quant(x)
        assert torch.equal(O.unpack(q.cpu()), ref[0]) and torch.equal(s.cpu(), ref[1])
    odd = big[::2, 1:257]  # rows no 16-byte load can start at
    q, s = mxfp4.quant(odd)
    assert torch.equal(s.cpu(), O.quant(odd.cpu())[1])
    q = torch.zeros(40, 200, dtype=torch.uint8, device=DEV)
    s = torch.zeros(40, 9, dtype=torch.uint8, device=DEV)
    mxfp4.quant(big[:, 8:264], out=(q[:, :128], s[:, :8]))
    assert torch.equal(O.unpack(q[:, :128].cpu()), ref[0]) and torch.equal(s[:, :8].cpu(), ref[1])
    assert not q[:, 128:].any() and not s[:, 8:].any()


def test_quant_of_nothing():
    q, s = mxfp4.quant(torch.empty(0, 64, dtype=BF16, device=DEV))
    assert q.shape == (0, 32) and s.shape == (0, 2)
    assert mxfp4.dequant(q, s).shape == (0, 64)


def test_mxfp8_dequant_gives_its_numbers():
    x = torch.randn(37, 416, generator=_gen(3)).to(BF16)
    q, s = mxfp8.quant(x.to(DEV))
    for out in (BF16, F16, F32):
        assert torch.equal(mxfp8.dequant(q, s, out).cpu(), O.values(q.cpu(), s.cpu()).to(out))


# ------------------------------------------------------------------ the product


def _operand(rows, k, wide, g, spread=6):
    """Random codes with scales a few powers of two apart."""
    s = torch.randint(127 - spread, 128 + spread, (rows, k // 32), generator=g).to(torch.uint8)
    if wide:
        return torch.randn(rows, k, generator=g).to(torch.float8_e4m3fn), s
    return torch.randint(0, 256, (rows, k // 2), generator=g).to(torch.uint8), s


def _check(a, b, sa, sb, bias=None, silu_mul=False, out=None):
    dev = [t.to(DEV) if t is not None else None for t in (a, b, sa, sb, bias)]
    c = mxfp4.gemm(*dev[:4], bias=dev[4], silu_mul=silu_mul, out=out)
    ref, err = O.gemm(a, b, sa, sb, bias, silu_mul)
    off = (c.cpu().double() - ref).abs()
    assert c.dtype == BF16 and c.shape == ref.shape
    bad = ~(off <= err)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, first at "
                           f"{bad.nonzero()[0].tolist()}: {c.cpu()[bad][0]} for {ref[bad][0]}")
    return c


SHAPES = [
    (1, 1, 32), (1, 16, 64), (1, 129, 4096), (2, 4096, 512), (3, 100, 2976), (4, 640, 96),
    (7, 1001, 1056), (16, 2048, 4096), (16, 33, 12288), (17, 512, 2048), (31, 257, 800),
    (32, 1024, 1024), (33, 200, 992), (37, 1001, 2976), (48, 512, 4096), (64, 768, 7168),
    (65, 130, 288), (100, 1000, 1504), (128, 256, 256), (200, 384, 8192), (255, 512, 1312),
    (257, 770, 640), (300, 300, 320), (512, 1024, 2048), (700, 640, 32), (1025, 520, 544),
]


@pytest.mark.parametrize("wide", [False, True], ids=["a4", "a8"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm(m, n, k, wide):
    print(f"case gemm {m}x{n}x{k} wide={wide}", flush=True)
    g = _gen(m, n, k)
    a, sa = _operand(m, k, wide, g)
    b, sb = _operand(n, k, False, g)
    bias = torch.randn(n, generator=g).to(BF16) if (m + n) % 2 else None
    _check(a, b, sa, sb, bias)


@pytest.mark.parametrize("wide", [False, True], ids=["a4", "a8"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 64), (1, 512, 4096), (4, 65, 96), (16, 1000, 2048), (29, 130, 1600),
                                   (37, 500, 2976), (64, 96, 4096), (130, 200, 352), (300, 512, 1024),
                                   (600, 257, 736)])
def test_gemm_silu_mul(m, n, k, wide):
    print(f"case silu_mul {m}x{n}x{k} wide={wide}", flush=True)
    g = _gen(m, n, k, 2)
    a, sa = _operand(m, k, wide, g, 2)
    b, sb = _operand(2 * n, k, False, g, 2)
    sb -= 6  # gates of a few units
    bias = torch.randn(2 * n, generator=g).to(F32) if m % 2 else None
    _check(a, b, sa, sb, bias, True)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_gemm_bias_types(m, dtype):
    g = _gen(m)
    a, sa = _operand(m, 512, False, g)
    b, sb = _operand(96, 512, False, g)
    _check(a, b, sa, sb, torch.randn(96, generator=g).to(dtype))


@pytest.mark.parametrize("wide", [False, True], ids=["a4", "a8"])
@pytest.mark.parametrize("m", [1, 16, 40, 300, 600])
def test_gemm_reads_nothing_past_k(m, wide):
    """Rows wider than K, a row of NaNs next to others: only its own outputs are NaN. The operands'
    bytes past K are e4m3 NaNs, their scales past K/32 the NaN scale."""
    k, n = 352, 520
    g = _gen(m, 9)
    a, sa = _operand(m, k, wide, g)
    b, sb = _operand(n, k, False, g)
    per = 1 if wide else 2
    ga = torch.full((m, 1024 // per), 0x7f, dtype=torch.uint8)
    ga[:, :k // per] = a.view(torch.uint8)
    gb = torch.full((n, 512), 0x7f, dtype=torch.uint8)
    gb[:, :k // 2] = b
    gsa, gsb = torch.full((m, 32), 255, dtype=torch.uint8), torch.full((n, 32), 255, dtype=torch.uint8)
    gsa[:, :k // 32], gsb[:, :k // 32] = sa, sb
    ga, gb, gsa, gsb = (t.to(DEV) for t in (ga, gb, gsa, gsb))
    av = ga[:, :k // per].view(torch.float8_e4m3fn) if wide else ga[:, :k // per]
    c = mxfp4.gemm(av, gb[:, :k // 2], gsa[:, :k // 32], gsb[:, :k // 32])
    ref, err = O.gemm(a, b, sa, sb)
    assert ((c.cpu().double() - ref).abs() <= err).all()
    # a whole row of NaN scales (and codes, where A has NaNs), and one of B
    row, col = m // 2, 77
    gsa[row, :k // 32] = 255
    if wide:
        ga[row] = 0x7f
    gsb[col, :k // 32] = 255
    c = mxfp4.gemm(av, gb[:, :k // 2], gsa[:, :k // 32], gsb[:, :k // 32]).cpu().double()
    nan = torch.zeros(m, n, dtype=torch.bool)
    nan[row], nan[:, col] = True, True
    assert torch.equal(torch.isnan(c), nan)
    assert ((c - ref).abs() <= err)[~nan].all()


@pytest.mark.parametrize("m", [2, 300])
def test_gemm_scales_of_a_block_reach_its_products_alone(m):
    """One block of one row of each side scaled by 32: the outputs it feeds change by its share."""
    n, k = 256, 800
    g = _gen(m, 4)
    a, sa = _operand(m, k, False, g)
    b, sb = _operand(n, k, False, g)
    sa[m - 1, 9] += 5
    sb[201, 24] += 5
    _check(a, b, sa, sb)


def test_gemm_of_extreme_scales():
    """Scale bytes 0 and 254 on opposite sides: the product of the scales is taken before fp32."""
    g = _gen(5)
    for m in (3, 70, 300):
        a, sa = _operand(m, 256, False, g, 1)
        b, sb = _operand(64, 256, False, g, 1)
        _check(a, b, torch.full_like(sa, 0), torch.full_like(sb, 254))


@pytest.mark.parametrize("m", [5, 80, 400])
def test_gemm_takes_strides_and_unaligned_scales(m):
    g = _gen(m, 6)
    k, n = 416, 200
    a, sa = _operand(2 * m, k, True, g)
    b, sb = _operand(n, k, False, g)
    ref, err = O.gemm(a[::2], b, sa[::2], sb)
    wide = torch.zeros(n, 240, dtype=torch.uint8, device=DEV)
    wide[:, 3:211] = b.to(DEV)  # rows no 16-byte load can start at
    out = torch.zeros(m, n + 5, dtype=BF16, device=DEV)
    c = mxfp4.gemm(a.to(DEV)[::2], wide[:, 3:211], sa.to(DEV)[::2], sb.to(DEV), out=out[:, 2:n + 2])
    assert ((c.cpu().double() - ref).abs() <= err).all()
    assert c.data_ptr() == out[:, 2:].data_ptr() and not out[:, :2].any() and not out[:, n + 2:].any()
    # float4 and e8m0 views of the same bytes
    c2 = mxfp4.gemm(a.to(DEV)[::2].contiguous(), b.to(DEV).view(torch.float4_e2m1fn_x2),
                    sa.to(DEV)[::2].contiguous().view(torch.float8_e8m0fnu), sb.to(DEV))
    assert torch.equal(c, c2)


def test_gemm_is_the_same_every_time_and_on_another_stream():
    g = _gen(7)
    for m, n, k in ((1, 512, 4096), (37, 1001, 2976), (300, 512, 8192)):
        a, sa = _operand(m, k, True, g)
        b, sb = _operand(n, k, False, g)
        dev = [t.to(DEV) for t in (a, b, sa, sb)]
        first = mxfp4.gemm(*dev)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            other = [mxfp4.gemm(*dev) for _ in range(3)]
        side.synchronize()
        assert all(torch.equal(first, o) for o in other)


def test_gemm_in_a_graph():
    g = _gen(8)
    cases = []
    for m, n, k in ((1, 256, 1024), (40, 200, 4096), (300, 512, 8192)):
        a, sa = _operand(m, k, False, g)
        b, sb = _operand(n, k, False, g)
        cases.append([t.to(DEV) for t in (a, b, sa, sb)])
    want = [mxfp4.gemm(*c) for c in cases]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [mxfp4.gemm(*c) for c in cases]
    for _ in range(3):
        for o in got:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(w, o) for w, o in zip(want, got))
        assert torch.equal(mxfp4.gemm(*cases[1]), want[1])


def test_linear_quantizes_the_activation():
    g = _gen(10)
    x = torch.randn(19, 512, generator=g).to(BF16)
    w, ws = mxfp4.quant((torch.randn(96, 512, generator=g) * 0.05).to(DEV))
    bias = torch.randn(96, generator=g).to(BF16)
    for act, q in (("mxfp8", mxfp8.quant), ("mxfp4", mxfp4.quant)):
        xq, xs = q(x.to(DEV))
        y = mxfp4.linear(x.to(DEV), w, ws, bias=bias.to(DEV), act=act)
        ref, err = O.gemm(xq.cpu(), w.cpu(), xs.cpu(), ws.cpu(), bias)
        assert ((y.cpu().double() - ref).abs() <= err).all()


def test_leading_dimensions():
    g = _gen(11)
    a, sa = _operand(30, 416, True, g)
    b, sb = _operand(24, 416, False, g)
    c = mxfp4.gemm(a.to(DEV), b.to(DEV), sa.to(DEV), sb.to(DEV))
    for lead in ((2, 3, 5), (30,), (1, 30)):
        a3, s3 = a.to(DEV).view(*lead, 416), sa.to(DEV).view(*lead, 13)
        for _ in range(2):  # the first call of a layout, and one that knows it
            assert torch.equal(mxfp4.gemm(a3, b.to(DEV), s3, sb.to(DEV)), c.view(*lead, 24))
        assert torch.equal(mxfp8.dequant(a3, s3).view(30, 416), mxfp8.dequant(a.to(DEV), sa.to(DEV)))
    one = mxfp4.gemm(a.to(DEV)[3], b.to(DEV), sa.to(DEV)[3], sb.to(DEV))
    assert torch.equal(one, mxfp4.gemm(a.to(DEV)[3:4], b.to(DEV), sa.to(DEV)[3:4], sb.to(DEV))[0])


def test_gemm_of_nothing():
    b, sb = torch.zeros(8, 32, dtype=torch.uint8, device=DEV), torch.zeros(8, 2, dtype=torch.uint8, device=DEV)
    c = mxfp4.gemm(b[:0], b, sb[:0], sb)
    assert c.shape == (0, 8)
    assert mxfp4.gemm(b, b[:0], sb, sb[:0]).shape == (8, 0)


def test_refusals():
    u8 = torch.uint8
    a, sa = torch.zeros(4, 64, dtype=u8, device=DEV), torch.zeros(4, 4, dtype=u8, device=DEV)
    b, sb = torch.zeros(6, 64, dtype=u8, device=DEV), torch.zeros(6, 4, dtype=u8, device=DEV)
    x = torch.zeros(4, 64, dtype=BF16, device=DEV)
    with pytest.raises(TypeError):
        mxfp4.gemm(a.float(), b, sa, sb)
    with pytest.raises(TypeError):
        mxfp4.gemm(a, b, sa.int(), sb)
    with pytest.raises(ValueError):
        mxfp4.gemm(a[:, :32], b, sa, sb)
    with pytest.raises(ValueError):
        mxfp4.gemm(a, b, sa[:, :3], sb)
    with pytest.raises(ValueError):
        mxfp4.gemm(a, b.cpu(), sa, sb)
    with pytest.raises(ValueError):
        mxfp4.gemm(a, b, sa, sb.cpu())
    with pytest.raises(ValueError):
        mxfp4.gemm(a, b[:5], sa, sb[:5], silu_mul=True)
    with pytest.raises(ValueError):
        mxfp4.gemm(a, b, sa, sb, bias=torch.zeros(5, device=DEV))
    with pytest.raises(ValueError):
        mxfp4.gemm(a, b, sa, sb, out=torch.zeros(4, 5, dtype=BF16, device=DEV))
    with pytest.raises(ValueError):
        mxfp4.gemm(a[:, :8], b[:, :8], sa[:, :1], sb[:, :1])
    with pytest.raises(TypeError):
        mxfp4.quant(x.int())
    with pytest.raises(ValueError):
        mxfp4.quant(x[:, :40])
    with pytest.raises(ValueError):
        mxfp4.quant(x.cpu())
    with pytest.raises(ValueError):
        mxfp4.dequant(a, sa[:2])
    with pytest.raises(TypeError):
        mxfp4.dequant(a, sa, torch.int32)
    with pytest.raises(ValueError):
        mxfp4.linear(x, b, sb, act="int8")
    g = nat.HkxMx4GemmArgs()
    with pytest.raises(nat.HkxError):
        nat.check(nat.lib().hkx_mx4_gemm(g, None))
    assert hk.ops.mxfp4 is mxfp4


def _forced(kernel, splits, a, b, sa, sb, bias=None, silu_mul=False):
    """A product on a kernel and split given (hk.ops.mxfp4.gemm picks them)."""
    import ctypes

    m, n = a.shape[0], b.shape[0] // (2 if silu_mul else 1)
    g = nat.HkxMx4GemmArgs()
    g.size = ctypes.sizeof(g)
    g.a_dtype = nat.FP8E4M3 if a.dtype == torch.float8_e4m3fn else nat.FP4E2M1
    out = torch.empty(m, n, dtype=BF16, device=DEV)
    g.a, g.b, g.sa, g.sb, g.c = (t.data_ptr() for t in (a, b, sa, sb, out))
    g.lda, g.ldb, g.ldc = a.stride(0), b.stride(0), n
    g.sa_ld, g.sb_ld = (t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 3) // 4 * 4 for t in (sa, sb))
    g.m, g.n, g.k, g.silu_mul, g.kernel, g.splits = m, n, 2 * b.shape[1], int(silu_mul), kernel, splits
    if bias is not None:
        g.bias, g.bias_dtype = bias.data_ptr(), nat.dtype_code(bias.dtype)
    need = nat.lib().hkx_mx4_gemm_workspace(g)
    ws = torch.full((need // 4 + 4,), float("nan"), device=DEV)
    g.ws, g.ws_bytes = ws.data_ptr(), need
    nat.check(nat.lib().hkx_mx4_gemm(g, nat.stream_of(a.device)))
    return out


@pytest.mark.parametrize("kernel", [nat.MX4_TILE64, nat.MX4_TILE128, nat.MX4_QUAD, nat.MX4_SKINNY])
@pytest.mark.parametrize("wide", [False, True], ids=["a4", "a8"])
@pytest.mark.parametrize("m,n,k,splits,pair", [
    (1, 8, 32, 1, False), (5, 40, 256, 1, True), (1, 300, 2080, 1, False), (13, 1050, 4096, 1, True),
    (16, 16400, 1120, 1, False), (9, 9001, 2976, 1, True), (16, 200, 12320, 1, False), (3, 70, 8192, 1, True),
    (32, 4100, 4096, 1, False), (29, 130, 2208, 1, True), (32, 600, 9952, 1, False), (27, 65, 5120, 1, True), (8, 5000, 6432, 1, True),
    (5, 48, 16448, 1, False), (48, 1001, 2976, 1, False), (64, 136, 4096, 1, True), (37, 2100, 1984, 1, False),
    (61, 72, 9000 // 32 * 32, 1, True), (47, 4101, 6144, 1, False), (300, 300, 288, 1, False), (260, 513, 1120, 3, False),
    (129, 130, 2048, 4, True), (520, 1000, 768, 1, True), (513, 264, 4096, 8, False), (700, 1032, 544, 2, False),
    (2304, 2560, 96, 1, False), (2100, 4352, 512, 1, False), (1500, 2400, 1312, 1, True)])
def test_every_kernel_takes_every_shape(m, n, k, splits, pair, wide, kernel):
    """Also several tiles a workgroup of the persistent kernel (2304 x 2560 and more), each K unit
    count from one, and both forms of its stores (N a multiple of 8 or not)."""
    print(f"case forced {kernel} {m}x{n}x{k}/{splits} pair={pair} wide={wide}", flush=True)
    g = _gen(m, n, k, 3)
    a, sa = _operand(m, k, wide, g, 2)
    b, sb = _operand(2 * n if pair else n, k, False, g, 2)
    if pair:
        sb -= 6
    bias = torch.randn(b.shape[0], generator=g).to([BF16, F16, F32][m % 3]) if n % 2 == 0 else None
    dev = [t.to(DEV) if t is not None else None for t in (a, b, sa, sb, bias)]
    c = _forced(kernel, splits, *dev, pair)
    ref, err = O.gemm(a, b, sa, sb, bias, pair)
    bad = ~((c.cpu().double() - ref).abs() <= err)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"
