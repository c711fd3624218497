"""Calls of more threads than one launch takes (2^32), on the GPU: their last rows are what they are in a
call of their own."""

import pytest
import torch

import hk
from hk.ops import mxfp4, mxfp8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _hand_the_memory_back():
    yield
    torch.cuda.empty_cache()


def _free(need):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < need * 2 ** 30:
        pytest.skip(f"needs {need} GiB")


def test_quantization_and_numbers_back():
    """2^35 values: pieces of 8, a thread each (two in mxfp8.quant)."""
    _free(200)
    m, k = (1 << 30) + 40, 32
    x = torch.zeros(m, k, device=DEV, dtype=BF16)
    ends = [slice(0, 64), slice(m // 2 - 32, m // 2 + 32), slice(m - 2200, m - 2136), slice(m - 64, m)]
    for p in ends:
        x[p] = torch.randn(64, k, device=DEV).to(BF16)
    for quant, dequant in ((mxfp4.quant, mxfp4.dequant), (lambda t: mxfp8.quant(t, nan_blocks=True), mxfp8.dequant)):
        q, s = quant(x)
        back = dequant(q, s)
        for p in ends:
            q1, s1 = quant(x[p].clone())
            assert torch.equal(q[p].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[p], s1)
            assert torch.equal(back[p], dequant(q1, s1)) and back[p].any()
        del q, s, back


@pytest.mark.parametrize("rows,d", [((1 << 26) + 37, 8), ((1 << 26) + 6, 3)])
def test_block_norm_of_many_rows(rows, d):
    """A wave a row: 2^26 rows are 2^32 threads. Forward (two launches), a gate a row of each, and backward."""
    _free(40)
    x = torch.empty(rows, d, device=DEV, dtype=BF16)
    x[:] = torch.randn(1, d, device=DEV).to(BF16)
    x *= torch.linspace(0.5, 2, 1024, device=DEV).to(BF16).repeat(rows // 1024 + 1)[:rows, None]
    gate = torch.linspace(0.25, 1, 999, device=DEV).to(BF16).repeat(rows // 999 + 1)[:rows, None]
    w = torch.linspace(0.9, 1.1, d, device=DEV).to(BF16)
    h, y = hk.ops.block_norm(x, x, post=w, pre=w, gate=gate)
    edge = (1 << 26) - 4
    ends = [slice(0, 40), slice(edge - 40, edge + 4), slice(rows - 40, rows)]
    for p in ends:
        h1, y1 = hk.ops.block_norm(x[p].clone(), x[p].clone(), post=w, pre=w, gate=gate[p].clone())
        assert torch.equal(h[p], h1) and torch.equal(y[p], y1)
    a = x.detach().requires_grad_()
    _, y2 = hk.ops.block_norm(a, x, post=w, pre=w, gate=gate)
    dx, = torch.autograd.grad(y2, a, y)
    for p in ends:
        a1 = x[p].clone().requires_grad_()
        _, y1 = hk.ops.block_norm(a1, x[p].clone(), post=w, pre=w, gate=gate[p].clone())
        assert torch.equal(dx[p], torch.autograd.grad(y1, a1, y[p].clone())[0])


@pytest.mark.parametrize("m,n,k,pair", [(1, 32770 * 4096 + 16, 32, False), (3, 32770 * 2048 + 8, 32, True),
                                        ((1 << 24) + 300, 64, 32, False)])
def test_products_of_many_columns_or_rows(m, n, k, pair):
    """The decode kernel's blocks of 16 columns (8 paired), 512 threads each, and 65536 tiles of 256 rows."""
    _free(20)
    rows = 2 * n if pair else n
    g = torch.Generator(device=DEV).manual_seed(n)
    a, b = (torch.randint(0, 256, (r, k // 2), generator=g, device=DEV, dtype=torch.uint8) for r in (m, rows))
    sa, sb = (torch.randint(125, 129, (r, k // 32), generator=g, device=DEV, dtype=torch.uint8) for r in (m, rows))
    c = mxfp4.gemm(a, b, sa, sb, silu_mul=pair)
    torch.cuda.synchronize()
    for p in (slice(0, 48), slice(n // 2, n // 2 + 48), slice(n - 48, n)) if m < 100 else (slice(0, n),):
        w = torch.cat([b[:n][p], b[n:][p]]) if pair else b[p].clone()
        ws = torch.cat([sb[:n][p], sb[n:][p]]) if pair else sb[p].clone()
        for r in (slice(0, 40), slice(m - 40, m)) if m > 100 else (slice(0, m),):
            # (32 products: exact in fp32 in any order)
            assert torch.equal(c[r, p], mxfp4.gemm(a[r].clone(), w, sa[r].clone(), ws, silu_mul=pair))
