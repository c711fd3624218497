"""Calls of more threads than one launch takes (2^32), on the GPU: their last rows are what they are in a
call of their own."""

import pytest
import torch

import hk
from hk.ops import mxfp4, mxfp8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


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
