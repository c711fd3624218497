"""hk.ops.block_norm on the GPU by the way it is called -- many gates, kept layouts, factors of the norms --
against the float64 oracle, with the tolerances of test_block_norm_gpu.py."""

import pytest
import torch

import hk
import test_block_norm_gpu as T
from oracle import mxfp4_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("gate_dtype", [BF16, F32])
@pytest.mark.parametrize("shape,one", [((70000, 2, 64), False), ((66000, 3, 37), False), ((70000, 2, 40), True),
                                       ((2100, 5, 1032), False), ((4099, 2, 130), True)])
def test_gradients_of_more_gates_than_workers(shape, one, gate_dtype):
    """A gate shared by a few rows (by the heads of a token, say), a value a column or one for all."""
    print(f"case gates {shape} one={one} {gate_dtype}", flush=True)
    a = T._inputs(shape, (BF16, F32, F32), "sequence", 21, gate_dtype)
    if one:
        a["gate"] = a["gate"][..., :1].clone()
    T._check_grads(a, 22, **T.SCALES)
