"""hk.ops: the GEMM entry points of this build -- `matmul` (bf16), `scaled_mm` (fp8 with
per-token x per-channel dequant), `mxfp8` (MX block-scaled fp8), `mxfp4` (4-bit weights) and the
gfx950 route (`gemm_cdna`); and `block_norm`, what stands between two blocks' products."""

from . import gemm_cdna, mxfp4, mxfp8  # noqa: F401
from .gemm import matmul, scaled_mm  # noqa: F401
from .norm import block_norm  # noqa: F401

__all__ = ["matmul", "scaled_mm", "gemm_cdna", "mxfp4", "mxfp8", "block_norm"]
