// The block norm's kernels of fp32 x (hkx_norm.hpp).
#include "hkx_norm.hpp"

namespace hkx {

hipError_t launch_norm_fp32(const NormArgs& a, hipStream_t s) { return launch_norm_typed<HKX_FP32, HKX_FP32, HKX_FP32>(a, s); }

hipError_t launch_norm_grad_fp32(const NormGradArgs& a, hipStream_t s) {
  return launch_norm_grad_typed<HKX_FP32, HKX_FP32, HKX_FP32>(a, s);
}

}  // namespace hkx
