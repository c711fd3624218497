// The block norm's kernels of fp16 x (hkx_norm.hpp).
#include "hkx_norm.hpp"

namespace hkx {

hipError_t launch_norm_fp16(const NormArgs& a, bool r32, bool w32, hipStream_t s) {
  if (r32) return w32 ? launch_norm_typed<HKX_FP16, HKX_FP32, HKX_FP32>(a, s) : launch_norm_typed<HKX_FP16, HKX_FP32, HKX_FP16>(a, s);
  return w32 ? launch_norm_typed<HKX_FP16, HKX_FP16, HKX_FP32>(a, s) : launch_norm_typed<HKX_FP16, HKX_FP16, HKX_FP16>(a, s);
}

hipError_t launch_norm_grad_fp16(const NormGradArgs& a, bool r32, bool w32, hipStream_t s) {
  if (r32)
    return w32 ? launch_norm_grad_typed<HKX_FP16, HKX_FP32, HKX_FP32>(a, s) : launch_norm_grad_typed<HKX_FP16, HKX_FP32, HKX_FP16>(a, s);
  return w32 ? launch_norm_grad_typed<HKX_FP16, HKX_FP16, HKX_FP32>(a, s) : launch_norm_grad_typed<HKX_FP16, HKX_FP16, HKX_FP16>(a, s);
}

}  // namespace hkx
