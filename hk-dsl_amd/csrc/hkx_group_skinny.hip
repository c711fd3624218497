// The experts' forward product for few rows an expert (hkx_group_skinny.hpp).
#include "hkx_group_launch.hpp"
#include "hkx_group_skinny.hpp"

namespace hkx {
namespace {

template <bool FP8, bool PAIR>
hipError_t launch(const GroupArgs& a, int bm, hipStream_t s) {
  constexpr int CN = PAIR ? 16 : 32;
  dim3 grid;
  if (!group_grid(group_tiles(a.rows, a.experts, bm) * ((a.n + CN - 1) / CN), 256, grid)) return hipErrorInvalidConfiguration;
  if (bm == 16) hipLaunchKernelGGL((group_skinny_kernel<FP8, PAIR, 1>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((group_skinny_kernel<FP8, PAIR, 2>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_group_skinny(const GroupArgs& a, bool fp8, bool pair, int bm, hipStream_t s) {
  if (fp8) return pair ? launch<true, true>(a, bm, s) : launch<true, false>(a, bm, s);
  return pair ? launch<false, true>(a, bm, s) : launch<false, false>(a, bm, s);
}

}  // namespace hkx
