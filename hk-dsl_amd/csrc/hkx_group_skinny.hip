// The experts' forward product for few rows an expert (hkx_group_skinny.hpp).
#include <algorithm>

#include "hkx_group_launch.hpp"
#include "hkx_group_skinny.hpp"

namespace hkx {
namespace {

template <bool FP8, bool PAIR>
hipError_t launch(const GroupArgs& a, int bm, int blocks, hipStream_t s) {
  const int cn = (PAIR ? 16 : 32) * blocks;
  dim3 grid;
  if (!group_grid(group_tiles(a.rows, a.experts, bm) * ((a.n + cn - 1) / cn), 256, grid)) return hipErrorInvalidConfiguration;
  if (bm == 16) hipLaunchKernelGGL((group_skinny_kernel<FP8, PAIR, 1>), grid, dim3(256), 0, s, a, blocks);
  else hipLaunchKernelGGL((group_skinny_kernel<FP8, PAIR, 2>), grid, dim3(256), 0, s, a, blocks);
  return hipGetLastError();
}

// Blocks a workgroup: 128 KB of W, while two workgroups a CU are left.
int skinny_blocks(const GroupArgs& a, bool fp8, bool pair, int cus) {
  const int64_t row = (int64_t)a.k * (fp8 ? 1 : 2), cn = pair ? 16 : 32;
  const int64_t groups = std::min<int64_t>(a.experts, a.rows), all = groups * ((a.n + cn - 1) / cn);
  int b = 1;
  while (b < 8 && 2 * b * 32 * row <= 128 * 1024 && all / (2 * b) >= 2 * cus) b *= 2;
  return b;
}

}  // namespace

hipError_t launch_group_skinny(const GroupArgs& a, bool fp8, bool pair, int bm, int cus, hipStream_t s) {
  const int b = skinny_blocks(a, fp8, pair, cus);
  if (fp8) return pair ? launch<true, true>(a, bm, b, s) : launch<true, false>(a, bm, b, s);
  return pair ? launch<false, true>(a, bm, b, s) : launch<false, false>(a, bm, b, s);
}

}  // namespace hkx
