// The experts' forward products on 256 x 256 tiles (hkx_group_quad.hpp).
#include "hkx_group_launch.hpp"
#include "hkx_group_quad.hpp"

namespace hkx {

hipError_t launch_group_quad_nt(const GroupArgs& a, bool fp8, bool pair, int cus, hipStream_t s) {
  const int cn = pair ? 128 : 256;
  const int64_t tiles = group_tiles(a.rows, a.experts, 256) * ((a.n + cn - 1) / cn);
  dim3 grid;
  if (!group_quad_grid(tiles, cus, grid)) return hipErrorInvalidConfiguration;
  const dim3 block(512);
#define HKX_QUAD(FP8, PAIR)                                                                                            \
  do {                                                                                                                 \
    hipLaunchKernelGGL((group_quad_kernel<kGroupNT, FP8, PAIR>), grid, block, 0, s, a);                                \
    if (a.ws)                                                                                                          \
      hipLaunchKernelGGL((group_quad_join_kernel<kGroupNT, FP8, PAIR>), dim3(4 * (grid.x / 2)), block, 0, s, a, (int)grid.x); \
  } while (0)
  if (fp8 && pair) HKX_QUAD(true, true);
  else if (fp8) HKX_QUAD(true, false);
  else if (pair) HKX_QUAD(false, true);
  else HKX_QUAD(false, false);
#undef HKX_QUAD
  return hipGetLastError();
}

}  // namespace hkx
