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
  if (fp8 && pair) hipLaunchKernelGGL((group_quad_kernel<kGroupNT, true, true>), grid, block, 0, s, a);
  else if (fp8) hipLaunchKernelGGL((group_quad_kernel<kGroupNT, true, false>), grid, block, 0, s, a);
  else if (pair) hipLaunchKernelGGL((group_quad_kernel<kGroupNT, false, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((group_quad_kernel<kGroupNT, false, false>), grid, block, 0, s, a);
  return hipGetLastError();
}

}  // namespace hkx
