// The experts' gradient products on 256 x 256 tiles (hkx_group_quad.hpp).
#include "hkx_group_launch.hpp"
#include "hkx_group_quad.hpp"

namespace hkx {

hipError_t launch_group_quad_grad(const GroupArgs& a, int op, int cus, hipStream_t s) {
  const int64_t tn = (a.n + 255) / 256;
  const int64_t tiles = op == kGroupTN ? (int64_t)a.experts * ((a.m + 255) / 256) * tn : group_tiles(a.rows, a.experts, 256) * tn;
  dim3 grid;
  if (!group_quad_grid(tiles, cus, grid)) return hipErrorInvalidConfiguration;
  const dim3 block(512);
  if (op == kGroupTN) hipLaunchKernelGGL((group_quad_kernel<kGroupTN, false, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((group_quad_kernel<kGroupNN, false, false>), grid, block, 0, s, a);
  if (op == kGroupNN && a.ws)
    hipLaunchKernelGGL((group_quad_join_kernel<kGroupNN, false, false>), dim3(4 * (grid.x / 2)), block, 0, s, a, (int)grid.x);
  return hipGetLastError();
}

}  // namespace hkx
