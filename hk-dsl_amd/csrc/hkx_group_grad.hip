// The experts' gradient products on tiles (hkx_group.hpp), and the launch of whichever kernel a call takes.
#include "hkx_group_launch.hpp"

namespace hkx {

hipError_t launch_group_grad(const GroupArgs& a, int op, int bm, hipStream_t s) {
  if (op == kGroupTN) return launch_group_tile<kGroupTN, false, false, 128, 2, 2, 4, 4>(a, s);
  if (bm == 16) return launch_group_tile<kGroupNN, false, false, 16, 1, 4, 2, 4>(a, s);
  if (bm == 64) return launch_group_tile<kGroupNN, false, false, 64, 1, 4, 2, 3>(a, s);
  return launch_group_tile<kGroupNN, false, false, 128, 2, 2, 4, 4>(a, s);
}

hipError_t launch_group(const GroupArgs& a, int op, bool fp8, bool pair, int kernel, int cus, hipStream_t s) {
  if (kernel == kGroupQuad) return op == kGroupNT ? launch_group_quad_nt(a, fp8, pair, cus, s) : launch_group_quad_grad(a, op, cus, s);
  if (kernel >= kGroupSkinny16) return launch_group_skinny(a, fp8, pair, kernel == kGroupSkinny16 ? 16 : 32, s);
  const int bm = kernel == kGroupTile16 ? 16 : kernel == kGroupTile64 ? 64 : 128;
  return op == kGroupNT ? launch_group_nt(a, fp8, pair, bm, s) : launch_group_grad(a, op, bm, s);
}

}  // namespace hkx
