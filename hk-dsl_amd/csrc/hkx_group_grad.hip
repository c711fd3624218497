// The experts' gradient products on tiles (hkx_group.hpp), and the choice of a kernel.
#include "hkx_group_launch.hpp"

namespace hkx {

hipError_t launch_group_grad(const GroupArgs& a, int op, int bm, hipStream_t s) {
  if (op == kGroupTN) return launch_group_tile<kGroupTN, false, false, 128, 2, 2, 4, 4>(a, s);
  if (bm == 16) return launch_group_tile<kGroupNN, false, false, 16, 1, 4, 2, 4>(a, s);
  if (bm == 64) return launch_group_tile<kGroupNN, false, false, 64, 1, 4, 2, 3>(a, s);
  return launch_group_tile<kGroupNN, false, false, 128, 2, 2, 4, 4>(a, s);
}

hipError_t launch_group(const GroupArgs& a, int op, bool fp8, bool pair, int kernel, int cus, hipStream_t s) {
  // rows an expert, were they even (the host does not know the counts)
  const int64_t each = a.rows / a.experts;
  if (kernel == HKX_EXPERTS_QUAD || (kernel == HKX_EXPERTS_AUTO && each >= 128 && group_quad_ok(a)))
    return op == kGroupNT ? launch_group_quad_nt(a, fp8, pair, cus, s) : launch_group_quad_grad(a, op, cus, s);
  const int bm = kernel == HKX_EXPERTS_TILE16 ? 16 : kernel == HKX_EXPERTS_TILE64 ? 64 : kernel == HKX_EXPERTS_TILE128 ? 128
                 : each <= 16 ? 16 : each <= 64 ? 64 : 128;
  return op == kGroupNT ? launch_group_nt(a, fp8, pair, bm, s) : launch_group_grad(a, op, bm, s);
}

}  // namespace hkx
