// The experts' forward products on tiles (hkx_group.hpp).
#include "hkx_group_launch.hpp"

namespace hkx {
namespace {

template <bool FP8, bool PAIR>
hipError_t tiles(const GroupArgs& a, int bm, hipStream_t s) {
  if (bm == 16) return launch_group_tile<kGroupNT, FP8, PAIR, 16, 1, 4, 2, 4>(a, s);
  if (bm == 64) return launch_group_tile<kGroupNT, FP8, PAIR, 64, 1, 4, 2, 3>(a, s);
  return launch_group_tile<kGroupNT, FP8, PAIR, 128, 2, 2, 4, 4>(a, s);
}

}  // namespace

hipError_t launch_group_nt(const GroupArgs& a, bool fp8, bool pair, int bm, hipStream_t s) {
  if (fp8) return pair ? tiles<true, true>(a, bm, s) : tiles<true, false>(a, bm, s);
  return pair ? tiles<false, true>(a, bm, s) : tiles<false, false>(a, bm, s);
}

}  // namespace hkx
