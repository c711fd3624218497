// The MXFP4 tile kernel's forms (hkx_mx4.hpp).
#include "hkx_mx4.hpp"

namespace hkx {

template <int BM, bool A8, bool PAIR, bool SHARE>
static hipError_t launch(const Mx4Args& a, bool two, dim3 grid, hipStream_t s) {
  if constexpr (BM == 64 || !A8) {  // (two stages of 128 rows of an 8-bit A do not fit half the LDS)
    if (two) {
      hipLaunchKernelGGL((mx4_tile_kernel<BM, 128, A8, PAIR, SHARE, 2>), grid, dim3(256), 0, s, a);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((mx4_tile_kernel<BM, 128, A8, PAIR, SHARE, 1>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int BM, bool A8>
static hipError_t launch_form(const Mx4Args& a, bool pair, bool share, bool two, dim3 grid, hipStream_t s) {
  if (pair) return share ? launch<BM, A8, true, true>(a, two, grid, s) : launch<BM, A8, true, false>(a, two, grid, s);
  return share ? launch<BM, A8, false, true>(a, two, grid, s) : launch<BM, A8, false, false>(a, two, grid, s);
}

hipError_t launch_mx4_tile(const Mx4Args& a, bool a8, bool pair, bool share, int bm, bool two, dim3 grid, hipStream_t s) {
  if (bm == 64)
    return a8 ? launch_form<64, true>(a, pair, share, two, grid, s) : launch_form<64, false>(a, pair, share, two, grid, s);
  return a8 ? launch_form<128, true>(a, pair, share, two, grid, s) : launch_form<128, false>(a, pair, share, two, grid, s);
}

}  // namespace hkx
