// The MXFP4 tile kernel's forms (hkx_mx4.hpp).
#include "hkx_mx4.hpp"

namespace hkx {

template <int BM, bool A8, bool PAIR, bool SHARE>
static hipError_t launch(const Mx4Args& a, dim3 grid, hipStream_t s) {
  hipLaunchKernelGGL((mx4_tile_kernel<BM, 128, A8, PAIR, SHARE, 1>), grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int BM, bool A8>
static hipError_t launch_form(const Mx4Args& a, bool pair, bool share, dim3 grid, hipStream_t s) {
  if (pair) return share ? launch<BM, A8, true, true>(a, grid, s) : launch<BM, A8, true, false>(a, grid, s);
  return share ? launch<BM, A8, false, true>(a, grid, s) : launch<BM, A8, false, false>(a, grid, s);
}

hipError_t launch_mx4_tile(const Mx4Args& a, bool a8, bool pair, bool share, int bm, dim3 grid, hipStream_t s) {
  if (bm == 64) return a8 ? launch_form<64, true>(a, pair, share, grid, s) : launch_form<64, false>(a, pair, share, grid, s);
  return a8 ? launch_form<128, true>(a, pair, share, grid, s) : launch_form<128, false>(a, pair, share, grid, s);
}

}  // namespace hkx
