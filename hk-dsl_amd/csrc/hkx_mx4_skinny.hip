// The MXFP4 decode kernel's forms (hkx_mx4_skinny.hpp).
#include <algorithm>

#include "hkx_mx4_skinny.hpp"

namespace hkx {

template <int MF, bool A8, bool PAIR>
static hipError_t launch(const Mx4SkinnyArgs& a, dim3 grid, hipStream_t s) {
  if (a.units <= 8) {
    hipLaunchKernelGGL((mx4_skinny_kernel<MF, A8, PAIR, 1>), grid, dim3(512), 0, s, a);
    return hipGetLastError();
  }
  if (a.units <= 16) {
    hipLaunchKernelGGL((mx4_skinny_kernel<MF, A8, PAIR, 2>), grid, dim3(512), 0, s, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((mx4_skinny_kernel<MF, A8, PAIR, 0>), grid, dim3(512), 0, s, a);
  return hipGetLastError();
}

template <int MF>
static hipError_t launch_form(const Mx4SkinnyArgs& a, bool a8, bool pair, dim3 grid, hipStream_t s) {
  if (a8) return pair ? launch<MF, true, true>(a, grid, s) : launch<MF, true, false>(a, grid, s);
  return pair ? launch<MF, false, true>(a, grid, s) : launch<MF, false, false>(a, grid, s);
}

hipError_t launch_mx4_skinny(Mx4SkinnyArgs a, bool a8, bool pair, int cus, hipStream_t s) {
  const int chunks = (a.M + 63) / 64;  // of 64 rows, each its own workgroups
  cus = std::max(1, cus / chunks);
  // the most blocks a workgroup, up to 4, that leave the CUs full and the blocks as even over them as
  // one each
  const int nq = a.units <= 8 ? 1 : a.units <= 16 ? 2 : 0;
  const int mf = chunks > 1 ? 4 : (a.M + 15) / 16;
  const int resident = mx4_skinny_resident(mf, a8, pair, nq);
  const int blocks = (a.N + (pair ? 7 : 15)) / (pair ? 8 : 16), least = (blocks + cus - 1) / cus;
  a.nb = 1;
  for (int nb = 2; nb <= 4; ++nb) {
    const int wgs = (blocks + nb - 1) / nb;
    if (wgs >= resident * cus && nb * ((wgs + cus - 1) / cus) <= least) a.nb = nb;
  }
  // (a grid past 2^32 threads is cut short, with no error; 2^28 rows of W, the most of 4 GiB, are 2^24 blocks)
  while ((int64_t)((blocks + a.nb - 1) / a.nb) * 512 >= (int64_t)1 << 32) ++a.nb;
  const dim3 grid((unsigned)((blocks + a.nb - 1) / a.nb), (unsigned)chunks);
  switch (mf) {
    case 1: return launch_form<1>(a, a8, pair, grid, s);
    case 2: return launch_form<2>(a, a8, pair, grid, s);
    case 3: return launch_form<3>(a, a8, pair, grid, s);
    default: return launch_form<4>(a, a8, pair, grid, s);
  }
}

}  // namespace hkx
