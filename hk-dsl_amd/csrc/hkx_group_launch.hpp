// Host-side launchers of the experts' products, one translation unit a kind of tile.
#pragma once

#include <algorithm>

#include "hkx_group.hpp"

namespace hkx {

// (kernel: group_kernel's) hipErrorInvalidConfiguration: more tiles than a launch takes.
hipError_t launch_group(const GroupArgs& a, int op, bool fp8, bool pair, int kernel, int cus, hipStream_t s);

// bm: 16, 64 or 128 rows (TN: 128)
hipError_t launch_group_nt(const GroupArgs& a, bool fp8, bool pair, int bm, hipStream_t s);
hipError_t launch_group_grad(const GroupArgs& a, int op, int bm, hipStream_t s);

// the decode kernel, bm 16 or 32 rows
hipError_t launch_group_skinny(const GroupArgs& a, bool fp8, bool pair, int bm, hipStream_t s);
// 256 x 256 tiles, at most `cus` workgroups
hipError_t launch_group_quad_nt(const GroupArgs& a, bool fp8, bool pair, int cus, hipStream_t s);
hipError_t launch_group_quad_grad(const GroupArgs& a, int op, int cus, hipStream_t s);
// C's rows are stored 16 bytes a lane
inline bool group_quad_ok(const GroupArgs& a) {
  auto whole = [](const void* p, int64_t ld) { return !p || ((uintptr_t)p % 16 == 0 && ld % 16 == 0); };
  return whole(a.c, a.ldc) && a.c_group % 16 == 0 && whole(a.z, a.ldz) && (!a.bias || a.bias_ld * (a.bias_dt == HKX_FP32 ? 4 : 2) % 16 == 0);
}

// The kernel of a call: the one asked for (of the forward product's decode kernels a gradient has none, of tiles TN
// has 128 and 256 rows), or the one that its shape picks.
inline int group_kernel(const GroupArgs& a, int op, bool fp8, bool pair, int kernel, int cus) {
  if (op != kGroupNT && kernel >= kGroupSkinny16) kernel = HKX_EXPERTS_AUTO;
  if (op == kGroupTN && kernel != HKX_EXPERTS_AUTO) return kernel == kGroupQuad ? kGroupQuad : kGroupTile128;
  if (kernel != HKX_EXPERTS_AUTO) return kernel;
  return group_pick({op, fp8, a.experts, a.rows, a.m, pair ? 2 * (int64_t)a.n : a.n, a.k}, group_quad_ok(a), cus);
}

// The 256-row kernel may split its last round along K: the bytes of workspace that takes (0: none; 24 units of K are
// some 36 us a round). Whether it does goes by the counts of rows, which the host does not know: the second launch, that of
// the sums, comes in any case, 5 us of it where no tile is split.
inline size_t group_ws_bytes(const GroupArgs& a, int op, bool fp8, bool pair, int kernel, int cus) {
  if (op == kGroupTN || (int64_t)a.k * (fp8 ? 1 : 2) < 24 * 128 || group_kernel(a, op, fp8, pair, kernel, cus) != kGroupQuad) return 0;
  return (size_t)std::max(cus / 256 * 256, 256) * 256 * 256 * 4;
}

// A grid of `tiles` workgroups and the places that their order over the XCDs leaves open (group_place).
inline bool group_grid(int64_t tiles, int threads, dim3& grid) {
  const int64_t n = (tiles + 255) / 256 * 256;
  if (n * threads >= ((int64_t)1 << 32) || n > INT32_MAX) return false;
  grid = dim3((unsigned)n);
  return true;
}

// The persistent kernel's: a workgroup a CU, whole rounds of places.
inline bool group_quad_grid(int64_t tiles, int cus, dim3& grid) {
  if (tiles > INT32_MAX - 65536) return false;
  grid = dim3((unsigned)std::max(cus / 256 * 256, 256));
  return true;
}

template <int OP, bool FP8, bool PAIR, int BM, int WM, int WN, int FN, int S>
hipError_t launch_group_tile(const GroupArgs& a, hipStream_t s) {
  constexpr int CN = 16 * FN * WN / (PAIR ? 2 : 1);
  const int64_t tn = (a.n + CN - 1) / CN;
  dim3 grid;
  const int64_t tiles = OP == kGroupTN ? (int64_t)a.experts * ((a.m + BM - 1) / BM) * tn : group_tiles(a.rows, a.experts, BM) * tn;
  if (!group_grid(tiles, 64 * WM * WN, grid)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((group_tile_kernel<OP, FP8, PAIR, BM, WM, WN, FN, S>), grid, dim3(64 * WM * WN), 0, s, a);
  return hipGetLastError();
}

}  // namespace hkx
