// The experts' gradient products on tiles (hkx_group.hpp), and the choice of a kernel.
#include "hkx_group_launch.hpp"

namespace hkx {

hipError_t launch_group_grad(const GroupArgs& a, int op, int bm, hipStream_t s) {
  if (op == kGroupTN) return launch_group_tile<kGroupTN, false, false, 128, 2, 2, 4, 4>(a, s);
  if (bm == 16) return launch_group_tile<kGroupNN, false, false, 16, 1, 4, 2, 4>(a, s);
  if (bm == 64) return launch_group_tile<kGroupNN, false, false, 64, 1, 4, 2, 3>(a, s);
  return launch_group_tile<kGroupNN, false, false, 128, 2, 2, 4, 4>(a, s);
}

namespace {

// rows an expert, were they even (the host does not know the counts), and the tiles that such groups would make
int64_t each_rows(const GroupArgs& a) { return (a.rows + a.experts - 1) / a.experts; }
int64_t even_tiles(const GroupArgs& a, int op, int64_t bm, int64_t cn) {
  const int64_t tn = (a.n + cn - 1) / cn;
  return op == kGroupTN ? a.experts * ((a.m + bm - 1) / bm) * tn : std::min<int64_t>(a.experts, a.rows) * ((each_rows(a) + bm - 1) / bm) * tn;
}

}  // namespace

// 256-row tiles where they fill most of the CUs and a group more than a quarter of one (64 groups of 64 rows, 2048 x 2048:
// 139 us against 119 on 64-row tiles; 16 of 100 rows, N = 4096: 58 against 68, their 128 tiles of 2048 columns with K =
// 4096: 97 against 50), 128-row tiles where those fill the CUs, 64-row and, where a group has few rows, 16-row ones.
bool group_quad_takes(const GroupArgs& a, int op, bool pair, int kernel, int cus) {
  if (kernel != HKX_EXPERTS_AUTO) return kernel == HKX_EXPERTS_QUAD;
  return even_tiles(a, op, 256, pair ? 128 : 256) * 5 >= (int64_t)cus * 4 && (each_rows(a) > 64 || op == kGroupTN) && group_quad_ok(a);
}

hipError_t launch_group(const GroupArgs& a, int op, bool fp8, bool pair, int kernel, int cus, hipStream_t s) {
  if (group_quad_takes(a, op, pair, kernel, cus))
    return op == kGroupNT ? launch_group_quad_nt(a, fp8, pair, cus, s) : launch_group_quad_grad(a, op, cus, s);
  const int64_t each = each_rows(a);
  // The decode kernel for up to 8 rows an expert and 2048 bytes along K (64 experts, 8 rows each: 98 us against 103 on
  // 16-row tiles; 16 each 117 against 103; 8 each over 1024 bytes 39 against 30 on 64-row tiles, which read a favoured
  // expert's W once and, with as little to do, have fewer workgroups to start).
  const int64_t row = (int64_t)a.k * (fp8 ? 1 : 2);
  const bool few = kernel == HKX_EXPERTS_AUTO && each <= 8 && row >= 2048;
  if (op == kGroupNT && (kernel == HKX_EXPERTS_SKINNY16 || kernel == HKX_EXPERTS_SKINNY32 || few))
    return launch_group_skinny(a, fp8, pair, kernel == HKX_EXPERTS_SKINNY16 || (few && each <= 4) ? 16 : 32, cus, s);
  const int bm = kernel == HKX_EXPERTS_TILE16 ? 16 : kernel == HKX_EXPERTS_TILE64 ? 64 : kernel == HKX_EXPERTS_TILE128 ? 128
                 : each <= 4 || (each <= 16 && row >= 2048) ? 16 : each > 64 && even_tiles(a, op, 128, pair ? 64 : 128) >= cus ? 128 : 64;
  return op == kGroupNT ? launch_group_nt(a, fp8, pair, bm, s) : launch_group_grad(a, op, bm, s);
}

}  // namespace hkx
