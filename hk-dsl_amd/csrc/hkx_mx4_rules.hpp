// The MXFP4 product's choice between its kernels, by shape and CUs alone: plain C++, no HIP, so that a
// host program can ask it.
#pragma once

#include <algorithm>
#include <cstdint>

namespace hkx {

// The kernels (HKX_MX4_* of hkx.h).
constexpr int kMx4Tile64 = 1, kMx4Tile128 = 2, kMx4Quad = 3, kMx4Skinny = 4;

struct Mx4Plan {
  int kernel, splits;
};

inline int mx4_rows(int kernel) { return kernel == kMx4Quad ? 256 : kernel == kMx4Tile128 ? 128 : 64; }
inline int mx4_cols(int kernel, bool pair) { return (kernel == kMx4Quad ? 256 : 128) / (pair ? 2 : 1); }

// 256-K units a split of at most s: the quadrant kernel's start at whole chunks of two units.
inline int mx4_split_units(int kernel, int units, int s) {
  const int per = (units + s - 1) / s;
  return kernel == kMx4Quad && s > 1 ? (per + 1) / 2 * 2 : per;
}
// The splits that leaves, none empty.
inline int mx4_splits(int kernel, int units, int s) {
  const int per = mx4_split_units(kernel, units, s);
  return (units + per - 1) / per;
}

// Whether a call runs on the decode kernel (workgroups of 16 rows of B and up to 64 of A). How many times its
// time the plan takes that mx4_cost picks among the other kernels, from the least to the most of 1772 shapes
// (512-28672 rows of B, K 1024-14336, cold weights; rows of B are twice the columns in the paired form):
// * to 64 rows of A, K to 4096: 1.08-2.46 to 16384 rows of B; 20480 and 28672 rows 1.05-1.86 and 0.87-1.82
//   (medians 1.1, 1.0) to M = 16, 0.38-0.99 past it;
// * K past 4096, where A is streamed with every 16 rows of B, M to 8: 4-bit A 1.03-1.72 to 16384 rows, 0.65-1.23
//   past them, 8-bit A 1.06-1.56 to 8192, 0.57-1.36 past; M = 9-16: 0.99-1.71 to 4096 rows, at 8192 0.97-1.15 to
//   K = 8192 and 0.90-1.16 past it, 0.51-1.31 from 12288 on; M = 17-32 to 4096 rows: 4-bit A 1.06-1.48 to K =
//   8192, 0.82-1.21 past it, 8-bit A 0.91-1.17 to 6144, 0.69-1.12 past it; more rows 0.30-1.25; M = 33-64: 4-bit
//   A 0.99-1.51 to 4096 rows and K = 8192, else 0.36-1.10; 8-bit A 0.28-1.21. Where it is above 1 and not
//   taken it is mostly the pick's split: the best other plan of 12288 rows and more takes 1.15 at most;
// * 65 to 512 rows of A, K to 4096: to one workgroup a CU 1.32-2.24, to two 1.12-1.58 (4-bit A), 0.86-1.46 (8-bit
//   to 256 rows of A) and 0.88-1.41 (past them), past two 0.26-1.18; K 5120-8192 of 4 bits to one a CU
//   0.95-1.35 to 256 rows of A and 1.15-1.27 past them, to two 0.67-1.02; 8-bit A 0.52-1.03.
// Both choices together take 1.03 times the best plan's time on average, 1.22 at the 95th hundredth (1.015 and
// 1.09 past 64 rows of A).
inline bool mx4_skinny_wins(int m, int rows, int k, bool a8, int cus) {
  const int64_t wgs = (int64_t)((m + 63) / 64) * ((rows + 15) / 16);
  if (m > 64 && k <= 4096) return m <= 512 && wgs <= (a8 && m > 256 ? cus : 2 * cus);
  if (m > 64) return !a8 && m <= 256 && wgs <= cus && k <= 8192;
  if (k <= 4096) return m <= 16 || rows <= 16384;
  if (m > 32) return !a8 && rows <= 4096 && k <= 8192;
  if (m > 16) return rows <= 4096 && k <= (a8 ? 6144 : 8192);
  if (m > 8) return rows <= 4096 || (rows <= 8192 && k <= 8192);
  return rows <= (a8 ? 8192 : 16384);
}

// A plan's estimated time in us: a launch, more for each further wave of workgroups, a time a 256-K unit
// and wave and one for its share of the memory's traffic, and where it goes through fp32 shares their
// sum's launch and their round trip. Fitted to 1740 timed plans (M 33-4096, N 512-24576, K 512-12288,
// weights past the cache); over 2168 timed since the tiles' scales come by four threads a row: medians
// 1.00-1.02 of the times, 0.85-0.94 and 1.13-1.24 at the tenths; the plans it picks take 1.005 times the best
// one's on average, 1.04 at the 95th hundredth (M to 32, not fitted: 1.07 and 1.33). Waves are whole ones also
// where two workgroups share a CU (0.83 of their number past one, as fitted before, picked plans of 1.02
// times: 777 x 4096 x 12288 of 4 bits as 448 workgroups 45.1 us, as 224 38.7). A C of odd columns or alignment goes through
// shares on the quadrant kernel always (stored from its registers two bytes at a time 3000 x 1001 took 25
// us more).
inline double mx4_cost(int kernel, int m, int n, int k, bool a8, bool pair, bool vec, int splits, int cus) {
  static const double kC[2][3][6] = {
      // launch, wave, unit, unit x filled, sum, share bytes
      {{4.3, 0.0, 0.437, 0.155, 2.1, 1.10}, {5.5, 0.2, 0.646, 0.116, 2.3, 0.88}, {10.3, 8.2, 1.296, 0.539, 5.5, 0.64}},
      {{4.5, 0.0, 0.552, 0.194, 2.0, 1.00}, {5.4, 2.8, 0.977, 0.172, 2.5, 0.86}, {10.0, 7.7, 1.980, 0.638, 5.5, 0.63}}};
  const double* c = kC[a8][kernel - 1];
  const int bm = mx4_rows(kernel), bn = mx4_cols(kernel, pair);
  const int per = mx4_split_units(kernel, (k + 255) / 256, splits);
  const double w = (double)((m + bm - 1) / bm) * ((n + bn - 1) / bn) * splits / cus;
  const double waves = w <= 1 ? 1.0 : (double)(int64_t)(w + 0.9999);
  double t = c[0] + c[1] * (waves - 1) + c[2] * per * waves + c[3] * per * std::min(w, 1.0);
  if (splits > 1 || (kernel == kMx4Quad && !vec)) t += c[4] + c[5] * splits * m * (pair ? 2.0 : 1.0) * n * 8.0 / 5e6;
  return t;
}

// quad_ok: the quadrant kernel takes the call; vec: C's rows are whole 16-byte pieces.
inline Mx4Plan mx4_plan(int m, int n, int k, bool a8, bool pair, bool quad_ok, bool vec, int cus) {
  if (mx4_skinny_wins(m, pair ? 2 * n : n, k, a8, cus)) return {kMx4Skinny, 1};
  const int units = (k + 255) / 256;
  Mx4Plan best{kMx4Tile64, 1};
  double t = 1e30;
  for (int kernel = kMx4Tile64; kernel <= kMx4Quad; ++kernel) {
    if ((kernel == kMx4Quad && (!quad_ok || m <= 128)) || (kernel == kMx4Tile128 && m <= 64)) continue;
    for (int s = 1; s <= 8; s *= 2) {
      if (s > 1 && (units < 2 * s || mx4_splits(kernel, units, s) != s)) continue;
      const double e = mx4_cost(kernel, m, n, k, a8, pair, vec, s, cus);
      if (e < t) t = e, best = {kernel, s};
    }
  }
  return best;
}

}  // namespace hkx
