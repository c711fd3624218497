// The experts' products' choice between their kernels, by shape and CUs alone: plain C++, no HIP, so that a host program
// can ask it.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace hkx {

// The products and the kernels (HKX_EXPERTS_* of hkx.h).
constexpr int kGroupNT = 0, kGroupNN = 1, kGroupTN = 2;
constexpr int kGroupTile16 = 1, kGroupTile64 = 2, kGroupTile128 = 3, kGroupQuad = 4, kGroupSkinny16 = 5, kGroupSkinny32 = 6;

// n: C's columns, of the paired form its gate and up rows of B together; k: the contraction (not TN); m: TN's rows of C.
struct GroupShape {
  int op;
  bool fp8;
  int64_t experts, rows, m, n, k;
};

// A kernel's estimated time in us: a launch and a chain of K units (of 128 bytes; a decode kernel's waves share them), more as
// the tiles that the groups make by estimate fill the CUs; joined (as the 4th powers) with the
// operands' bytes at 6 TB/s. The host does not know the counts of rows. Fitted to 1615 timed calls (2-256 experts of 1-8192
// rows, N 64-28672, K 64-14400, random counts, cold weights, all kernels of each; within 15-21% of the times).
struct GroupCost {
  double launch, chain, unit, fill;
};
inline double group_cost(const GroupShape& s, int kernel, int cus) {
  static constexpr GroupCost fp8[] = {{3.36, 1.19, 0.354, 2.02}, {3.43, 1.77, 0.442, 2.45}, {2.12, 4.43, 0.520, 1.68},
                                      {10.52, 1.81, 0.839, 2.34}, {4.58, 0.33, 0.234, 5.95}, {5.24, 0.24, 0.186, 9.57}};
  static constexpr GroupCost bf16[] = {{2.98, 1.12, 0.305, 2.05}, {2.80, 1.75, 0.439, 2.07}, {0.88, 4.78, 0.528, 1.27},
                                       {9.60, 3.07, 0.725, 2.03}, {4.17, 0.40, 0.267, 4.76}, {4.52, 0.46, 0.312, 5.25}};
  static constexpr GroupCost nn[] = {{2.38, 1.41, 0.307, 1.82}, {2.46, 1.65, 0.408, 2.01}, {1.01, 4.07, 0.520, 1.19},
                                     {12.40, 0.46, 0.461, 3.65}};
  static constexpr GroupCost tn[] = {{2.69, 2.72, 0.821, 1.16}, {7.78, 0.08, 1.164, 1.76}};
  static constexpr double rows_of[] = {16, 64, 128, 256, 16, 32}, cols_of[] = {128, 128, 128, 256, 32, 32}, resident[] = {2, 2, 1, 1, 2, 2};
  const int i = kernel - 1;
  const GroupCost& c = s.op == kGroupTN ? tn[i - 2] : s.op == kGroupNN ? nn[i] : s.fp8 ? fp8[i] : bf16[i];
  const double groups = (double)std::min(s.experts, s.rows), each = std::ceil((double)s.rows / (double)s.experts);
  const double es = s.fp8 ? 1 : 2, across = std::ceil((double)s.n / cols_of[i]);
  double tiles, units, bytes;
  if (s.op == kGroupTN) {
    tiles = (double)s.experts * std::ceil((double)s.m / rows_of[i]) * across;
    units = (double)s.rows / (double)s.experts / 64 + 0.5;
    bytes = 2 * ((double)s.experts * s.m * s.n + (double)s.rows * (double)(s.m + s.n));
  } else {
    // (few rows a group: some groups have none; many: a ragged tile and an imbalance)
    tiles = groups * (each / rows_of[i] + 1 - 0.5 * std::exp(-2 * each / rows_of[i])) * across;
    units = std::ceil((double)s.k * es / 128);
    bytes = groups * (double)s.n * (double)s.k * es;
  }
  if (kernel == kGroupQuad) units = std::max(units, 5.0);
  if (kernel >= kGroupSkinny16) units = std::ceil(units / 4);
  const double full = c.fill * tiles / (resident[i] * cus);
  const double work = (c.chain + c.unit * units) * std::sqrt(1 + full * full), memory = bytes / 6e6;
  return c.launch + std::sqrt(std::sqrt(work * work * work * work + memory * memory * memory * memory));
}

// The kernel of a call; quad: whether its rows suit the 256-row kernel. Up to 8 rows an expert of 24 units of K or more a
// decode kernel: of 87 such calls to 4 rows it took 0.38-1.16 times the 16-row tiles' time (median 0.89), with fewer units
// 0.55-2.34, where the cost decides as for all else. Of 749 other calls, not in the fit, the pick takes 1.02 times the best
// kernel's time on average and 1.14 at the 95th hundredth (NN 1.03 and 1.22, TN 1.00 and 1.04). Steps at sizes in place
// of the cost (256-row tiles where they fill four fifths of the CUs, then 128 rows where those fill them, then 64) had 1.10 and
// 1.47 (NN 1.06 and 1.29, TN 1.04 and 1.37).
inline int group_pick(const GroupShape& s, bool quad, int cus) {
  const int64_t each = (s.rows + s.experts - 1) / s.experts;
  if (s.op == kGroupNT && each <= 8 && s.k * (s.fp8 ? 1 : 2) > 23 * 128) return each <= 4 ? kGroupSkinny16 : kGroupSkinny32;
  int best = 0;
  double least = 0;
  for (int k = s.op == kGroupTN ? kGroupTile128 : kGroupTile16; k <= (s.op == kGroupNT ? kGroupSkinny32 : kGroupQuad); ++k) {
    if (k == kGroupQuad && !quad) continue;
    const double c = group_cost(s, k, cus);
    if (!best || c < least) best = k, least = c;
  }
  return best;
}

}  // namespace hkx
