// The experts' forward product for few rows an expert (decode): 16 or 32 rows of C a tile, W read once.
//
// Bound by HBM: the touched experts' weights. A short workgroup of 4 waves owns 32 rows of an expert's W (paired: 16 gate
// and the 16 up rows of the same columns); the waves cut K, wave w the units of 128 bytes w, w + 4, ..., each with its own four slots
// of LDS that its own DMA fills (non-temporal, whole lines) and its own rows of A straight to registers: no barrier until the
// waves' sums meet. Two workgroups a CU, 128 KB of W in flight. One token's 8 of 64 experts, 2048 columns of 2048: 14.8 us;
// 128 workgroups of 128 rows with a barrier a unit, 48 KB in flight on half the CUs, took 20.7. A short K makes a workgroup
// little more than its start; such calls go to the tiles by their cost (64 experts of 2048 rows, 1024 bytes each, 64 tokens: 52
// us here, 27-30 on 64-row tiles).
//
// Which expert a tile is, is found by each wave from the offsets (a map in LDS and its barriers come before the first load).
#pragma once

#include "hkx_group.hpp"

namespace hkx {

// The group of tile row i of BM rows, and the tile's first row in it; -1: no such tile.
template <int BM>
HKX_DEV int group_find(const GroupArgs& p, int i, int& m0) {
  const int lane = threadIdx.x & 63, groups = p.experts + 1;
  int before = 0;
  for (int g = 0; g < groups; g += 64) {
    int n = 0;
    if (g + lane < groups) {
      int lo, hi;
      group_rows(p, g + lane, lo, hi);
      n = (hi - lo + BM - 1) / BM;
    }
    int sum = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(sum, d);
      if (lane >= d) sum += u;
    }
    const unsigned long long past = __ballot(before + sum > i);
    if (past) {
      const int who = __builtin_ctzll(past);
      m0 = (i - (before + __builtin_amdgcn_readlane(sum - n, who))) * BM;
      return g + who;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return -1;
}

template <bool FP8, bool PAIR, int MF>
__global__ void __launch_bounds__(256) group_skinny_kernel(const GroupArgs p) {
  constexpr int BM = 16 * MF, BN = 32, CN = PAIR ? 16 : 32, S = 4;
  constexpr int ES = FP8 ? 1 : 2, KU = 128 / ES, KH = FP8 ? 1 : 2;
  constexpr int NV = 4 + 2 * MF;  // loads of a unit
  constexpr int PART = 4 * S * 4096;  // then the waves' sums
  __shared__ __attribute__((aligned(16))) uint8_t smem[PART + 4 * MF * 2 * 1024];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rf = lane & 15, q = lane >> 4;
  const int tiles_n = (p.n + CN - 1) / CN;
  const int place = group_place((int)blockIdx.x);
  int m0;
  const int e = group_find<BM>(p, place / tiles_n, m0);
  if (e < 0) return;
  const int n0 = place % tiles_n * CN;
  int lo, hi;
  group_rows(p, e, lo, hi);
  const int64_t row0 = (int64_t)lo + m0;
  const int rows = min(hi - (int)row0, BM);
  const bool rest = e == p.experts;  // the rows behind the last group
  const uint32_t k_row = (uint32_t)p.k * ES;
  const int nku = rest ? 0 : (p.k + KU - 1) / KU;

  // ---- W: instruction i moves rows 8 i + [0, 8): lane l row l / 8, its 16-byte chunk (l % 8) ^ (row % 8)
  const uint32_t chunk = (uint32_t)((lane % 8) ^ (lane / 8)) * 16u;
  const __amdgpu_buffer_rsrc_t rb = group_rsrc(p.b + (rest ? 0 : e) * p.b_group + n0 * p.ldb, (PAIR ? p.n : 0) + min(p.n - n0, CN), p.ldb, k_row);
  uint32_t vb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) vb[i] = (uint32_t)(PAIR ? 8 * (i & 1) + lane / 8 + (i >> 1) * p.n : 8 * i + lane / 8) * (uint32_t)p.ldb + chunk;
  uint8_t* const mine = smem + wave * (S * 4096);
  // ---- A: lane (rf, q) 16 bytes of each half unit of row rf
  const __amdgpu_buffer_rsrc_t ra = p.index ? group_rsrc(p.a, p.a_rows, p.lda, k_row) : group_rsrc(p.a + row0 * p.lda, rows, p.lda, k_row);
  uint32_t va[MF];

  // Unit u's W into slot s, its A into registers. Past the contraction's end (a ragged last unit's lanes, units past the
  // wave's last) an offset is out of range, with no branch: behind one the compiler's count of the loads in flight is short.
  const uint32_t k_end = rest ? 0u : k_row;
  auto fill = [&](int u, int s) {
    const uint32_t so = (uint32_t)u * 128u, at = min(so, k_row);
    const bool in = so + chunk < k_end;
#pragma unroll
    for (int i = 0; i < 4; ++i) buf_load16_lds<kNonTemporal>(rb, mine + s * 4096 + i * 1024, in ? vb[i] : kGroupOut, at);
  };
  i32x4 a[S][MF][2];
  auto load_a = [&](int u, int s) {
    const uint32_t so = (uint32_t)u * 128u, at = min(so, k_row);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool in = so + 64u * h + 16u * q < k_end;
#pragma unroll
      for (int m = 0; m < MF; ++m) a[s][m][h] = buf_load16(ra, in ? va[m] + 64u * h : kGroupOut, at);
    }
  };
  // (W does not wait for the row numbers)
#pragma unroll
  for (int s = 0; s < S; ++s) fill(wave + 4 * s, s);
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    const int r = 16 * m + rf;
    int64_t at = r < rows ? r : -1;
    if (p.index) {
      const int j = r < rows ? p.index[row0 + r] : -1;
      at = (uint32_t)j < (uint32_t)p.a_rows ? j : -1;
    }
    va[m] = at < 0 ? kGroupOut - 64u : (uint32_t)(at * p.lda) + 16u * q;  // (out also 64 bytes on)
  }
#pragma unroll
  for (int s = 0; s < S; ++s) load_a(wave + 4 * s, s);

  using Frag = typename std::conditional<FP8, i32x8, bf16x8>::type;
  f32x4 acc[MF][2] = {};
  auto eight = [](i32x4 x, i32x4 y) { return i32x8{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w}; };
  // The units in the slots and registers; in their place units un + 4 s.
  auto round = [&](int un) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      // (all but the three later units' loads; the first round's W is older than any A, which its registers wait for)
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(wait_vm((S - 1) * NV));
      __builtin_amdgcn_sched_barrier(0);
      const uint8_t* w = mine + s * 4096;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const uint8_t* row = w + (16 * g + rf) * 128;
        const i32x4 x = *(const i32x4*)(row + ((q ^ (rf & 7)) << 4)), y = *(const i32x4*)(row + (((4 + q) ^ (rf & 7)) << 4));
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          if constexpr (FP8) {
            acc[m][g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(eight(x, y), eight(a[s][m][0], a[s][m][1]), acc[m][g], 0, 0, 0, 0, 0, 0);
          } else {
            acc[m][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, a[s][m][0]), acc[m][g], 0, 0, 0);
            acc[m][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, y), __builtin_bit_cast(bf16x8, a[s][m][1]), acc[m][g], 0, 0, 0);
          }
        }
      }
      // the slot is read: its next unit's fill may land
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(wait_lgkm0());
      __builtin_amdgcn_sched_barrier(0);
      fill(un + 4 * s, s);
      load_a(un + 4 * s, s);
    }
  };
  // A wave's rounds, at least one (of zeros, where K has no unit for it). (The first by itself: its loads came in another
  // order, and one wait that held for both would be the shorter.)
  const int rounds = max(1, (nku - wave + 4 * S - 1) / (4 * S));
  round(wave + 4 * S);
  for (int t = 1; t < rounds; ++t) round(wave + 4 * S * (t + 1));
  // The waves' sums, in order; lane (rf, q) holds row rf, columns 4 q + [0, 4) of each fragment. (No wait for the
  // fills in flight, as __syncthreads has it.)
  f32x4* const part = (f32x4*)(smem + PART);
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int g = 0; g < 2; ++g) part[(wave * 2 * MF + 2 * m + g) * 64 + lane] = acc[m][g];
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(wait_lgkm0());
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  auto sum = [&](int f) {
    f32x4 v = part[f * 64 + lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) v += part[(w * 2 * MF + f) * 64 + lane];
    return v;
  };
  const int m = PAIR ? wave : wave >> 1, g = wave & 1;  // a wave's fragment (paired: both of a row block)
  const int r = 16 * m + rf, n = n0 + (PAIR ? 0 : 16 * g) + 4 * q;
  if (m < MF && r < rows && n < p.n) {
    const float sa = FP8 && !rest ? group_row_scale(p, row0 + r) : 1.0f;
    group_store<true, FP8, PAIR>(p, e, rest, p.c + (row0 + r) * p.ldc, PAIR ? p.z + (row0 + r) * p.ldz : nullptr, n,
                                 sum(PAIR ? 2 * m : 2 * m + g), PAIR ? sum(2 * m + 1) : f32x4{}, sa);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no fill lands in LDS after the exit
}

}  // namespace hkx
