// The experts' products on 256 x 256 tiles: one persistent workgroup of 8 waves a CU, in the quadrant kernel's order
// (hkx_quad.hpp: its wave map, whole-line fills, phases and waits), over the tiles of all groups one after another.
//
// What the groups add:
// * A tile's group, rows and columns are found once, in the tile before it (at its first K unit), from the map of tile
//   rows in LDS; a tile therefore has at least 5 K units, shorter ones (few rows of an expert in TN, the rows behind the
//   last) padded with units that read as zeros and cost no memory traffic.
// * Fills go through a resource a tile from 64-bit addresses. Operands that lie along K (NN's B, TN's A and B) move on by
//   64 rows a unit, and their fragments are turned on the way from LDS (hkx_group.hpp).
// * NT's rows by index: a tile's 256 row numbers reach LDS by DMA during the tile before it, where the fills' offsets
//   are made from them; 8-bit rows' scales by a DMA of one word a lane from the same numbers.
// * Vectors (scales, bias) of a tile stand in slot (tile % 3), filled when its first fills are issued.
//
// K past its end: K-contiguous pieces out of range, rows along K past the resource: zeros in both operands.
#pragma once

#include "hkx_group.hpp"

namespace hkx {

constexpr int kQuadUnits = 5;  // K units a tile at least

// The kernel's arguments, read anew: what only a tile's beginning and end take of them is not held through the K loop
// (held, they filled the scalar registers, and what was moved to vector lanes cost a lane's read a use).
HKX_DEV const GroupArgs& args_anew() {
  auto k = (const __attribute__((address_space(4))) GroupArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(k));
  return *(const GroupArgs*)k;
}

template <int OP, bool FP8, bool PAIR>
__global__ void __launch_bounds__(512, 1) group_quad_kernel(const GroupArgs p) {
  constexpr bool TA = OP == kGroupTN, TB = OP != kGroupNT, NT = OP == kGroupNT;
  constexpr int BM = 256, BN = PAIR ? 128 : 256;  // BN: C columns of a tile
  constexpr int ES = FP8 ? 1 : 2, KU = 128 / ES, KH = FP8 ? 1 : 2;
  constexpr int QB = 128 * 128;
  constexpr int VEC = 8 * QB;              // [tile % 3][row scales 1 KB, column scales 1 KB, bias 2 KB]
  constexpr int IDX = VEC + 3 * 4096;      // [tile % 2][256 row numbers]
  constexpr int MAP = NT ? IDX + 2 * 1024 : VEC;
  constexpr int STARTS = MAP + (TA ? 0 : (int)sizeof(GroupMap));
  constexpr int SMEM = STARTS + 4 * (kMaxExperts + 1);
  static_assert(SMEM <= 160 * 1024, "LDS");
  // (one array: beside a second one the compiler waits for every fill before each LDS read)
  __shared__ __attribute__((aligned(16))) uint8_t smem[SMEM];
  GroupMap& map = *(GroupMap*)(smem + MAP);
  int* const starts = (int*)(smem + STARTS);  // the groups' first rows (from memory a read would wait for the fills)

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave >> 2, wc = wave & 3;
  const int tiles_n = (p.n + BN - 1) / BN;

  for (int g = tid; g <= p.experts; g += 512) starts[g] = min(max(p.offsets[g], 0), p.rows);
  if constexpr (TA) __syncthreads();
  else group_map<BM>(map, p, tid, 512);
  auto rows_of = [&](int g, int& lo, int& hi) {  // (group_rows)
    const GroupArgs& p = args_anew();
    lo = starts[g];
    hi = g < p.experts ? max(starts[g + 1], lo) : p.tail ? p.rows : lo;
  };
  const int total = __builtin_amdgcn_readfirstlane(TA ? p.experts * ((p.m + BM - 1) / BM) * tiles_n
                                                      : map.first[p.experts + 1] * tiles_n);
  // the workgroup's tiles: places of v, v + grid, ... (grid a multiple of 8, so all on its XCD's stretch)
  const int per = (total + 7) >> 3, x = (int)blockIdx.x & 7, y0 = (int)blockIdx.x >> 3, step = (int)gridDim.x >> 3;
  const int my_tiles = max(0, (min(per, total - x * per) - y0 + step - 1) / step);
  if (my_tiles == 0) return;
  auto tile_at = [&](int lt) {
    const GroupArgs& p = args_anew();
    GroupTile t = group_tile_at<OP, BM, BN>(map, p, x * per + y0 + lt * step, tiles_n, rows_of);
    t.e = __builtin_amdgcn_readfirstlane(t.e);
    t.m0 = __builtin_amdgcn_readfirstlane(t.m0);
    t.n0 = __builtin_amdgcn_readfirstlane(t.n0);
    t.rows = __builtin_amdgcn_readfirstlane(t.rows);
    t.klen = __builtin_amdgcn_readfirstlane(t.klen);
    t.row0 = (int64_t)__builtin_amdgcn_readfirstlane((int)t.row0);
    return t;
  };
  auto units = [&](const GroupTile& t) { return max((t.klen + KU - 1) / KU, kQuadUnits); };

  // ---- fills. Instruction k (0, 1) of wave w: K-contiguous rows 16 w + 8 k + [0, 8) of a quarter, lane l row l % 32 / 4,
  // K-half l / 32, its 16-byte piece (l % 4) ^ swz4(row); rows along K 8 w + 4 k + [0, 4), lane l row l / 16.
  uint32_t la[2], lb[2], lch[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t r = (uint32_t)(16 * wave + 8 * k + (lane & 31) / 4);
    const uint32_t rb = PAIR ? (uint32_t)(16 * (wave >> 1) + 8 * k + (lane & 31) / 4 + ((wave & 1) ? p.n : 0)) : r;
    lch[k] = (uint32_t)(64 * (lane >> 5) + 16 * ((lane & 3) ^ ((wave & 1) | (k << 1))));
    const uint32_t kr = (uint32_t)(8 * wave + 4 * k + lane / 16), kc = (uint32_t)((lane % 16) ^ (group_swz(kr) << 1)) * 16u;
    la[k] = TA ? kr * (uint32_t)p.lda + kc : r * (uint32_t)p.lda + lch[k];
    lb[k] = TB ? kr * (uint32_t)p.ldb + kc : rb * (uint32_t)p.ldb + lch[k];
  }
  const uint32_t k_row = (uint32_t)p.k * ES;  // NT, NN: bytes of a K-contiguous row

  // The two fill streams: s1 a unit ahead (A1), s2 two (A0, B0, B1).
  struct Ahead {
    int t, nkt, par;           // its unit in its tile, the tile's units, its slot
    int left;                  // TN, NN: rows along K that are left
    const uint8_t *a, *b;
    uint32_t ba, bb;           // the resources' bytes; of rows along K a row's
    uint32_t b1;               // B's second half behind the first (0: past N, the first again: it is never stored)
    uint32_t va[2];            // offsets of A's half
  };
  const bool gathered = NT && p.index != nullptr;
  const int32_t* const idx_lds = (const int32_t*)(smem + IDX);
  auto rows_bytes = [](int rows, int64_t ld, uint32_t row) { return rows > 0 ? (uint32_t)((rows - 1) * ld) + row : 0u; };
  // a lane's row of a half, instruction k (made where a tile begins: held through the K loop it would spill)
  auto row_a = [&](int k) {
    int l = lane;
    asm volatile("" : "+v"(l));
    return 16 * wave + 8 * k + (l & 31) / 4;
  };
  // A's offsets of half i from its row numbers
  auto offset_of = [&](int j, int k) { return (uint32_t)j < (uint32_t)p.a_rows ? (uint32_t)j * (uint32_t)p.lda + lch[k] : kGroupOut; };
  auto begin_a = [&](Ahead& s, const GroupTile& t, int i) {
    const GroupArgs& p = args_anew();
    if constexpr (TA) {
      const int m = t.m0 + (t.rows > 128 * i ? 128 * i : 0);  // (a half past M: the first again)
      s.a = p.a + t.row0 * p.lda + (int64_t)m * 2;
      s.ba = (uint32_t)(p.m - m) * 2u;
      s.left = t.klen;
    } else if (gathered) {
      s.a = p.a;
      s.ba = t.klen ? rows_bytes(p.a_rows, p.lda, k_row) : 0u;
    } else {
      s.a = p.a + (t.row0 + 128 * i) * p.lda;
      s.ba = t.klen ? rows_bytes(t.rows - 128 * i, p.lda, k_row) : 0u;
    }
  };
  auto begin_b = [&](Ahead& s, const GroupTile& t) {
    const GroupArgs& p = args_anew();
    const int e = t.klen ? t.e : 0;
    constexpr int HB = PAIR ? 64 : 128;
    s.b1 = t.n0 + HB < p.n ? (TB ? HB * 2u : (uint32_t)HB * (uint32_t)p.ldb) : 0u;
    s.bb = (uint32_t)(p.n - t.n0) * 2u;
    if constexpr (TA) {
      s.b = p.b + t.row0 * p.ldb + (int64_t)t.n0 * 2;
    } else if constexpr (TB) {
      s.b = p.b + e * p.b_group + (int64_t)t.n0 * 2;
      s.left = t.klen;
    } else {
      s.b = p.b + e * p.b_group + t.n0 * p.ldb;
      s.bb = t.klen ? rows_bytes((PAIR ? p.n : 0) + min(p.n - t.n0, BN), p.ldb, k_row) : 0u;
    }
  };
  auto fill2 = [&](const uint8_t* base, uint32_t bytes, uint8_t* slot, const uint32_t (&v)[2], uint32_t so, bool straight, bool ends) {
    const __amdgpu_buffer_rsrc_t r = make_rsrc(base, bytes);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      buf_load16_lds(r, slot + wave * 2048 + k * 1024, straight && ends && so + lch[k] >= k_row ? kGroupOut : v[k], so);
  };
  // half i of A (B) of stream s's unit into its slot
  auto fill_a = [&](const Ahead& s, int i) {
    uint8_t* slot = smem + (s.par * 4 + i) * QB;
    if constexpr (TA) {
      fill2(s.a, rows_bytes(min(s.left, 64), p.lda, s.ba), slot, la, 0, false, false);
    } else {
      const uint32_t so = (uint32_t)s.t * 128u;
      const bool in = s.ba != 0 && so < k_row;
      const bool ends = in && so + 128u > k_row;
      fill2(s.a, in ? s.ba : 0u, slot, NT ? s.va : la, in ? so : 0u, true, ends);
    }
  };
  auto fill_b = [&](const Ahead& s, int j) {
    uint8_t* slot = smem + (s.par * 4 + 2 + j) * QB;
    const uint32_t c = j ? s.b1 : 0u;
    if constexpr (TB) {
      fill2(s.b + c, rows_bytes(min(s.left, 64), p.ldb, s.bb - c), slot, lb, 0, false, false);
    } else {
      const uint32_t so = (uint32_t)s.t * 128u;
      const bool in = s.bb != 0 && so < k_row;
      fill2(s.b + c, in ? s.bb - c : 0u, slot, lb, in ? so : 0u, true, in && so + 128u > k_row);
    }
  };

  // ---- a tile's vectors and row numbers
  uint8_t* const vecs = smem + VEC;
  [[maybe_unused]] auto fill_index = [&](const GroupTile& t, int lt) {  // wave 7
    if (!gathered || wave != 7) return;
    const GroupArgs& p = args_anew();
    const __amdgpu_buffer_rsrc_t r = make_rsrc(p.index + t.row0, (uint32_t)t.rows * 4u);
#pragma unroll
    for (int i = 0; i < 4; ++i)  // (a word a lane: a tile's first row number may stand anywhere)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(smem + IDX + (lt & 1) * 1024 + i * 256), 4,
                                               (uint32_t)(64 * i + lane) * 4u, 0, 0, 0);
  };
  [[maybe_unused]] auto fill_vectors = [&](const GroupTile& t, int lt, const int32_t* index) {
    uint8_t* s = vecs + (lt % 3) * 4096;
    if (t.klen == 0) return;
    const GroupArgs& p = args_anew();
    const int32_t bias_es = p.bias_dt == HKX_FP32 ? 4 : 2;
    if constexpr (FP8) {
      if (wave < 4 && p.sa_ld) {  // a word a lane: rows 64 w + l
        const int r = 64 * wave + lane;
        uint32_t at = kGroupOut;
        if (r < t.rows) at = gathered ? ((uint32_t)index[r] < (uint32_t)p.a_rows ? (uint32_t)index[r] * 4u : kGroupOut) : (uint32_t)r * 4u;
        const __amdgpu_buffer_rsrc_t rs = gathered ? make_rsrc(p.sa, (uint32_t)p.a_rows * 4u) : make_rsrc(p.sa + t.row0, (uint32_t)t.rows * 4u);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(s + wave * 256), 4, at, 0, 0, 0);
      }
      if (wave == 4 && p.sb_col) {  // columns, or 128 gate and 128 up columns
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.sb + t.e * p.sb_ld, (uint32_t)p.n * (PAIR ? 8u : 4u));
        const uint32_t at = PAIR ? (uint32_t)(t.n0 + (lane & 31) * 4 + (lane >> 5) * p.n) * 4u : (uint32_t)(t.n0 + lane * 4) * 4u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(s + 1024), 16, at, 0, 0, 0);
      }
    }
    if (p.bias && (wave == 5 || (PAIR && wave == 6))) {
      const int up = wave == 6;
      const __amdgpu_buffer_rsrc_t rs = make_rsrc((const uint8_t*)p.bias + (t.e * p.bias_ld + (up ? p.n : 0)) * bias_es, (uint32_t)(p.n * bias_es));
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)(s + 2048 + up * 1024), 16,
                                               (uint32_t)(t.n0 * bias_es + lane * 16), 0, 0, 0);
    }
  };

  // ---- fragments
  const int rf = lane & 15, q = lane >> 4;
  uint32_t rdo[2];
#pragma unroll
  for (int par = 0; par < 2; ++par) rdo[par] = (uint32_t)((rf >> 3) * 1024 + (rf & 7) * 64 + ((q ^ (par | ((rf >> 3) << 1))) << 4));
  constexpr int NA = 4, NB = 2;
  using Frag = typename std::conditional<FP8, i32x8, bf16x8>::type;
  Frag af[NA][2], bf0[NB][2], bf1[NB][2], bfn[NB][2];
  auto straight = [&](const uint8_t* s, int r0, int h, int par) -> Frag {
    if constexpr (FP8) {
      const i32x4 lo = *(const i32x4*)(s + r0 * 128 + rdo[par]), hi = *(const i32x4*)(s + r0 * 128 + 512 + rdo[par]);
      return i32x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    } else {
      return *(const bf16x8*)(s + r0 * 128 + h * 512 + rdo[par]);
    }
  };
  auto read_b = [&](int slot, int j, Frag (&bf)[NB][2]) {
    const uint8_t* s = smem + (slot * 4 + 2 + j) * QB;
    if constexpr (TB) {
      uint32_t at[NB];
#pragma unroll
      for (int g = 0; g < NB; ++g) at[g] = lds_address(s) + turned_at(lane, wc * 2 + g);
      read_turned<NB>(at, bf);
    } else {
#pragma unroll
      for (int g = 0; g < NB; ++g)
#pragma unroll
        for (int h = 0; h < KH; ++h) bf[g][h] = straight(s, wc * 32 + 16 * g, h, g & 1);
    }
  };
  // A's half i, and half j of B in slot sb, into af and bf
  auto read_ab = [&](int slot, int i, int sb, int j, Frag (&bf)[NB][2]) {
    const uint8_t *sa = smem + (slot * 4 + i) * QB, *s2 = smem + (sb * 4 + 2 + j) * QB;
    if constexpr (TA) {
      uint32_t at[NA + NB];
      Frag both[NA + NB][2];
#pragma unroll
      for (int f = 0; f < NA; ++f) at[f] = lds_address(sa) + turned_at(lane, grp * 4 + f);
#pragma unroll
      for (int g = 0; g < NB; ++g) at[NA + g] = lds_address(s2) + turned_at(lane, wc * 2 + g);
      read_turned<NA + NB>(at, both);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int f = 0; f < NA; ++f) af[f][h] = both[f][h];
#pragma unroll
        for (int g = 0; g < NB; ++g) bf[g][h] = both[NA + g][h];
      }
    } else {
#pragma unroll
      for (int f = 0; f < NA; ++f)
#pragma unroll
        for (int h = 0; h < KH; ++h) af[f][h] = straight(sa, grp * 64 + 16 * f, h, f & 1);
      read_b(sb, j, bf);
    }
  };

  f32x4 acc[2][2][NA][NB];
  auto math = [&](int i, int j, const Frag (&bf)[NB][2]) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int h = 0; h < KH; ++h)
#pragma unroll
      for (int f = 0; f < NA; ++f)
#pragma unroll
        for (int g = 0; g < NB; ++g) {
          const f32x4 c = acc[i][j][f][g];
          if constexpr (FP8) acc[i][j][f][g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[g][h], af[f][h], c, 0, 0, 0, 0, 0, 0);
          else acc[i][j][f][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[g][h], af[f][h], c, 0, 0, 0);
        }
    __builtin_amdgcn_s_setprio(0);
  };

  // ---- the epilogue: lane (rf, q) holds row rf, columns 4 q + [0, 4) of each fragment; two fragments trade quarters so
  // that a lane stores 16 bytes
  auto epilogue = [&](const GroupTile& t, int lt) __attribute__((always_inline)) {
    // (values the compiler cannot see through: what the stores need of the lane is made here, once a tile, instead of
    // held in registers through the K loop, which spilled)
    const GroupArgs& p = args_anew();
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));
    const int rf = lane & 15, q = lane >> 4;
    const uint8_t* ev = vecs + (lt % 3) * 4096;
    const int64_t row0 = TA ? t.m0 : t.row0;
    const __amdgpu_buffer_rsrc_t rc = make_rsrc(p.c + (TA ? t.e * p.c_group : 0) + row0 * p.ldc, rows_bytes(t.rows, p.ldc, (uint32_t)p.n * 2u));
    auto store = [&](const __amdgpu_buffer_rsrc_t& r, i32x4 v, int n, uint32_t off) {
      if (n < p.n) __builtin_amdgcn_raw_buffer_store_b128(v, r, off, 0, 0);
    };
    [[maybe_unused]] float rs[2][4];
    [[maybe_unused]] f32x4 cs[2][2], bv[2][2];
    if constexpr (FP8) {
      const float one = p.sa_ld || !t.klen ? 0.0f : p.sa[0], col = p.sb_col || !t.klen ? 0.0f : p.sb[t.e * p.sb_ld];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int f = 0; f < 4; ++f) rs[i][f] = p.sa_ld ? ((const float*)ev)[128 * i + 64 * grp + 16 * f + rf] : one;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int c = PAIR ? 128 * g + 64 * j + 16 * wc + 4 * q : 128 * j + 32 * wc + 16 * g + 4 * q;
          cs[j][g] = p.sb_col ? *(const f32x4*)(ev + 1024 + 4 * c) : f32x4{col, col, col, col};
        }
    }
    const bool bias = NT && p.bias && t.klen;
    if constexpr (NT) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint8_t* b = ev + 2048 + (PAIR ? 1024 * g : 0);
          const int c = PAIR ? 64 * j + 16 * wc + 4 * q : 128 * j + 32 * wc + 16 * g + 4 * q;
          bv[j][g] = bias ? ld4(b, p.bias_dt, c) : f32x4{};
        }
    }
    // (a tile without a contraction, the rows behind the last: what its vectors' slots hold is not used)
    auto value = [&](int i, int j, int f, int g) {
      f32x4 v = acc[i][j][f][g];
      if constexpr (FP8) v = t.klen ? v * (cs[j][g] * rs[i][f]) : f32x4{};
      if constexpr (NT) {
        if (bias) v += bv[j][g];
      }
      return v;
    };
    // two fragments' values to 16 bytes a lane
    auto join = [&](f32x4 a, f32x4 b) {
      const u32x2 wa = pack4<2>(HKX_BF16, a), wb = pack4<2>(HKX_BF16, b);
      uint32_t x0 = wa.x, x1 = wb.x, y0 = wa.y, y1 = wb.y;
      swap16(x0, x1);
      swap16(y0, y1);
      return i32x4{(int)x0, (int)y0, (int)x1, (int)y1};
    };
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (PAIR) {
          // fragments 2 a and 2 a + 1 of the rows: a lane ends with 8 columns of a row of one of them
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            __builtin_amdgcn_sched_barrier(0);
            const f32x4 g0 = value(i, j, 2 * a, 0), u0 = value(i, j, 2 * a, 1), g1 = value(i, j, 2 * a + 1, 0), u1 = value(i, j, 2 * a + 1, 1);
            const int n = t.n0 + 64 * j + 16 * wc + 8 * (lane >> 5), m = 128 * i + 64 * grp + 32 * a + 16 * (q & 1) + rf;
            store(rc, join(silu_mul4(g0, u0), silu_mul4(g1, u1)), n, (uint32_t)m * (uint32_t)p.ldc + (uint32_t)n * 2u);
            if (p.z) {
              const __amdgpu_buffer_rsrc_t rz = make_rsrc(p.z + t.row0 * p.ldz, rows_bytes(t.rows, p.ldz, (uint32_t)p.n * 4u));
              store(rz, join(g0, g1), n, (uint32_t)m * (uint32_t)p.ldz + (uint32_t)n * 2u);
              store(rz, join(u0, u1), n, (uint32_t)m * (uint32_t)p.ldz + (uint32_t)(n + p.n) * 2u);
            }
          }
        } else {
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            __builtin_amdgcn_sched_barrier(0);
            const int n = t.n0 + 128 * j + 32 * wc + 16 * (q & 1) + 8 * (q >> 1), m = 128 * i + 64 * grp + 16 * f + rf;
            store(rc, join(value(i, j, f, 0), value(i, j, f, 1)), n, (uint32_t)m * (uint32_t)p.ldc + (uint32_t)n * 2u);
          }
        }
      }
  };

  // ---- the K loop
  auto sync = [&](bool lds) {
    __builtin_amdgcn_sched_barrier(0);
    if (lds) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
    else __builtin_amdgcn_s_waitcnt(wait_vm(8));
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  GroupTile cur = tile_at(0), nxt = cur;
  Ahead s1{}, s2{};
  s1.va[0] = s2.va[0] = la[0];
  s1.va[1] = s2.va[1] = la[1];
  if (gathered) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r0 = row_a(k), r1 = r0 + 128;
      s2.va[k] = r0 < cur.rows ? offset_of(p.index[cur.row0 + r0], k) : kGroupOut;
      s1.va[k] = r1 < cur.rows ? offset_of(p.index[cur.row0 + r1], k) : kGroupOut;
    }
  }
  // the row numbers of tile lt are in LDS from the tile before on; the first's are read here, for its scales
  begin_a(s1, cur, 1);
  begin_a(s2, cur, 0);
  begin_b(s2, cur);
  s1.nkt = s2.nkt = units(cur);
  int l1 = 0, l2 = 0;
  if constexpr (NT) fill_vectors(cur, 0, p.index ? p.index + cur.row0 : nullptr);
  auto step_on = [&](Ahead& s) {
    ++s.t;
    s.par ^= 1;
    if constexpr (TA) s.a += 64 * p.lda;
    if constexpr (TB) s.b += 64 * p.ldb;
    if constexpr (TB) s.left -= 64;
  };
  // Past a stream's last unit its next tile begins (found at the current tile's first unit), or nothing is left.
  auto next1 = [&]() {
    step_on(s1);
    if (s1.t < s1.nkt) return;
    s1.t = 0;
    if (++l1 >= my_tiles) {  // nothing is left: zeros
      s1.ba = 0;
      s1.left = 0;
      return;
    }
    const GroupTile& t1 = nxt;
    s1.nkt = units(t1);
    if (gathered) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
      {
        const int r = row_a(k) + 128;
        s1.va[k] = r < t1.rows ? offset_of(idx_lds[(l1 & 1) * 256 + r], k) : kGroupOut;
      }
    }
    begin_a(s1, t1, 1);
  };
  auto next2 = [&]() {
    step_on(s2);
    if (s2.t < s2.nkt) return;
    s2.t = 0;
    if (++l2 >= my_tiles) {
      s2.ba = s2.bb = s2.b1 = 0;
      s2.left = 0;
      return;
    }
    const GroupTile& t2 = nxt;
    s2.nkt = units(t2);
    if (gathered) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
      {
        const int r = row_a(k);
        s2.va[k] = r < t2.rows ? offset_of(idx_lds[(l2 & 1) * 256 + r], k) : kGroupOut;
      }
    }
    begin_a(s2, t2, 0);
    begin_b(s2, t2);
    if constexpr (NT) fill_vectors(t2, l2, idx_lds + (l2 & 1) * 256);
  };
  // unit 0 whole and unit 1 but A1, in the steady state's order (a tile has 5 units or more)
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    fill_b(s2, 1);
    fill_b(s2, 0);
    fill_a(s2, 0);
    if (r == 0) {
      fill_a(s1, 1);
      next1();
    }
    next2();
  }
  __builtin_amdgcn_s_waitcnt(wait_vm(8));  // A0, B0 and B1 of unit 0
  __builtin_amdgcn_s_barrier();
  read_b(0, 1, bf1);  // B1 of unit 0, read by every wave before any refill of it
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
  __builtin_amdgcn_s_barrier();
  if (grp == 1) __builtin_amdgcn_s_barrier();

  // unit t of tile lt: b1 holds its B1 fragments, nb1 takes the next unit's. Group 1's last barrier of a tile is after
  // its epilogue.
  auto unit = [&](int lt, int t, int nkt, int slot, Frag (&b1)[NB][2], Frag (&nb1)[NB][2]) {
    // (rows along K are read, and waited for, behind the fills; the fills' quarters are none that is read here)
    if constexpr (!TB) read_ab(slot, 0, slot, 0, bf0);
    if (t == 0 && lt + 1 < my_tiles) {
      nxt = tile_at(lt + 1);
      if constexpr (NT) fill_index(nxt, lt + 1);
    }
    fill_a(s1, 1);
    next1();
    fill_b(s2, 1);
    if constexpr (TB) read_ab(slot, 0, slot, 0, bf0);
    sync(true);
    math(0, 0, bf0);
    math(0, 1, b1);
    sync(false);
    if constexpr (!TB) read_ab(slot, 1, slot ^ 1, 1, nb1);
    fill_b(s2, 0);
    fill_a(s2, 0);
    next2();
    if constexpr (TB) read_ab(slot, 1, slot ^ 1, 1, nb1);
    sync(true);
    math(1, 0, bf0);
    math(1, 1, b1);
    if (grp == 0 || t + 1 < nkt) sync(false);
  };
  int slot = 0;
  for (int lt = 0; lt < my_tiles; ++lt) {
    const int nkt = units(cur);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int f = 0; f < NA; ++f)
#pragma unroll
          for (int g = 0; g < NB; ++g) acc[i][j][f][g] = f32x4{};
    int t = 0;
    // (unpeeled: TN's first units on their own spilled)
#pragma clang loop unroll(disable)
    for (; t + 1 < nkt; t += 2) {
      unit(lt, t, nkt, slot, bf1, bfn);
      unit(lt, t + 1, nkt, slot ^ 1, bfn, bf1);
    }
    if (t < nkt) {  // an odd count: the last unit, and the next tile's B1 back in bf1
      unit(lt, t, nkt, slot, bf1, bfn);
      slot ^= 1;
#pragma unroll
      for (int f = 0; f < NB; ++f)
#pragma unroll
        for (int h = 0; h < 2; ++h) bf1[f][h] = bfn[f][h];
    }
    epilogue(cur, lt);
    cur = nxt;
    if (grp == 1) sync(false);
  }
  if (grp == 0) __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no fill lands in LDS after the exit
}

}  // namespace hkx
