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
//
// Bound by MFMAs and by the rows that ragged groups leave empty in their last tiles. 4096 tokens to 2 of 8 experts, bf16, gate and
// up of 14336 rows, K = 4096: 755 us, 1.27 PFLOP/s of useful products (a library's 8192 cubed, no groups: 1.40); 2047 to 8 of
// 64, e4m3, 2048 rows, K = 4096: 180 us, 1.5 of 2.86, 64% of the tiles' rows being rows of A. On 128 x 128 tiles of a kernel
// without the schedule the first took 2313.
#pragma once

#include "hkx_group.hpp"

namespace hkx {

constexpr int kQuadUnits = 5;  // K units a tile at least
constexpr int kQuadMostParts = 8, kQuadPartUnits = 8;
constexpr size_t kQuadPartBytes = 256 * 256 * 4;

// The last round of `total` tiles on `grid` workgroups, where it fills at most half of them: its `rem` tiles in `parts`
// along K each (1: whole), a workgroup one part, the fp32 sums through memory. A round of nku units takes some 1.5 nku us, a
// part's sums written and read 0.13 us of the whole: parts while their square times rem is below 12 nku. (Gradient of
// 8192 rows, 36 tile rows of 8 tiles, K = 8192: 335 us, with the 32 tiles over in parts 236.)
struct QuadRound {
  int full, rem, parts;
};
HKX_DEV QuadRound quad_round(int total, int grid, int nku, bool ws) {
  QuadRound r{total / grid * grid, total % grid, 1};
  if (!ws || r.rem == 0) return r;
  while (r.parts < kQuadMostParts && (r.parts + 1) * r.rem <= grid && (r.parts + 1) * (r.parts + 1) * r.rem <= 12 * nku &&
         (r.parts + 1) * kQuadPartUnits <= nku)
    ++r.parts;
  return r;
}

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
                                                      : group_total(map, p, tiles_n));
  // the workgroup's tiles: one at its place in every round of the grid
  const int place = group_place((int)blockIdx.x), step = (int)gridDim.x;
  const int nku = TA ? 0 : (p.k + KU - 1) / KU;
  const QuadRound round = quad_round(total, step, nku, !TA && p.ws != nullptr);
  const int whole = round.full / step;  // rounds before the last
  const int my_tiles = whole + (place < round.rem * round.parts ? 1 : 0);
  if (my_tiles == 0) return;
  struct Tile : GroupTile {
    int u0, u1;  // its units (at least kQuadUnits: what is past K reads as zeros)
    bool part;   // of a tile's units: the sums go to memory
  };
  auto tile_at = [&](int lt) {
    const GroupArgs& p = args_anew();
    const bool last = lt == whole;
    const int at = place + lt * step, part = last && round.parts > 1 ? place / round.rem : 0;
    Tile t;
    (GroupTile&)t = group_tile_at<OP, BM, BN>(map, p, last && round.parts > 1 ? round.full + place % round.rem : at, tiles_n, rows_of);
    t.e = __builtin_amdgcn_readfirstlane(t.e);
    t.m0 = __builtin_amdgcn_readfirstlane(t.m0);
    t.n0 = __builtin_amdgcn_readfirstlane(t.n0);
    t.rows = __builtin_amdgcn_readfirstlane(t.rows);
    t.klen = __builtin_amdgcn_readfirstlane(t.klen);
    t.row0 = (int64_t)__builtin_amdgcn_readfirstlane((int)t.row0);
    t.part = last && round.parts > 1;
    const int real = (t.klen + KU - 1) / KU, each = t.part ? (real + round.parts - 1) / round.parts : real;
    t.u0 = __builtin_amdgcn_readfirstlane(part * each);
    t.u1 = __builtin_amdgcn_readfirstlane(max(min(real, t.u0 + each), t.u0 + kQuadUnits));
    return t;
  };

  // ---- fills. Instruction k (0, 1) of wave w: K-contiguous rows 16 w + 8 k + [0, 8) of a quarter, lane l row l % 32 / 4,
  // K-half l / 32, its 16-byte piece (l % 4) ^ swz4(row); rows along K 8 w + 4 k + [0, 4), lane l row l / 16.
  //
  // Two streams walk the workgroup's units: one a unit ahead (A1), one two (A0, B0, B1). A unit's fills are loads at a
  // scalar offset from a resource made once a tile (rows along K: moved on a unit at a time) into the stream's slot; what
  // is not every unit's, a ragged last unit, units past K and the next tile, is told by one comparison with the stream's
  // `edge` (scalar work between two barriers is time that no MFMA covers: 140 instructions of it a phase took NT from 1380
  // to 1100 TFLOP/s).
  auto lane_anew = [&]() {  // (made where a tile begins: held through the K loop it would spill)
    int l = tid & 63;
    asm volatile("" : "+v"(l));
    return l;
  };
  auto row_of = [&](int l, int k) { return 16 * wave + 8 * k + (l & 31) / 4; };
  auto piece_of = [&](int l, int k) { return (uint32_t)(64 * (l >> 5) + 16 * ((l & 3) ^ ((wave & 1) | (k << 1)))); };
  auto along_of = [&](int l, int k, int64_t ld) {
    const uint32_t kr = (uint32_t)(8 * wave + 4 * k + l / 16);
    return kr * (uint32_t)ld + (uint32_t)((l % 16) ^ (group_swz(kr) << 1)) * 16u;
  };
  struct Walk {
    int t, nkt, edge;     // its unit in its tile; the tile's units; the unit at which something changes
    uint32_t slot;        // its slot, bytes
    uint32_t so, inc;     // K-contiguous operands: the unit's offset along K
    int lt, klen;         // its tile, and that tile's contraction
  };
  const bool gathered = NT && p.index != nullptr;
  const int32_t* const idx_lds = (const int32_t*)(smem + IDX);
  auto rows_bytes = [](int rows, int64_t ld, uint32_t row) { return rows > 0 ? (uint32_t)((rows - 1) * ld) + row : 0u; };
  Walk w1{}, w2{};
  __amdgpu_buffer_rsrc_t ra1 = make_rsrc(nullptr, 0), ra2 = ra1, rb = ra1;
  uint32_t va1[2], va2[2], vb[2];
  const uint8_t *pa1 = nullptr, *pa2 = nullptr, *pb = nullptr;  // rows along K: the unit's first
  uint32_t na1 = 0, na2 = 0, nb = 0;                            // and the resource's bytes
  uint32_t b1 = 0;  // B's second half behind the first (0: past N, the first again: it is never stored)
  Tile cur = tile_at(0), nxt = cur;

  auto load = [&](__amdgpu_buffer_rsrc_t r, uint32_t slot, const uint32_t (&v)[2], uint32_t so, int k) {
    uint8_t* s = smem + slot + wave * 2048;
    if (k != 1) buf_load16_lds(r, s, v[0], so);
    if (k != 0) buf_load16_lds(r, s + 1024, v[1], so);
  };
  // (k: instruction 0 or 1, or both)
  auto fill_a1 = [&](int k = 2) { load(ra1, w1.slot + QB, va1, TA ? 0u : w1.so, k); };
  auto fill_a0 = [&](int k = 2) { load(ra2, w2.slot, va2, TA ? 0u : w2.so, k); };
  auto fill_b = [&](int j, int k = 2) { load(rb, w2.slot + (2 + j) * QB, vb, (TB ? 0u : w2.so) + (j ? b1 : 0u), k); };

  // A's half i of tile t: offsets, and the resource of a K-contiguous A or the first rows and bytes of one along K
  auto begin_a = [&](const Tile& t, int i, const int32_t* index, uint32_t (&v)[2], __amdgpu_buffer_rsrc_t& r,
                     const uint8_t*& base, uint32_t& bytes) {
    const GroupArgs& p = args_anew();
    const int l = lane_anew();
    if constexpr (TA) {
      const int m = t.m0 + (t.rows > 128 * i ? 128 * i : 0);  // (a half past M: the first again)
      base = p.a + (t.row0 + 64 * (int64_t)t.u0) * p.lda + (int64_t)m * 2;
      bytes = rows_bytes(64, p.lda, (uint32_t)(p.m - m) * 2u);
      v[0] = along_of(l, 0, p.lda), v[1] = along_of(l, 1, p.lda);
    } else {
      const uint32_t k_row = (uint32_t)p.k * ES;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = row_of(l, k);
        v[k] = (uint32_t)row * (uint32_t)p.lda + piece_of(l, k);
        if (gathered) {
          const int j = row + 128 * i < t.rows ? index[row + 128 * i] : -1;
          v[k] = (uint32_t)j < (uint32_t)p.a_rows ? (uint32_t)j * (uint32_t)p.lda + piece_of(l, k) : kGroupOut;
        }
      }
      r = gathered ? make_rsrc(p.a, rows_bytes(p.a_rows, p.lda, k_row))
                   : make_rsrc(p.a + (t.row0 + 128 * i) * p.lda, rows_bytes(t.rows - 128 * i, p.lda, k_row));
      // (no row of the half: every offset is out, as a resource of nothing is at any offset along K)
      if (!gathered && t.rows <= 128 * i) r = make_rsrc(p.a, k_row), v[0] = v[1] = kGroupOut;
    }
  };
  auto begin_b = [&](const Tile& t) {
    const GroupArgs& p = args_anew();
    const int l = lane_anew();
    constexpr int HB = PAIR ? 64 : 128;
    b1 = t.n0 + HB < p.n ? (TB ? HB * 2u : (uint32_t)HB * (uint32_t)p.ldb) : 0u;
    if constexpr (TB) {
      pb = p.b + (TA ? t.row0 * p.ldb : t.e * p.b_group) + 64 * (int64_t)t.u0 * p.ldb + (int64_t)t.n0 * 2;
      nb = rows_bytes(64, p.ldb, (uint32_t)(p.n - t.n0) * 2u);
      vb[0] = along_of(l, 0, p.ldb), vb[1] = along_of(l, 1, p.ldb);
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int row = PAIR ? 16 * (wave >> 1) + 8 * k + (l & 31) / 4 + ((wave & 1) ? p.n : 0) : row_of(l, k);
        vb[k] = (uint32_t)row * (uint32_t)p.ldb + piece_of(l, k);
      }
      rb = make_rsrc(p.b + t.e * p.b_group + t.n0 * p.ldb, rows_bytes((PAIR ? p.n : 0) + min(p.n - t.n0, BN), p.ldb, (uint32_t)p.k * ES));
    }
  };
  // At unit w.t: a ragged last unit, units past K (nothing), or nothing special until the
  // edge. out(k): what lanes past K of K-contiguous rows do; rows(n): rows along K that are left; none(): zeros.
  auto at_edge = [&](Walk& w, auto out, auto rows, auto none) {
    const int real = (w.klen + KU - 1) / KU, ragged = w.klen % KU;
    if (w.t >= real) {
      none();
      w.so = w.inc = 0;
      w.edge = w.nkt;
    } else if (ragged && w.t == real - 1) {
      if (TB) rows(ragged);
      if (!TA) {
        const int l = lane_anew();
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (piece_of(l, k) >= (uint32_t)(ragged * ES)) out(k);
      }
      w.edge = min(real, w.nkt);
    } else {
      w.edge = min(ragged ? real - 1 : real, w.nkt);
    }
  };
  auto edge1 = [&]() {
    at_edge(w1, [&](int k) { va1[k] = kGroupOut; },
            [&](int n) { if (TA) na1 -= (uint32_t)(64 - n) * (uint32_t)args_anew().lda; },
            [&]() { na1 = 0; ra1 = make_rsrc(nullptr, 0); });
  };
  auto edge2 = [&]() {
    at_edge(w2, [&](int k) { va2[k] = kGroupOut; if (!TB) vb[k] = kGroupOut; },
            [&](int n) {
              if (TA) na2 -= (uint32_t)(64 - n) * (uint32_t)args_anew().lda;
              nb -= (uint32_t)(64 - n) * (uint32_t)args_anew().ldb;
            },
            [&]() { na2 = nb = b1 = 0; ra2 = rb = make_rsrc(nullptr, 0); });
  };
  auto begin1 = [&](const Tile& t, const int32_t* index) {
    w1.t = t.u0, w1.so = (uint32_t)t.u0 * 128u, w1.inc = 128, w1.nkt = t.u1, w1.klen = t.klen;
    begin_a(t, 1, index, va1, ra1, pa1, na1);
    edge1();
    if (TA) ra1 = make_rsrc(pa1, na1);
  };
  auto begin2 = [&](const Tile& t, const int32_t* index) {
    w2.t = t.u0, w2.so = (uint32_t)t.u0 * 128u, w2.inc = 128, w2.nkt = t.u1, w2.klen = t.klen;
    begin_a(t, 0, index, va2, ra2, pa2, na2);
    begin_b(t);
    edge2();
    if (TA) ra2 = make_rsrc(pa2, na2);
    if (TB) rb = make_rsrc(pb, nb);
  };

  // ---- a tile's vectors and row numbers
  uint8_t* const vecs = smem + VEC;
  [[maybe_unused]] auto fill_index = [&](const Tile& t, int lt) {  // wave 7
    if (!gathered || wave != 7) return;
    const GroupArgs& p = args_anew();
    const __amdgpu_buffer_rsrc_t r = make_rsrc(p.index + t.row0, (uint32_t)t.rows * 4u);
#pragma unroll
    for (int i = 0; i < 4; ++i)  // (a word a lane: a tile's first row number may stand anywhere)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(smem + IDX + (lt & 1) * 1024 + i * 256), 4,
                                               (uint32_t)(64 * i + lane) * 4u, 0, 0, 0);
  };
  [[maybe_unused]] auto fill_vectors = [&](const Tile& t, int lt, const int32_t* index) {
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
  // (a quarter is a multiple of 256 bytes: fragments f on are 32 f bytes away under an exclusive or, as the swizzle is)
  const uint32_t ta = turned_at(lane, grp * 4), tb = turned_at(lane, wc * 2);
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
      for (int g = 0; g < NB; ++g) at[g] = (lds_address(s) + tb) ^ (32u * g);
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
      for (int f = 0; f < NA; ++f) at[f] = (lds_address(sa) + ta) ^ (32u * f);
#pragma unroll
      for (int g = 0; g < NB; ++g) at[NA + g] = (lds_address(s2) + tb) ^ (32u * g);
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
  // TN issues its fills here, an instruction behind four MFMAs: before its reads, twice as many as the others', they held
  // those up (8192 even rows of 8 groups, 8192 x 2048: 253 us, like this 239; NT and NN got 6-13% slower by it).
  auto math = [&](int i, int j, const Frag (&bf)[NB][2], auto fill) {
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
          if (TA && g == 1 && (h * NA + f) % 4 == 1) {
            __builtin_amdgcn_sched_barrier(0);
            fill(h);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
    __builtin_amdgcn_s_setprio(0);
  };

  // ---- the epilogue: lane (rf, q) holds row rf, columns 4 q + [0, 4) of each fragment; two fragments trade quarters so
  // that a lane stores 16 bytes
  auto epilogue = [&](const Tile& t, int lt) __attribute__((always_inline)) {
    // (values the compiler cannot see through: what the stores need of the lane is made here, once a tile, instead of
    // held in registers through the K loop, which spilled)
    const GroupArgs& p = args_anew();
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));
    const int rf = lane & 15, q = lane >> 4;
    if (!TA && t.part) {
      f32x4* const w = (f32x4*)p.ws + (int64_t)place * (kQuadPartBytes / 16) + 64 * wave + lane;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int f = 0; f < NA; ++f)
#pragma unroll
            for (int g = 0; g < NB; ++g) w[(((i * 2 + j) * 4 + f) * 2 + g) * 512] = acc[i][j][f][g];
      return;
    }
    const uint8_t* ev = vecs + (lt % 3) * 4096;
    const int64_t row0 = TA ? t.m0 : t.row0;
    const __amdgpu_buffer_rsrc_t rc = make_rsrc(p.c + (TA ? t.e * p.c_group : 0) + row0 * p.ldc, rows_bytes(t.rows, p.ldc, (uint32_t)p.n * (OP == kGroupNN && p.c_f32 ? 4u : 2u)));
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
        for (int f = 0; f < 4; ++f) rs[i][f] = p.sa_ld && t.klen ? ((const float*)ev)[128 * i + 64 * grp + 16 * f + rf] : one;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const int c = PAIR ? 128 * g + 64 * j + 16 * wc + 4 * q : 128 * j + 32 * wc + 16 * g + 4 * q;
          cs[j][g] = p.sb_col && t.klen ? *(const f32x4*)(ev + 1024 + 4 * c) : f32x4{col, col, col, col};
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
    // (a tile without a contraction, the rows behind the last: its sums and scales are 0)
    auto value = [&](int i, int j, int f, int g, auto biased) {
      f32x4 v = acc[i][j][f][g];
      if constexpr (FP8) v *= cs[j][g] * rs[i][f];
      if constexpr (NT && decltype(biased)::value) v += bv[j][g];
      return v;
    };
    const bool z = PAIR && p.z != nullptr;
    const __amdgpu_buffer_rsrc_t rz = make_rsrc(z ? p.z + t.row0 * p.ldz : nullptr, z ? rows_bytes(t.rows, p.ldz, (uint32_t)p.n * 4u) : 0u);
    // two fragments' values to 16 bytes a lane
    auto join = [&](f32x4 a, f32x4 b) {
      const u32x2 wa = pack4<2>(HKX_BF16, a), wb = pack4<2>(HKX_BF16, b);
      uint32_t x0 = wa.x, x1 = wb.x, y0 = wa.y, y1 = wb.y;
      swap16(x0, x1);
      swap16(y0, y1);
      return i32x4{(int)x0, (int)y0, (int)x1, (int)y1};
    };
    if (OP == kGroupNN && p.c_f32) {  // (16 bytes a lane as they are)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int n = t.n0 + 128 * j + 32 * wc + 16 * g + 4 * q, m = 128 * i + 64 * grp + 16 * f + rf;
              store(rc, __builtin_bit_cast(i32x4, acc[i][j][f][g]), n, (uint32_t)m * (uint32_t)p.ldc + (uint32_t)n * 4u);
            }
      return;
    }
    auto stores = [&](auto biased) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (PAIR) {
            // fragments 2 a and 2 a + 1 of the rows: a lane ends with 8 columns of a row of one of them
#pragma unroll
            for (int a = 0; a < 2; ++a) {
              __builtin_amdgcn_sched_barrier(0);
              const f32x4 g0 = value(i, j, 2 * a, 0, biased), u0 = value(i, j, 2 * a, 1, biased), g1 = value(i, j, 2 * a + 1, 0, biased), u1 = value(i, j, 2 * a + 1, 1, biased);
              const int n = t.n0 + 64 * j + 16 * wc + 8 * (lane >> 5), m = 128 * i + 64 * grp + 32 * a + 16 * (q & 1) + rf;
              store(rc, join(silu_mul4(g0, u0), silu_mul4(g1, u1)), n, (uint32_t)m * (uint32_t)p.ldc + (uint32_t)n * 2u);
              if (z) {
                store(rz, join(g0, g1), n, (uint32_t)m * (uint32_t)p.ldz + (uint32_t)n * 2u);
                store(rz, join(u0, u1), n, (uint32_t)m * (uint32_t)p.ldz + (uint32_t)(n + p.n) * 2u);
              }
            }
          } else {
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              __builtin_amdgcn_sched_barrier(0);
              const int n = t.n0 + 128 * j + 32 * wc + 16 * (q & 1) + 8 * (q >> 1), m = 128 * i + 64 * grp + 16 * f + rf;
              store(rc, join(value(i, j, f, 0, biased), value(i, j, f, 1, biased)), n, (uint32_t)m * (uint32_t)p.ldc + (uint32_t)n * 2u);
            }
          }
        }
    };
    if (bias) stores(std::true_type{});
    else stores(std::false_type{});
  };

  // ---- the K loop
  auto sync = [&](bool lds) {
    __builtin_amdgcn_sched_barrier(0);
    // (TN's own fills of the phase come after this)
    if (lds) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(TA ? 4 : 8));
    else __builtin_amdgcn_s_waitcnt(wait_vm(8));
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  // A step: the next unit, at an edge what changes there. Past a tile's last unit the next one begins (found at the current
  // tile's first unit); past the last tile's there is nothing.
  auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };  // (kept in scalar registers)
  auto over = [](Walk& w) {
    w.klen = w.t = 0;
    w.nkt = 0x7fffffff;
  };
  auto next1 = [&]() {
    w1.t = (int)uniform((uint32_t)w1.t + 1);
    w1.slot ^= 4 * QB;
    if constexpr (TA) pa1 += 64 * p.lda;
    else w1.so = uniform(w1.so + w1.inc);
    if (w1.t == w1.edge) {
      if (w1.t == w1.nkt && ++w1.lt < my_tiles) {
        begin1(nxt, idx_lds + (w1.lt & 1) * 256);
      } else {
        if (w1.t == w1.nkt) over(w1);
        edge1();
      }
    }
    if constexpr (TA) ra1 = make_rsrc(pa1, na1);
  };
  auto next2 = [&]() {
    w2.t = (int)uniform((uint32_t)w2.t + 1);
    w2.slot ^= 4 * QB;
    if constexpr (TA) pa2 += 64 * p.lda;
    else w2.so = uniform(w2.so + w2.inc);
    if constexpr (TB) pb += 64 * p.ldb;
    if (w2.t == w2.edge) {
      if (w2.t == w2.nkt && ++w2.lt < my_tiles) {
        begin2(nxt, idx_lds + (w2.lt & 1) * 256);
        if constexpr (NT) fill_vectors(nxt, w2.lt, idx_lds + (w2.lt & 1) * 256);
      } else {
        if (w2.t == w2.nkt) over(w2);
        edge2();
      }
    }
    if constexpr (TA) ra2 = make_rsrc(pa2, na2);
    if constexpr (TB) rb = make_rsrc(pb, nb);
  };
  {
    const int32_t* const index = gathered ? p.index + cur.row0 : nullptr;
    begin1(cur, index);
    begin2(cur, index);
    if constexpr (NT) fill_vectors(cur, 0, index);
  }
  // unit 0 whole and unit 1 but A1, in the steady state's order (a tile has 5 units or more)
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    fill_b(1);
    fill_b(0);
    fill_a0();
    if (r == 0) {
      fill_a1();
      next1();
    }
    if (!TA || r == 0) next2();
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
    // (NN: rows along K are read, and waited for, behind the fills; the fills' quarters are none that is read here)
    if constexpr (!TB || TA) read_ab(slot, 0, slot, 0, bf0);
    if constexpr (TA) next2();
    if (t == 0 && lt + 1 < my_tiles) {
      nxt = tile_at(lt + 1);
      if constexpr (NT) fill_index(nxt, lt + 1);
    }
    if constexpr (!TA) {
      fill_a1();
      next1();
      fill_b(1);
    }
    if constexpr (TB && !TA) read_ab(slot, 0, slot, 0, bf0);
    sync(true);
    math(0, 0, bf0, [&](int k) { fill_a1(k); });
    math(0, 1, b1, [&](int k) { fill_b(1, k); });
    sync(false);
    if constexpr (!TB || TA) read_ab(slot, 1, slot ^ 1, 1, nb1);
    if constexpr (TA) next1();
    if constexpr (!TA) {
      fill_b(0);
      fill_a0();
      next2();
    }
    if constexpr (TB && !TA) read_ab(slot, 1, slot ^ 1, 1, nb1);
    sync(true);
    math(1, 0, bf0, [&](int k) { fill_b(0, k); });
    math(1, 1, b1, [&](int k) { fill_a0(k); });
    if (grp == 0 || t + 1 < nkt) sync(false);
  };
  int slot = 0;
  for (int lt = 0; lt < my_tiles; ++lt) {
    const int nkt = cur.u1 - cur.u0;
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

// The last round's parts, summed in order: a workgroup a quarter (i, j) of a tile, its threads where the product's were.
template <int OP, bool FP8, bool PAIR>
__global__ void __launch_bounds__(512) group_quad_join_kernel(const GroupArgs p, const int grid) {
  constexpr int BM = 256, BN = PAIR ? 128 : 256, KU = FP8 ? 128 : 64;
  __shared__ GroupMap map;
  const int tiles_n = (p.n + BN - 1) / BN;
  group_map<BM>(map, p, threadIdx.x, 512);
  const QuadRound round = quad_round(group_total(map, p, tiles_n), grid, (p.k + KU - 1) / KU, true);
  const int tile = (int)blockIdx.x >> 2, i = ((int)blockIdx.x >> 1) & 1, j = (int)blockIdx.x & 1;
  if (round.parts < 2 || tile >= round.rem) return;
  const GroupTile t = group_tile_at<OP, BM, BN>(map, p, round.full + tile, tiles_n,
                                                [&](int g, int& lo, int& hi) { group_rows(p, g, lo, hi); });
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rf = lane & 15, q = lane >> 4;
  const bool rest = t.klen == 0;
  const f32x4* const w = (const f32x4*)p.ws + (int64_t)tile * (kQuadPartBytes / 16) + threadIdx.x;
#pragma unroll
  for (int f = 0; f < 4; ++f) {
    const int r = 128 * i + 64 * (wave >> 2) + 16 * f + rf;
    if (r >= t.rows) continue;
    f32x4 v[2] = {};
    for (int k = 0; k < round.parts; ++k) {
      const f32x4* at = w + (int64_t)k * round.rem * (kQuadPartBytes / 16) + ((i * 2 + j) * 4 + f) * 2 * 512;
      v[0] += at[0];
      v[1] += at[512];
    }
    const float sa = FP8 && !rest ? group_row_scale(p, t.row0 + r) : 1.0f;
    uint8_t *const c = p.c + (t.row0 + r) * p.ldc, *const z = PAIR ? p.z + (t.row0 + r) * p.ldz : nullptr;
#pragma unroll
    for (int g = 0; g < (PAIR ? 1 : 2); ++g) {
      const int n = t.n0 + (PAIR ? 64 * j + 16 * (wave & 3) : 128 * j + 32 * (wave & 3) + 16 * g) + 4 * q;
      if (n < p.n) group_store<OP == kGroupNT, FP8, PAIR>(p, t.e, rest, c, z, n, v[g], PAIR ? v[1] : f32x4{}, sa);
    }
  }
}

}  // namespace hkx
