// Products of ragged groups of rows, each with its expert's matrix: rows offsets[e] .. offsets[e + 1] of R are
// expert e's, and the counts are known to the GPU alone.
//
//   NT  C[r] = A[r or index[r]] . B_e^T (+ bias_e), B_e (N, K): the experts' products, silu(gate) up of B_e's two
//       halves, fp8 operands with a scale a row of A and a row of B_e
//   NN  C[r] = A[r] . B_e,                          B_e (K, N): the gradient of their rows
//   TN  C_e  = sum over the group's rows of A[r]^T B[r], (M, N): the gradient of their weights
//
// K is the contracted size; in TN it is a group's rows. A tile of C belongs to one expert: a group's last tile
// may be ragged, and a grid is sized for the most tiles that R rows in E groups can make; where the counts
// make fewer, the rest end at once. The rows behind the last group are one more group, whose A reads as
// zeros.
//
// Operands reach LDS by 16-byte DMA through a buffer resource a tile, made from 64-bit addresses (an operand may
// be larger than 4 GiB) and bounded by the tile's own rows: what lies past a group's rows, past N or past K reads 0.
// Bad offsets are clamped to 0 .. R and an index past A's rows reads 0: no access leaves an operand.
#pragma once

#include "hkx_device.hpp"
#include "hkx_group_rules.hpp"
#include "hkx_ring.hpp"

namespace hkx {

constexpr int kMaxExperts = 1024;

struct GroupArgs {
  const uint8_t* a;
  const uint8_t* b;
  uint8_t* c;
  uint8_t* z;              // the paired form's product before silu(gate) up (nullptr: not kept)
  const int32_t* offsets;  // E + 1
  const int32_t* index;    // NT: the row of A of each row (nullptr: its own)
  const void* bias;        // (E, N), N in the paired form 2 N
  const float* sa;         // fp8: a scale a row of A (sa_ld 1) or one (0)
  const float* sb;         // fp8: sb[e sb_ld + n sb_col]
  float* ws;               // the 256-row kernel's parts of tiles (nullptr: none)
  int64_t lda, ldb, ldc, ldz;  // bytes a row
  int64_t b_group, c_group;    // bytes an expert (NT and NN: B; TN: C)
  int64_t bias_ld, sb_ld;      // elements an expert
  int32_t experts, rows, a_rows;
  int32_t m, n, k;   // m: TN's rows of C; n: C's columns (paired: of silu(gate) up); k: NT's and NN's contraction
  int32_t tail;      // 1: the rows behind the last group are written too, with zeros
  int32_t bias_dt, sa_ld, sb_col;
  int32_t c_f32;     // NN: C is fp32
};

// ---------------------------------------------------------------- which tile is whose
//
// LDS: the first tile row of each group (first[0 .. groups]), made once a workgroup from the offsets.

struct GroupMap {
  int first[kMaxExperts + 2];
};

// Group g's rows of R; group `experts` are the rows behind the last.
HKX_DEV void group_rows(const GroupArgs& p, int g, int& lo, int& hi) {
  lo = min(max(p.offsets[g], 0), p.rows);
  hi = g < p.experts ? min(max(p.offsets[g + 1], lo), p.rows) : p.tail ? p.rows : lo;
}

// `threads` threads build the map of tiles of BM rows; ends with a barrier.
template <int BM>
HKX_DEV void group_map(GroupMap& s, const GroupArgs& p, int tid, int threads) {
  const int groups = p.experts + 1;
  for (int g = tid; g < groups; g += threads) {
    int lo, hi;
    group_rows(p, g, lo, hi);
    s.first[g + 1] = (hi - lo + BM - 1) / BM;
  }
  if (tid == 0) s.first[0] = 0;
  __syncthreads();
  if (tid < 64) {
    int sum = 0;
    for (int g = 0; g < groups; g += 64) {
      int v = g + tid < groups ? s.first[g + tid + 1] : 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(v, d);
        if (tid >= d) v = __builtin_elementwise_add_sat(v, u);
      }
      v = __builtin_elementwise_add_sat(v, sum);
      if (g + tid < groups) s.first[g + tid + 1] = v;
      sum = __shfl(v, 63);
    }
  }
  __syncthreads();
}

// All tiles of the map. (Offsets out of order can make groups that overlap, and more tiles than a launch has or an int
// counts: what is past them is not computed.)
HKX_DEV int group_total(const GroupMap& s, const GroupArgs& p, int tiles_n) {
  return (int)min((int64_t)s.first[p.experts + 1] * tiles_n, (int64_t)1 << 30);
}

// The group of tile row i (a wave's lanes look together).
HKX_DEV int group_of(const GroupMap& s, int groups, int i) {
  int e = 0;
  const int lane = threadIdx.x & 63;
  for (int g = 0; g < groups; g += 64)
    e += __popcll(__ballot(g + lane < groups && s.first[g + lane + 1] <= i));
  return __builtin_amdgcn_readfirstlane(e);
}

// 32 consecutive tiles on one XCD at a time (workgroup v runs on XCD v % 8, and each has 32 CUs): they share panels in
// its L2, and all XCDs are at work on neighbouring tiles, so that none has the longest group to itself (an eighth of all
// tiles an XCD: TN of 8 groups, the longest with 1.8 times the mean's rows, 383 us, like this 265).
HKX_DEV int group_place(int v) { return (v & ~255) + (v & 7) * 32 + ((v >> 3) & 31); }

// A tile: group e, its rows (columns of A in TN) from m0 on, C's columns from n0 on, `rows` of them in C; row0: the
// first row of R (TN: of the contraction), klen: the contraction's length.
struct GroupTile {
  int e, m0, n0, rows, klen;
  int64_t row0;
};

// Tile `in` of tm x tn: eight tile rows at a time, down them first, so that the tiles in flight on an XCD share panels
// of A and of B.
HKX_DEV void group_raster(int in, int tm, int tn, int& tr, int& tc) {
  const int g = in / (8 * tn), first = 8 * g, gm = min(tm - first, 8), r = in - g * 8 * tn;
  tr = first + r % gm;
  tc = r / gm;
}

// rows_of(e, lo, hi): group e's rows.
template <int OP, int BM, int CN, typename Rows>
HKX_DEV GroupTile group_tile_at(const GroupMap& map, const GroupArgs& p, int at, int tiles_n, Rows rows_of) {
  GroupTile t;
  int lo, hi, tr, tc;
  if constexpr (OP == kGroupTN) {
    const int tiles_m = (p.m + BM - 1) / BM, per = tiles_m * tiles_n;
    t.e = at / per;
    group_raster(at - t.e * per, tiles_m, tiles_n, tr, tc);
    rows_of(t.e, lo, hi);
    t.m0 = tr * BM;
    t.rows = min(p.m - t.m0, BM);
    t.row0 = lo;
    t.klen = hi - lo;
  } else {
    t.e = group_of(map, p.experts + 1, at / tiles_n);
    const int t0 = map.first[t.e];
    group_raster(at - t0 * tiles_n, map.first[t.e + 1] - t0, tiles_n, tr, tc);
    rows_of(t.e, lo, hi);
    t.m0 = tr * BM;
    t.row0 = lo + t.m0;
    t.rows = min(hi - (int)t.row0, BM);
    t.klen = t.e == p.experts ? 0 : p.k;
  }
  t.n0 = tc * CN;
  return t;
}

constexpr uint32_t kGroupOut = 0xfffffff0u;  // an offset past every resource: reads 0

// A resource of `rows` rows of `row` bytes, `ld` apart, from a 64-bit address (0 rows: reads 0).
HKX_DEV __amdgpu_buffer_rsrc_t group_rsrc(const uint8_t* p, int rows, int64_t ld, uint32_t row) {
  return make_rsrc(p, rows > 0 ? (uint32_t)((rows - 1) * ld) + row : 0u);
}

// ---------------------------------------------------------------- C
//
// What row r of R (a tile's, not `rest`) is scaled by, and four columns n of C from the sums v (paired: gate v, up u).

HKX_DEV float group_row_scale(const GroupArgs& p, int64_t r) {
  int64_t at = p.index ? p.index[r] : r;
  const bool in = !p.index || (uint32_t)at < (uint32_t)p.a_rows;
  return in ? p.sa[at * p.sa_ld] : 0.0f;
}

template <bool NT, bool FP8, bool PAIR>
HKX_DEV void group_store(const GroupArgs& p, int e, bool rest, uint8_t* c, uint8_t* z, int n, f32x4 v, f32x4 u, float sa) {
  auto finish = [&](f32x4 v, int n) {  // n: B_e's row
    if (FP8 && !rest) {
      const float* sb = p.sb + e * p.sb_ld;
      if (p.sb_col) v *= *(const f32x4*)(sb + n) * sa;
      else v *= sb[0] * sa;
    }
    if (NT && p.bias && !rest) v += ld4(p.bias, p.bias_dt, e * p.bias_ld + n);
    return v;
  };
  v = finish(v, n);
  if constexpr (PAIR) {
    u = finish(u, n + p.n);
    if (p.z) {
      store4(z, HKX_BF16, n, v);
      store4(z, HKX_BF16, n + p.n, u);
    }
    v = silu_mul4(v, u);
  }
  store4(c, !NT && p.c_f32 ? HKX_FP32 : HKX_BF16, n, v);
}

// ---------------------------------------------------------------- fragments in LDS
//
// A K unit is 128 bytes: 64 bf16 or 128 fp8.
// * K-contiguous rows: 128 bytes a row, its 16-byte chunk c at c ^ (row % 8). A fill instruction moves 8 rows.
// * rows along K (NN's B, TN's A and B): 64 rows of 128 values, 256 bytes; the 32-byte pair of chunks j (16 values, a
//   fragment's columns) at j ^ group_swz(row), so that the four rows that 16 lanes read, and those of the next
//   16, lie in different banks. A fill instruction moves 4 rows. ds_read_b64_tr_b16 turns them: of 16 lanes, lane i names
//   row i / 4, values 4 (i % 4) + [0, 4), and is given value i of the four rows.

HKX_DEV uint32_t group_swz(uint32_t k) { return (k & 3) | ((k >> 1) & 4); }

// Fragments of 16 values from a quarter of rows along K: `at` their LDS addresses (turned_at, 8 KB a K-half on, 1 KB the
// half's later rows), out[f] the K-halves of fragment f. The reads and their wait are one block: behind the compiler's own
// instruction for them stands a wait for every fill in flight.
template <int N>
HKX_DEV void read_turned(const uint32_t (&at)[N], bf16x8 (&out)[N][2]) {
  u32x2 v[4 * N];
  static_assert(N == 2 || N == 4 || N == 6, "fragments");
  if constexpr (N == 2) {
    asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:0\n"
      "ds_read_b64_tr_b16 %1, %8 offset:1024\n"
      "ds_read_b64_tr_b16 %2, %8 offset:8192\n"
      "ds_read_b64_tr_b16 %3, %8 offset:9216\n"
      "ds_read_b64_tr_b16 %4, %9 offset:0\n"
      "ds_read_b64_tr_b16 %5, %9 offset:1024\n"
      "ds_read_b64_tr_b16 %6, %9 offset:8192\n"
      "ds_read_b64_tr_b16 %7, %9 offset:9216\n"
      "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
        : "v"(at[0]), "v"(at[1])
        : "memory");
  }
  if constexpr (N == 4) {
    asm volatile(
      "ds_read_b64_tr_b16 %0, %16 offset:0\n"
      "ds_read_b64_tr_b16 %1, %16 offset:1024\n"
      "ds_read_b64_tr_b16 %2, %16 offset:8192\n"
      "ds_read_b64_tr_b16 %3, %16 offset:9216\n"
      "ds_read_b64_tr_b16 %4, %17 offset:0\n"
      "ds_read_b64_tr_b16 %5, %17 offset:1024\n"
      "ds_read_b64_tr_b16 %6, %17 offset:8192\n"
      "ds_read_b64_tr_b16 %7, %17 offset:9216\n"
      "ds_read_b64_tr_b16 %8, %18 offset:0\n"
      "ds_read_b64_tr_b16 %9, %18 offset:1024\n"
      "ds_read_b64_tr_b16 %10, %18 offset:8192\n"
      "ds_read_b64_tr_b16 %11, %18 offset:9216\n"
      "ds_read_b64_tr_b16 %12, %19 offset:0\n"
      "ds_read_b64_tr_b16 %13, %19 offset:1024\n"
      "ds_read_b64_tr_b16 %14, %19 offset:8192\n"
      "ds_read_b64_tr_b16 %15, %19 offset:9216\n"
      "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]), "=&v"(v[8]), "=&v"(v[9]), "=&v"(v[10]), "=&v"(v[11]), "=&v"(v[12]), "=&v"(v[13]), "=&v"(v[14]), "=&v"(v[15])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
        : "memory");
  }
  if constexpr (N == 6) {
    asm volatile(
      "ds_read_b64_tr_b16 %0, %24 offset:0\n"
      "ds_read_b64_tr_b16 %1, %24 offset:1024\n"
      "ds_read_b64_tr_b16 %2, %24 offset:8192\n"
      "ds_read_b64_tr_b16 %3, %24 offset:9216\n"
      "ds_read_b64_tr_b16 %4, %25 offset:0\n"
      "ds_read_b64_tr_b16 %5, %25 offset:1024\n"
      "ds_read_b64_tr_b16 %6, %25 offset:8192\n"
      "ds_read_b64_tr_b16 %7, %25 offset:9216\n"
      "ds_read_b64_tr_b16 %8, %26 offset:0\n"
      "ds_read_b64_tr_b16 %9, %26 offset:1024\n"
      "ds_read_b64_tr_b16 %10, %26 offset:8192\n"
      "ds_read_b64_tr_b16 %11, %26 offset:9216\n"
      "ds_read_b64_tr_b16 %12, %27 offset:0\n"
      "ds_read_b64_tr_b16 %13, %27 offset:1024\n"
      "ds_read_b64_tr_b16 %14, %27 offset:8192\n"
      "ds_read_b64_tr_b16 %15, %27 offset:9216\n"
      "ds_read_b64_tr_b16 %16, %28 offset:0\n"
      "ds_read_b64_tr_b16 %17, %28 offset:1024\n"
      "ds_read_b64_tr_b16 %18, %28 offset:8192\n"
      "ds_read_b64_tr_b16 %19, %28 offset:9216\n"
      "ds_read_b64_tr_b16 %20, %29 offset:0\n"
      "ds_read_b64_tr_b16 %21, %29 offset:1024\n"
      "ds_read_b64_tr_b16 %22, %29 offset:8192\n"
      "ds_read_b64_tr_b16 %23, %29 offset:9216\n"
      "s_waitcnt lgkmcnt(0)"
        : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]), "=&v"(v[8]), "=&v"(v[9]), "=&v"(v[10]), "=&v"(v[11]), "=&v"(v[12]), "=&v"(v[13]), "=&v"(v[14]), "=&v"(v[15]), "=&v"(v[16]), "=&v"(v[17]), "=&v"(v[18]), "=&v"(v[19]), "=&v"(v[20]), "=&v"(v[21]), "=&v"(v[22]), "=&v"(v[23])
        : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5])
        : "memory");
  }
#pragma unroll
  for (int f = 0; f < N; ++f)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const u32x2 lo = v[4 * f + 2 * h], hi = v[4 * f + 2 * h + 1];
      out[f][h] = __builtin_bit_cast(bf16x8, i32x4{(int)lo.x, (int)lo.y, (int)hi.x, (int)hi.y});
    }
}

HKX_DEV uint32_t lds_address(const uint8_t* s) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)s; }

// What a lane adds to a quarter's address for the fragment of values 16 j + [0, 16).
HKX_DEV uint32_t turned_at(int lane, uint32_t j) {
  const uint32_t rf = lane & 15, k = 8 * (lane >> 4) + rf / 4;
  return k * 256 + (j ^ group_swz(k)) * 32 + (rf % 4) * 8;
}

// The product on BM x BN tiles, BN = 16 FN WN rows of B: WM x WN waves of BM / WM rows and 16 FN columns, S stages
// of a K unit. For groups that 256-row tiles would leave mostly empty: bound by the weights' reads (64 tokens to 8 of 64
// experts, e4m3, 2048 x 1024: 134 MB in 26-30 us, 64-row tiles) or by the few workgroups that there are, each a chain of units with
// a barrier (333 tokens to 2 of 5 experts, 904 x 1112 bf16: 14.7 us, rows' gradient 10.9, weights' 14.3).
template <int OP, bool FP8, bool PAIR, int BM, int WM, int WN, int FN, int S>
__global__ void __launch_bounds__(64 * WM * WN) group_tile_kernel(const GroupArgs p) {
  constexpr int NW = WM * WN, BN = 16 * FN * WN, CN = PAIR ? BN / 2 : BN;
  constexpr int FM = BM / WM / 16;
  constexpr bool TA = OP == kGroupTN, TB = OP != kGroupNT;
  constexpr int ES = FP8 ? 1 : 2, KU = 128 / ES;  // values a K unit
  constexpr int AB = BM * 128, BB = BN * 128, STAGE = AB + BB;
  constexpr int IA = AB / 1024, IB = BB / 1024;                 // fill instructions of a stage
  constexpr int WA = (IA + NW - 1) / NW, WB = (IB + NW - 1) / NW;  // and of a wave
  constexpr int KH = FP8 ? 1 : 2;
  static_assert(!FP8 || OP == kGroupNT, "8-bit operands: the forward product");
  static_assert(!TB || BN == 128, "rows along K: 128 values");
  static_assert(!TA || BM == 128, "rows along K: 128 values");
  static_assert(!PAIR || (FN % 2 == 0 && OP == kGroupNT), "gate and up fragments of one wave");
  // (one array: beside a second one the compiler waits for every fill before each LDS read)
  __shared__ __attribute__((aligned(16))) uint8_t smem[S * STAGE + (TA ? 0 : sizeof(GroupMap))];
  GroupMap& map = *(GroupMap*)(smem + (TA ? 0 : S * STAGE));

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wave / WN, wc = wave % WN;
  const int tiles_n = (p.n + CN - 1) / CN;

  if constexpr (!TA) group_map<BM>(map, p, tid, 64 * NW);
  const int total = TA ? p.experts * ((p.m + BM - 1) / BM) * tiles_n : group_total(map, p, tiles_n);
  const int place = group_place((int)blockIdx.x);
  if (place >= total) return;
  const GroupTile tile = group_tile_at<OP, BM, CN>(
      map, p, place, tiles_n, [&](int g, int& lo, int& hi) { group_rows(p, g, lo, hi); });
  const int e = tile.e, m0 = tile.m0, mrows = tile.rows, n0 = tile.n0, klen = tile.klen;
  const int64_t row0 = tile.row0;
  const bool rest = e == p.experts;  // the rows behind the last group
  const int nku = (klen + KU - 1) / KU;

  // ---- fills
  __amdgpu_buffer_rsrc_t ra, rb;
  uint32_t va[WA], vb[WB], ca[WA], cb[WB];  // offsets; bytes along K of K-contiguous rows
#pragma unroll
  for (int i = 0; i < WA; ++i) {
    const int ins = (wave + NW * i) % IA;
    if constexpr (TA) {
      const uint32_t k = 4 * ins + lane / 16, c = (lane % 16) ^ (group_swz(k) << 1);
      va[i] = k * (uint32_t)p.lda + c * 16;
    } else {
      const int r = 8 * ins + lane / 8;
      ca[i] = ((lane % 8) ^ (r % 8)) * 16;
      int64_t at = r;
      if (OP == kGroupNT && p.index) {
        const int j = r < mrows ? p.index[row0 + r] : -1;
        at = (uint32_t)j < (uint32_t)p.a_rows ? j : -1;
      }
      va[i] = at < 0 ? kGroupOut : (uint32_t)(at * p.lda) + ca[i];
    }
  }
  if constexpr (TA) {
    ra = make_rsrc(nullptr, 0);
    rb = make_rsrc(nullptr, 0);
  } else {
    const uint32_t row = (uint32_t)p.k * ES;
    ra = OP == kGroupNT && p.index ? group_rsrc(p.a, p.a_rows, p.lda, row) : group_rsrc(p.a + row0 * p.lda, mrows, p.lda, row);
    if constexpr (TB) rb = make_rsrc(nullptr, 0);
    else rb = group_rsrc(p.b + (rest ? 0 : e) * p.b_group + n0 * p.ldb, (PAIR ? p.n : 0) + min(p.n - n0, CN), p.ldb, row);
  }
#pragma unroll
  for (int i = 0; i < WB; ++i) {
    const int ins = (wave + NW * i) % IB;
    if constexpr (TB) {
      const uint32_t k = 4 * ins + lane / 16, c = (lane % 16) ^ (group_swz(k) << 1);
      vb[i] = k * (uint32_t)p.ldb + c * 16;
    } else {
      const int r = 8 * ins + lane / 8, f = r / 16;
      cb[i] = ((lane % 8) ^ (r % 8)) * 16;
      // paired: fragments of gate rows and up rows by turns
      const int at = PAIR ? 16 * (f / 2) + r % 16 + (f & 1) * p.n : r;
      vb[i] = (uint32_t)at * (uint32_t)p.ldb + cb[i];
    }
  }
  // rows along K: a resource a unit, of the rows that are left
  auto along = [&](const uint8_t* base, int64_t first, int left, int64_t ld, int cols, int col0) {
    return group_rsrc(base + first * ld + (int64_t)col0 * 2, min(left, 64), ld, (uint32_t)(cols - col0) * 2u);
  };
  auto fill = [&](int t) {
    uint8_t* s = smem + (t % S) * STAGE;
    const bool in = t < nku;
    const uint32_t k0 = (uint32_t)t * 128u;  // bytes along K
    if constexpr (TA) ra = along(p.a, row0 + 64 * (int64_t)t, in ? klen - 64 * t : 0, p.lda, p.m, m0);
    if constexpr (TB) {
      const int64_t first = (int64_t)64 * t;
      rb = TA ? along(p.b, row0 + first, in ? klen - 64 * t : 0, p.ldb, p.n, n0)
              : along(p.b + (rest ? 0 : e) * p.b_group, first, in ? klen - 64 * t : 0, p.ldb, p.n, n0);
    }
    const uint32_t row = (uint32_t)klen * ES;
#pragma unroll
    for (int i = 0; i < WA; ++i) {
      const int ins = (wave + NW * i) % IA;
      if constexpr (TA) buf_load16_lds(ra, s + ins * 1024, va[i], 0);
      else buf_load16_lds(ra, s + ins * 1024, in && k0 + ca[i] < row ? va[i] : kGroupOut, in ? k0 : 0);
    }
#pragma unroll
    for (int i = 0; i < WB; ++i) {
      const int ins = (wave + NW * i) % IB;
      if constexpr (TB) buf_load16_lds(rb, s + AB + ins * 1024, vb[i], 0);
      else buf_load16_lds(rb, s + AB + ins * 1024, in && k0 + cb[i] < row ? vb[i] : kGroupOut, in ? k0 : 0);
    }
  };

  // ---- fragments: lane (rf, q) row rf, K 8 q + [0, 8) of a K-half (fp8: 16 bytes of each half)
  const int rf = lane & 15, q = lane >> 4;
  using Frag = typename std::conditional<FP8, i32x8, bf16x8>::type;
  auto straight = [&](const uint8_t* s, int r0, int h) -> Frag {  // r0 a multiple of 16
    const uint8_t* row = s + (r0 + rf) * 128;
    if constexpr (FP8) {
      const i32x4 lo = *(const i32x4*)(row + ((q ^ (rf & 7)) << 4)), hi = *(const i32x4*)(row + (((4 + q) ^ (rf & 7)) << 4));
      return i32x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    } else {
      return *(const bf16x8*)(row + (((4 * h + q) ^ (rf & 7)) << 4));
    }
  };
  // both K-halves of a wave's fragments: along r0 + [0, 16 N) of an operand's rows
  auto read = [&](const uint8_t* s, int r0, auto along, auto& out) {
    constexpr int N = sizeof(out) / sizeof(out[0]);
    if constexpr (decltype(along)::value) {
      uint32_t at[N];
#pragma unroll
      for (int f = 0; f < N; ++f) at[f] = lds_address(s) + turned_at(lane, r0 / 16 + f);
      read_turned<N>(at, out);
    } else {
#pragma unroll
      for (int f = 0; f < N; ++f)
#pragma unroll
        for (int h = 0; h < KH; ++h) out[f][h] = straight(s, r0 + 16 * f, h);
    }
  };

  f32x4 acc[FM][FN] = {};
  constexpr int NF = WA + WB;
#pragma unroll
  for (int t = 0; t < S - 1; ++t) fill(t);
  for (int t = 0; t < nku; ++t) {
    // stage t has landed in every wave, and stage t - 1 is read
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0((S - 2) * NF));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    fill(t + S - 1);
    const uint8_t* s = smem + (t % S) * STAGE;
    Frag af[FM][2], bf[FN][2];
    read(s, wr * (BM / WM), std::bool_constant<TA>{}, af);
    read(s + AB, wc * FN * 16, std::bool_constant<TB>{}, bf);
#pragma unroll
    for (int h = 0; h < KH; ++h)
#pragma unroll
      for (int f = 0; f < FM; ++f)
#pragma unroll
        for (int g = 0; g < FN; ++g) {
          if constexpr (FP8) acc[f][g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[g][h], af[f][h], acc[f][g], 0, 0, 0, 0, 0, 0);
          else acc[f][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[g][h], af[f][h], acc[f][g], 0, 0, 0);
        }
  }
  __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no fill lands in LDS after the exit

  // ---- C: lane (rf, q) holds row rf, columns 4 q + [0, 4) of each fragment
  const int64_t c_row = TA ? (int64_t)m0 : row0;
  uint8_t* const c0 = p.c + (TA ? e * p.c_group : 0);
#pragma unroll
  for (int f = 0; f < FM; ++f) {
    const int r = wr * (BM / WM) + 16 * f + rf;
    if (r >= mrows) continue;
    const float sa = FP8 && !rest ? group_row_scale(p, row0 + r) : 1.0f;
#pragma unroll
    for (int g = 0; g < FN; g += PAIR ? 2 : 1) {
      const int n = n0 + (PAIR ? (wc * FN + g) / 2 * 16 : (wc * FN + g) * 16) + 4 * q;
      if (n < p.n)
        group_store<OP == kGroupNT, FP8, PAIR>(p, e, rest, c0 + (c_row + r) * p.ldc, PAIR ? p.z + (c_row + r) * p.ldz : nullptr, n,
                                               acc[f][g], PAIR ? acc[f][g + 1] : f32x4{}, sa);
    }
  }
}

// The tiles that R rows in E groups can make at most, of bm rows (and the rows behind them).
inline int64_t group_tiles(int64_t rows, int64_t experts, int64_t bm) {
  return rows / bm + (rows < experts ? rows : experts) + 1;
}

}  // namespace hkx
