// The MXFP4 product's kernels: C (M, N) = (sa . A)(sb . B)^T (+ bias), B 4-bit e2m1 with an
// E8M0 scale a row and 32 K, A the same or 8-bit e4m3, C bf16; or the paired form C =
// silu(Z[:, :N]) * Z[:, N:] over B's 2N rows.
//
// Every product runs on gfx950's scaled MFMAs, which take either operand as 4- or 8-bit and a
// scale byte a lane: v_mfma_scale_f32_32x32x64_f8f6f4 reads K 32 h + [0, 32) of row l % 32 from
// lane half h = l / 32 where the operand is 4-bit (16 bytes), and K 16 h + [0, 16) and 32 + 16 h +
// [0, 16) where it is 8-bit (two 16-byte pieces); the scale byte of lane half h is that of 32-K
// block h in both. 16 x 16 x 128 is the same with four lane groups of 16: K 32 g + [0, 32), or
// 16 g + [0, 16) and 64 + 16 g + [0, 16). Sums are fp32 throughout and rounded to bf16 once.
//
// A K unit is 256 K: one 128-byte line of a 4-bit row, two of an 8-bit one, 8 scale bytes. K is any
// multiple of 32: past it a unit's lines hold the next row's bytes, whose scales are masked to byte
// 0 on both sides -- 2^-254 of a 4-bit value, which no fp32 sum holds -- and an 8-bit A's pieces
// past K, which could be NaN, are read out of range, as zeros.
#pragma once

#include "hkx_tile.hpp"

namespace hkx {

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Mx4Args {
  const uint8_t* a;
  const uint8_t* b;
  const uint8_t* sa;
  const uint8_t* sb;
  void* c;           // bf16 C, or a split's fp32 shares
  const void* bias;  // one value a row of B (nullptr: none), of type bias_dt
  uint32_t a_bytes, b_bytes, sa_bytes, sb_bytes;  // bounds of the buffer resources
  uint32_t lda, ldb, sa_ld, sb_ld;                // row strides in bytes
  int64_t ldc;                                    // elements
  int64_t split_stride;                           // fp32 elements from a split's shares to the next's
  int32_t M, N, K;   // N: columns of C; the paired form's B has 2N rows
  int32_t bias_dt;
  int32_t units, units_split;  // 256-K units in all and of a split (blockIdx.y)
  int32_t tiles_m, tiles_n, wgm;
  int32_t c_vec;     // C's rows are 16-byte aligned and N a multiple of 8: 16-byte stores
  int32_t share_up;  // the paired form's shares: columns from a gate sum to its up sum
};

constexpr uint32_t kMx4Out = 0xfffffff0u;  // an offset past every buffer's end

// The masks of a unit's 8 scale bytes (two dwords) where `left` blocks of 32 K are left.
HKX_DEV uint32_t mx4_mask(int left) { return left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u; }

// Tiles of BM x BN by 4 waves (2 x 2) of 32 x 32 x 64 fragments.
//
// * LDS: stages of one K unit: A's lines (one panel of BM rows x 128 bytes a line), then B's, each
//   row's eight 16-byte pieces XOR-swizzled (piece c of row r at c ^ swz(r % 16)) so that the
//   fragment reads of 16 rows hit distinct banks; filled by 16-byte DMA of whole lines, the swizzle
//   applied on the global side.
// * Scales: four threads a row, 64 bytes of it (eight units) at a time into registers, as aligned dwords,
//   one more where rows are off a multiple of 4 bytes; a chunk of two units goes to one of two LDS buffers a
//   unit ahead, joined and masked past K where it needs it. (A thread a row, 16 bytes every two units, asked
//   for a line a row and piece, half as many as the fills, and with joins and masks always, 128 x 4096 x
//   12288 of 4 bits unsplit took 37.0 us on 64 x 128 tiles against 28.6, and on 128 x 128 ones 44.6 against
//   38.4.)
// * Fragment reads run a k-step of 64 K ahead of their MFMAs, the next unit's first ones under the last
//   k-step, after the unit's one barrier (read just before them, 4096 x 4096 of 4-bit K = 12288 at M =
//   777 took 39.6 us). After that barrier the unit's stage takes the fills of unit t + NST; a wave
//   waits for its own fills of the next unit only (buffer loads land in order).
// * Measured: 777 x 4096 x 12288 of 4 bits 38.0 us on 128 x 128 tiles (2.1 PFLOP/s), 128 x 4096 x 12288 in
//   four splits on 64 x 128 ones 16.9. Bound by what a unit's fills and scales take beside its MFMAs, a SIMD
//   having one wave and nothing else to run: copies with work left out, where the whole took 44.8 (64 x 128
//   tiles 46.2): no fills 30.7 (31.0), no scales 33.9 (41.0), neither 25.3 (24.4), no fragment reads 39.8
//   (43.9), the MFMAs alone 20.5 (20.2).
// * RES = 2: two workgroups a CU, for grids of more than one a CU, in half the LDS.
template <int BM, int BN, bool A8, bool PAIR, bool SHARE, int RES>
__global__ void __launch_bounds__(256, RES) mx4_tile_kernel(const Mx4Args p) {
  constexpr int TM = BM / 2, TN = BN / 2;
  constexpr int FM = TM / 32, FN = TN / 32;
  constexpr int AL = A8 ? 2 : 1;
  constexpr int LINES = BM * AL + BN;  // 128-byte lines a stage
  constexpr int NCH = LINES / 32;      // 16-byte fills a thread and stage
  constexpr int NA = BM * AL / 32;     // of which A's
  constexpr int STAGE = LINES * 128;
  constexpr int ROWS = BM + BN;
  static_assert(BM % 64 == 0 && BN % 64 == 0, "64 rows of scales a load");
  constexpr int OUTW = PAIR ? BN / 2 : BN;
  constexpr int RS = OUTW * 2 + 16;  // staging row stride
  constexpr int BESIDE = BN * 4 + 2 * ROWS * 16;
  constexpr int LDS = 160 * 1024 / RES;
  constexpr int NST = 4 * STAGE + BESIDE <= LDS ? 4 : 3 * STAGE + BESIDE <= LDS ? 3 : 2;
  constexpr int BODY = NST * STAGE > (SHARE ? 0 : BM * RS) ? NST * STAGE : BM * RS;
  constexpr int SCO = BODY + BN * 4;
  constexpr int SMEM = SCO + 2 * ROWS * 16;
  static_assert(SMEM <= LDS, "LDS");
  static_assert(!PAIR || FN % 2 == 0, "gate and up fragments side by side");
  __shared__ __attribute__((aligned(16))) uint8_t smem[SMEM];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;

  // the tile: consecutive ones on one XCD, in groups of wgm tile rows
  const int total = p.tiles_m * p.tiles_n;
  int L = blockIdx.x;
  if ((total & 7) == 0) L = (L & 7) * (total >> 3) + (L >> 3);
  const int per = p.wgm * p.tiles_n;
  const int first = L / per * p.wgm;
  const int gm = min(p.tiles_m - first, p.wgm);
  const int in = L % per;
  const int m0 = (first + in % gm) * BM, n0 = in / gm * OUTW;

  const int kt0 = blockIdx.y * p.units_split;
  const int nkt = min(p.units_split, p.units - kt0);

  // row of B of tile row v: the paired form's 32-row fragments alternate gate and up
  auto brow = [&](int v) {
    if constexpr (PAIR) return n0 + (v >> 6) * 32 + (v & 31) + (v & 32 ? p.N : 0);
    else return n0 + v;
  };

  const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a, p.a_bytes), rb = make_rsrc(p.b, p.b_bytes);
  const int lrow = tid >> 3;
  const uint32_t lch = (uint32_t)(((tid & 7) ^ swz(lrow & 15)) << 4);
  uint32_t voff[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int r = lrow + 32 * i;
    voff[i] = i < NA ? (uint32_t)(m0 + r % BM) * p.lda + (uint32_t)(r / BM) * 128u + lch
                     : (uint32_t)brow(r - BM * AL) * p.ldb + lch;
  }
  auto fill = [&](int kt, int s) {
    uint8_t* base = smem + s * STAGE + wave * 1024;
    const uint32_t kb = __builtin_amdgcn_readfirstlane((uint32_t)(kt0 + kt) * 128u);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (i < NA && A8) {
        const uint32_t k = 2 * kb + (uint32_t)((lrow + 32 * i) / BM) * 128u + lch;
        buf_load16_lds(ra, base + i * 4096, k < (uint32_t)p.K ? voff[i] : kMx4Out, 2 * kb);
      } else {
        buf_load16_lds(i < NA ? ra : rb, base + i * 4096, voff[i], kb);
      }
    }
  };
  // scales: thread t's piece t % 4 (of a chunk of two units) of rows t / 4 + 64 i, A's and then B's
  constexpr int NS = ROWS / 64;
  const uint32_t k32 = (uint32_t)p.K / 32;
  const uint32_t s0a = (uint32_t)((uintptr_t)p.sa & 3), s0b = (uint32_t)((uintptr_t)p.sb & 3);
  const __amdgpu_buffer_rsrc_t rsa = make_rsrc((const void*)((uintptr_t)p.sa & ~(uintptr_t)3),
                                               (s0a + (uint32_t)(p.M - 1) * p.sa_ld + k32 + 3) & ~3u);
  const __amdgpu_buffer_rsrc_t rsb = make_rsrc((const void*)((uintptr_t)p.sb & ~(uintptr_t)3),
                                               (s0b + (uint32_t)((PAIR ? 2 : 1) * p.N - 1) * p.sb_ld + k32 + 3) & ~3u);
  const uint32_t fifth_a = ((p.sa_ld | s0a) & 3) ? 0u : kMx4Out, fifth_b = ((p.sb_ld | s0b) & 3) ? 0u : kMx4Out;
  uint32_t sat[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int r = 64 * i + (tid >> 2);
    sat[i] = (64 * i < BM ? s0a + (uint32_t)(m0 + r) * p.sa_ld : s0b + (uint32_t)brow(r - BM) * p.sb_ld) +
             (uint32_t)kt0 * 8u + (uint32_t)(tid & 3) * 16u;
  }
  struct Scales {  // of four chunks: four dwords a piece and, off a multiple of 4 bytes, a fifth
    i32x4 d[NS];
    uint32_t e[NS];
  };
  auto load_scales = [&](int c, Scales& s) {  // chunks c to c + 3
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const uint32_t at = (sat[i] + (uint32_t)c * 16u) & ~3u;
      s.d[i] = buf_load16(64 * i < BM ? rsa : rsb, at, 0);
      s.e[i] = __builtin_amdgcn_raw_buffer_load_b32(64 * i < BM ? rsa : rsb, (at + 16u) | (64 * i < BM ? fifth_a : fifth_b), 0, 0);
    }
  };
  auto write_scales = [&](int c, const Scales& s) {
    const int left = (int)k32 - 8 * kt0 - 16 * c;
    uint8_t* at = smem + SCO + (c & 1) * ROWS * 16 + (tid >> 2) * 16;
    if ((fifth_a & fifth_b) && left >= 16) {  // nothing to join or mask
      if ((tid & 3) == (c & 3)) {
#pragma unroll
        for (int i = 0; i < NS; ++i) *(i32x4*)(at + 1024 * i) = s.d[i];
      }
      return;
    }
    if ((tid & 3) != (c & 3)) return;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      i32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = (int)(__builtin_amdgcn_alignbyte(j < 3 ? (uint32_t)s.d[i][(j + 1) & 3] : s.e[i], (uint32_t)s.d[i][j], sat[i] & 3) &
                     mx4_mask(left - 4 * j));
      *(i32x4*)(at + 1024 * i) = v;
    }
  };

  const int rf = lane & 31, h = lane >> 5, sw = swz(rf & 15);
  using AFrag = typename std::conditional<A8, i32x8, i32x4>::type;
  auto piece = [&](const uint8_t* panel, int row, int c) {
    return *(const i32x4*)(panel + (row + rf) * 128 + ((c ^ sw) << 4));
  };
  auto wide = [](i32x4 v) { return i32x8{v.x, v.y, v.z, v.w, 0, 0, 0, 0}; };
  auto read = [&](int s, int ks, AFrag (&af)[FM], i32x4 (&bf)[FN]) {
    const uint8_t* st = smem + s * STAGE;
#pragma unroll
    for (int j = 0; j < FN; ++j) bf[j] = piece(st + BM * AL * 128, wn * TN + 32 * j, 2 * ks + h);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      if constexpr (A8) {
        const uint8_t* line = st + (ks >> 1) * BM * 128;
        const i32x4 lo = piece(line, wm * TM + 32 * i, 4 * (ks & 1) + h);
        const i32x4 hi = piece(line, wm * TM + 32 * i, 4 * (ks & 1) + 2 + h);
        af[i] = i32x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      } else {
        af[i] = piece(st, wm * TM + 32 * i, 2 * ks + h);
      }
    }
  };
  using ScaleA = uint32_t[FM][2];
  using ScaleB = uint32_t[FN][2];
  auto read_scales = [&](int kt, ScaleA& sca, ScaleB& scb) {
    const uint8_t* sc = smem + SCO + ((kt >> 1) & 1) * ROWS * 16 + (kt & 1) * 8 + rf * 16;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const u32x2 v = *(const u32x2*)(sc + (wm * TM + 32 * i) * 16);
      sca[i][0] = v.x >> (8 * h);
      sca[i][1] = v.y >> (8 * h);
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const u32x2 v = *(const u32x2*)(sc + (BM + wn * TN + 32 * j) * 16);
      scb[j][0] = v.x >> (8 * h);
      scb[j][1] = v.y >> (8 * h);
    }
  };
  f32x16 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x16{};
  ScaleA sca, nsca;
  ScaleB scb, nscb;
  auto mma = [&](const AFrag (&af)[FM], const i32x4 (&bf)[FN], int ks) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int q = ks >> 1;
        i32x8 a;
        if constexpr (A8) a = af[i];
        else a = wide(af[i]);
        if (ks & 1)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(bf[j]), a, acc[i][j], 4, A8 ? 0 : 4, 2,
                                                                     (int)scb[j][q], 2, (int)sca[i][q]);
        else
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(bf[j]), a, acc[i][j], 4, A8 ? 0 : 4, 0,
                                                                     (int)scb[j][q], 0, (int)sca[i][q]);
      }
  };

  float* bias = (float*)(smem + BODY);  // one a tile row of B
  if (!SHARE && tid < BN) {
    const int r = brow(tid);
    bias[tid] = p.bias && r < (PAIR ? 2 * p.N : p.N) ? ld1(p.bias, p.bias_dt, r) : 0.0f;
  }

  // this wave's LDS reads are done and all but its newest (NST - 2) NCH fills landed
  auto sync = [&]() {
    constexpr int n = (NST - 2) * NCH;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((n & 15) | ((n >> 4) << 14) | (7 << 4));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  // one LDS read or two after each MFMA of a k-step, then what is left of either
  auto interleave = [&]() {
    constexpr int reads = FN + FM * AL, mfmas = FM * FN, each = (reads + mfmas - 1) / mfmas;
#pragma unroll
    for (int q = 0; q < mfmas; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x100, each, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    }
  };
  // all stages; unit 0 landed. (A fill past the last unit fetches that unit again.)
  Scales scales;
  load_scales(0, scales);
#pragma unroll
  for (int s = 0; s < NST; ++s) fill(min(s, nkt - 1), s);
  write_scales(0, scales);
  __builtin_amdgcn_s_waitcnt((((NST - 1) * NCH) & 15) | ((((NST - 1) * NCH) >> 4) << 14) | (7 << 4));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  AFrag a0[FM], a1[FM];
  i32x4 b0[FN], b1[FN];
  read(0, 0, a0, b0);
  read_scales(0, sca, scb);
  auto unit = [&](int kt, bool odd) {
    const int s = kt % NST;
    if (odd) {
      const int c = (kt + 1) >> 1;
      write_scales(c, scales);  // (its buffer's last reads were two barriers ago)
      if ((c & 3) == 3) load_scales(c + 1, scales);  // (past the last unit: masked, or another row's, never used)
    }
    read(s, 1, a1, b1);
    mma(a0, b0, 0);
    interleave();
    __builtin_amdgcn_sched_barrier(0);
    read(s, 2, a0, b0);
    mma(a1, b1, 1);
    interleave();
    __builtin_amdgcn_sched_barrier(0);
    read(s, 3, a1, b1);
    mma(a0, b0, 2);
    interleave();
    sync();  // every wave is past stage s, and unit kt + 1 landed
    fill(min(kt + NST, nkt - 1), s);
    read((kt + 1) % NST, 0, a0, b0);  // (past the last unit: never used)
    read_scales(kt + 1, nsca, nscb);
    mma(a1, b1, 3);
    interleave();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < FM; ++i) sca[i][0] = nsca[i][0], sca[i][1] = nsca[i][1];
#pragma unroll
    for (int j = 0; j < FN; ++j) scb[j][0] = nscb[j][0], scb[j][1] = nscb[j][1];
  };
  for (int kt = 0;; kt += 2) {
    unit(kt, false);
    if (kt + 1 >= nkt) break;
    unit(kt + 1, true);
    if (kt + 2 >= nkt) break;
  }
  __builtin_amdgcn_s_waitcnt(0x3f70);  // the last fills land before LDS is reused
  __syncthreads();

  // lane l holds, of fragment (i, j) and run g, row wm TM + 32 i + l % 32 and tile columns
  // wn TN + 32 j + 8 g + 4 h + [0, 4)
  if constexpr (SHARE) {
    float* out = (float*)p.c + (int64_t)blockIdx.y * p.split_stride;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = m0 + wm * TM + 32 * i + rf;
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int v = wn * TN + 32 * j + 8 * g + 4 * h;
          const int col = PAIR ? n0 + (v >> 6) * 32 + (v & 31) : n0 + v;
          if (m < p.M && col < p.N)
            *(f32x4*)(out + (int64_t)m * p.ldc + col + (PAIR && (v & 32) ? p.share_up : 0)) =
                f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        }
    }
  } else {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; j += PAIR ? 2 : 1)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int v = wn * TN + 32 * j + 8 * g + 4 * h;
          f32x4 x = f32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]} +
                    *(const f32x4*)(bias + v);
          int col = v;
          if constexpr (PAIR) {
            const f32x4 u = f32x4{acc[i][j + 1][4 * g], acc[i][j + 1][4 * g + 1], acc[i][j + 1][4 * g + 2],
                                  acc[i][j + 1][4 * g + 3]} +
                            *(const f32x4*)(bias + v + 32);
            x = silu_mul4(x, u);
            col = (v >> 6) * 32 + (v & 31);
          }
          *(u32x2*)(smem + (wm * TM + 32 * i + rf) * RS + col * 2) = pack4<2>(HKX_BF16, x);
        }
    __syncthreads();
    constexpr int CPR = OUTW / 8;  // 16-byte pieces a row
    for (int q = tid; q < BM * CPR; q += 256) {
      const int row = q / CPR, ch = q % CPR;
      const int m = m0 + row, n = n0 + 8 * ch;
      if (m >= p.M || n >= p.N) continue;
      const uint8_t* src = smem + row * RS + ch * 16;
      uint16_t* dst = (uint16_t*)p.c + (int64_t)m * p.ldc + n;
      if (p.c_vec) {
        *(i32x4*)dst = *(const i32x4*)src;
      } else {
        for (int x = 0; x < min(8, p.N - n); ++x) dst[x] = ((const uint16_t*)src)[x];
      }
    }
  }
}

// The sum of a K split's shares, in split order, then bias, silu(gate) * up and the one rounding.
struct Mx4ReduceArgs {
  const float* ws;
  int64_t ws_ld, split_stride;
  void* c;
  int64_t ldc;
  const void* bias;
  int32_t bias_dt, splits, M, N, share_up, pair, c_vec;
};

// two: two workgroups a CU.
hipError_t launch_mx4_tile(const Mx4Args& a, bool a8, bool pair, bool share, int bm, bool two, dim3 grid, hipStream_t s);
hipError_t launch_mx4_reduce(const Mx4ReduceArgs& r, hipStream_t s);

}  // namespace hkx
