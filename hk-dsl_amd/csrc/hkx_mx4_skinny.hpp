// The MXFP4 product at decode sizes: C (M, N) from X . W^T, 64 rows of X a workgroup (blockIdx.y: which),
// W read once for them, in the 8-bit decode kernel's plan (hkx_skinny.hpp): short workgroups whose 8
// waves cut K, each wave's share of W by non-temporal DMA of whole lines into slots of its own, X in
// registers. Bound by HBM and, where W is small, by the latency of a round: W of 12288 x 4096 (26.7 MB)
// at M = 1 7.5 us, 24576 x 4096 (53.5 MB) paired at M = 16 11.8 us, 4.5 TB/s; 37 x 1001 x 2976 5.7 us.
//
// * A block is 16 rows of W (a 16 x 16 x 128 MFMA fragment): 16 columns of C, or in the paired form 8
//   gate rows and the 8 up rows of the same columns, whose sums meet by a shuffle. A workgroup owns nb
//   (1-4) blocks and 8 waves cut K: in round q of a block wave w takes K unit 8 q + w, 256 K: a line of
//   each row of W and one (4-bit) or two (8-bit) of each row of X.
// * Two rounds are in flight, four of a long K (a workgroup a CU at 4096 columns: two took 4096 x 12288
//   at M = 16 from 9 to 14 us). One fragment of tokens (M <= 16) fits three workgroups a CU, 96 KB of W in
//   flight (two rounds of two units, two workgroups a CU and one unit each with 8-bit X before: 12288 x
//   4096 at M = 1 took 10.9 us). Up to NQ = 2 rounds a block (K = 4096) X stays in registers for all the
//   workgroup's blocks; past that it is streamed with the rounds.
// * X is read in whole lines and turned into the MFMA's layout through the slot, a line at a time.
// * Scales: lane r < 16 (of X: r < 16 MF) reads row r's bytes of the round as dwords, at any
//   alignment (one dword more, joined by the byte offset), masks those past K, and hands them to the
//   lanes by ds_bpermute.
// * K's ragged end reads past the row, into finite 4-bit codes under scales of 0; an 8-bit X's pieces
//   past K, and rows past M and N, are read out of range, as zeros.
#pragma once

#include "hkx_mx4.hpp"
#include "hkx_mx4_rules.hpp"
#include "hkx_skinny.hpp"

namespace hkx {

struct Mx4SkinnyArgs {
  const uint8_t* a;  // X (M, K)
  const uint8_t* b;  // W (N or 2N, K)
  const uint8_t* sa;
  const uint8_t* sb;
  void* c;
  const void* bias;
  uint32_t a_bytes, b_bytes, lda, ldb, sa_ld, sb_ld;
  int64_t ldc;
  int32_t M, N, K, units;
  int32_t nb;  // blocks a workgroup, 1 to 4
  int32_t bias_dt;
  int32_t c_vec;  // C's rows 8-byte aligned and N a multiple of 4: 8-byte stores
};

// Workgroups a CU, as the registers allow: three where a round's X is few, one where it is many.
constexpr int mx4_skinny_resident(int mf, bool a8, bool pair, int nq) {
  if (mf == 1) return nq > 0 && (!a8 || nq == 1 || !pair) ? 3 : a8 && nq == 0 ? 1 : 2;
  return mf == 2 && nq > 0 ? 2 : 1;
}

template <int MF, bool A8, bool PAIR, int NQ>
__global__ void __launch_bounds__(512, 2 * mx4_skinny_resident(MF, A8, PAIR, NQ)) mx4_skinny_kernel(const Mx4SkinnyArgs p) {
  constexpr int NW = 8;
  constexpr int NL = A8 ? 2 : 1;          // lines of a row of X a unit
  constexpr int SLOT = 16 * 128;          // 16 rows of W, or of X as a line is turned
  constexpr int NS = NQ || MF > 2 ? 2 : 4;  // rounds in flight, a slot each
  constexpr int RED = NW * NS * SLOT;     // then the waves' sums of a block: [wave][fragment][lane]
  constexpr int BC = PAIR ? 8 : 16;       // columns a block
  __shared__ __attribute__((aligned(16))) uint8_t lds[RED + NW * MF * 1024];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rf = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * BC * p.nb;
  // blockIdx.y: 64 rows of X and C (all of them where M is no more)
  const int mb = blockIdx.y * 64, rows = min(p.M - mb, 16 * MF);
  const int nb = min(p.nb, (p.N - n0 + BC - 1) / BC);
  const int nq = NQ ? NQ : (p.units + NW - 1) / NW;
  const int nu = nb * nq;  // steps: (block, round)
  uint8_t* own = lds + wave * NS * SLOT;

  const __amdgpu_buffer_rsrc_t rw = make_rsrc(p.b, p.b_bytes), rx = make_rsrc(p.a + (int64_t)mb * p.lda, p.a_bytes - (uint32_t)mb * p.lda);
  // the scales' buffers begin at an aligned dword and end with the one that holds the last byte
  const uint8_t* const sa = p.sa + (int64_t)mb * p.sa_ld;
  const uint32_t sx0 = (uint32_t)((uintptr_t)sa & 3), sw0 = (uint32_t)((uintptr_t)p.sb & 3);
  const uint32_t k32 = (uint32_t)p.K / 32;
  const __amdgpu_buffer_rsrc_t rsx =
      make_rsrc((const void*)((uintptr_t)sa & ~(uintptr_t)3), (sx0 + (uint32_t)(rows - 1) * p.sa_ld + k32 + 3) & ~3u);
  const __amdgpu_buffer_rsrc_t rsw = make_rsrc((const void*)((uintptr_t)p.sb & ~(uintptr_t)3),
                                               (sw0 + (uint32_t)((PAIR ? 2 : 1) * p.N - 1) * p.sb_ld + k32 + 3) & ~3u);

  // W's row of row r of block j
  auto wrow = [&](int j, int r) -> uint32_t {
    if constexpr (PAIR) return (uint32_t)(n0 + 8 * j + (r & 7) + (r & 8 ? p.N : 0));
    else return (uint32_t)(n0 + 16 * j + r);
  };

  // the bias of the workgroup's columns, one a lane (paired: gates, then ups from lane 32 on), as
  // 32 and as 16 bits, without a branch
  const int bc = PAIR ? n0 + (lane & 31) + (lane & 32 ? p.N : 0) : n0 + lane;
  const __amdgpu_buffer_rsrc_t rbias = make_rsrc(p.bias, p.bias ? (uint32_t)((PAIR ? 2 : 1) * p.N) * (p.bias_dt == HKX_FP32 ? 4u : 2u) : 0u);
  float bias32 = 0.0f;
  uint16_t bias16 = 0;
  auto load_bias = [&]() {
    const uint32_t o32 = p.bias_dt == HKX_FP32 ? 0u : kMx4Out, o16 = p.bias_dt == HKX_FP32 ? kMx4Out : 0u;
    bias32 = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rbias, ((uint32_t)bc * 4u) | o32, 0, 0));
    bias16 = __builtin_amdgcn_raw_buffer_load_b16(rbias, ((uint32_t)bc * 2u) | o16, 0, 0);
  };
  load_bias();
  __builtin_amdgcn_sched_barrier(0);

  auto fresh = [](int v) {  // (as in the 8-bit kernel: offsets made again a round, not held)
    asm volatile("" : "+v"(v));
    return v;
  };
  // The row's dwords of a unit from the aligned one on: two, and the next one's part. (Three: of a load of
  // four the compiler used the fourth's register at once, and so waited for the load there.)
  typedef int Scales __attribute__((ext_vector_type(3)));
  auto load_scales = [](__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_bit_cast(Scales, __builtin_amdgcn_raw_buffer_load_b96(r, off, 0, 0));
  };
  constexpr int WLOADS = 3;
  constexpr int XLOADS = 2 * NL * MF + 1;
  struct XRegs {
    i32x4 x[MF][NL][2];
    Scales s;
  };
  // dword d of a unit's row, in place: bytes 4 d .. of it, those past K 0
  auto scale_dword = [&](const Scales& s, uint32_t at, int d, int left) -> uint32_t {
    return __builtin_amdgcn_alignbyte((uint32_t)s[d + 1], (uint32_t)s[d], at & 3) & mx4_mask(left - 4 * d);
  };
  // (Out of range by or-ed bits, not branches. Rows past M and past B's last are out of range by
  // themselves; the paired form's gate rows past N are up rows, whose columns are never stored.)
  // step u's fills into its slot (8 rows x 128 bytes each), and W's scales
  auto issue_w = [&](int u, Scales& sw) {
    const int j = NQ == 1 ? u : u / nq;
    const int k = (u - j * nq) * NW + wave;  // its unit
    const uint32_t out = u < nu && k < p.units ? 0u : kMx4Out;
    uint8_t* slot = own + (u & (NS - 1)) * SLOT;
    __builtin_amdgcn_sched_barrier(0);
    const int ln = fresh(lane);
    sw = load_scales(rsw, ((sw0 + wrow(j, ln & 15) * p.sb_ld + (uint32_t)k * 8u) & ~3u) | out | (ln < 16 ? 0u : kMx4Out));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 8 * i + (ln >> 3), piece = (ln & 7) ^ ((row >> 1) & 7);
      buf_load16_lds<kNonTemporal>(rw, slot + i * 1024,
                                   (wrow(j, row) * p.ldb + (uint32_t)k * 128u + (uint32_t)piece * 16u) | out, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // round q of X in line order, and its scales
  auto issue_x = [&](int q, XRegs& r) {
    const int k = q * NW + wave;
    const int ln = fresh(lane);
    const uint32_t out = k < p.units ? 0u : kMx4Out;
    r.s = load_scales(rsx, ((sx0 + (uint32_t)ln * p.sa_ld + (uint32_t)k * 8u) & ~3u) | out);
#pragma unroll
    for (int f = 0; f < MF; ++f)
#pragma unroll
      for (int l = 0; l < NL; ++l)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = 16 * f + 8 * i + (ln >> 3);
          const uint32_t at = (uint32_t)(k * NL + l) * 128u + (uint32_t)(ln & 7) * 16u;
          r.x[f][l][i] = buf_load16(rx, ((uint32_t)row * p.lda + at) | out | (!A8 || at < (uint32_t)p.K ? 0u : kMx4Out), 0);
        }
    __builtin_amdgcn_sched_barrier(0);
  };
  // into the MFMA's layout: x[f][l][i] the 16-byte piece 4 i + g of row rf's line l
  const uint32_t wr = (uint32_t)((lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 4) & 7)) << 4));
  const uint32_t rd0 = (uint32_t)(rf * 128 + ((g ^ ((rf >> 1) & 7)) << 4)), rd1 = (uint32_t)(rf * 128 + (((4 + g) ^ ((rf >> 1) & 7)) << 4));
  auto turn_x = [&](int u, XRegs& r) {
    uint8_t* slot = own + (u & (NS - 1)) * SLOT;
#pragma unroll
    for (int f = 0; f < MF; ++f)
#pragma unroll
      for (int l = 0; l < NL; ++l) {
        *(i32x4*)(slot + wr) = r.x[f][l][0];  // rows 0-7, and 8-15 with the piece's other half
        *(i32x4*)(slot + 1024 + (wr ^ 64)) = r.x[f][l][1];
        r.x[f][l][0] = *(const i32x4*)(slot + rd0);
        r.x[f][l][1] = *(const i32x4*)(slot + rd1);
      }
  };

  f32x4 acc[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  i32x4 w[2];  // [K-half]
  auto read_w = [&](int u) {
    const uint8_t* slot = own + (u & (NS - 1)) * SLOT;
    w[0] = *(const i32x4*)(slot + rd0);
    w[1] = *(const i32x4*)(slot + rd1);
  };
  auto wide = [](i32x4 v) { return i32x8{v.x, v.y, v.z, v.w, 0, 0, 0, 0}; };
  // W's registers of a step (round q) against X's
  auto mma = [&](int q, const XRegs& r, const Scales& sw) {
    const int left = (int)k32 - 8 * (q * NW + wave);
    // (only their last two bits count, which a block's first row and a unit's first byte leave alone)
    const int ln = fresh(lane);
    const uint32_t atw = sw0 + (uint32_t)(PAIR ? (ln & 7) + (ln & 8 ? p.N : 0) : ln & 15) * p.sb_ld;
    const uint32_t atx = sx0 + (uint32_t)ln * p.sa_ld;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int wsc = (int)((uint32_t)__builtin_amdgcn_ds_bpermute(4 * rf, (int)scale_dword(sw, atw, h, left)) >> (8 * g));
      const uint32_t xd = scale_dword(r.s, atx, h, left);
#pragma unroll
      for (int f = 0; f < MF; ++f) {
        const int xsc = (int)((uint32_t)__builtin_amdgcn_ds_bpermute(4 * (16 * f + rf), (int)xd) >> (8 * g));
        i32x8 x;
        if constexpr (A8) {
          const i32x4 lo = r.x[f][NL - 1 ? h : 0][0], hi = r.x[f][NL - 1 ? h : 0][1];
          x = i32x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        } else {
          x = wide(r.x[f][0][h]);
        }
        acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(w[h]), x, acc[f], 4, A8 ? 0 : 4, 0, wsc, 0, xsc);
      }
    }
  };
  // the sums of block j meet: wave f finishes fragment f's 16 tokens
  const int m_out = 16 * wave + rf;
  auto finish = [&](int j) {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): this wave's reads of the last sums
    if (j > 0) __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int f = 0; f < MF; ++f) {
      *(f32x4*)(lds + RED + ((wave * MF + f) * 64 + lane) * 16) = acc[f];
      acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    if (wave >= MF) return;
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int h = 0; h < NW; h += 4) {
      f32x4 part[4];
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) part[w2] = *(const f32x4*)(lds + RED + (((h + w2) * MF + wave) * 64 + lane) * 16);
#pragma unroll
      for (int w2 = 0; w2 < 4; ++w2) v += part[w2];
    }
    if (p.bias) {
      const float b = p.bias_dt == HKX_FP32 ? bias32
                      : p.bias_dt == HKX_BF16 ? bf16_to_f32(bias16) : (float)__builtin_bit_cast(_Float16, bias16);
      const int from = PAIR ? 8 * j + 4 * (g & 1) + 32 * (g >> 1) : 16 * j + 4 * g;
      v += f32x4{__shfl(b, from), __shfl(b, from + 1), __shfl(b, from + 2), __shfl(b, from + 3)};
    }
    int n = n0 + BC * j + 4 * g;
    if constexpr (PAIR) {
      const f32x4 up = f32x4{__shfl_down(v.x, 32), __shfl_down(v.y, 32), __shfl_down(v.z, 32), __shfl_down(v.w, 32)};
      v = silu_mul4(v, up);
      if (g > 1) n = p.N;
    }
    if (m_out >= rows || n >= p.N) return;
    const u32x2 o = pack4<2>(HKX_BF16, v);
    uint16_t* dst = (uint16_t*)p.c + (int64_t)(mb + m_out) * p.ldc + n;
    if (p.c_vec) {
      *(u32x2*)dst = o;
    } else {
      const uint32_t h[4] = {o.x, o.x >> 16, o.y, o.y >> 16};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) dst[i] = (uint16_t)h[i];
    }
  };
  auto wait0 = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(skinny_vmcnt(0));
    __builtin_amdgcn_sched_barrier(0);
  };
#define HKX_SKINNY_WAIT(N)                       \
  do {                                           \
    __builtin_amdgcn_sched_barrier(0);           \
    __builtin_amdgcn_s_waitcnt(skinny_vmcnt(N)); \
    __builtin_amdgcn_sched_barrier(0);           \
  } while (0)

  Scales s0{}, s1{};
  XRegs x0, x1;  // NQ = 1: x0 alone; 2: round 0's and 1's; 0: turning with the steps, as x2 and x3
  // a step: its fills landed (the newest are the next one's), W read, X turned in its first block
  if constexpr (NQ > 0) {
    auto odd = [&]() -> XRegs& {
      if constexpr (NQ == 2) return x1;
      else return x0;
    };
    issue_x(0, x0);
    issue_w(0, s0);
    if constexpr (NQ == 2) issue_x(1, x1);
    issue_w(1, s1);
    HKX_SKINNY_WAIT(WLOADS + (NQ == 2 ? XLOADS : 0));
    read_w(0);
    turn_x(0, x0);
    mma(0, x0, s0);
    if (NQ == 1 && nu == 1) {
      finish(0);
      wait0();
      return;
    }
    // (past the last step the fills go on, out of range, so that every path waits for one count)
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the slot is free
    issue_w(2, s0);
    if (NQ == 1) finish(0);
    HKX_SKINNY_WAIT(WLOADS);
    read_w(1);
    if constexpr (NQ == 2) turn_x(1, x1);
    mma(NQ == 1 ? 0 : 1, odd(), s1);
    if (nu > 2) {
      __builtin_amdgcn_s_waitcnt(0xc07f);
      issue_w(3, s1);
      finish(NQ == 1 ? 1 : 0);
      auto step = [&](int u, const XRegs& x, Scales& sw) {
        HKX_SKINNY_WAIT(WLOADS);
        read_w(u);
        __builtin_amdgcn_s_waitcnt(0xc07f);
        mma(NQ == 1 ? 0 : u & 1, x, sw);
        issue_w(u + 2, sw);
        if (NQ == 1 || (u & 1)) finish(NQ == 1 ? u : u >> 1);
      };
      for (int u = 2;; u += 2) {
        step(u, x0, s0);
        if (u + 1 >= nu) break;
        step(u + 1, odd(), s1);
        if (u + 2 >= nu) break;
      }
    } else {
      finish(NQ == 1 ? 1 : 0);
    }
  } else {
    [[maybe_unused]] Scales s2{}, s3{};
    [[maybe_unused]] XRegs x2, x3;
    auto round_of = [&](int u) { return u < nq ? u : u % nq; };
    issue_x(0, x0);
    issue_w(0, s0);
    issue_x(round_of(1), x1);
    issue_w(1, s1);
    if constexpr (NS == 4) {
      issue_x(round_of(2), x2);
      issue_w(2, s2);
      issue_x(round_of(3), x3);
      issue_w(3, s3);
    }
    int j = 0, q = 0;      // step u's block and round
    int qx = round_of(NS);  // round of step u + NS
    auto step = [&](int u, XRegs& x, Scales& sw) {
      HKX_SKINNY_WAIT((NS - 1) * (WLOADS + XLOADS));
      read_w(u);
      turn_x(u, x);
      mma(q, x, sw);
      __builtin_amdgcn_s_waitcnt(0xc07f);
      issue_x(qx, x);
      issue_w(u + NS, sw);
      if (++qx == nq) qx = 0;
      if (++q == nq) {
        finish(j++);
        q = 0;
      }
    };
    for (int u = 0;; u += NS) {  // (each exit leaves the loop: a step the compiler sees skipped costs waits)
      step(u, x0, s0);
      if (u + 1 >= nu) break;
      step(u + 1, x1, s1);
      if (u + 2 >= nu) break;
      if constexpr (NS == 4) {
        step(u + 2, x2, s2);
        if (u + 3 >= nu) break;
        step(u + 3, x3, s3);
        if (u + 4 >= nu) break;
      }
    }
  }
#undef HKX_SKINNY_WAIT
  wait0();  // no fill lands in LDS after the exit
}

hipError_t launch_mx4_skinny(Mx4SkinnyArgs a, bool a8, bool pair, int cus, hipStream_t s);

}  // namespace hkx
