// The MXFP4 product on 256 x 256 tiles: one persistent workgroup of 8 waves a CU, in the quadrant
// kernel's order (hkx_quad.hpp), 16 x 16 x 128 scaled MFMAs.
//
// * A tile's A rows are two halves of 128 (A0, A1), its B rows likewise. Wave w of the 2 x 4 grid (r,
//   c) = (w / 4, w % 4) owns rows 64 r + 128 i and columns 32 c + 128 j for i, j in {0, 1}: each half of
//   A or B is read by all eight waves in one phase and free for its next fill right after.
// * Slots of quarters, 128 rows x 128 bytes = 16 KB: a 4-bit quarter holds a 256-K unit, an 8-bit A's
//   half a unit (a step of 128 K; a 4-bit A's step is the unit). LDS holds A0 and A1 of two steps and
//   B0 and B1 of two units, 128 KB either way, three rotating buffers of scales (two units of the
//   tile's 512 rows) and the bias of three tiles.
// * A step t is two phases, each LDS reads, fills, a barrier, 32 MFMAs (16 of twice the cycles with an
//   8-bit A), a barrier; the two groups of four waves run one barrier apart, one's reads under the
//   other's MFMAs. With a 4-bit A (B1 is read a step ahead, so that each phase reads 12 fragments):
//     1: read A0(t), B0(t);     fill A1(t + 1), B1(t + 2);  math (0, 0), (0, 1)
//     2: read A1(t), B1(t + 1); fill B0(t + 2), A0(t + 2);  math (1, 0), (1, 1)
//   With an 8-bit A, whose steps are half a unit (B's K-half of the unit):
//     1: read A0(t), B0, B1; fill A1(t + 1);                                        math (0, 0), (0, 1)
//     2: read A1(t);         fill A0(t + 2), and B0, B1 two units on at a unit's last; math (1, 0), (1, 1)
//   A quarter is refilled only after both groups read it. Before a barrier a wave waits for all but
//   its newest fills, those since the quarter that the next phase reads: 8 instructions, or with an
//   8-bit A 4 after a step that filled no B.
// * The next tile's fills run on under a tile's last phases and its epilogue, and group 1 runs its
//   epilogue before the barrier that ends its last phase, so that the groups' epilogues overlap.
// * Scales: packed beforehand (mx4_pack_kernel) so that a lane's bytes of a unit are 16 (A) and 8 (B)
//   consecutive ones, read in two LDS loads and picked by the MFMA's byte select; from the OCP layout a
//   unit took 24 loads, masks and shifts, and 16 bytes a row by DMA were half as many cache lines as
//   the operands themselves. Bytes past K are 0 there.
//
// Measured: 4096 x 12288 x 4096 of 4 bits 102-110 us (3.8-4.0 PFLOP/s; 8192 cubed 261, 4.2), 2048 x 12288 x
// 4096 paired with an 8-bit A 138 (3.0). Register-only loops of these MFMAs on random operands reach 6.97
// and 4.26 PFLOP/s. Two bounds lie close together: the power-limited clock (8192 cubed with operands of zeros
// takes 205 us) and fills with LDS reads (without its MFMAs 183-185, zeros or not, where the MFMAs alone need
// 158 at that rate); without its fills 218 (zeros: 161), without fills and MFMAs 101.
//
// K past its end: as in hkx_mx4.hpp (scales of 0, an 8-bit A's pieces out of range); an 8-bit A
// takes two steps of a unit even where K ends in its first.
#pragma once

#include "hkx_mx4.hpp"
#include "hkx_ring.hpp"

namespace hkx {

template <bool A8, bool PAIR, bool SHARE>
__global__ void __launch_bounds__(512, 1) mx4_quad_kernel(const Mx4Args p) {
  constexpr int BM = 256, BN = PAIR ? 128 : 256;  // BN: C columns of a tile
  constexpr int QB = 128 * 128;
  constexpr int SCO = 8 * QB;            // packed scales: [chunk of two units % 3][A's 4 KB, B's 4 KB]
  constexpr int EPV = SCO + 3 * 8192;    // bias: [tile % 3][B rows' halves of the paired form][1 KB]
  constexpr int SMEM = EPV + 3 * 2048;
  constexpr int SPU = A8 ? 2 : 1;  // steps a unit
  constexpr int KH = A8 ? 1 : 2;   // MFMA K-steps a step
  static_assert(SMEM <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) uint8_t smem[SMEM];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave >> 2, wc = wave & 3;

  const int total = p.tiles_m * p.tiles_n;
  const int G = gridDim.x;
  const int my_tiles = (total - (int)blockIdx.x + G - 1) / G;
  const int u0 = SHARE ? (int)blockIdx.y * p.units_split : 0;
  const int nst = SPU * (SHARE ? min(p.units_split, p.units - u0) : p.units);  // steps a tile
  const int ns = my_tiles * nst;                                              // of this workgroup

  auto tile_at = [&](int lt, int& m0, int& n0) {
    int L = (int)blockIdx.x + lt * G;
    if ((total & 7) == 0) L = (L & 7) * (total >> 3) + (L >> 3);
    const int per = p.wgm * p.tiles_n;
    const int gi = L / per;
    const int first = gi * p.wgm;
    const int gm = min(p.tiles_m - first, p.wgm);
    const int in = L - gi * per;
    m0 = (first + in % gm) * BM;
    n0 = (in / gm) * BN;
  };

  // ---- fills. Instruction k (0, 1) of wave w moves rows 16 w + 8 k + [0, 8) of a quarter: lane l row
  // l % 32 / 4, K-half l / 32, its 16-byte piece (l % 4) ^ swz4(row). Paired: B's tile row 16 F + x is
  // row x of the gate (F even) or up (F odd) block of C columns 16 (F / 2) + [0, 16).
  const __amdgpu_buffer_rsrc_t ra = make_rsrc(p.a, p.a_bytes), rb = make_rsrc(p.b, p.b_bytes);
  uint32_t voff_a[2], voff_b[2], lch[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t row = (uint32_t)(16 * wave + 8 * k + (lane & 31) / 4);
    const uint32_t row_b = PAIR ? (uint32_t)(16 * (wave >> 1) + 8 * k + (lane & 31) / 4 + ((wave & 1) ? p.N : 0)) : row;
    lch[k] = (uint32_t)(64 * (lane >> 5) + 16 * ((lane & 3) ^ ((wave & 1) | (k << 1))));
    voff_a[k] = row * p.lda + lch[k];
    voff_b[k] = row_b * p.ldb + lch[k];
  }
  // The fills walk the workgroup's steps: what they need of a step are scalar offsets, 128 bytes a step
  // on, made anew where a tile begins (the scalar work between two barriers is time that no MFMA
  // covers: streams that made them from the tile's origin, with a remainder by 3 for the scales'
  // buffers, took a third of a step). A half past M or N takes the tile's first rows: they are never stored.
  struct Ahead {
    int t, lt;            // its step (A) or unit (B) in its tile, and the tile
    uint32_t lo, hi, sc;  // A0 and A1, or B0 and B1; the wave's packed scales
  };
  auto at_a = [&](Ahead& s) {
    int m0, n0;
    tile_at(s.lt, m0, n0);
    const uint32_t k = (uint32_t)(SPU * u0) * 128u;
    s.lo = (uint32_t)m0 * p.lda + k;
    s.hi = (uint32_t)(m0 + 128 < p.M ? m0 + 128 : m0) * p.lda + k;
  };
  auto at_b = [&](Ahead& s) {
    int m0, n0;
    tile_at(s.lt, m0, n0);
    constexpr int HB = PAIR ? 64 : 128;
    s.lo = (uint32_t)n0 * p.ldb + (uint32_t)u0 * 128u;
    s.hi = (uint32_t)(n0 + HB < p.N ? n0 + HB : n0) * p.ldb + (uint32_t)u0 * 128u;
    s.sc = ((uint32_t)(wave < 4 ? m0 / BM : n0 / BN) * (uint32_t)((p.units + 1) >> 1) + (uint32_t)(u0 >> 1)) * 4096u;
  };
  // The next step, or past the last the same again, into a slot that nothing reads any more.
  auto next_of = [&](Ahead& s, int per, auto begin, bool scales) {
    if (s.t + 1 < per) {
      ++s.t;
      s.lo += 128u;
      s.hi += 128u;
      if (scales && !(s.t & 1)) s.sc += 4096u;
    } else if (s.lt + 1 < my_tiles) {
      s.t = 0;
      ++s.lt;
      begin(s);
    }
  };
  // A's half i of a step at scalar offset so into the slot at byte `slot` (0 or 2 QB); k: its first K
  auto fill_a = [&](int i, uint32_t slot, uint32_t so, [[maybe_unused]] uint32_t k0) {
    uint8_t* base = smem + slot + i * QB + wave * 2048;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      buf_load16_lds(ra, base + k * 1024, !A8 || k0 + lch[k] < (uint32_t)p.K ? voff_a[k] : kMx4Out, so);
  };
  auto fill_b = [&](int j, uint32_t slot, uint32_t so) {
    uint8_t* base = smem + 4 * QB + slot + j * QB + wave * 2048;
#pragma unroll
    for (int k = 0; k < 2; ++k) buf_load16_lds(rb, base + k * 1024, voff_b[k], so);
  };
  const int upt = nst / SPU;  // units a tile
  // with B0 of a chunk's first unit: wave w a KB of the tile's packed scales (A's, then B's)
  const __amdgpu_buffer_rsrc_t rsc = make_rsrc(wave < 4 ? p.sa : p.sb, wave < 4 ? p.sa_bytes : p.sb_bytes);
  uint32_t sc_fill = 0, sc_read = 0;  // the rotating buffers' offsets
  auto turn = [](uint32_t& o) { o = o == 2 * 8192u ? 0u : o + 8192u; };
  auto fill_scales = [&](const Ahead& s) {
    if (s.t & 1) return;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rsc, (__attribute__((address_space(3))) void*)(smem + SCO + sc_fill + wave * 1024), 16,
        (uint32_t)((wave & 3) * 1024 + lane * 16), (uint32_t)s.sc, 0, 0);
    turn(sc_fill);
  };
  // a tile's bias, raw, into slot lt % 3 during the tile before (waves 0 and, paired, 1: the up half)
  const uint32_t bias_es = p.bias_dt == HKX_FP32 ? 4u : 2u;
  const bool bias = !SHARE && p.bias != nullptr;
  auto fill_bias = [&](int lt) {
    if (!bias || wave > (PAIR ? 1 : 0)) return;
    int cols = p.N;
    asm volatile("" : "+v"(cols));  // (as in the epilogue)
    cols = __builtin_amdgcn_readfirstlane(cols);
    const __amdgpu_buffer_rsrc_t rbias = make_rsrc(
        (const uint8_t*)p.bias + (PAIR && wave == 1 ? (uint64_t)cols * bias_es : 0u), (uint32_t)cols * bias_es);
    int m0, n0;
    tile_at(lt, m0, n0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rbias, (__attribute__((address_space(3))) void*)(smem + EPV + (lt % 3) * 2048 + wave * 1024), 16,
        (uint32_t)lane * 16u + (uint32_t)n0 * bias_es, 0, 0, 0);
  };

  // ---- fragment reads: row l % 16, piece l / 16 of a K-half (rows r0.. at r0 * 128 + 512 half + rdo)
  const int rf = lane & 15, q = lane >> 4;
  uint32_t rdo[2];
#pragma unroll
  for (int par = 0; par < 2; ++par)
    rdo[par] = (uint32_t)((rf >> 3) * 1024 + (rf & 7) * 64 + ((q ^ (par | ((rf >> 3) << 1))) << 4));
  auto piece = [&](const uint8_t* s, int r0, int h) { return *(const i32x4*)(s + r0 * 128 + 512 * h + rdo[(r0 >> 4) & 1]); };
  constexpr int NA = 4, NB = 2;
  using AFrag = typename std::conditional<A8, i32x8, i32x4>::type;
  AFrag af[NA][KH];
  i32x4 b0[NB][KH], b1[NB][KH], bn[NB][KH];  // B0, B1, and with a 4-bit A the next step's B1
  auto read_a = [&](uint32_t slot, int i) {
    const uint8_t* s = smem + slot + i * QB;
#pragma unroll
    for (int f = 0; f < NA; ++f) {
      const i32x4 lo = piece(s, grp * 64 + 16 * f, 0), hi = piece(s, grp * 64 + 16 * f, 1);
      if constexpr (A8) af[f][0] = i32x8{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      else af[f][0] = lo, af[f][1] = hi;
    }
  };
  auto read_b = [&](uint32_t slot, int j, int half, i32x4 (&bf)[NB][KH]) {  // half: an 8-bit A's step of the unit
#pragma unroll
    for (int g = 0; g < NB; ++g)
#pragma unroll
      for (int h = 0; h < KH; ++h) bf[g][h] = piece(smem + 4 * QB + slot + j * QB, wc * 32 + 16 * g, A8 ? half : h);
  };
  // a unit's scale bytes of this lane: A's dword 2 h + i byte f, B's dword h byte 2 j + g
  i32x4 sca;
  u32x2 scb;
  auto read_scales = [&](int odd) {  // the unit's place in its chunk
    const uint8_t* s = smem + SCO + sc_read + 2048 * odd;
    sca = *(const i32x4*)(s + (grp * 64 + lane) * 16);
    scb = *(const u32x2*)(s + 4096 + (wc * 64 + lane) * 8);
  };

  f32x4 acc[2][2][NA][NB];
  auto wide = [](i32x4 v) { return i32x8{v.x, v.y, v.z, v.w, 0, 0, 0, 0}; };
  // block (i, j): the K-half h of the unit is the MFMA's K-step (4-bit A) or the step (8-bit)
  auto block = [&](auto ic, auto jc, int half, const i32x4 (&bf)[NB][KH], bool zero) {
    constexpr int i = decltype(ic)::value, j = decltype(jc)::value;
    auto one = [&](auto hc, auto fc, auto gc) {
      constexpr int h = decltype(hc)::value, f = decltype(fc)::value, g = decltype(gc)::value;
      const f32x4 c = (zero && h == 0) ? f32x4{} : acc[i][j][f][g];
      i32x8 a;
      if constexpr (A8) a = af[f][h];
      else a = wide(af[f][h]);
      const int sb = (int)(A8 ? (half ? scb.y : scb.x) : (h ? scb.y : scb.x));
      const int sa = A8 ? (half ? sca[2 + i] : sca[i]) : sca[2 * h + i];
      acc[i][j][f][g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(bf[g][h]), a, c, 4, A8 ? 0 : 4, 2 * j + g, sb,
                                                                         f, sa);
    };
    auto row = [&](auto hc, auto fc) {
      one(hc, fc, std::integral_constant<int, 0>{});
      one(hc, fc, std::integral_constant<int, 1>{});
    };
    auto kstep = [&](auto hc) {
      row(hc, std::integral_constant<int, 0>{});
      row(hc, std::integral_constant<int, 1>{});
      row(hc, std::integral_constant<int, 2>{});
      row(hc, std::integral_constant<int, 3>{});
    };
    kstep(std::integral_constant<int, 0>{});
    if constexpr (KH == 2) kstep(std::integral_constant<int, 1>{});
  };
  auto math = [&](auto ic, int half, const i32x4 (&bj1)[NB][KH], bool zero) {
    constexpr int i = decltype(ic)::value;
    __builtin_amdgcn_s_setprio(1);
    block(ic, std::integral_constant<int, 0>{}, half, b0, zero);
    block(ic, std::integral_constant<int, 1>{}, half, bj1, zero);
    // (the sums are made here: left alone, the compiler moved whole phases of MFMAs past the
    // branches of the next fills, to their results' next use, and spilled what they read)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int f = 0; f < NA; ++f)
#pragma unroll
        for (int g = 0; g < NB; ++g) asm volatile("" : "+v"(acc[i][j][f][g]));
    __builtin_amdgcn_s_setprio(0);
  };
  constexpr std::integral_constant<int, 0> I0{};
  constexpr std::integral_constant<int, 1> I1{};

  // ---- the epilogue of local tile lt: lane (rf, q) holds row rf, columns 4 q + [0, 4) of each 16 x 16
  // fragment; two fragments trade quarters (v_permlane16_swap) so that a lane stores 16 bytes (C's rows
  // are whole 16-byte pieces; others leave as shares)
  auto bias4 = [&](int lt, int half, int col) -> f32x4 {
    const uint8_t* s = smem + EPV + (lt % 3) * 2048 + half * 1024;
    if (p.bias_dt == HKX_FP32) return *(const f32x4*)(s + 4 * col);
    const u32x2 w = *(const u32x2*)(s + 2 * col);
    return p.bias_dt == HKX_BF16 ? unpack_bf16x4(w) : unpack_f16x4(w);
  };
  auto epilogue = [&](int lt) {
    // (values the compiler cannot see through: what the stores need of the lane and the arguments is
    // made here, once a tile, instead of held in registers through the K loop, which spilled)
    int ln = lane, rows = p.M;
    asm volatile("" : "+v"(ln), "+v"(rows));
    rows = __builtin_amdgcn_readfirstlane(rows);
    const int rf = ln & 15, q = ln >> 4;
    const uint32_t row_b = (uint32_t)p.ldc * (SHARE ? 4u : 2u);
    const __amdgpu_buffer_rsrc_t rc = make_rsrc(
        SHARE ? (const void*)((const float*)p.c + (int64_t)blockIdx.y * p.split_stride) : p.c, (uint32_t)rows * row_b);
    int m0, n0;
    tile_at(lt, m0, n0);
    m0 += 64 * grp;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if constexpr (SHARE) {
#pragma unroll
          for (int f = 0; f < NA; ++f)
#pragma unroll
            for (int g = 0; g < NB; ++g) {
              __builtin_amdgcn_sched_barrier(0);
              const int n = n0 + (PAIR ? 64 * j + 16 * wc : 128 * j + 32 * wc + 16 * g) + 4 * q;
              if (n < p.N)
                __builtin_amdgcn_raw_buffer_store_b128(
                    __builtin_bit_cast(i32x4, acc[i][j][f][g]), rc,
                    (uint32_t)(m0 + 128 * i + 16 * f + rf) * row_b + (uint32_t)(n + (PAIR && g ? p.share_up : 0)) * 4u, 0, 0);
            }
        } else if constexpr (PAIR) {
          // fragments 2 a and 2 a + 1: a lane ends with 8 columns of a row of one of them
          const int col = 64 * j + 16 * wc;
          f32x4 bg = {}, bu = {};
          if (bias) bg = bias4(lt, 0, col + 4 * q), bu = bias4(lt, 1, col + 4 * q);
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            __builtin_amdgcn_sched_barrier(0);
            u32x2 w[2];
#pragma unroll
            for (int f = 0; f < 2; ++f)
              w[f] = pack4<2>(HKX_BF16, silu_mul4(acc[i][j][2 * a + f][0] + bg, acc[i][j][2 * a + f][1] + bu));
            uint32_t ax = w[0].x, ay = w[0].y, bx = w[1].x, by = w[1].y;
            swap16(ax, bx);
            swap16(ay, by);
            const int n = n0 + col + 8 * (ln >> 5);
            if (n < p.N)
              __builtin_amdgcn_raw_buffer_store_b128(
                  i32x4{(int)ax, (int)ay, (int)bx, (int)by}, rc,
                  (uint32_t)(m0 + 128 * i + 32 * a + 16 * (q & 1) + rf) * row_b + (uint32_t)n * 2u, 0, 0);
          }
        } else {
          const int col = 128 * j + 32 * wc;
          f32x4 b0 = {}, b1 = {};
          if (bias) b0 = bias4(lt, 0, col + 4 * q), b1 = bias4(lt, 0, col + 16 + 4 * q);
#pragma unroll
          for (int f = 0; f < NA; ++f) {
            __builtin_amdgcn_sched_barrier(0);
            const u32x2 wa = pack4<2>(HKX_BF16, acc[i][j][f][0] + b0), wb = pack4<2>(HKX_BF16, acc[i][j][f][1] + b1);
            const int m = m0 + 128 * i + 16 * f + rf;
            uint32_t x0 = wa.x, x1 = wb.x, y0 = wa.y, y1 = wb.y;
            swap16(x0, x1);
            swap16(y0, y1);
            const int n = n0 + col + 16 * (q & 1) + 8 * (q >> 1);
            if (n < p.N)
              __builtin_amdgcn_raw_buffer_store_b128(i32x4{(int)x0, (int)y0, (int)x1, (int)y1}, rc,
                                                     (uint32_t)m * row_b + (uint32_t)n * 2u, 0, 0);
          }
        }
      }
  };

  // ---- the K loop
  auto sync = [&](int newest, bool lds) {  // newest: 4 or 8, a constant at every call
    __builtin_amdgcn_sched_barrier(0);
    if (newest == 8) {
      if (lds) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
      else __builtin_amdgcn_s_waitcnt(wait_vm(8));
    } else {
      if (lds) __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(4));
      else __builtin_amdgcn_s_waitcnt(wait_vm(4));
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  Ahead sa{0, 0, 0, 0, 0}, sb{0, 0, 0, 0, 0};
  at_a(sa);
  at_b(sb);
  uint32_t a1 = sa.hi, ka1 = 0, ka = 0;  // A1's step, one behind A0's: its offset; the two's first K (8-bit A)
  auto next_a = [&]() {
    a1 = sa.hi;
    ka1 = ka;
    next_of(sa, nst, at_a, false);
    ka = (uint32_t)(SPU * u0 + sa.t) * 128u;
  };
  auto next_b = [&]() { next_of(sb, upt, at_b, true); };
  if constexpr (A8) ka = ka1 = (uint32_t)(SPU * u0) * 128u;
  fill_bias(0);
  // before step 0, in the steady state's order: B of unit 0 and A0, A1 of step 0, B of unit 1 and A0 of
  // step 1
  uint32_t sl = 0;  // the slot of the current step's A (4-bit: and B); of an 8-bit A's unit's B
  if constexpr (!A8) fill_b(1, 0, sb.hi);
  fill_b(0, 0, sb.lo);
  fill_scales(sb);
  if constexpr (A8) fill_b(1, 0, sb.hi);
  next_b();
  fill_a(0, 0, sa.lo, ka);
  next_a();
  fill_a(1, 0, a1, ka1);
  if constexpr (!A8) fill_b(1, 2 * QB, sb.hi);
  fill_b(0, 2 * QB, sb.lo);
  fill_scales(sb);
  if constexpr (A8) fill_b(1, 2 * QB, sb.hi);
  next_b();
  fill_a(0, 2 * QB, sa.lo, ka);
  next_a();
  // all but A1 of step 0 and what follows it (one more, a chunk of scales, where a tile is one unit)
  __builtin_amdgcn_s_waitcnt(wait_vm(8));
  __builtin_amdgcn_s_barrier();
  if constexpr (!A8) {  // B1 of step 0, read by every wave before any refill of it
    read_b(0, 1, 0, b1);
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(8));
    __builtin_amdgcn_s_barrier();
  }
  if (grp == 1) __builtin_amdgcn_s_barrier();

  // a step of a 4-bit A: cur holds its B1, next takes the next one's. Group 1's last barrier of a tile
  // is after its epilogue.
  auto step4 = [&](int lt, int t, int odd, i32x4 (&cur)[NB][KH], i32x4 (&next)[NB][KH]) {
    read_a(sl, 0);
    read_b(sl, 0, 0, b0);
    read_scales(odd);
    if (t == 0 && lt + 1 < my_tiles) fill_bias(lt + 1);
    fill_a(1, sl ^ (2 * QB), a1, 0);
    fill_b(1, sl, sb.hi);
    sync(8, true);
    math(I0, 0, cur, t == 0);
    sync(8, false);
    read_a(sl, 1);
    read_b(sl ^ (2 * QB), 1, 0, next);
    fill_b(0, sl, sb.lo);
    fill_scales(sb);
    fill_a(0, sl, sa.lo, 0);
    next_b();
    next_a();
    sl ^= 2 * QB;
    sync(8, true);
    math(I1, 0, cur, t == 0);
    if (grp == 0 || t + 1 < nst) sync(8, false);
  };
  // a step of an 8-bit A, half (0, 1) of a unit, whose A slot is the half
  auto step8 = [&](int lt, int u, auto hc) {
    constexpr int half = decltype(hc)::value;
    constexpr int n1 = half ? 4 : 8, n2 = half ? 8 : 4;
    read_a(half * 2 * QB, 0);
    read_b(sl, 0, half, b0);
    read_b(sl, 1, half, b1);
    if (half == 0) read_scales(u & 1);
    if (half == 0 && u == 0 && lt + 1 < my_tiles) fill_bias(lt + 1);
    fill_a(1, (half ^ 1) * 2 * QB, a1, ka1);
    sync(n1, true);
    math(I0, half, b1, half == 0 && u == 0);
    sync(n1, false);
    read_a(half * 2 * QB, 1);
    if (half) {
      fill_b(0, sl, sb.lo);
      fill_scales(sb);
      fill_b(1, sl, sb.hi);
      next_b();
      sl ^= 2 * QB;
    }
    fill_a(0, half * 2 * QB, sa.lo, ka);
    next_a();
    sync(n2, true);
    math(I1, half, b1, half == 0 && u == 0);
    if (half == 0 || grp == 0 || u + 1 < upt) sync(n2, false);
  };
  for (int lt = 0; lt < my_tiles; ++lt) {
    if constexpr (A8) {
      for (int u = 0; u < upt; ++u) {
        step8(lt, u, I0);
        step8(lt, u, I1);
        if ((u & 1) || u + 1 == upt) turn(sc_read);
      }
    } else {
      int t = 0;
      for (; t + 1 < nst; t += 2) {
        step4(lt, t, 0, b1, bn);
        step4(lt, t + 1, 1, bn, b1);
        turn(sc_read);
      }
      if (t < nst) {  // an odd count: the last step, and the next tile's B1 back in b1
        step4(lt, t, 0, b1, bn);
        turn(sc_read);
#pragma unroll
        for (int f = 0; f < NB; ++f)
#pragma unroll
          for (int h = 0; h < KH; ++h) b1[f][h] = bn[f][h];
      }
    }
    epilogue(lt);
    if (grp == 1) sync(8, false);
  }
  if (grp == 0) __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_s_waitcnt(wait_vm(0));  // no fill lands in LDS after the exit
}

// The quadrant kernel's scales, from E8M0 rows (any alignment) to [tile of 256 rows][chunk of two
// units][4 KB]: A's [unit][row group][lane][16 bytes], byte 8 h + 4 i + f of lane (rf, q) the scale of
// row 128 i + 64 grp + 16 f + rf, block 8 unit + 4 h + q; B's [unit][column group][lane][8 bytes], byte
// 4 h + 2 j + g that of tile row 128 j + 32 c + 16 g + rf. Rows past the last and blocks past K are 0.
// (4096 + 12288 rows of 128 bytes take 4.8-5.3 us, half of it a launch's latency.)
struct Mx4PackArgs {
  const uint8_t* s;
  uint8_t* out;
  uint32_t ld, rows;       // rows of s (paired: of the gate; the up rows follow)
  int32_t k32, chunks;     // blocks a row; chunks of 16 blocks
  int32_t tiles;
  int32_t is_b, pair;
};
hipError_t launch_mx4_pack(const Mx4PackArgs& a, const Mx4PackArgs& b, hipStream_t s);

hipError_t launch_mx4_quad(const Mx4Args& a, bool a8, bool pair, bool share, dim3 grid, hipStream_t s);

}  // namespace hkx
