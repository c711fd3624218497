// Between two blocks of a decoder layer, one pass over a row: the norm after a block, its gated,
// scaled residual add and the norm before the next block,
//   u = x rsqrt(mean x^2 + eps) post,  h = rs r + bs g u,  y = h rsqrt(mean h^2 + eps) pre,
// y as numbers or quantized (MXFP8, MXFP4); and its backward pass. Bound by HBM: forward reads x and
// r and writes h and y once, backward reads x, r, dh, dy and writes dx and dr; a row stays in
// registers between its two reductions, so nothing is read twice. h is rounded for its store only:
// the second norm takes the fp32 h, and the backward pass computes it again from x and r (the same
// bytes as reading the rounded h would be).
//
// A row is held by T threads (a wave, or a workgroup of up to 16), 8 C elements a thread: C pieces of
// 8 (16-byte loads), or single ones T apart where D or a row's address is no multiple of 8.
//
// Measured, 8192 rows of 4096 bf16 with fp32 weights and a gate a sequence: forward 54 us (268 MB, 5.0
// TB/s; a copy of 1 GiB reaches 5.25), backward 83-86 (403 MB, 4.8) and the sum of its partial sums 5.1;
// 4096 rows with an fp32 stream, y as MXFP8, 37 (185 MB, 5.0); 16 rows 4; 999 rows of 1111 fp32 (single
// elements) 6.6, 14.5 and 3.9.
#pragma once

#include <algorithm>

#include "hkx_api.hpp"
#include "hkx_device.hpp"
#include "hkx_mx_block.hpp"

namespace hkx {

struct NormArgs {
  const void* x;
  const void* res;
  const void* post;  // nullptr: u = x
  const void* pre;   // nullptr: no y
  const void* gate;  // nullptr: 1
  void* h;
  void* y;
  uint8_t* ys;   // the scale bytes of a quantized y
  float* rstd;   // [rows][2]: the two norms' factors (nullptr: not kept)
  int64_t ldx, ldr, ldh, ldy, lds;
  int32_t rows, d;
  int32_t gate_dt;
  int32_t gate_rows;  // rows that share a gate's row
  int32_t gate_col;   // 1: a gate a column, 0: one a row
  int32_t quant;      // 0: y as x's type, 1: MXFP8, 2: MXFP4
  float bs, rs, eps;
  double inv_d;  // 1 / d
  int32_t row0;  // the launch's first row (forward)
};

// The elements a thread (8 c, in pieces of 8 where vec), and the row's threads (64: a wave a row, else
// the workgroup).
struct NormShape {
  int c, threads;
  bool vec;
};

struct NormGradArgs {
  NormArgs f;        // x, res, post, pre, gate, rstd and their strides
  const void* dh;    // nullptr: zero
  const void* dy;    // nullptr: zero
  void* dx;
  void* dr;
  void* dgate;       // written here where a worker has whole groups (parts 1), else summed from pgate
  float* ppost;      // [workers][d] partial sums (nullptr: not wanted), likewise ppre
  float* ppre;
  float* pgate;      // [groups][parts][d or 1] (parts past 1)
  int64_t lddh, lddy, lddx, lddr;
  int32_t workers;
  int32_t parts;     // workers a group of gate_rows rows (groups <= workers), or 1
  int32_t groups;    // rows / gate_rows (1 without a gate)
  int32_t group_rows;  // gate_rows (rows without a gate)
  NormShape shape;
};

// ---------------------------------------------------------------- loads and stores of a thread's elements
//
// Through a buffer resource over the row: an element past d reads 0 and is not written, with no
// predicate and 32-bit offsets (pointers a lane and branches cost the backward pass its registers).

// Row elements of thread t of T: piece c of 8 at 8 (t + T c), or element i at t + T i.
template <int C, bool VEC>
struct Cols {
  static constexpr int E = 8 * C;
  struct Row {
    float v[E];
  };
  int t, T, d;

  template <int DT>
  HKX_DEV __amdgpu_buffer_rsrc_t row(const void* p, int64_t at) const {
    constexpr int es = DT == HKX_FP32 ? 4 : 2;
    return make_rsrc((const uint8_t*)p + at * es, p ? (uint32_t)d * es : 0u);  // (nothing: zeros)
  }
  template <int DT>
  HKX_DEV Row load(const void* p, int64_t at) const {
    const __amdgpu_buffer_rsrc_t r = row<DT>(p, at);
    Row o;
    if constexpr (VEC) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        f32x4 a, b;
        if constexpr (DT == HKX_FP32) {
          a = __builtin_bit_cast(f32x4, buf_load16(r, 32u * (uint32_t)(t + T * c), 0));
          b = __builtin_bit_cast(f32x4, buf_load16(r, 32u * (uint32_t)(t + T * c) + 16u, 0));
        } else {
          const i32x4 w = buf_load16(r, 16u * (uint32_t)(t + T * c), 0);
          const u32x2 lo = u32x2{(uint32_t)w.x, (uint32_t)w.y}, hi = u32x2{(uint32_t)w.z, (uint32_t)w.w};
          a = DT == HKX_BF16 ? unpack_bf16x4(lo) : unpack_f16x4(lo);
          b = DT == HKX_BF16 ? unpack_bf16x4(hi) : unpack_f16x4(hi);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) o.v[8 * c + j] = a[j], o.v[8 * c + 4 + j] = b[j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if constexpr (DT == HKX_FP32) {
          o.v[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, 4u * (uint32_t)(t + T * i), 0, 0));
        } else {
          const uint16_t w = __builtin_amdgcn_raw_buffer_load_b16(r, 2u * (uint32_t)(t + T * i), 0, 0);
          o.v[i] = DT == HKX_BF16 ? bf16_to_f32(w) : (float)__builtin_bit_cast(_Float16, w);
        }
      }
    }
    return o;
  }
  template <int DT>
  HKX_DEV void store(void* p, int64_t at, const Row& o) const {
    const __amdgpu_buffer_rsrc_t r = row<DT>(p, at);
    if constexpr (VEC) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if constexpr (DT == HKX_FP32) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const f32x4 w = f32x4{o.v[8 * c + 4 * k], o.v[8 * c + 4 * k + 1], o.v[8 * c + 4 * k + 2], o.v[8 * c + 4 * k + 3]};
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, w), r, 32u * (uint32_t)(t + T * c) + 16u * k, 0, 0);
          }
        } else {
          i32x4 w;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[j] = (int)(DT == HKX_BF16 ? pack_bf16x2(o.v[8 * c + 2 * j], o.v[8 * c + 2 * j + 1])
                                        : pack_f16x2(o.v[8 * c + 2 * j], o.v[8 * c + 2 * j + 1]));
          __builtin_amdgcn_raw_buffer_store_b128(w, r, 16u * (uint32_t)(t + T * c), 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if constexpr (DT == HKX_FP32)
          __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, o.v[i]), r, 4u * (uint32_t)(t + T * i), 0, 0);
        else
          __builtin_amdgcn_raw_buffer_store_b16(
              (uint16_t)(DT == HKX_BF16 ? pack_bf16x2(o.v[i], 0.0f) : pack_f16x2(o.v[i], 0.0f)), r, 2u * (uint32_t)(t + T * i), 0, 0);
      }
    }
  }
};

// ---------------------------------------------------------------- sums over a row's threads

template <int CTRL>
HKX_DEV float add_dpp(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}

HKX_DEV float wave_sum(float x) {
  x = add_dpp<0xb1>(x);   // lane ^ 1
  x = add_dpp<0x4e>(x);   // lane ^ 2
  x = add_dpp<0x141>(x);  // row_half_mirror: the other quad of 8
  x = add_dpp<0x140>(x);  // row_mirror: the other half of 16
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = __builtin_bit_cast(float, (uint32_t)a[0]) + __builtin_bit_cast(float, (uint32_t)a[1]);
  const uint32_t w = __builtin_bit_cast(uint32_t, x);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __builtin_bit_cast(float, (uint32_t)b[0]) + __builtin_bit_cast(float, (uint32_t)b[1]);
}

// A sum over the row's threads, the same bits on each; `red`: 16 floats that no other sum uses
// until a barrier has passed (unused where a row is a wave).
template <bool WAVE>
HKX_DEV float row_sum(float x, float* red) {
  x = wave_sum(x);
  if constexpr (!WAVE) {
    const int w = threadIdx.x >> 6, n = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) red[w] = x;
    __syncthreads();
    x = 0.0f;
    for (int i = 0; i < n; ++i) x += red[i];
  }
  return x;
}

// A norm's factor 1 / sqrt(sum / d + eps), rounded once. v_rsq_f32 alone is up to 0.72 of a step off, for every
// value of the row alike, and takes a subnormal mean for 0. A Newton step leaves 3/2 of the square of
// v_rsq_f64's error (some 2^-26); of a mean of 0 or infinity the step is NaN and the seed is exact.
HKX_DEV float row_factor(float sum, const NormArgs& p) {
  const double m = (double)sum * p.inv_d + (double)p.eps;
  const double y = __builtin_amdgcn_rsq(m);
  const double e = __builtin_fma(-m * y, y, 1.0);
  return (float)(e == e ? __builtin_fma(0.5 * e, y, y) : y);
}

// ---------------------------------------------------------------- quantized stores (whole quads of 8-value pieces)

// 8 values of a row at column i (a multiple of 8) and their block's scale byte: MXFP8, or MXFP4.
HKX_DEV void store_quant(int quant, uint8_t* q, uint8_t* s, int i, const float (&v)[8]) {
  const uint32_t top = mx_block_top(v);
  uint32_t sc;
  if (quant == 1) {
    u32x2 w;
    sc = mx8_block(v, top, w);
    *(u32x2*)(q + i) = w;
  } else {
    uint32_t w;
    sc = mx4_block(v, top, w);
    *(uint32_t*)(q + i / 2) = w;
  }
  if ((i & 31) == 0) s[i / 32] = (uint8_t)sc;
}

// The gate's values of a row: a column each, or one for all.
template <int XT, int C, bool VEC>
HKX_DEV typename Cols<C, VEC>::Row load_gate(const NormArgs& p, const Cols<C, VEC>& cols, int row) {
  const int64_t grp = row / p.gate_rows;
  if (p.gate_col) {
    if (p.gate_dt == XT) return cols.template load<XT>(p.gate, grp * p.d);
    return cols.template load<HKX_FP32>(p.gate, grp * p.d);
  }
  const float v = ld1(p.gate, p.gate_dt, grp);
  typename Cols<C, VEC>::Row g;
#pragma unroll
  for (int i = 0; i < Cols<C, VEC>::E; ++i) g.v[i] = v;
  return g;
}

HKX_DEV void store_one(void* p, int dt, int64_t i, float v) {
  if (dt == HKX_FP32) ((float*)p)[i] = v;
  else ((uint16_t*)p)[i] = (uint16_t)(dt == HKX_BF16 ? pack_bf16x2(v, 0.0f) : pack_f16x2(v, 0.0f));
}

// ---------------------------------------------------------------- forward

template <int XT, int RT, int WT, int C, bool VEC, bool WAVE>
__global__ void __launch_bounds__(WAVE ? 256 : 1024) norm_kernel(const NormArgs p) {
  constexpr int E = Cols<C, VEC>::E;
  __shared__ float red[2][16];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row = p.row0 + (WAVE ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x);
  if (row >= p.rows) return;
  const Cols<C, VEC> cols{WAVE ? (int)(threadIdx.x & 63) : (int)threadIdx.x, WAVE ? 64 : (int)blockDim.x, p.d};
  using Row = typename Cols<C, VEC>::Row;
  Row x = cols.template load<XT>(p.x, row * p.ldx);
  Row r = cols.template load<RT>(p.res, row * p.ldr);
  Row w1, w2, g;
  if (p.post) w1 = cols.template load<WT>(p.post, 0);
  if (p.pre) w2 = cols.template load<WT>(p.pre, 0);
  if (p.gate) g = load_gate<XT>(p, cols, row);
  float rx = 1.0f;
  if (p.post) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += x.v[i] * x.v[i];
    rx = row_factor(row_sum<WAVE>(s, red[0]), p);
#pragma unroll
    for (int i = 0; i < E; ++i) x.v[i] *= rx * w1.v[i];
  }
  if (p.gate) {
#pragma unroll
    for (int i = 0; i < E; ++i) x.v[i] *= g.v[i];
  }
#pragma unroll
  for (int i = 0; i < E; ++i) r.v[i] = p.rs * r.v[i] + p.bs * x.v[i];
  cols.template store<RT>(p.h, row * p.ldh, r);
  float rh = 1.0f;
  if (p.pre) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += r.v[i] * r.v[i];
    rh = row_factor(row_sum<WAVE>(s, red[1]), p);
#pragma unroll
    for (int i = 0; i < E; ++i) r.v[i] *= rh * w2.v[i];
    if (VEC && p.quant) {
#pragma unroll
      for (int c = 0; c < E / 8; ++c) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = r.v[8 * c + j];
        const int i = 8 * (cols.t + cols.T * c);
        if (i < p.d) store_quant(p.quant, (uint8_t*)p.y + row * p.ldy, p.ys + row * p.lds, i, v);
      }
    } else {
      cols.template store<XT>(p.y, row * p.ldy, r);
    }
  }
  if (p.rstd && cols.t == 0) {
    p.rstd[2 * (int64_t)row] = rx;
    p.rstd[2 * (int64_t)row + 1] = rh;
  }
}

// ---------------------------------------------------------------- backward
//
// With xh = x rx, u = xh post, h as above, hh = h rh:
//   dpre = sum over rows of dy hh;  dH = dh + rh (t - hh mean(t hh)), t = dy pre;  dr = rs dH
//   dg = bs dH u, summed over what the gate is broadcast over;  du = bs g dH
//   dpost = sum over rows of du xh;  dx = rx (t2 - xh mean(t2 xh)), t2 = du post
// A worker (a workgroup, or a wave) takes a run of rows that share a gate's row, or whole such runs,
// and keeps its sums of dpost, dpre and the gate in registers; a second launch adds the workers'
// sums in order: no atomics, the same bits every time.

//
// Single elements keep those sums in LDS, one slot an element that only its thread touches (in
// registers they spilled): TM is the most threads of a row there.

template <int XT, int RT, int WT, int C, bool VEC, bool WAVE, int TM = 512>
__global__ void __launch_bounds__(WAVE ? 256 : TM) norm_grad_kernel(const NormGradArgs p) {
  constexpr int E = Cols<C, VEC>::E;
  constexpr int SLOTS = (WAVE ? 64 : TM) * E;
  __shared__ float red[3][16];
  __shared__ float held_sums[VEC ? 1 : (WAVE ? 4 : 1) * 3 * SLOTS];
  const NormArgs& f = p.f;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int worker = WAVE ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x;
  if (worker >= p.workers) return;
  const Cols<C, VEC> cols{WAVE ? (int)(threadIdx.x & 63) : (int)threadIdx.x, WAVE ? 64 : (int)blockDim.x, f.d};
  using Row = typename Cols<C, VEC>::Row;
  // dpost, dpre and the gate: sums 0, 1 and 2
  Row sums[VEC ? 3 : 1];
  float* const own_sums = held_sums + (WAVE && !VEC ? wave * 3 * SLOTS : 0) + cols.t;
  auto sum = [&](int k, int i) -> float& {
    if constexpr (VEC) return sums[k].v[i];
    else return own_sums[k * SLOTS + cols.T * i];
  };
  auto store_sum = [&](int k, float* to, int64_t at) {
    Row o;
#pragma unroll
    for (int i = 0; i < E; ++i) o.v[i] = sum(k, i);
    cols.template store<HKX_FP32>(to, at, o);
  };
  Row w1, w2, g;
#pragma unroll
  for (int i = 0; i < E; ++i) w1.v[i] = w2.v[i] = g.v[i] = 1.0f, sum(0, i) = sum(1, i) = sum(2, i) = 0.0f;
  float ags = 0.0f;
  // (read again every row by single elements, which have no registers to hold them)
  auto weights = [&]() {
    if (f.post) w1 = cols.template load<WT>(f.post, 0);
    if (f.pre) w2 = cols.template load<WT>(f.pre, 0);
  };
  if (VEC) weights();
  const float inv_d = 1.0f / (float)f.d;

  // this worker's rows [row, end): a part of one group, or whole groups
  const int rpg = p.group_rows;
  int row, end;
  if (p.parts > 1) {
    const int grp = worker / p.parts, part = worker % p.parts, chunk = (rpg + p.parts - 1) / p.parts;
    row = grp * rpg + min(part * chunk, rpg);
    end = grp * rpg + min((part + 1) * chunk, rpg);
  } else {
    const int per = (p.groups + p.workers - 1) / p.workers;
    row = min(worker * per, p.groups) * rpg;
    end = min((worker + 1) * per, p.groups) * rpg;
  }
  const bool own_gate = f.gate && f.gate_rows == 1;  // every row its own: written row by row
  const bool group_gate = p.pgate || (f.gate && p.dgate && !own_gate);
  auto flush = [&](int grp) {  // the gate's sums of a group (or of this worker's part of it)
    if (f.gate_col) {
      if (p.pgate) {
        store_sum(2, p.pgate, (int64_t)worker * f.d);
      } else {
        Row o;
#pragma unroll
        for (int i = 0; i < E; ++i) o.v[i] = sum(2, i);
        if (f.gate_dt == XT) cols.template store<XT>(p.dgate, (int64_t)grp * f.d, o);
        else cols.template store<HKX_FP32>(p.dgate, (int64_t)grp * f.d, o);
      }
    } else if (cols.t == 0) {
      if (p.pgate) p.pgate[worker] = ags;
      else store_one(p.dgate, f.gate_dt, grp, ags);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) sum(2, i) = 0.0f;
    ags = 0.0f;
  };
  if (p.pgate && row >= end) flush(0);  // an empty part: zeros
  int held = -1;  // the group whose gate is in g
  for (; row < end; ++row) {
    Row x = cols.template load<XT>(f.x, row * f.ldx);
    Row r = cols.template load<RT>(f.res, row * f.ldr);
    Row dy = cols.template load<XT>(p.dy, row * p.lddy);
    Row dh = cols.template load<RT>(p.dh, row * p.lddh);
    if (f.gate && row / rpg != held) {
      held = row / rpg;
      g = load_gate<XT>(f, cols, row);
    }
    if (!VEC) weights();
    const float rx = f.rstd[2 * (int64_t)row], rh = f.rstd[2 * (int64_t)row + 1];
    float s1 = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      x.v[i] *= rx;                                              // xh (x itself without a post norm: rx = 1)
      r.v[i] = (f.rs * r.v[i] + f.bs * g.v[i] * (x.v[i] * w1.v[i])) * rh;  // hh
      sum(1, i) += dy.v[i] * r.v[i];
      dy.v[i] *= w2.v[i];
      s1 += dy.v[i] * r.v[i];
    }
    if (f.pre) {
      s1 = row_sum<WAVE>(s1, red[0]) * inv_d;
#pragma unroll
      for (int i = 0; i < E; ++i) dh.v[i] += rh * (dy.v[i] - r.v[i] * s1);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) r.v[i] = f.rs * dh.v[i];
    cols.template store<RT>(p.dr, row * p.lddr, r);
    if (f.gate) {
      float sg = 0.0f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        r.v[i] = f.bs * dh.v[i] * (x.v[i] * w1.v[i]);
        sg += r.v[i];
        sum(2, i) += r.v[i];
      }
      if (!f.gate_col) {
        sg = row_sum<WAVE>(sg, red[1]);
        ags += sg;
        if (own_gate && p.dgate && cols.t == 0) store_one(p.dgate, f.gate_dt, row, sg);
      } else if (own_gate && p.dgate) {
        if (f.gate_dt == XT) cols.template store<XT>(p.dgate, (int64_t)row * f.d, r);
        else cols.template store<HKX_FP32>(p.dgate, (int64_t)row * f.d, r);
      }
    }
    float s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float du = f.bs * g.v[i] * dh.v[i];
      sum(0, i) += du * x.v[i];
      dh.v[i] = du * w1.v[i];
      s2 += dh.v[i] * x.v[i];
    }
    if (f.post) {
      s2 = row_sum<WAVE>(s2, red[2]) * inv_d;
#pragma unroll
      for (int i = 0; i < E; ++i) dh.v[i] = rx * (dh.v[i] - x.v[i] * s2);
    }
    cols.template store<XT>(p.dx, row * p.lddx, dh);
    if (group_gate && (row + 1 == end || (row + 1) % rpg == 0)) flush(row / rpg);
    if (!WAVE) __syncthreads();  // (the sums' slots are free for the next row)
  }
  if (p.ppost) store_sum(0, p.ppost, (int64_t)worker * f.d);
  if (p.ppre) store_sum(1, p.ppre, (int64_t)worker * f.d);
}

// By the types of x and the residual, and whether the weights are fp32 (else x's type).
hipError_t launch_norm_bf16(const NormArgs& a, bool r32, bool w32, hipStream_t s);
hipError_t launch_norm_fp16(const NormArgs& a, bool r32, bool w32, hipStream_t s);
hipError_t launch_norm_fp32(const NormArgs& a, hipStream_t s);
hipError_t launch_norm_grad_bf16(const NormGradArgs& a, bool r32, bool w32, hipStream_t s);
hipError_t launch_norm_grad_fp16(const NormGradArgs& a, bool r32, bool w32, hipStream_t s);
hipError_t launch_norm_grad_fp32(const NormGradArgs& a, hipStream_t s);

// ---------------------------------------------------------------- host: the form of a row

inline bool norm_vec_ok(const NormArgs& a, int xs, int rs, int ws, int gs) {
  auto ok = [](const void* p, int64_t ld, int es) { return !p || (api_aligned(p, 16) && ld * es % 16 == 0); };
  return a.d % 8 == 0 && ok(a.x, a.ldx, xs) && ok(a.res, a.ldr, rs) && ok(a.h, a.ldh, rs) &&
         (a.quant || ok(a.y, a.ldy, xs)) && ok(a.post, 0, ws) && ok(a.pre, 0, ws) &&
         (!a.gate || !a.gate_col || ok(a.gate, a.d, gs));
}

// Two pieces a thread past 512 columns (a wave a row up to 1024).
inline NormShape norm_shape(int d, bool vec) {
  const int c = d <= 512 ? 1 : 2;
  return {c, (d + 512 * c - 1) / (512 * c) * 64, vec};
}

constexpr int kNormMaxD = 16384;     // 16 waves of 64 x 16 elements
constexpr int kNormGradMaxD = 8192;  // 8 waves of 64 x 16: ten registers an element

// A launch's threads stay under 2^32 (a grid past that is cut short, with no error): more rows go launch by
// launch, whole workgroups each.
template <int XT, int RT, int WT>
hipError_t launch_norm_typed(NormArgs a, hipStream_t s) {
  auto es = [](int dt) { return dt == HKX_FP32 ? 4 : 2; };
  const NormShape f = norm_shape(a.d, norm_vec_ok(a, es(XT), es(RT), es(WT), es(a.gate_dt)));
  const bool wave = f.threads == 64;
  const int most = (int)((((int64_t)1 << 32) - 1) / f.threads) & ~3;
  for (int64_t r = 0; r < a.rows; r += most) {
    const int rows = (int)std::min<int64_t>(most, a.rows - r);
    a.row0 = (int)r;
    const dim3 grid(wave ? (rows + 3) / 4 : rows), block(wave ? 256 : f.threads);
#define HKX_NORM(C, V, W) hipLaunchKernelGGL((norm_kernel<XT, RT, WT, C, V, W>), grid, block, 0, s, a)
    if (f.vec) {
      if (!wave) HKX_NORM(2, true, false);
      else if (f.c == 1) HKX_NORM(1, true, true);
      else HKX_NORM(2, true, true);
    } else {
      if (!wave) HKX_NORM(2, false, false);
      else if (f.c == 1) HKX_NORM(1, false, true);
      else HKX_NORM(2, false, true);
    }
#undef HKX_NORM
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

template <int XT, int RT, int WT>
hipError_t launch_norm_grad_typed(const NormGradArgs& a, hipStream_t s) {
  const NormShape f = a.shape;
  const bool wave = f.threads == 64;
  const dim3 grid(wave ? (a.workers + 3) / 4 : a.workers), block(wave ? 256 : f.threads);
#define HKX_NORM(...) hipLaunchKernelGGL((norm_grad_kernel<XT, RT, WT, __VA_ARGS__>), grid, block, 0, s, a)
  if (f.vec) {
    if (!wave) HKX_NORM(2, true, false);
    else if (f.c == 1) HKX_NORM(1, true, true);
    else HKX_NORM(2, true, true);
  } else {
    if (!wave && f.threads <= 128) HKX_NORM(2, false, false, 128);
    else if (!wave && f.threads <= 256) HKX_NORM(2, false, false, 256);
    else if (!wave) HKX_NORM(2, false, false, 512);
    else if (f.c == 1) HKX_NORM(1, false, true);
    else HKX_NORM(2, false, true);
  }
#undef HKX_NORM
  return hipGetLastError();
}

}  // namespace hkx
