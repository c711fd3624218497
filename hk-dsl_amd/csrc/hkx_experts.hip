// The router and the way back: which experts a token goes to, the order of the rows by expert, and the weighted sum of a
// token's rows; their gradients.
#include <algorithm>

#include "hkx_api.hpp"
#include "hkx_device.hpp"
#include "hkx_norm.hpp"

namespace hkx {
namespace {

constexpr int kMaxRouted = 1024;  // experts a wave's lanes hold (16 each)
constexpr int kMaxChosen = 64;    // a lane each
constexpr int kChunk = 64;        // tokens whose places are found together: a bit each

// ---------------------------------------------------------------- the k largest
//
// A wave a token; lane l holds logits J l .. J l + J - 1 as keys: 32 bits that order as the numbers do (-0 as 0, NaN above
// all; 0: no logit), so that the lowest lane of the largest key has the lowest expert. A round: each lane's largest, the
// wave's, the first lane that has it.
//
// Bound by latency: k rounds, one after another, of a wave's largest. 16 tokens of 64 experts, k = 8: 5.2 us, one launch with
// the plan behind it in LDS (up to 64 tokens: a bit of a 64-bit mask each); 16384 of 128: 18 us for the choices (4 tokens a
// wave, 16 waves a workgroup, one after another), 5 for the sums, 5 for the places.

struct RouteArgs {
  const void* logits;
  int64_t ld;
  int32_t dt, t, e, k, renormalize;
  float* weights;
  int32_t* chosen;
  int32_t* offsets;
  int32_t* rows;
  int32_t* slots;
  int32_t* hist;   // [chunks][e]: a chunk's tokens of an expert, then those of the chunks before it
  int32_t* total;  // [e]
  int32_t chunks;
};

HKX_DEV uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
HKX_DEV float of_key(uint32_t k) {
  if (k == 0xffffffffu) return __builtin_nanf("");
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kMinusInf = 0x007fffffu;

// A token's choices: lane j < k writes the j-th (weight, expert) and returns its expert, or -1.
template <int J>
HKX_DEV int choose(const RouteArgs& p, int token) {
  const int lane = threadIdx.x & 63;
  uint32_t key[J];
  const int64_t at = (int64_t)token * p.ld;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = J * lane + j;
    key[j] = e < p.e ? key_of(ld1(p.logits, p.dt, at + e)) : 0u;
  }
  uint32_t best = key[0];
#pragma unroll
  for (int j = 1; j < J; ++j) best = max(best, key[j]);
  float sum = 0.0f;
  const uint32_t first = wave_max(best);
  const float top = of_key(first);
  if (!p.renormalize) {
    // over all experts, from the largest on (a token of -inf alone has no weight)
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (key[j] > kMinusInf) sum += expf(of_key(key[j]) - top);
    sum = wave_sum(sum);
  }
  int expert = -1;
  float value = 0.0f;
  for (int r = 0; r < p.k; ++r) {
    const uint32_t m = r ? wave_max(best) : first;
    if (m <= kMinusInf) break;
    const int who = __builtin_ctzll(__ballot(best == m));
    int mine = 0;
    if (lane == who) {
      bool taken = false;
      best = 0;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (!taken && key[j] == m) {
          taken = true;
          mine = J * lane + j;
          key[j] = 0;
        }
        best = max(best, key[j]);
      }
    }
    const int e = __builtin_amdgcn_readlane(mine, who);
    if (lane == r) {
      expert = e;
      value = expf(of_key(m) - top);
    }
  }
  if (p.renormalize) sum = wave_sum(value);
  if (lane < p.k) {
    const int64_t o = (int64_t)token * p.k + lane;
    p.weights[o] = expert < 0 ? 0.0f : value / sum;
    p.chosen[o] = expert;
  }
  return lane < p.k ? expert : -1;
}

// ---------------------------------------------------------------- many tokens: choices and counts, sums, places

// A chunk a workgroup of 16 waves, 4 tokens a wave.
template <int J>
__global__ void __launch_bounds__(1024) route_choose_kernel(const RouteArgs p) {
  __shared__ int count[64 * J];
  for (int e = threadIdx.x; e < p.e; e += 1024) count[e] = 0;
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  for (int i = wave; i < kChunk; i += 16) {
    const int64_t token = (int64_t)blockIdx.x * kChunk + i;
    if (token >= p.t) break;
    const int e = choose<J>(p, (int)token);
    if (e >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.e; e += 1024) p.hist[(int64_t)blockIdx.x * p.e + e] = count[e];
}

// 16 experts a workgroup: each chunk's count becomes the sum of those before it. Thread (s, e): segment s of 64.
__global__ void __launch_bounds__(1024) route_sum_kernel(const RouteArgs p) {
  __shared__ int part[64][17];
  const int le = threadIdx.x & 15, s = threadIdx.x >> 4, e = blockIdx.x * 16 + le;
  const int per = (p.chunks + 63) / 64, lo = min(s * per, p.chunks), hi = min(lo + per, p.chunks);
  int sum = 0;
  if (e < p.e) {
    for (int c = lo; c < hi; ++c) sum += p.hist[(int64_t)c * p.e + e];
  }
  part[s][le] = sum;
  __syncthreads();
  int before = 0, all = 0;
  for (int i = 0; i < 64; ++i) {
    const int v = part[i][le];
    if (i < s) before += v;
    all += v;
  }
  if (e >= p.e) return;
  for (int c = lo; c < hi; ++c) {
    const int64_t at = (int64_t)c * p.e + e;
    const int v = p.hist[at];
    p.hist[at] = before;
    before += v;
  }
  if (s == 0) p.total[e] = all;
}

// The exclusive sums of count[0 .. e) by the first wave; returns the whole (to that wave).
HKX_DEV int exclusive(int* count, int e) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int g = 0; g < e; g += 64) {
    const int own = g + lane < e ? count[g + lane] : 0;
    int v = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(v, d);
      if (lane >= d) v += u;
    }
    if (g + lane < e) count[g + lane] = sum + v - own;
    sum += __shfl(v, 63);
  }
  return sum;
}

// A token's place among its chunk's tokens of an expert is the number of lower bits of the expert's mask: the rows
// stand in the order of their tokens, and no atomic's order matters.
__global__ void __launch_bounds__(256) route_place_kernel(const RouteArgs p) {
  __shared__ int first[kMaxRouted + 1];
  __shared__ unsigned long long mask[kMaxRouted];
  for (int e = threadIdx.x; e < p.e; e += 256) {
    first[e] = p.total[e];
    mask[e] = 0;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int all = exclusive(first, p.e);
    if (threadIdx.x == 0) first[p.e] = all;
  }
  const int64_t t0 = (int64_t)blockIdx.x * kChunk;
  const int n = (int)min((int64_t)kChunk, p.t - t0) * p.k;
  const int64_t at0 = t0 * p.k;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int e = p.chosen[at0 + i];
    if (e >= 0) atomicOr(&mask[e], 1ull << (i / p.k));
  }
  __syncthreads();
  const int all = first[p.e];
  for (int i = threadIdx.x; i < n; i += 256) {
    const int e = p.chosen[at0 + i], t = i / p.k;
    int slot = -1;
    if (e >= 0) {
      slot = first[e] + p.hist[(int64_t)blockIdx.x * p.e + e] + __popcll(mask[e] & ((1ull << t) - 1));
      p.rows[slot] = (int)(t0 + t);
    }
    p.slots[at0 + i] = slot;
    if (at0 + i >= all) p.rows[at0 + i] = -1;
  }
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= p.e; e += 256) p.offsets[e] = first[e];
}

// ---------------------------------------------------------------- a chunk at most: one launch

template <int J>
__global__ void __launch_bounds__(1024) route_small_kernel(const RouteArgs p) {
  __shared__ int first[64 * J + 1];
  __shared__ unsigned long long mask[64 * J];
  __shared__ int picked[kChunk * kMaxChosen];
  for (int e = threadIdx.x; e < p.e; e += 1024) mask[e] = 0;
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  for (int t = wave; t < p.t; t += 16) {
    const int e = choose<J>(p, t);
    if (e >= 0) atomicOr(&mask[e], 1ull << t);
    if (lane < p.k) picked[t * p.k + lane] = e;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.e; e += 1024) first[e] = __popcll(mask[e]);
  __syncthreads();
  if (threadIdx.x < 64) {
    const int all = exclusive(first, p.e);
    if (threadIdx.x == 0) first[p.e] = all;
  }
  __syncthreads();
  const int all = first[p.e], n = p.t * p.k;
  for (int i = threadIdx.x; i < n; i += 1024) {
    const int e = picked[i], t = i / p.k;
    int slot = -1;
    if (e >= 0) {
      slot = first[e] + __popcll(mask[e] & ((1ull << t) - 1));
      p.rows[slot] = t;
    }
    p.slots[i] = slot;
    if (i >= all) p.rows[i] = -1;
  }
  for (int e = threadIdx.x; e <= p.e; e += 1024) p.offsets[e] = first[e];
}

// ---------------------------------------------------------------- the logits' gradient
//
// A wave a token. Of the chosen alone: w (dw - sum w dw), else 0. Of a softmax over all: p_e (dw_e or 0 - sum w dw), with
// p made again from the logits. 16384 tokens of 128 experts, bf16: 6.6 us, 1.3 TB/s: four waves a workgroup, two barriers.

struct RouteGradArgs {
  const void* logits;
  int64_t ld;
  const float* weights;
  const int32_t* chosen;
  const float* dw;
  void* dl;
  int64_t lddl;
  int32_t dt, t, e, k, renormalize;
};

template <int J>
__global__ void __launch_bounds__(256) route_grad_kernel(const RouteGradArgs p) {
  __shared__ float at[4][64 * J];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t token = (int64_t)blockIdx.x * 4 + wave;
  const bool in = token < p.t;
  float* g = at[wave];
  for (int e = lane; e < p.e; e += 64) g[e] = 0.0f;
  __syncthreads();
  float w = 0.0f, dw = 0.0f;
  int e = -1;
  if (in && lane < p.k) {
    e = p.chosen[token * p.k + lane];
    if ((uint32_t)e < (uint32_t)p.e) {
      w = p.weights[token * p.k + lane];
      dw = p.dw[token * p.k + lane];
    } else {
      e = -1;
    }
  }
  const float dot = wave_sum(w * dw);
  if (e >= 0) g[e] = p.renormalize ? w * (dw - dot) : dw;
  __syncthreads();
  if (!in) return;
  float top = 0.0f, sum = 1.0f;
  if (!p.renormalize) {
    uint32_t best = 0;
    for (int i = lane; i < p.e; i += 64) best = max(best, key_of(ld1(p.logits, p.dt, token * p.ld + i)));
    best = wave_max(best);
    top = of_key(best);
    sum = 0.0f;
    if (best > kMinusInf)
      for (int i = lane; i < p.e; i += 64) sum += expf(ld1(p.logits, p.dt, token * p.ld + i) - top);
    sum = wave_sum(sum);
    if (best <= kMinusInf) sum = 0.0f;
  }
  for (int i = lane; i < p.e; i += 64) {
    float v = g[i];
    if (!p.renormalize) v = sum == 0.0f ? 0.0f : expf(ld1(p.logits, p.dt, token * p.ld + i) - top) / sum * (v - dot);
    store_one(p.dl, p.dt, token * p.lddl + i, v);
  }
}

// ---------------------------------------------------------------- the way back
//
// A workgroup 2048 columns of a token, a thread 8 (pieces of 16 bytes of a 16-bit type, or single elements 256 apart). Bound
// by HBM: 8192 tokens of 4 rows of 4096 bf16, 335 MB in 77-79 us, 4.3 TB/s; four rows in flight. A gathered x's gradient is
// the same sum of fp32 rows: 4096 tokens of 2 rows of 2048 into bf16, 84 MB in 14.6 us, 5.7 TB/s (the rows' product has just
// written them).

struct CombineArgs {
  const void* y;
  const void* dout;
  const int32_t* slots;
  const int32_t* owner;  // the gradient's
  const int32_t* other;
  const float* weights;
  void* out;
  float* dw;
  int64_t ldy, ldo, lddy;
  int32_t t, k, rows, d;
};

// (OT: out's type)
template <int DT, bool VEC, int OT = DT>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs p) {
  const int per = (p.d + 2047) / 2048;
  const int64_t token = blockIdx.x / per;
  const int part = (int)(blockIdx.x - token * per), c0 = part * 2048;
  const Cols<1, VEC> cols{(int)threadIdx.x, 256, min(p.d - c0, 2048)};
  float sum[8] = {};
  const int32_t* slots = p.slots + token * p.k;
  const float* w = p.weights ? p.weights + token * p.k : nullptr;
#pragma unroll 4
  for (int j = 0; j < p.k; ++j) {
    const int s = slots[j];
    const bool in = (uint32_t)s < (uint32_t)p.rows;
    const float f = in ? (w ? w[j] : 1.0f) : 0.0f;
    const auto v = cols.template load<DT>(in ? p.y : nullptr, (in ? s : 0) * p.ldy + c0);  // (nothing: zeros)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += f * v.v[i];
  }
  typename Cols<1, VEC>::Row o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o.v[i] = sum[i];
  cols.template store<OT>(p.out, token * p.ldo + c0, o);
}

// The gradient: a workgroup a token, its k rows of dy and k dot products. A row that no slot names gets zeros (from the
// token whose choices have its number), one that several name the sum of theirs, in order, from one of them.
//
// Which is which takes one launch and no cleared memory. owner[r] ends as a choice that names r; of what stands in it
// beforehand nothing is assumed, as slots says whether a choice names a row. A choice that finds another one that names its
// row in its place keeps it in other[]: of several at least the last has one, and the last is the owner.
//
// Bound by HBM: 8192 tokens of 4 rows of 4096 bf16, 604 MB in 107 us, 5.6 TB/s (one choice after another, its barriers and
// dout again for each, 130).

__global__ void __launch_bounds__(256) combine_owner_kernel(const int32_t* slots, int32_t* owner, int32_t* other, int rows) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= rows) return;
  const int i = (int)at, s = slots[i];
  int found = -1;
  if ((uint32_t)s < (uint32_t)rows) {
    const int before = atomicExch(&owner[s], i);
    if ((uint32_t)before < (uint32_t)rows && before != i && slots[before] == s) found = before;
  }
  other[i] = found;
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(256) combine_grad_kernel(const CombineArgs p) {
  constexpr int B = 4;
  __shared__ float red[B][4];
  const int64_t token = blockIdx.x, first = token * p.k;
  const int lane = threadIdx.x & 63;
  auto piece = [&](int c0) { return Cols<1, VEC>{(int)threadIdx.x, 256, min(p.d - c0, 2048)}; };
  auto sum_all = [&](int s) {  // row s of dy: its choices, in order
    for (int c0 = 0; c0 < p.d; c0 += 2048) {
      const auto cols = piece(c0);
      typename Cols<1, VEC>::Row sum{};
      for (int64_t i = 0; i < p.rows; i += 64) {
        for (uint64_t m = __ballot(i + lane < p.rows && p.slots[min(i + lane, (int64_t)p.rows - 1)] == s); m; m &= m - 1) {
          const int64_t from = i + __builtin_ctzll(m);
          const float w = p.weights ? p.weights[from] : 1.0f;
          const auto g = cols.template load<DT>(p.dout, from / p.k * p.ldo + c0);
#pragma unroll
          for (int c = 0; c < 8; ++c) sum.v[c] += w * g.v[c];
        }
      }
      cols.template store<DT>(p.out, s * p.lddy + c0, sum);
    }
  };
  for (int j0 = 0; j0 < p.k; j0 += 64) {
    // a lane a choice: its row, and whose rows the choice's row and the row of its own number are
    const int n = min(p.k - j0, 64);
    int slot = -1, kind = 0;  // kind: 1 its row is this choice's alone, 2 others' too and this one's to write; 4 a row of zeros
    float weight = 0.0f;
    if (lane < n) {
      const int i = (int)first + j0 + lane;
      slot = p.slots[i];
      const bool in = (uint32_t)slot < (uint32_t)p.rows;
      if (in) weight = p.weights ? p.weights[i] : 1.0f;
      if (p.out) {
        const int other = p.other[i], here = p.owner[i];
        if (in && p.owner[slot] == i) kind = other < 0 ? 1 : 2;
        if ((uint32_t)here >= (uint32_t)p.rows || p.slots[here] != i) kind |= 4;
      }
      if (!in) slot = -1;
    }
    // B choices at a time: their rows of y are in flight together, and dout is read once
    for (int jb = 0; jb < n; jb += B) {
      int s[B], what[B];
      float f[B], dot[B] = {};
#pragma unroll
      for (int b = 0; b < B; ++b) {  // (past n: no row)
        s[b] = __builtin_amdgcn_readlane(slot, jb + b);
        what[b] = __builtin_amdgcn_readlane(kind, jb + b);
        f[b] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), jb + b));
      }
      for (int c0 = 0; c0 < p.d; c0 += 2048) {
        const auto cols = piece(c0);
        const auto g = cols.template load<DT>(p.dout, token * p.ldo + c0);
        if (p.dw) {
          typename Cols<1, VEC>::Row y[B];
#pragma unroll
          for (int b = 0; b < B; ++b) y[b] = cols.template load<DT>(s[b] >= 0 ? p.y : nullptr, max(s[b], 0) * p.ldy + c0);
#pragma unroll
          for (int b = 0; b < B; ++b)
#pragma unroll
            for (int i = 0; i < 8; ++i) dot[b] += g.v[i] * y[b].v[i];
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
          typename Cols<1, VEC>::Row o;
#pragma unroll
          for (int i = 0; i < 8; ++i) o.v[i] = g.v[i] * f[b];
          if (what[b] & 1) cols.template store<DT>(p.out, s[b] * p.lddy + c0, o);
          if (what[b] & 4) cols.template store<DT>(p.out, (first + j0 + jb + b) * p.lddy + c0, typename Cols<1, VEC>::Row{});
        }
      }
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (what[b] & 2) sum_all(s[b]);
      if (p.dw) {
        __syncthreads();  // (the last ones are read)
#pragma unroll
        for (int b = 0; b < B; ++b) {
          dot[b] = wave_sum(dot[b]);
          if (lane == 0) red[b][threadIdx.x >> 6] = s[b] >= 0 ? dot[b] : 0.0f;
        }
        __syncthreads();
        const int b = threadIdx.x;
        if (b < B && jb + b < n) p.dw[first + j0 + jb + b] = red[b][0] + red[b][1] + red[b][2] + red[b][3];
      }
    }
  }
}

// ---------------------------------------------------------------- rows to 8 bits
//
// A workgroup a row, a thread 8 columns of every 2048; up to 16384 columns stay in registers between the largest and
// the codes (P pieces a thread), past that they are read again. Bound by HBM for many rows (8192 of 14336 bf16: 65.7 us,
// 5.36 TB/s, where a copy has 4.8; of fp32 109, 5.4), by a launch for few (512 rows of 1024 bf16: 4 us). The scale is the row's
// largest / 448, so that no value is clamped.

struct QuantArgs {
  const void* x;
  uint8_t* q;
  float* s;
  int64_t ldx, ldq;
  int32_t k;
};

template <int DT, int P, bool VEC>
__global__ void __launch_bounds__(256) fp8_quant_kernel(const QuantArgs p) {
  __shared__ uint32_t red[4];
  const int64_t row = blockIdx.x;
  constexpr int es = DT == HKX_FP32 ? 4 : 2;
  const int pieces = P ? P : (p.k + 2047) / 2048;
  using Row = typename Cols<1, VEC>::Row;
  // (a piece past the row has no columns: zeros)
  auto cols_at = [&](int c) { return Cols<1, VEC>{(int)threadIdx.x, 256, min(max(p.k - 2048 * c, 0), 2048)}; };
  const uint8_t* x = (const uint8_t*)p.x + row * p.ldx * es;
  Row v[P ? P : 1];
  uint32_t top = 0;  // |x|'s bits order as the numbers do, a NaN's above an infinity's
  auto largest = [&](const Row& r) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __builtin_bit_cast(uint32_t, r.v[i]) & 0x7fffffffu);
  };
  if constexpr (P > 0) {
#pragma unroll
    for (int c = 0; c < P; ++c) v[c] = cols_at(c).template load<DT>(x, 2048 * c);
#pragma unroll
    for (int c = 0; c < P; ++c) largest(v[c]);
  } else {
    for (int c = 0; c < pieces; ++c) largest(cols_at(c).template load<DT>(x, 2048 * c));
  }
  top = wave_max(top);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
  __syncthreads();
  top = max(max(red[0], red[1]), max(red[2], red[3]));
  const float s = fp8_row_scale(top);
  auto put = [&](const Row& r, int c) { cols_at(c).store8(p.q + row * p.ldq, 2048 * c, r.v, 0, s); };
  if constexpr (P > 0) {
#pragma unroll
    for (int c = 0; c < P; ++c) put(v[c], c);
  } else {
    for (int c = 0; c < pieces; ++c) put(cols_at(c).template load<DT>(x, 2048 * c), c);
  }
  if (threadIdx.x == 0) p.s[row] = s;
}

template <int DT, bool VEC>
hipError_t launch_quant(const QuantArgs& a, int m, hipStream_t st) {
  const int most = ((1 << 24) - 1);  // rows a launch: under 2^32 threads
  for (int64_t r = 0; r < m; r += most) {
    QuantArgs b = a;
    b.x = (const uint8_t*)a.x + r * a.ldx * (DT == HKX_FP32 ? 4 : 2);
    b.q += r * a.ldq;
    b.s += r;
    const dim3 grid((unsigned)std::min<int64_t>(most, m - r));
#define HKX_QUANT(P) hipLaunchKernelGGL((fp8_quant_kernel<DT, P, VEC>), grid, dim3(256), 0, st, b)
    if (a.k <= 2048) HKX_QUANT(1);
    else if (a.k <= 4096) HKX_QUANT(2);
    else if (a.k <= 8192) HKX_QUANT(4);
    else if (a.k <= 16384) HKX_QUANT(8);
    else HKX_QUANT(0);
#undef HKX_QUANT
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

bool floating(int dt) { return dt == HKX_BF16 || dt == HKX_FP16 || dt == HKX_FP32; }
int es(int dt) { return dt == HKX_FP32 ? 4 : 2; }

int route_chunks(int t) { return (t + kChunk - 1) / kChunk; }

size_t route_bytes(int t, int e) {
  return t <= kChunk ? 0 : ((size_t)route_chunks(t) * e + e) * 4;
}

// the logits a lane holds
template <typename F>
hipError_t by_lane(int e, F f) {
  if (e <= 64) return f(std::integral_constant<int, 1>{});
  if (e <= 128) return f(std::integral_constant<int, 2>{});
  if (e <= 256) return f(std::integral_constant<int, 4>{});
  if (e <= 512) return f(std::integral_constant<int, 8>{});
  return f(std::integral_constant<int, 16>{});
}

template <typename F>
hipError_t by_type(int dt, F f) {
  if (dt == HKX_BF16) return f(std::integral_constant<int, HKX_BF16>{});
  if (dt == HKX_FP16) return f(std::integral_constant<int, HKX_FP16>{});
  return f(std::integral_constant<int, HKX_FP32>{});
}

bool whole(const void* p, int64_t ld, int dt) { return !p || (api_aligned(p, 16) && ld * es(dt) % 16 == 0); }

}  // namespace
}  // namespace hkx

extern "C" {

size_t hkx_experts_route_workspace(const HkxExpertsRouteArgs* args) {
  if (!args || args->size != sizeof *args || args->t < 1 || args->e < 1 || args->e > hkx::kMaxRouted) return 0;
  return hkx::route_bytes(args->t, args->e);
}

int hkx_experts_route(const HkxExpertsRouteArgs* args, void* stream) {
  using namespace hkx;
  api_clear();
  if (!args) return api_fail(HKX_ERR_ARG, "experts_route: null args");
  if (args->size != sizeof *args)
    return api_fail(HKX_ERR_ARG, "experts_route: args of %d bytes, the library's have %zu", args->size, sizeof *args);
  const HkxExpertsRouteArgs& g = *args;
  if (!g.logits || !g.weights || !g.chosen || !g.offsets || !g.rows || !g.slots) return api_fail(HKX_ERR_ARG, "experts_route: a null pointer");
  if (!floating(g.dtype)) return api_fail(HKX_ERR_DTYPE, "experts_route: logits are bf16, fp16 or fp32");
  if (g.t < 1 || g.e < 1 || g.e > kMaxRouted || g.k < 1 || g.k > kMaxChosen || g.k > g.e || g.ld < g.e || (int64_t)g.t * g.k > INT32_MAX)
    return api_fail(HKX_ERR_SHAPE, "experts_route: t=%d e=%d (at most %d) k=%d (at most %d and e)", g.t, g.e, kMaxRouted, g.k, kMaxChosen);
  const size_t need = route_bytes(g.t, g.e);
  if (need && (!g.ws || g.ws_bytes < need || !api_aligned(g.ws, 16)))
    return api_fail(HKX_ERR_WORKSPACE, "experts_route: needs %zu bytes of 16-byte aligned workspace, got %zu", need, g.ws ? g.ws_bytes : (size_t)0);
  RouteArgs a{};
  a.logits = g.logits;
  a.ld = g.ld;
  a.dt = g.dtype;
  a.t = g.t;
  a.e = g.e;
  a.k = g.k;
  a.renormalize = g.renormalize != 0;
  a.weights = g.weights;
  a.chosen = g.chosen;
  a.offsets = g.offsets;
  a.rows = g.rows;
  a.slots = g.slots;
  a.chunks = route_chunks(g.t);
  a.hist = (int32_t*)g.ws;
  a.total = a.hist + (int64_t)a.chunks * g.e;
  const hipStream_t s = (hipStream_t)stream;
  if (g.t <= kChunk)
    return api_launched(by_lane(g.e, [&](auto j) {
      hipLaunchKernelGGL((route_small_kernel<decltype(j)::value>), dim3(1), dim3(1024), 0, s, a);
      return hipGetLastError();
    }), "experts route");
  // (2^22 chunks of 1024 threads are a launch's 2^32)
  if (a.chunks >= 1 << 22) return api_fail(HKX_ERR_SHAPE, "experts_route: t=%d tokens are more than a launch takes; split the call", g.t);
  return api_launched(by_lane(g.e, [&](auto j) {
    hipLaunchKernelGGL((route_choose_kernel<decltype(j)::value>), dim3(a.chunks), dim3(1024), 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(route_sum_kernel, dim3((a.e + 15) / 16), dim3(1024), 0, s, a);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL(route_place_kernel, dim3(a.chunks), dim3(256), 0, s, a);
    return hipGetLastError();
  }), "experts route");
}

int hkx_experts_route_backward(const void* logits, int64_t ld, int32_t dtype, const float* weights, const int32_t* chosen,
                               const float* dweights, void* dlogits, int64_t lddl, int32_t t, int32_t e, int32_t k,
                               int32_t renormalize, void* stream) {
  using namespace hkx;
  api_clear();
  if (!logits || !weights || !chosen || !dweights || !dlogits) return api_fail(HKX_ERR_ARG, "experts_route_backward: a null pointer");
  if (!floating(dtype)) return api_fail(HKX_ERR_DTYPE, "experts_route_backward: logits are bf16, fp16 or fp32");
  if (t < 1 || e < 1 || e > kMaxRouted || k < 1 || k > kMaxChosen || k > e || ld < e || lddl < e)
    return api_fail(HKX_ERR_SHAPE, "experts_route_backward: t=%d e=%d k=%d", t, e, k);
  return api_launched(by_lane(e, [&](auto j) {
    constexpr int64_t most = 1 << 25;  // tokens a launch: under 2^32 threads
    for (int64_t i = 0; i < t; i += most) {
      const int n = (int)std::min(most, t - i);
      const RouteGradArgs a{(const uint8_t*)logits + i * ld * es(dtype), ld, weights + i * k, chosen + i * k, dweights + i * k,
                            (uint8_t*)dlogits + i * lddl * es(dtype), lddl, dtype, n, e, k, renormalize != 0};
      hipLaunchKernelGGL((route_grad_kernel<decltype(j)::value>), dim3((n + 3) / 4), dim3(256), 0, (hipStream_t)stream, a);
      if (hipError_t rc = hipGetLastError()) return rc;
    }
    return hipSuccess;
  }), "experts route backward");
}

int hkx_experts_combine(const void* y, int64_t ldy, int32_t dtype, const int32_t* slots, const float* weights, void* out,
                        int64_t ldo, int32_t t, int32_t k, int32_t rows, int32_t d, void* stream) {
  using namespace hkx;
  api_clear();
  if (!y || !slots || !out) return api_fail(HKX_ERR_ARG, "experts_combine: a null pointer");
  if (!floating(dtype)) return api_fail(HKX_ERR_DTYPE, "experts_combine: y is bf16, fp16 or fp32");
  if (t < 0 || k < 1 || rows < 0 || d < 1 || ldy < d || ldo < d) return api_fail(HKX_ERR_SHAPE, "experts_combine: t=%d k=%d rows=%d d=%d", t, k, rows, d);
  if (t == 0) return HKX_OK;
  const int64_t grid = (int64_t)t * ((d + 2047) / 2048);
  if (grid >= 1 << 24) return api_fail(HKX_ERR_SHAPE, "experts_combine: t=%d of d=%d are more than a launch takes; split the call", t, d);
  CombineArgs a{};
  a.y = y;
  a.slots = slots;
  a.weights = weights;
  a.out = out;
  a.ldy = ldy;
  a.ldo = ldo;
  a.t = t;
  a.k = k;
  a.rows = rows;
  a.d = d;
  const bool vec = d % 8 == 0 && whole(y, ldy, dtype) && whole(out, ldo, dtype);
  return api_launched(by_type(dtype, [&](auto dt) {
    if (vec) hipLaunchKernelGGL((combine_kernel<decltype(dt)::value, true>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((combine_kernel<decltype(dt)::value, false>), dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, a);
    return hipGetLastError();
  }), "experts combine");
}

int hkx_experts_gather_grad(const float* dr, int64_t lddr, const int32_t* slots, void* dx, int64_t lddx, int32_t t, int32_t k,
                            int32_t rows, int32_t d, void* stream) {
  using namespace hkx;
  api_clear();
  if (!dr || !slots || !dx) return api_fail(HKX_ERR_ARG, "experts_gather_grad: a null pointer");
  if (t < 0 || k < 1 || rows < 0 || d < 1 || lddr < d || lddx < d)
    return api_fail(HKX_ERR_SHAPE, "experts_gather_grad: t=%d k=%d rows=%d d=%d", t, k, rows, d);
  if (!api_aligned(dr, 4) || !api_aligned(dx, 2)) return api_fail(HKX_ERR_SHAPE, "experts_gather_grad: the operands need their elements' alignment");
  if (t == 0) return HKX_OK;
  CombineArgs a{};
  a.y = dr;
  a.ldy = lddr;
  a.ldo = lddx;
  a.k = k;
  a.rows = rows;
  a.d = d;
  const bool vec = d % 8 == 0 && whole(dr, lddr, HKX_FP32) && whole(dx, lddx, HKX_BF16);
  const int64_t per = ((int64_t)d + 2047) / 2048, most = std::max<int64_t>(((1 << 24) - 1) / per, 1);  // under 2^32 threads a launch
  for (int64_t i = 0; i < t; i += most) {
    a.t = (int)std::min(most, t - i);
    a.slots = slots + i * k;
    a.out = (uint16_t*)dx + i * lddx;
    const dim3 grid((unsigned)(a.t * per));
    if (vec) hipLaunchKernelGGL((combine_kernel<HKX_FP32, true, HKX_BF16>), grid, dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((combine_kernel<HKX_FP32, false, HKX_BF16>), grid, dim3(256), 0, (hipStream_t)stream, a);
    if (hipError_t e = hipGetLastError()) return api_launched(e, "experts gather grad");
  }
  return api_launched(hipSuccess, "experts gather grad");
}

int hkx_experts_combine_backward(const void* y, int64_t ldy, const void* dout, int64_t lddo, int32_t dtype, const int32_t* slots,
                                 const float* weights, void* dy, int64_t lddy, float* dweights, void* ws, int32_t t,
                                 int32_t k, int32_t rows, int32_t d, void* stream) {
  using namespace hkx;
  api_clear();
  if ((dweights && !y) || !dout || !slots || (!dy && !dweights) || (dy && !ws)) return api_fail(HKX_ERR_ARG, "experts_combine_backward: a null pointer");
  if (!floating(dtype)) return api_fail(HKX_ERR_DTYPE, "experts_combine_backward: y is bf16, fp16 or fp32");
  if (t < 0 || k < 1 || rows != (int64_t)t * k || d < 1 || (dweights && ldy < d) || lddo < d || (dy && (lddy < d || !api_aligned(ws, 4))) || t >= 1 << 24)
    return api_fail(HKX_ERR_SHAPE, "experts_combine_backward: t=%d k=%d rows=%d d=%d", t, k, rows, d);
  if (t == 0) return HKX_OK;
  CombineArgs a{};
  a.y = y;
  a.dout = dout;
  a.slots = slots;
  a.owner = (const int32_t*)ws;
  a.other = a.owner + rows;
  a.weights = weights;
  a.out = dy;
  a.dw = dweights;
  a.ldy = ldy;
  a.ldo = lddo;
  a.lddy = lddy;
  a.t = t;
  a.k = k;
  a.rows = rows;
  a.d = d;
  const hipStream_t st = (hipStream_t)stream;
  if (dy) {
    const dim3 grid((unsigned)(((int64_t)rows + 255) / 256));
    hipLaunchKernelGGL(combine_owner_kernel, grid, dim3(256), 0, st, slots, (int32_t*)ws, (int32_t*)ws + rows, rows);
    if (hipError_t e = hipGetLastError()) return api_launched(e, "experts combine backward");
  }
  const bool vec = d % 8 == 0 && whole(dweights ? y : nullptr, ldy, dtype) && whole(dout, lddo, dtype) && whole(dy, lddy, dtype);
  return api_launched(by_type(dtype, [&](auto dt) {
    if (vec) hipLaunchKernelGGL((combine_grad_kernel<decltype(dt)::value, true>), dim3(t), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((combine_grad_kernel<decltype(dt)::value, false>), dim3(t), dim3(256), 0, st, a);
    return hipGetLastError();
  }), "experts combine backward");
}

int hkx_fp8_quant(const void* x, int64_t ldx, int32_t x_dtype, void* q, int64_t ldq, float* s, int32_t m, int32_t k, void* stream) {
  using namespace hkx;
  api_clear();
  if (!x || !q || !s) return api_fail(HKX_ERR_ARG, "fp8_quant: a null pointer");
  if (!floating(x_dtype)) return api_fail(HKX_ERR_DTYPE, "fp8_quant: x is bf16, fp16 or fp32");
  if (m < 0 || k < 1 || ldx < k || ldq < k) return api_fail(HKX_ERR_SHAPE, "fp8_quant: M=%d K=%d, row strides of at least K", m, k);
  if (!api_aligned(x, es(x_dtype)) || !api_aligned(s, 4)) return api_fail(HKX_ERR_SHAPE, "fp8_quant: x and s need their elements' alignment");
  if (m == 0) return HKX_OK;
  const QuantArgs a{x, (uint8_t*)q, s, ldx, ldq, k};
  return api_launched(by_type(x_dtype, [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const bool vec = k % 8 == 0 && whole(x, ldx, x_dtype) && api_aligned(q, 8) && ldq % 8 == 0;
    return vec ? launch_quant<DT, true>(a, m, (hipStream_t)stream) : launch_quant<DT, false>(a, m, (hipStream_t)stream);
  }), "fp8 quant");
}

}  // extern "C"
