// The block norm's C ABI: argument checks, the workers of a backward pass, the sum of their parts.
#include <algorithm>

#include "hkx_norm.hpp"

namespace hkx {
namespace {

// Sums of rows of fp32 partial sums: out[g][c] = sum over i < count of src[g][i][c], in order and in 64 bits (in 32
// dpost and dpre of 999 rows were 1.4e-7 off of their norm, so 7e-8; the same time).
struct SumJob {
  const float* src;
  void* dst;
  int32_t dst_dt, count, width, groups;
};
struct SumArgs {
  SumJob job[3];
};

// A workgroup 64 columns of one sum, 16 waves a sixteenth of the rows each, joined in wave order.
__global__ void __launch_bounds__(1024) norm_sum_kernel(const SumArgs p) {
  __shared__ double part[16][64];
  int y = blockIdx.y, k = 0;
  while (k < 2 && y >= p.job[k].groups) y -= p.job[k++].groups;
  const SumJob& j = p.job[k];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
  if ((int)blockIdx.x * 64 >= j.width || y >= j.groups) return;
  const int per = (j.count + 15) / 16, lo = min(wave * per, j.count), hi = min(lo + per, j.count);
  const float* src = j.src + (int64_t)y * j.count * j.width + col;
  double s = 0.0;
  if (col < j.width) {
    int i = lo;
    for (; i + 8 <= hi; i += 8) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = src[(int64_t)(i + u) * j.width];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
    for (; i < hi; ++i) s += src[(int64_t)i * j.width];
  }
  part[wave][lane] = s;
  __syncthreads();
  if (wave || col >= j.width) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += part[w][lane];
  store_one(j.dst, j.dst_dt, (int64_t)y * j.width + col, (float)s);
}

int es(int dt) { return dt == HKX_FP32 ? 4 : 2; }
bool floating(int dt) { return dt == HKX_BF16 || dt == HKX_FP16 || dt == HKX_FP32; }

// What forward and backward check alike; the kernels' arguments.
int forward_args(const HkxBlockNormArgs& g, const char* what, NormArgs& a) {
  if (!g.x || !g.residual) return api_fail(HKX_ERR_ARG, "%s: a null pointer", what);
  // (row numbers, and a worker's past the last, are 32-bit)
  if (g.rows < 0 || g.rows > INT32_MAX - 65536 || g.d < 1)
    return api_fail(HKX_ERR_SHAPE, "%s: rows=%d d=%d", what, g.rows, g.d);
  if (!floating(g.x_dtype) || (g.r_dtype != g.x_dtype && g.r_dtype != HKX_FP32))
    return api_fail(HKX_ERR_DTYPE, "%s: x is bf16, fp16 or fp32, the residual the same or fp32", what);
  if ((g.post || g.pre) && g.w_dtype != g.x_dtype && g.w_dtype != HKX_FP32)
    return api_fail(HKX_ERR_DTYPE, "%s: the weights have x's type or are fp32", what);
  if (g.gate && g.gate_dtype != g.x_dtype && g.gate_dtype != HKX_FP32)
    return api_fail(HKX_ERR_DTYPE, "%s: the gate has x's type or is fp32", what);
  if (g.gate && (g.gate_rows < 1 || g.rows % g.gate_rows))
    return api_fail(HKX_ERR_SHAPE, "%s: %d rows do not divide into gates of %d rows", what, g.rows, g.gate_rows);
  if (g.ldx < g.d || g.ldr < g.d) return api_fail(HKX_ERR_SHAPE, "%s: row strides below d", what);
  a.x = g.x;
  a.res = g.residual;
  a.post = g.post;
  a.pre = g.pre;
  a.gate = g.gate;
  a.h = g.h;
  a.y = g.y;
  a.ys = g.y_scales;
  a.rstd = g.rstd;
  a.ldx = g.ldx;
  a.ldr = g.ldr;
  a.ldh = g.ldh;
  a.ldy = g.ldy;
  a.lds = g.ldys;
  a.rows = g.rows;
  a.d = g.d;
  a.gate_dt = g.gate_dtype;
  a.gate_rows = g.gate ? g.gate_rows : g.rows;
  a.gate_col = g.gate_col != 0;
  a.quant = g.quant;
  a.bs = g.branch_scale;
  a.rs = g.residual_scale;
  a.eps = g.eps;
  a.inv_d = 1.0 / g.d;
  return HKX_OK;
}

// A backward call's workers: two waves a SIMD of the GPU, at least 2 rows each. (Their number, and so
// the workspace, goes by the shape alone, not by how a call's rows are aligned.)
struct Grad {
  int workers, parts, groups, group_rows;
  NormShape shape;
  size_t post, pre, gate;  // floats of each partial sum
};

Grad grad_plan(const HkxBlockNormGradArgs& g, bool vec) {
  const HkxBlockNormArgs& f = g.f;
  Grad q{};
  q.shape = norm_shape(f.d, vec);
  const int most = api_cus() * std::max(1, 512 / q.shape.threads);
  q.group_rows = f.gate ? f.gate_rows : std::max(1, f.rows);
  q.groups = std::max(1, f.rows / q.group_rows);
  const int p = std::max(1, std::min(most, (f.rows + 1) / 2));
  q.parts = std::max(1, std::min(p / q.groups, q.group_rows));
  q.workers = q.groups <= p ? q.groups * q.parts : p;
  auto pad = [](size_t n) { return (n + 3) / 4 * 4; };
  q.post = f.post && g.dpost ? pad((size_t)q.workers * f.d) : 0;
  q.pre = f.pre && g.dpre ? pad((size_t)q.workers * f.d) : 0;
  q.gate = f.gate && g.dgate && q.parts > 1 ? pad((size_t)q.workers * (f.gate_col ? f.d : 1)) : 0;
  return q;
}

bool grad_vec(const HkxBlockNormGradArgs& g) {
  const HkxBlockNormArgs& f = g.f;
  NormArgs a{};
  if (forward_args(f, "block_norm_backward", a)) return false;
  a.h = a.y = nullptr;
  a.quant = 0;
  auto ok = [](const void* p, int64_t ld, int e) { return !p || (api_aligned(p, 16) && ld * e % 16 == 0); };
  return norm_vec_ok(a, es(f.x_dtype), es(f.r_dtype), es(f.w_dtype), es(f.gate_dtype)) &&
         ok(g.dh, g.lddh, es(f.r_dtype)) && ok(g.dy, g.lddy, es(f.x_dtype)) && ok(g.dx, g.lddx, es(f.x_dtype)) &&
         ok(g.dresidual, g.lddr, es(f.r_dtype)) && ok(g.dgate, 0, 1);
}

}  // namespace
}  // namespace hkx

extern "C" {

int hkx_block_norm(const HkxBlockNormArgs* args, void* stream) {
  using namespace hkx;
  api_clear();
  if (!args) return api_fail(HKX_ERR_ARG, "block_norm: null args");
  if (args->size != sizeof *args)
    return api_fail(HKX_ERR_ARG, "block_norm: args of %d bytes, the library's have %zu", args->size, sizeof *args);
  const HkxBlockNormArgs& g = *args;
  NormArgs a{};
  if (int rc = forward_args(g, "block_norm", a)) return rc;
  if (g.d > kNormMaxD) return api_fail(HKX_ERR_SHAPE, "block_norm: d=%d, at most %d", g.d, kNormMaxD);
  if (!g.h || (g.pre && !g.y)) return api_fail(HKX_ERR_ARG, "block_norm: a null output");
  if (g.quant < 0 || g.quant > 2) return api_fail(HKX_ERR_ARG, "block_norm: quant=%d", g.quant);
  if (g.quant && (!g.pre || !g.y_scales)) return api_fail(HKX_ERR_ARG, "block_norm: a quantized y needs pre and its scales");
  const int64_t ybytes = g.quant == 2 ? g.d / 2 : g.d;
  if (g.ldh < g.d || (g.pre && g.ldy < ybytes) || (g.quant && g.ldys < g.d / 32))
    return api_fail(HKX_ERR_SHAPE, "block_norm: row strides below d");
  if (g.rows == 0) return HKX_OK;
  if (g.quant) {
    if (g.d % 32) return api_fail(HKX_ERR_SHAPE, "block_norm: d=%d, a multiple of 32 where y is quantized", g.d);
    const int64_t al = g.quant == 2 ? 4 : 8;
    if (!norm_vec_ok(a, es(g.x_dtype), es(g.r_dtype), es(g.w_dtype), es(g.gate_dtype)) || !api_aligned(g.y, al) || g.ldy % al)
      return api_fail(HKX_ERR_SHAPE, "block_norm: a quantized y needs 16-byte aligned rows of every other operand");
  }
  const hipStream_t s = (hipStream_t)stream;
  const bool r32 = g.r_dtype == HKX_FP32, w32 = (g.post || g.pre) && g.w_dtype == HKX_FP32;
  return api_launched(g.x_dtype == HKX_BF16   ? launch_norm_bf16(a, r32, w32, s)
                      : g.x_dtype == HKX_FP16 ? launch_norm_fp16(a, r32, w32, s)
                                              : launch_norm_fp32(a, s),
                      "block norm");
}

size_t hkx_block_norm_backward_workspace(const HkxBlockNormGradArgs* args) {
  using namespace hkx;
  if (!args || args->size != sizeof *args || args->f.rows < 1 || args->f.d < 1 || args->f.d > kNormGradMaxD) return 0;
  if (args->f.gate && (args->f.gate_rows < 1 || args->f.rows % args->f.gate_rows)) return 0;
  const Grad q = grad_plan(*args, grad_vec(*args));
  return (q.post + q.pre + q.gate) * 4;
}

int hkx_block_norm_backward(const HkxBlockNormGradArgs* args, void* stream) {
  using namespace hkx;
  api_clear();
  if (!args) return api_fail(HKX_ERR_ARG, "block_norm_backward: null args");
  if (args->size != sizeof *args)
    return api_fail(HKX_ERR_ARG, "block_norm_backward: args of %d bytes, the library's have %zu", args->size, sizeof *args);
  const HkxBlockNormGradArgs& g = *args;
  const HkxBlockNormArgs& f = g.f;
  NormGradArgs a{};
  if (int rc = forward_args(f, "block_norm_backward", a.f)) return rc;
  if (f.d > kNormGradMaxD) return api_fail(HKX_ERR_SHAPE, "block_norm_backward: d=%d, at most %d", f.d, kNormGradMaxD);
  if (!f.rstd || !g.dx || !g.dresidual) return api_fail(HKX_ERR_ARG, "block_norm_backward: a null pointer");
  if ((g.dh && g.lddh < f.d) || (g.dy && g.lddy < f.d) || g.lddx < f.d || g.lddr < f.d)
    return api_fail(HKX_ERR_SHAPE, "block_norm_backward: row strides below d");
  if (f.rows == 0) return api_fail(HKX_ERR_SHAPE, "block_norm_backward: no rows");
  const Grad q = grad_plan(g, grad_vec(g));
  const size_t need = (q.post + q.pre + q.gate) * 4;
  if (need && (!g.ws || g.ws_bytes < need || !api_aligned(g.ws, 16)))
    return api_fail(HKX_ERR_WORKSPACE, "block_norm_backward: needs %zu bytes of 16-byte aligned workspace, got %zu", need,
                    g.ws ? g.ws_bytes : (size_t)0);
  a.f.h = a.f.y = nullptr;
  a.dh = g.dh;
  a.dy = f.pre ? g.dy : nullptr;
  a.dx = g.dx;
  a.dr = g.dresidual;
  a.lddh = g.lddh;
  a.lddy = g.lddy;
  a.lddx = g.lddx;
  a.lddr = g.lddr;
  a.workers = q.workers;
  a.parts = q.parts;
  a.groups = q.groups;
  a.group_rows = q.group_rows;
  a.shape = q.shape;
  float* ws = (float*)g.ws;
  a.ppost = q.post ? ws : nullptr;
  a.ppre = q.pre ? ws + q.post : nullptr;
  a.pgate = q.gate ? ws + q.post + q.pre : nullptr;
  a.dgate = f.gate && q.parts == 1 ? g.dgate : nullptr;
  const hipStream_t s = (hipStream_t)stream;
  const bool r32 = f.r_dtype == HKX_FP32, w32 = (f.post || f.pre) && f.w_dtype == HKX_FP32;
  int rc = api_launched(f.x_dtype == HKX_BF16   ? launch_norm_grad_bf16(a, r32, w32, s)
                        : f.x_dtype == HKX_FP16 ? launch_norm_grad_fp16(a, r32, w32, s)
                                                : launch_norm_grad_fp32(a, s),
                        "block norm backward");
  if (rc || !need) return rc;
  SumArgs j{};
  int k = 0, width = 0, groups = 0;
  auto add = [&](const float* src, void* dst, int dt, int count, int w, int n) {
    j.job[k++] = SumJob{src, dst, dt, count, w, n};
    width = std::max(width, w);
    groups += n;
  };
  if (q.post) add(a.ppost, g.dpost, f.w_dtype, q.workers, f.d, 1);
  if (q.pre) add(a.ppre, g.dpre, f.w_dtype, q.workers, f.d, 1);
  if (q.gate) add(a.pgate, g.dgate, f.gate_dtype, q.parts, f.gate_col ? f.d : 1, q.groups);
  // (no more groups than workers: where there are more, each worker has whole ones)
  hipLaunchKernelGGL(norm_sum_kernel, dim3((width + 63) / 64, groups), dim3(1024), 0, s, j);
  return api_launched(hipGetLastError(), "block norm backward (sums)");
}

}  // extern "C"
