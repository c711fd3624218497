// The experts' products: the C ABI's checks, the kernel a call takes, and the small passes of their gradient.
#include <algorithm>

#include "hkx_api.hpp"
#include "hkx_group.hpp"
#include "hkx_group_launch.hpp"

namespace hkx {
namespace {

// dz = (dy up silu'(gate), dy silu(gate)), a thread 8 columns. Bound by HBM: 3 reads and 2 writes of bf16 a gate column,
// 8192 rows of 4096: 336 MB in 55 us, 6.1 TB/s (z and dy partly from the 256 MB cache). dz is rounded to bf16, as the
// products that read it take it.
__global__ void __launch_bounds__(256) silu_grad_kernel(const uint8_t* z, int64_t ldz, const uint8_t* dy, int64_t lddy,
                                                        uint8_t* dz, int64_t lddz, const int32_t* offsets, int experts,
                                                        int rows, int n) {
  const int per = n / 8;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = at / per;
  const int c = (int)(at - r * per) * 8;
  if (r >= min(max(offsets[experts], 0), rows)) return;
  const i32x4 g = *(const i32x4*)(z + r * ldz + c * 2), u = *(const i32x4*)(z + r * ldz + (c + n) * 2),
              d = *(const i32x4*)(dy + r * lddy + c * 2);
  i32x4 dg, du;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float og[2], ou[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      auto half = [&](int w) { return bf16_to_f32(h ? (uint32_t)w >> 16 : (uint32_t)w & 0xffffu); };
      const float gv = half(g[j]), uv = half(u[j]), dv = half(d[j]), s = sigmoid(gv);
      // silu(g) = g s; where s is 0 (g past -88) the product is 0, also of an infinite g
      const float gs = s > 0.0f ? gv * s : 0.0f;
      og[h] = dv * uv * (s + gs * (1.0f - s));
      ou[h] = dv * gs;
    }
    dg[j] = (int)pack_bf16x2(og[0], og[1]);
    du[j] = (int)pack_bf16x2(ou[0], ou[1]);
  }
  *(i32x4*)(dz + r * lddz + c * 2) = dg;
  *(i32x4*)(dz + r * lddz + (c + n) * 2) = du;
}

// The sum of an expert's rows, 128 columns a workgroup (two a lane), a sixteenth of the rows a wave, joined in order: the same
// bits every time, and 64 bits, as a sum of many rows cancels. Bound by latency, eight rows in flight a wave: 600 rows of 904
// columns in 5 groups 4.0 us.
__global__ void __launch_bounds__(1024) bias_grad_kernel(const uint8_t* dz, int64_t ld, const int32_t* offsets, void* db,
                                                         int dt, int rows, int n) {
  __shared__ double part[16][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = blockIdx.y, c = blockIdx.x * 128 + 2 * lane;
  const int lo = min(max(offsets[e], 0), rows), hi = min(max(offsets[e + 1], lo), rows);
  const int per = (hi - lo + 15) / 16, from = min(lo + wave * per, hi), to = min(from + per, hi);
  double a = 0.0, b = 0.0;
  if (c < n) {
    const uint8_t* p = dz + (int64_t)from * ld + (int64_t)c * 2;
    int r = from;
    for (; r + 8 <= to; r += 8, p += 8 * ld) {
      uint32_t w[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) w[u] = *(const uint32_t*)(p + u * ld);
#pragma unroll
      for (int u = 0; u < 8; ++u) a += bf16_to_f32(w[u] & 0xffffu), b += bf16_to_f32(w[u] >> 16);
    }
    for (; r < to; ++r, p += ld) {
      const uint32_t w = *(const uint32_t*)p;
      a += bf16_to_f32(w & 0xffffu), b += bf16_to_f32(w >> 16);
    }
  }
  part[wave][2 * lane] = a;
  part[wave][2 * lane + 1] = b;
  __syncthreads();
  const int col = blockIdx.x * 128 + (int)threadIdx.x;
  if (threadIdx.x >= 128 || col >= n) return;
  double s = part[0][threadIdx.x];
#pragma unroll
  for (int w = 1; w < 16; ++w) s += part[w][threadIdx.x];
  const int64_t at = (int64_t)e * n + col;
  const float v = (float)s;
  if (dt == HKX_FP32) ((float*)db)[at] = v;
  else ((uint16_t*)db)[at] = (uint16_t)(dt == HKX_BF16 ? pack_bf16x2(v, 0.0f) : pack_f16x2(v, 0.0f));
}

// Rows of x by index, 16 bytes a thread, for the weights' gradient (its rows lie along K, where a fill reads 4 rows at
// one offset from a scalar base). 8192 rows of 2048 bf16: 14 us, 4.8 TB/s.
__global__ void __launch_bounds__(256) gather_kernel(const uint8_t* x, int64_t ldx, const int32_t* index, uint8_t* out,
                                                     int64_t ldo, int rows, int a_rows, int per) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t r = at / per, c = (at - r * per) * 16;
  if (r >= rows) return;
  const int j = index[r];
  i32x4 v = {};
  if ((uint32_t)j < (uint32_t)a_rows) v = *(const i32x4*)(x + (int64_t)j * ldx + c);
  *(i32x4*)(out + r * ldo + c) = v;
}

// A group's rows are counted in tiles by ints: rows + 255 is one.
constexpr int32_t kMostRows = INT32_MAX - 255;

bool floating(int dt) { return dt == HKX_BF16 || dt == HKX_FP16 || dt == HKX_FP32; }

// What a call asks for, refused where the kernels do not take it; the kernels' arguments.
int gemm_args(const HkxExpertsGemmArgs& g, GroupArgs& a) {
  const bool nt = g.op == HKX_EXPERTS_NT, tn = g.op == HKX_EXPERTS_TN, fp8 = g.ab_dtype == HKX_FP8E4M3;
  if (!nt && !tn && g.op != HKX_EXPERTS_NN) return api_fail(HKX_ERR_ARG, "experts_gemm: op %d", g.op);
  if (!fp8 && g.ab_dtype != HKX_BF16) return api_fail(HKX_ERR_DTYPE, "experts_gemm: operands are bf16 or e4m3");
  if (fp8 && !nt) return api_fail(HKX_ERR_DTYPE, "experts_gemm: no gradient of e4m3 operands");
  if (g.c_dtype != HKX_BF16 && (g.c_dtype != HKX_FP32 || g.op != HKX_EXPERTS_NN))
    return api_fail(HKX_ERR_DTYPE, "experts_gemm: C is bf16, or fp32 where op is NN");
  if (!g.a || !g.b || !g.c || !g.offsets || (fp8 && (!g.sa || !g.sb))) return api_fail(HKX_ERR_ARG, "experts_gemm: a null pointer");
  if (g.experts < 1 || g.experts > kMaxExperts || g.rows < 0 || g.rows > kMostRows || g.n < 1 || (tn ? g.m < 1 : g.k < 1))
    return api_fail(HKX_ERR_SHAPE, "experts_gemm: experts=%d (at most %d) rows=%d m=%d n=%d k=%d", g.experts, kMaxExperts, g.rows,
                    g.m, g.n, g.k);
  if (!nt && (g.silu_mul || g.z || g.index || g.bias)) return api_fail(HKX_ERR_ARG, "experts_gemm: silu_mul, z, index and bias go with NT");
  if (g.z && !g.silu_mul) return api_fail(HKX_ERR_ARG, "experts_gemm: z goes with silu_mul");
  if (g.bias && !floating(g.bias_dtype)) return api_fail(HKX_ERR_DTYPE, "experts_gemm: the bias is bf16, fp16 or fp32");
  if (g.index && g.a_rows < 1) return api_fail(HKX_ERR_SHAPE, "experts_gemm: an index into %d rows", g.a_rows);
  const int64_t es = fp8 ? 1 : 2, ces = g.c_dtype == HKX_FP32 ? 4 : 2, step = fp8 ? 16 : 8, brows = nt ? (g.silu_mul ? 2 * (int64_t)g.n : g.n) : g.k;
  if (g.n % 8 || (tn ? g.m % 8 : g.k % step) || brows > INT32_MAX)
    return api_fail(HKX_ERR_SHAPE, "experts_gemm: m=%d n=%d k=%d: multiples of 8, an e4m3 k of 16", g.m, g.n, g.k);
  const int64_t acols = tn ? g.m : g.k, bcols = nt ? g.k : g.n;
  if (g.lda < acols || g.ldb < bcols || g.ldc < g.n || (g.z && g.ldz < 2 * (int64_t)g.n) || (g.bias && g.bias_ld < brows))
    return api_fail(HKX_ERR_SHAPE, "experts_gemm: row strides below a row");
  if (g.lda % step || g.ldb % step || (!tn && g.b_expert % step) || !api_aligned(g.a, 16) || !api_aligned(g.b, 16))
    return api_fail(HKX_ERR_SHAPE, "experts_gemm: A's and B's rows and experts need 16-byte alignment");
  if (g.ldc % 4 || !api_aligned(g.c, 4 * ces) || (tn && g.c_expert % 4) || (g.z && (g.ldz % 4 || !api_aligned(g.z, 8))))
    return api_fail(HKX_ERR_SHAPE, "experts_gemm: C's and z's rows need 8-byte alignment, an fp32 C's 16");
  if (g.bias && (!api_aligned(g.bias, 16) || g.bias_ld % 4)) return api_fail(HKX_ERR_SHAPE, "experts_gemm: the bias needs 16-byte aligned rows");
  if (fp8 && (!api_aligned(g.sa, 4) || !api_aligned(g.sb, g.sb_col ? 16 : 4) || (g.sb_col && g.sb_ld % 4)))
    return api_fail(HKX_ERR_SHAPE, "experts_gemm: the scales' alignment");
  // offsets in a tile, in an expert of B, and in an A that an index picks from are 32-bit
  const int64_t lim = ((int64_t)1 << 32) - 4096;
  if (256 * g.lda * es > lim || 256 * g.ldc * ces > lim || 256 * g.ldz * 2 > lim || (nt ? brows : 256) * g.ldb * es > lim || (g.index && g.a_rows * g.lda * es > lim))
    return api_fail(HKX_ERR_SHAPE, "experts_gemm: an expert's B or an indexed A spans 4 GiB or more; split the call");
  if (g.kernel < 0 || g.kernel > HKX_EXPERTS_SKINNY32) return api_fail(HKX_ERR_ARG, "experts_gemm: kernel %d", g.kernel);
  a.a = (const uint8_t*)g.a;
  a.b = (const uint8_t*)g.b;
  a.c = (uint8_t*)g.c;
  a.z = (uint8_t*)g.z;
  a.offsets = g.offsets;
  a.index = g.index;
  a.bias = g.bias;
  a.sa = g.sa;
  a.sb = g.sb;
  a.lda = g.lda * es;
  a.ldb = g.ldb * es;
  a.ldc = g.ldc * ces;
  a.ldz = g.ldz * 2;
  a.b_group = g.b_expert * es;
  a.c_group = g.c_expert * 2;
  a.bias_ld = g.bias_ld;
  a.sb_ld = g.sb_ld;
  a.experts = g.experts;
  a.rows = g.rows;
  a.a_rows = g.a_rows;
  a.m = g.m;
  a.n = g.n;
  a.k = g.k;
  a.tail = g.zero_rest != 0;
  a.bias_dt = g.bias_dtype;
  a.sa_ld = g.sa_ld != 0;
  a.sb_col = g.sb_col != 0;
  a.c_f32 = g.c_dtype == HKX_FP32;
  if (g.kernel == HKX_EXPERTS_QUAD && !group_quad_ok(a))
    return api_fail(HKX_ERR_SHAPE, "experts_gemm: the 256-row kernel stores 16-byte aligned rows");
  return HKX_OK;
}

// Blocks of 256 threads, a thread one of `per` pieces of a row; 0 where a launch does not take them.
unsigned pieces(int64_t rows, int64_t per) {
  const int64_t n = (rows * per + 255) / 256;
  return n < ((int64_t)1 << 24) ? (unsigned)n : 0;
}

}  // namespace
}  // namespace hkx

extern "C" {

int hkx_experts_gemm(const HkxExpertsGemmArgs* args, void* stream) {
  using namespace hkx;
  api_clear();
  if (!args) return api_fail(HKX_ERR_ARG, "experts_gemm: null args");
  if (args->size != sizeof *args)
    return api_fail(HKX_ERR_ARG, "experts_gemm: args of %d bytes, the library's have %zu", args->size, sizeof *args);
  const HkxExpertsGemmArgs& g = *args;
  GroupArgs a{};
  if (int rc = gemm_args(g, a)) return rc;
  if (g.rows == 0 && g.op != HKX_EXPERTS_TN) return HKX_OK;
  const bool fp8 = g.ab_dtype == HKX_FP8E4M3, pair = g.silu_mul != 0;
  const int kernel = group_kernel(a, g.op, fp8, pair, g.kernel, api_cus());
  const size_t need = group_ws_bytes(a, g.op, fp8, pair, kernel, api_cus());
  if (need && (!g.ws || g.ws_bytes < need || !api_aligned(g.ws, 16)))
    return api_fail(HKX_ERR_WORKSPACE, "experts_gemm: needs %zu bytes of 16-byte aligned workspace, got %zu", need, g.ws ? g.ws_bytes : (size_t)0);
  a.ws = need ? (float*)g.ws : nullptr;
  const hipError_t e = launch_group(a, g.op, fp8, pair, kernel, api_cus(), (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return api_fail(HKX_ERR_SHAPE, "experts_gemm: rows=%d of n=%d are more tiles than a launch takes; split the call", g.rows, g.n);
  return api_launched(e, "experts gemm");
}

size_t hkx_experts_gemm_workspace(const HkxExpertsGemmArgs* args) {
  using namespace hkx;
  GroupArgs a{};
  if (!args || args->size != sizeof *args || gemm_args(*args, a) || args->rows == 0) return 0;
  return group_ws_bytes(a, args->op, args->ab_dtype == HKX_FP8E4M3, args->silu_mul != 0, args->kernel, api_cus());
}

int hkx_experts_silu_grad(const void* z, int64_t ldz, const void* dy, int64_t lddy, void* dz, int64_t lddz,
                          const int32_t* offsets, int32_t experts, int32_t rows, int32_t n, void* stream) {
  using namespace hkx;
  api_clear();
  if (!z || !dy || !dz || !offsets) return api_fail(HKX_ERR_ARG, "experts_silu_grad: a null pointer");
  if (experts < 1 || experts > kMaxExperts || rows < 0 || n < 1 || n % 8)
    return api_fail(HKX_ERR_SHAPE, "experts_silu_grad: experts=%d rows=%d n=%d, a multiple of 8", experts, rows, n);
  if (ldz < 2 * (int64_t)n || lddy < n || lddz < 2 * (int64_t)n || ldz % 8 || lddy % 8 || lddz % 8 || !api_aligned(z, 16) ||
      !api_aligned(dy, 16) || !api_aligned(dz, 16))
    return api_fail(HKX_ERR_SHAPE, "experts_silu_grad: rows need 16-byte alignment and strides of a row");
  if (rows == 0) return HKX_OK;
  const unsigned grid = pieces(rows, n / 8);
  if (!grid) return api_fail(HKX_ERR_SHAPE, "experts_silu_grad: rows=%d of n=%d are more than a launch takes; split the call", rows, n);
  hipLaunchKernelGGL(silu_grad_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)z, ldz * 2,
                     (const uint8_t*)dy, lddy * 2, (uint8_t*)dz, lddz * 2, offsets, experts, rows, n);
  return api_launched(hipGetLastError(), "experts silu grad");
}

int hkx_experts_bias_grad(const void* dz, int64_t lddz, const int32_t* offsets, void* db, int32_t db_dtype,
                          int32_t experts, int32_t rows, int32_t n, void* stream) {
  using namespace hkx;
  api_clear();
  if (!dz || !offsets || !db) return api_fail(HKX_ERR_ARG, "experts_bias_grad: a null pointer");
  if (!floating(db_dtype)) return api_fail(HKX_ERR_DTYPE, "experts_bias_grad: db is bf16, fp16 or fp32");
  if (experts < 1 || experts > kMaxExperts || rows < 0 || rows > kMostRows || n < 1 || n % 8 || lddz < n || lddz % 2 || !api_aligned(dz, 4))
    return api_fail(HKX_ERR_SHAPE, "experts_bias_grad: experts=%d rows=%d n=%d", experts, rows, n);
  hipLaunchKernelGGL(bias_grad_kernel, dim3((n + 127) / 128, experts), dim3(1024), 0, (hipStream_t)stream,
                     (const uint8_t*)dz, lddz * 2, offsets, db, db_dtype, rows, n);
  return api_launched(hipGetLastError(), "experts bias grad");
}

int hkx_experts_gather(const void* x, int64_t ldx, const int32_t* index, void* out, int64_t ldo, int32_t rows,
                       int32_t a_rows, int32_t k, void* stream) {
  using namespace hkx;
  api_clear();
  if (!x || !index || !out) return api_fail(HKX_ERR_ARG, "experts_gather: a null pointer");
  if (rows < 0 || a_rows < 0 || k < 1 || k % 8 || ldx < k || ldo < k || ldx % 8 || ldo % 8 || !api_aligned(x, 16) || !api_aligned(out, 16))
    return api_fail(HKX_ERR_SHAPE, "experts_gather: rows=%d k=%d, 16-byte aligned rows", rows, k);
  if (rows == 0) return HKX_OK;
  const unsigned grid = pieces(rows, k / 8);
  if (!grid) return api_fail(HKX_ERR_SHAPE, "experts_gather: rows=%d of k=%d are more than a launch takes; split the call", rows, k);
  hipLaunchKernelGGL(gather_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)x, ldx * 2, index,
                     (uint8_t*)out, ldo * 2, rows, a_rows, k / 8);
  return api_launched(hipGetLastError(), "experts gather");
}

}  // extern "C"
