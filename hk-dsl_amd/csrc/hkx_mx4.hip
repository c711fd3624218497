// The MXFP4 product's C ABI: argument checks, the plan, the launches; and the sum of a K split.
#include <algorithm>

#include "hkx_api.hpp"
#include "hkx_mx4_quad.hpp"
#include "hkx_mx4_skinny.hpp"

namespace hkx {

// A thread four columns of a row: the splits' shares in order, the bias, silu(gate) * up.
__global__ void __launch_bounds__(256) mx4_reduce_kernel(const Mx4ReduceArgs p) {
  const int n = ((int)blockIdx.x * 256 + (int)threadIdx.x) * 4;
  if (n >= p.N) return;
  for (int m = blockIdx.y; m < p.M; m += gridDim.y) {
    const float* w = p.ws + (int64_t)m * p.ws_ld + n;
    f32x4 z = *(const f32x4*)w, u = {};
    if (p.pair) u = *(const f32x4*)(w + p.share_up);
    for (int s = 1; s < p.splits; ++s) {
      z += *(const f32x4*)(w + s * p.split_stride);
      if (p.pair) u += *(const f32x4*)(w + s * p.split_stride + p.share_up);
    }
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) {
          z[i] += ld1(p.bias, p.bias_dt, n + i);
          if (p.pair) u[i] += ld1(p.bias, p.bias_dt, p.N + n + i);
        }
    }
    if (p.pair) z = silu_mul4(z, u);
    const u32x2 v = pack4<2>(HKX_BF16, z);
    uint16_t* dst = (uint16_t*)p.c + (int64_t)m * p.ldc + n;
    if (p.c_vec) {
      *(u32x2*)dst = v;
    } else {
      const uint16_t h[4] = {(uint16_t)v.x, (uint16_t)(v.x >> 16), (uint16_t)v.y, (uint16_t)(v.y >> 16)};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) dst[i] = h[i];
    }
  }
}

hipError_t launch_mx4_reduce(const Mx4ReduceArgs& r, hipStream_t s) {
  const dim3 grid((unsigned)(((r.N + 3) / 4 + 255) / 256), (unsigned)std::min(r.M, 65535));
  hipLaunchKernelGGL(mx4_reduce_kernel, grid, dim3(256), 0, s, r);
  return hipGetLastError();
}

namespace {

static_assert(kMx4Tile64 == HKX_MX4_TILE64 && kMx4Tile128 == HKX_MX4_TILE128 && kMx4Quad == HKX_MX4_QUAD &&
                  kMx4Skinny == HKX_MX4_SKINNY, "kernels");

// The quadrant kernel's epilogue: 32-bit offsets into C or the shares. (Any bias: C of odd columns leaves through
// shares, whose sum adds it.) And the scales' packing: a tile each of A and B along a grid's y.
bool quad_ok(const HkxMx4GemmArgs& g) {
  const int64_t rows = ((int64_t)g.m + 255) / 256 * 256;
  if (rows / 256 + g.n / mx4_cols(HKX_MX4_QUAD, g.silu_mul) >= 65535) return false;
  return rows * std::max(g.ldc * 2, ((int64_t)g.n + 3) / 4 * 4 * (g.silu_mul ? 8 : 4)) < ((int64_t)1 << 32) - 65536;
}

// C's rows are 16-byte aligned and N a multiple of 8. (By the row stride where C is not there yet: the
// workspace's size is asked before.)
bool c_vec(const HkxMx4GemmArgs& g) { return api_aligned(g.c, 16) && g.ldc % 8 == 0 && g.n % 8 == 0; }

Mx4Plan plan(const HkxMx4GemmArgs& g) {
  if (g.kernel == HKX_MX4_AUTO)
    return mx4_plan(g.m, g.n, g.k, g.a_dtype == HKX_FP8E4M3, g.silu_mul != 0, quad_ok(g), c_vec(g), api_cus());
  const int units = (g.k + 255) / 256;
  return {g.kernel, g.kernel == HKX_MX4_SKINNY ? 1 : mx4_splits(g.kernel, units, std::max(1, std::min(g.splits, units)))};
}

// Whether the sums leave through fp32 shares and a second pass.
bool shared(const HkxMx4GemmArgs& g, const Mx4Plan& q) { return q.splits > 1 || (q.kernel == HKX_MX4_QUAD && !c_vec(g)); }

int64_t share_ld(const HkxMx4GemmArgs& g, int& up) {
  up = (g.n + 3) / 4 * 4;
  return g.silu_mul ? 2 * (int64_t)up : up;
}

// The workspace: a split's shares, then A's and B's scales packed for the quadrant kernel.
struct Room {
  size_t shares, sa, sb;
  size_t all() const { return shares + sa + sb; }
};

Room room(const HkxMx4GemmArgs& g, const Mx4Plan& q) {
  Room r{};
  int up;
  if (shared(g, q)) r.shares = ((size_t)q.splits * g.m * share_ld(g, up) * 4 + 15) / 16 * 16;
  if (q.kernel == HKX_MX4_QUAD) {
    const size_t chunks = (size_t)(g.k + 511) / 512;
    r.sa = (size_t)((g.m + 255) / 256) * chunks * 4096;
    r.sb = (size_t)((g.n + mx4_cols(q.kernel, g.silu_mul) - 1) / mx4_cols(q.kernel, g.silu_mul)) * chunks * 4096;
  }
  return r;
}

}  // namespace
}  // namespace hkx

extern "C" {

size_t hkx_mx4_gemm_workspace(const HkxMx4GemmArgs* args) {
  if (!args || args->size != sizeof *args || args->m < 1 || args->n < 1 || args->k < 32) return 0;
  return hkx::room(*args, hkx::plan(*args)).all();
}

int hkx_mx4_gemm(const HkxMx4GemmArgs* args, void* stream) {
  using namespace hkx;
  api_clear();
  if (!args) return api_fail(HKX_ERR_ARG, "mx4_gemm: null args");
  if (args->size != sizeof *args)
    return api_fail(HKX_ERR_ARG, "mx4_gemm: args of %d bytes, the library's have %zu", args->size, sizeof *args);
  const HkxMx4GemmArgs& g = *args;
  if (!g.a || !g.b || !g.c || !g.sa || !g.sb) return api_fail(HKX_ERR_ARG, "mx4_gemm: a null pointer");
  if (g.a_dtype != HKX_FP4E2M1 && g.a_dtype != HKX_FP8E4M3) return api_fail(HKX_ERR_DTYPE, "mx4_gemm: A is packed 4-bit or e4m3");
  if (g.bias && g.bias_dtype != HKX_BF16 && g.bias_dtype != HKX_FP16 && g.bias_dtype != HKX_FP32)
    return api_fail(HKX_ERR_DTYPE, "mx4_gemm: the bias is bf16, fp16 or fp32");
  if (g.m < 1 || g.n < 1 || g.k < 1) return api_fail(HKX_ERR_SHAPE, "mx4_gemm: M=%d N=%d K=%d", g.m, g.n, g.k);
  if (g.k % 32) return api_fail(HKX_ERR_SHAPE, "mx4_gemm: K=%d, a multiple of 32", g.k);
  const bool a8 = g.a_dtype == HKX_FP8E4M3, pair = g.silu_mul != 0;
  const int64_t abytes = a8 ? g.k : g.k / 2, bbytes = g.k / 2, sbytes = g.k / 32;
  const int64_t brows = pair ? 2 * (int64_t)g.n : g.n;
  if (brows > INT32_MAX) return api_fail(HKX_ERR_SHAPE, "mx4_gemm: N=%d", g.n);
  if (g.lda < abytes || g.ldb < bbytes || g.ldc < g.n || g.sa_ld < sbytes || g.sb_ld < sbytes)
    return api_fail(HKX_ERR_SHAPE, "mx4_gemm: row strides below a row");
  if (!api_aligned(g.a, 16) || !api_aligned(g.b, 16) || g.lda % 16 || g.ldb % 16)
    return api_fail(HKX_ERR_SHAPE, "mx4_gemm: A and B need 16-byte aligned rows");
  // 32-bit byte offsets of the operands, up to the last row of a 256-row tile
  const int64_t mr = ((int64_t)g.m + 255) / 256 * 256, nr = (brows + 511) / 256 * 256;
  constexpr int64_t kMost = ((int64_t)1 << 32) - 65536;
  if (mr * g.lda >= kMost || nr * g.ldb >= kMost || mr * g.sa_ld >= kMost || nr * g.sb_ld >= kMost)
    return api_fail(HKX_ERR_SHAPE, "mx4_gemm: A, B or their scales span 4 GiB or more; split the call");
  if (g.kernel < HKX_MX4_AUTO || g.kernel > HKX_MX4_SKINNY || g.splits < 0)
    return api_fail(HKX_ERR_ARG, "mx4_gemm: kernel %d, splits %d", g.kernel, g.splits);
  if (g.bias && !api_aligned(g.bias, 16)) return api_fail(HKX_ERR_SHAPE, "mx4_gemm: the bias needs 16-byte alignment");
  if (g.kernel == HKX_MX4_QUAD && !quad_ok(g)) return api_fail(HKX_ERR_SHAPE, "mx4_gemm: the quadrant kernel does not take this call");
  const Mx4Plan q = plan(g);
  const Room rm = room(g, q);
  const size_t need = rm.all();
  if (need && (!g.ws || g.ws_bytes < need || !api_aligned(g.ws, 16)))
    return api_fail(HKX_ERR_WORKSPACE, "mx4_gemm: needs %zu bytes of 16-byte aligned workspace, got %zu", need,
                    g.ws ? g.ws_bytes : (size_t)0);
  Mx4Args t{};
  t.a = (const uint8_t*)g.a;
  t.b = (const uint8_t*)g.b;
  t.sa = g.sa;
  t.sb = g.sb;
  t.c = g.c;
  t.bias = g.bias;
  t.bias_dt = g.bias_dtype;
  // (a row's bytes past K, between rows, are read and not used; past the last row nothing is)
  t.a_bytes = (uint32_t)((g.m - 1) * g.lda + abytes);
  t.b_bytes = (uint32_t)((brows - 1) * g.ldb + bbytes);
  t.sa_bytes = (uint32_t)((g.m - 1) * g.sa_ld + (sbytes + 3) / 4 * 4);  // whole dwords, within an aligned one
  t.sb_bytes = (uint32_t)((brows - 1) * g.sb_ld + (sbytes + 3) / 4 * 4);
  t.lda = (uint32_t)g.lda;
  t.ldb = (uint32_t)g.ldb;
  t.sa_ld = (uint32_t)g.sa_ld;
  t.sb_ld = (uint32_t)g.sb_ld;
  t.ldc = g.ldc;
  t.M = g.m;
  t.N = g.n;
  t.K = g.k;
  t.units = t.units_split = (g.k + 255) / 256;
  t.wgm = 8;
  t.c_vec = c_vec(g);
  const hipStream_t s = (hipStream_t)stream;
  if (q.kernel == HKX_MX4_SKINNY) {
    Mx4SkinnyArgs d{};
    d.a = t.a;
    d.b = t.b;
    d.sa = t.sa;
    d.sb = t.sb;
    d.c = t.c;
    d.bias = t.bias;
    d.a_bytes = t.a_bytes;
    d.b_bytes = t.b_bytes;
    d.lda = t.lda;
    d.ldb = t.ldb;
    d.sa_ld = t.sa_ld;
    d.sb_ld = t.sb_ld;
    d.ldc = t.ldc;
    d.M = t.M;
    d.N = t.N;
    d.K = t.K;
    d.units = t.units;
    d.bias_dt = t.bias_dt;
    d.c_vec = api_aligned(g.c, 8) && g.ldc % 4 == 0 && g.n % 4 == 0;
    return api_launched(launch_mx4_skinny(d, a8, pair, api_cus(), s), "mx4 decode GEMM");
  }
  const int bm = mx4_rows(q.kernel), bn = mx4_cols(q.kernel, pair);
  t.tiles_m = (g.m + bm - 1) / bm;
  t.tiles_n = (g.n + bn - 1) / bn;
  // (a grid past 2^32 threads is cut short, with no error)
  if (q.kernel != HKX_MX4_QUAD && (int64_t)t.tiles_m * t.tiles_n >= (1 << 24) - 1)
    return api_fail(HKX_ERR_SHAPE, "mx4_gemm: M=%d N=%d is more tiles than a launch takes; split the call", g.m, g.n);
  if (q.kernel == HKX_MX4_QUAD) {
    Mx4PackArgs pa{}, pb{};
    pa.s = g.sa;
    pa.out = (uint8_t*)g.ws + rm.shares;
    pa.ld = t.sa_ld;
    pa.rows = (uint32_t)g.m;
    pa.k32 = pb.k32 = g.k / 32;
    pa.chunks = pb.chunks = (t.units + 1) / 2;
    pa.tiles = t.tiles_m;
    pb.s = g.sb;
    pb.out = pa.out + rm.sa;
    pb.ld = t.sb_ld;
    pb.rows = (uint32_t)g.n;
    pb.tiles = t.tiles_n;
    pb.is_b = 1;
    pb.pair = pair;
    if (int rc = api_launched(launch_mx4_pack(pa, pb, s), "mx4 GEMM (scales)")) return rc;
    t.sa = pa.out;
    t.sb = pb.out;
    t.sa_bytes = (uint32_t)rm.sa;
    t.sb_bytes = (uint32_t)rm.sb;
  }
  auto launch = [&](bool share) {
    const int tiles = t.tiles_m * t.tiles_n;
    if (q.kernel == HKX_MX4_QUAD)
      return launch_mx4_quad(t, a8, pair, share, dim3((unsigned)std::min(tiles, std::max(1, api_cus() / q.splits)), (unsigned)q.splits), s);
    // (two workgroups a CU past one a CU)
    return launch_mx4_tile(t, a8, pair, share, bm, tiles * q.splits > api_cus(), dim3((unsigned)tiles, (unsigned)q.splits), s);
  };
  if (!shared(g, q)) return api_launched(launch(false), "mx4 GEMM");
  Mx4ReduceArgs r{};
  r.ws = (const float*)g.ws;
  r.ws_ld = share_ld(g, r.share_up);
  r.split_stride = (int64_t)g.m * r.ws_ld;
  r.c = g.c;
  r.ldc = g.ldc;
  r.bias = g.bias;
  r.bias_dt = g.bias_dtype;
  r.splits = q.splits;
  r.M = g.m;
  r.N = g.n;
  r.pair = pair;
  r.c_vec = t.c_vec;
  t.c = g.ws;
  t.ldc = r.ws_ld;
  t.split_stride = r.split_stride;
  t.share_up = r.share_up;
  t.units_split = mx4_split_units(q.kernel, t.units, q.splits);
  int rc = api_launched(launch(true), "mx4 GEMM (split over K)");
  return rc ? rc : api_launched(launch_mx4_reduce(r, s), "mx4 GEMM (sum of the splits)");
}

}  // extern "C"
