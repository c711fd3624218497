// MXFP4 quantization of rows, and MX values (4- or 8-bit) back to numbers.
//
// quant: for each 32-column block, amax = max |x|, e = ceil(log2(amax / 6)) at least -127, codes x /
// 2^e rounded to the nearest e2m1 value (ties to the even code), scale byte e + 127. 6 is e2m1's
// largest value, so nothing is clamped (the same choice as MXFP8's quantization here: rounding amax
// up to the next scale costs a bit of resolution where the floor rule would clip values up to 25%).
// A block with an infinity or a NaN gets the scale 255, E8M0's NaN, and codes 0 (hkx_mx_block.hpp).
//
// Both bound by HBM, a thread 8 values so that a wave reads and writes whole lines: fp32 12288 x 4096 46 us
// (229 MB, 5.0 TB/s; a copy of 1 GiB 5.25), back to bf16 20 (129 MB, the codes from the cache).
#include <algorithm>

#include "hkx_api.hpp"
#include "hkx_device.hpp"
#include "hkx_mx_block.hpp"

namespace hkx {

// 8 consecutive values of row type DT as fp32
template <int DT>
HKX_DEV void load8(const void* p, int64_t idx, float (&v)[8]) {
  if constexpr (DT == HKX_FP32) {
    const f32x4 a = *(const f32x4*)((const float*)p + idx), b = *(const f32x4*)((const float*)p + idx + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const i32x4 w = *(const i32x4*)((const uint16_t*)p + idx);
    const u32x2 lo = u32x2{(uint32_t)w.x, (uint32_t)w.y}, hi = u32x2{(uint32_t)w.z, (uint32_t)w.w};
    const f32x4 a = DT == HKX_BF16 ? unpack_bf16x4(lo) : unpack_f16x4(lo);
    const f32x4 b = DT == HKX_BF16 ? unpack_bf16x4(hi) : unpack_f16x4(hi);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}

// A thread a piece of 8 values, the 4 threads of a block a quad.
template <int DT>
__global__ void __launch_bounds__(256) mx4_quant_kernel(const void* x, int64_t ldx, uint8_t* q, int64_t ldq,
                                                        uint8_t* sc, int64_t lds, int m, int k8) {
  const uint32_t p = blockIdx.x * 256 + threadIdx.x;
  if (p >= (uint32_t)m * (uint32_t)k8) return;  // (k8 is a multiple of 4: whole quads)
  const uint32_t row = p / (uint32_t)k8;
  const int g = (int)(p - row * (uint32_t)k8);
  float v[8];
  load8<DT>(x, (int64_t)row * ldx + 8 * g, v);
  uint32_t w;
  const uint32_t s = mx4_block(v, mx_block_top(v), w);
  *(uint32_t*)(q + (int64_t)row * ldq + 4 * g) = w;
  if ((g & 3) == 0) sc[(int64_t)row * lds + g / 4] = (uint8_t)s;
}

// MX values as numbers: a thread 8 of them, each an exact power-of-two scaling, rounded once to
// the output's type.
template <bool FP8, int DT>
__global__ void __launch_bounds__(256) mx_dequant_kernel(const uint8_t* q, int64_t ldq, const uint8_t* sc, int64_t lds,
                                                         void* y, int64_t ldy, int m, int k8) {
  const uint32_t p = blockIdx.x * 256 + threadIdx.x;
  if (p >= (uint32_t)m * (uint32_t)k8) return;
  const uint32_t row = p / (uint32_t)k8;
  const int g = (int)(p - row * (uint32_t)k8);
  const int s = sc[(int64_t)row * lds + g / 4];
  float v[8];
  if constexpr (FP8) {
    const u32x2 w = *(const u32x2*)(q + (int64_t)row * ldq + 8 * g);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = (int)(i ? w.y : w.x);
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
      v[4 * i] = lo.x; v[4 * i + 1] = lo.y; v[4 * i + 2] = hi.x; v[4 * i + 3] = hi.y;
    }
  } else {
    const uint32_t w = *(const uint32_t*)(q + (int64_t)row * ldq + 4 * g);
#define HKX_FP4_PAIR(i)                                                      \
  {                                                                          \
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, i);    \
    v[2 * i] = d.x;                                                          \
    v[2 * i + 1] = d.y;                                                      \
  }
    HKX_FP4_PAIR(0) HKX_FP4_PAIR(1) HKX_FP4_PAIR(2) HKX_FP4_PAIR(3)
#undef HKX_FP4_PAIR
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = s == 255 ? __builtin_nanf("") : __builtin_ldexpf(v[i], s - 127);
  const int64_t at = (int64_t)row * ldy + 8 * g;
  store4(y, DT, at, f32x4{v[0], v[1], v[2], v[3]});
  store4(y, DT, at + 4, f32x4{v[4], v[5], v[6], v[7]});
}

}  // namespace hkx

namespace {

// A launch's threads, a piece each, stay under 2^32 (a grid past that is cut short, with no error): more rows
// go launch by launch.
int64_t rows_a_launch(int k) { return (((int64_t)1 << 32) - 256) / (k / 8); }

template <int DT>
hipError_t quant(const void* x, int64_t ldx, void* q, int64_t ldq, uint8_t* s, int64_t lds, int m, int k, hipStream_t st) {
  constexpr int es = DT == HKX_FP32 ? 4 : 2;
  for (int64_t r = 0, most = rows_a_launch(k); r < m; r += most) {
    const int rows = (int)std::min(most, m - r);
    const dim3 grid((unsigned)(((int64_t)rows * (k / 8) + 255) / 256));
    hipLaunchKernelGGL((hkx::mx4_quant_kernel<DT>), grid, dim3(256), 0, st, (const uint8_t*)x + r * ldx * es, ldx,
                       (uint8_t*)q + r * ldq, ldq, s + r * lds, lds, rows, k / 8);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

template <bool FP8, int DT>
hipError_t dequant(const void* q, int64_t ldq, const uint8_t* s, int64_t lds, void* y, int64_t ldy, int m, int k, hipStream_t st) {
  constexpr int es = DT == HKX_FP32 ? 4 : 2;
  for (int64_t r = 0, most = rows_a_launch(k); r < m; r += most) {
    const int rows = (int)std::min(most, m - r);
    const dim3 grid((unsigned)(((int64_t)rows * (k / 8) + 255) / 256));
    hipLaunchKernelGGL((hkx::mx_dequant_kernel<FP8, DT>), grid, dim3(256), 0, st, (const uint8_t*)q + r * ldq, ldq,
                       s + r * lds, lds, (uint8_t*)y + r * ldy * es, ldy, rows, k / 8);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

}  // namespace

extern "C" {

int hkx_mx4_quant(const void* x, int64_t ldx, int32_t x_dtype, void* q, int64_t ldq, uint8_t* s, int64_t lds,
                  int32_t m, int32_t k, void* stream) {
  using namespace hkx;
  api_clear();
  if (!x || !q || !s) return api_fail(HKX_ERR_ARG, "mx4_quant: a null pointer");
  if (x_dtype != HKX_BF16 && x_dtype != HKX_FP16 && x_dtype != HKX_FP32)
    return api_fail(HKX_ERR_DTYPE, "mx4_quant: x is bf16, fp16 or fp32");
  if (m < 0 || k < 0 || k % 32) return api_fail(HKX_ERR_SHAPE, "mx4_quant: M=%d, K=%d a multiple of 32", m, k);
  if (ldx < k || ldq < k / 2 || lds < k / 32) return api_fail(HKX_ERR_SHAPE, "mx4_quant: row strides below K, K/2 or K/32");
  const int64_t es = x_dtype == HKX_FP32 ? 4 : 2;
  if (!api_aligned(x, 16) || ldx * es % 16 || !api_aligned(q, 4) || ldq % 4)
    return api_fail(HKX_ERR_SHAPE, "mx4_quant: x needs 16-byte and q 4-byte aligned rows");
  if (m == 0 || k == 0) return HKX_OK;
  const hipStream_t st = (hipStream_t)stream;
  return api_launched(x_dtype == HKX_BF16   ? quant<HKX_BF16>(x, ldx, q, ldq, s, lds, m, k, st)
                      : x_dtype == HKX_FP16 ? quant<HKX_FP16>(x, ldx, q, ldq, s, lds, m, k, st)
                                            : quant<HKX_FP32>(x, ldx, q, ldq, s, lds, m, k, st),
                      "mx4 quant");
}

int hkx_mx_dequant(const void* q, int64_t ldq, int32_t q_dtype, const uint8_t* s, int64_t lds, void* y, int64_t ldy,
                   int32_t y_dtype, int32_t m, int32_t k, void* stream) {
  using namespace hkx;
  api_clear();
  if (!q || !y || !s) return api_fail(HKX_ERR_ARG, "mx_dequant: a null pointer");
  const bool fp8 = q_dtype == HKX_FP8E4M3;
  if (!fp8 && q_dtype != HKX_FP4E2M1) return api_fail(HKX_ERR_DTYPE, "mx_dequant: q is packed 4-bit or e4m3");
  if (y_dtype != HKX_BF16 && y_dtype != HKX_FP16 && y_dtype != HKX_FP32)
    return api_fail(HKX_ERR_DTYPE, "mx_dequant: y is bf16, fp16 or fp32");
  if (m < 0 || k < 0 || k % 32) return api_fail(HKX_ERR_SHAPE, "mx_dequant: M=%d, K=%d a multiple of 32", m, k);
  if (ldq < (fp8 ? k : k / 2) || ldy < k || lds < k / 32) return api_fail(HKX_ERR_SHAPE, "mx_dequant: row strides below a row");
  const int64_t es = y_dtype == HKX_FP32 ? 4 : 2, qa = fp8 ? 8 : 4;
  if (!api_aligned(y, 16) || ldy * es % 16 || !api_aligned(q, qa) || ldq % qa)
    return api_fail(HKX_ERR_SHAPE, "mx_dequant: y needs 16-byte and q %d-byte aligned rows", (int)qa);
  if (m == 0 || k == 0) return HKX_OK;
  const hipStream_t st = (hipStream_t)stream;
  hipError_t e;
  if (fp8)
    e = y_dtype == HKX_BF16   ? dequant<true, HKX_BF16>(q, ldq, s, lds, y, ldy, m, k, st)
        : y_dtype == HKX_FP16 ? dequant<true, HKX_FP16>(q, ldq, s, lds, y, ldy, m, k, st)
                              : dequant<true, HKX_FP32>(q, ldq, s, lds, y, ldy, m, k, st);
  else
    e = y_dtype == HKX_BF16   ? dequant<false, HKX_BF16>(q, ldq, s, lds, y, ldy, m, k, st)
        : y_dtype == HKX_FP16 ? dequant<false, HKX_FP16>(q, ldq, s, lds, y, ldy, m, k, st)
                              : dequant<false, HKX_FP32>(q, ldq, s, lds, y, ldy, m, k, st);
  return api_launched(e, "mx dequant");
}

}  // extern "C"
