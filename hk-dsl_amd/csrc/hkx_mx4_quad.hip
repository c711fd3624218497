// The MXFP4 quadrant kernel's forms (hkx_mx4_quad.hpp).
#include "hkx_mx4_quad.hpp"

namespace hkx {

// A workgroup 4 chunks (64 blocks) of a tile's 256 rows: the rows' dwords into LDS, 16 at a time a row,
// then out in packed order. A row that starts off a multiple of 4 bytes joins two dwords.
__global__ void __launch_bounds__(256) mx4_pack_kernel(const Mx4PackArgs pa, const Mx4PackArgs pb) {
  constexpr int NC = 4;
  __shared__ uint32_t lds[256][NC * 4 + 1];
  const bool isb = (int)blockIdx.y >= pa.tiles;
  const Mx4PackArgs& p = isb ? pb : pa;
  const int tile = (int)blockIdx.y - (isb ? pa.tiles : 0);
  const int c0 = blockIdx.x * NC;
  const uintptr_t base = (uintptr_t)p.s & ~(uintptr_t)3;
  const uint32_t off0 = (uint32_t)((uintptr_t)p.s & 3);
  const uint32_t total = (p.pair ? 2 : 1) * p.rows;
  // (whole dwords up to the one that holds the last byte)
  const __amdgpu_buffer_rsrc_t r = make_rsrc((const void*)base, (off0 + (total - 1) * p.ld + (uint32_t)p.k32 + 3) & ~3u);
  const int w = threadIdx.x & 15;
  uint32_t v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int row = (threadIdx.x >> 4) + 16 * i;  // of the tile
    uint32_t g;
    bool ok;
    if (p.pair) {
      g = (uint32_t)(tile * 128 + 16 * (row >> 5) + (row & 15));
      ok = g < p.rows;
      g += row & 16 ? p.rows : 0;
    } else {
      g = (uint32_t)(tile * 256 + row);
      ok = g < p.rows;
    }
    const int blk = c0 * 16 + 4 * w;
    const uint32_t at = off0 + g * p.ld + (uint32_t)blk;
    ok = ok && blk < p.k32;
    const uint32_t lo = __builtin_amdgcn_raw_buffer_load_b32(r, ok ? at & ~3u : kMx4Out, 0, 0);
    const uint32_t hi = __builtin_amdgcn_raw_buffer_load_b32(r, ok && (at & 3) ? (at & ~3u) + 4 : kMx4Out, 0, 0);
    v[i] = __builtin_amdgcn_alignbyte(hi, lo, at & 3) & (ok ? mx4_mask(p.k32 - blk) : 0u);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) lds[(threadIdx.x >> 4) + 16 * i][w] = v[i];
  __syncthreads();
  const uint8_t* s = (const uint8_t*)lds;
  constexpr int RS = (NC * 4 + 1) * 4;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    if (c0 + c >= p.chunks) break;
    uint8_t* out = p.out + ((int64_t)tile * p.chunks + c0 + c) * 4096 + threadIdx.x * 16;
    uint32_t o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      uint32_t x = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int byte = threadIdx.x * 16 + 4 * d + b;  // of the chunk's 4 KB
        const int unit = byte >> 11, e = byte & 2047;
        int row, blk;
        if (p.is_b) {
          const int lane = (e >> 3) & 63, k = e & 7;
          row = 128 * ((k >> 1) & 1) + 32 * (e >> 9) + 16 * (k & 1) + (lane & 15);
          blk = 8 * unit + 4 * (k >> 2) + (lane >> 4);
        } else {
          const int lane = (e >> 4) & 63, k = e & 15;
          row = 128 * ((k >> 2) & 1) + 64 * (e >> 10) + 16 * (k & 3) + (lane & 15);
          blk = 8 * unit + 4 * (k >> 3) + (lane >> 4);
        }
        x |= (uint32_t)s[row * RS + 16 * c + blk] << (8 * b);
      }
      o[d] = x;
    }
    *(i32x4*)out = i32x4{(int)o[0], (int)o[1], (int)o[2], (int)o[3]};
  }
}

hipError_t launch_mx4_pack(const Mx4PackArgs& a, const Mx4PackArgs& b, hipStream_t s) {
  hipLaunchKernelGGL(mx4_pack_kernel, dim3((unsigned)((a.chunks + 3) / 4), (unsigned)(a.tiles + b.tiles)), dim3(256), 0, s, a, b);
  return hipGetLastError();
}

template <bool A8, bool PAIR>
static hipError_t launch(const Mx4Args& a, bool share, dim3 grid, hipStream_t s) {
  if (share) hipLaunchKernelGGL((mx4_quad_kernel<A8, PAIR, true>), grid, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((mx4_quad_kernel<A8, PAIR, false>), grid, dim3(512), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_mx4_quad(const Mx4Args& a, bool a8, bool pair, bool share, dim3 grid, hipStream_t s) {
  if (a8) return pair ? launch<true, true>(a, share, grid, s) : launch<true, false>(a, share, grid, s);
  return pair ? launch<false, true>(a, share, grid, s) : launch<false, false>(a, share, grid, s);
}

}  // namespace hkx
