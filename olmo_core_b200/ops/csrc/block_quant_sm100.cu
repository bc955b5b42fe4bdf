// Quantisation to e4m3 with one power-of-two scale per block of 128, for the GEMM of gemm_block_fp8_sm100.cu.
//
//   rows      block = 128 consecutive elements of a row         scale s_row[column / 128][row]
//   columns   block = 128 consecutive elements of a column      scale s_col[row / 128][column]
//   tiles     block = 128 x 128 elements                        scale s_tile[row / 128][column / 128]
//
// A block's scale is the smallest power of two (not below 2^-126) that brings its largest magnitude to 448 = 1.75 * 2^8 or
// below, so it follows from the exponent and the mantissa of that magnitude alone, dividing by it is exact, and the only
// rounding is the one to e4m3. A block of zeros has scale 1. NaN and infinity become NaN.
//
// One CTA holds a 128 x 128 tile in registers (16 threads across, 16 down, each 8 rows of 8 columns): the maxima over a row
// are shuffles within half a warp, those over a column go through shared memory. Rows and columns can come out of one launch,
// which reads the tensor once where a layer needs both (the activations of a training step and the output gradient).
// Memory bound: 2 bytes in, 1 byte out per orientation.

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ocb_api.h"

namespace ocb {
namespace blkq {

constexpr int B = 128;
constexpr int THREADS = 256;
enum : int { ROWS = 1, COLUMNS = 2, TILES = 4 };

struct Params {
  const __nv_bfloat16* x;
  uint8_t *q_row, *q_col, *q_tile;
  float *s_row, *s_col, *s_tile;
  int rows, cols;
  long long ldx, ldq;
  long long x_group, q_group;  // elements between the matrices of a stack (tiles only)
};

// Biased exponent of the scale of a block with the largest magnitude `amax`.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return bits == 0u ? 127 : min(max(e, 1), 253);
}
__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }

__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// x * inv; the product with zero turns an infinity into NaN, which the saturating cast would hide, and adds nothing otherwise.
__device__ __forceinline__ float scaled(float x, float inv) { return __fmaf_rn(x, 0.f, x * inv); }

__device__ __forceinline__ float lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

__device__ __forceinline__ void store8(uint8_t* dst, uint2 v, int n) {
  if (n >= 8) {
    *reinterpret_cast<uint2*>(dst) = v;
  } else {
    for (int j = 0; j < n; ++j) dst[j] = static_cast<uint8_t>((j < 4 ? v.x >> (8 * j) : v.y >> (8 * (j - 4))) & 0xffu);
  }
}

template <int MODE>
__global__ void __launch_bounds__(THREADS) quantize_block_kernel(const Params p, int vec) {
  __shared__ float red[8][B];  // column maxima of each warp; the tile form uses red[0][0..7]
  const int across = threadIdx.x & 15, down = threadIdx.x >> 4;
  const int warp = threadIdx.x >> 5;
  const int col = blockIdx.x * B + across * 8;
  const int n_col = min(8, p.cols - col);  // columns of this thread inside the matrix (may be <= 0)
  const long long row0 = static_cast<long long>(blockIdx.y) * B;
  const __nv_bfloat16* x = p.x + static_cast<long long>(blockIdx.z) * p.x_group;
  uint4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long long row = row0 + down + 16 * i;
    v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (row < p.rows && n_col > 0) {
      const __nv_bfloat16* src = x + row * p.ldx + col;
      if (vec && n_col == 8) {
        v[i] = *reinterpret_cast<const uint4*>(src);
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n_col) w[j >> 1] |= static_cast<uint32_t>(h[j]) << (16 * (j & 1));
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }

  if (MODE & ROWS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fmaxf(fabsf(lo(w[j])), fabsf(hi(w[j]))));
#pragma unroll
      for (int o = 8; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const int e = scale_exponent(amax);
      const float inv = pow2_biased(254 - e);
      const long long row = row0 + down + 16 * i;
      if (row < p.rows) {
        uint2 o;
        o.x = e4m3x2(scaled(lo(w[0]), inv), scaled(hi(w[0]), inv)) | (e4m3x2(scaled(lo(w[1]), inv), scaled(hi(w[1]), inv)) << 16);
        o.y = e4m3x2(scaled(lo(w[2]), inv), scaled(hi(w[2]), inv)) | (e4m3x2(scaled(lo(w[3]), inv), scaled(hi(w[3]), inv)) << 16);
        if (n_col > 0) store8(p.q_row + row * p.ldq + col, o, n_col);
        if (across == 0) p.s_row[static_cast<long long>(blockIdx.x) * p.rows + row] = pow2_biased(e);
      }
    }
  }

  if (MODE & (COLUMNS | TILES)) {
    float m[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[2 * j] = fmaxf(m[2 * j], fabsf(lo(w[j])));
        m[2 * j + 1] = fmaxf(m[2 * j + 1], fabsf(hi(w[j])));
      }
    }
    float inv[8];
    if (MODE & COLUMNS) {
#pragma unroll
      for (int j = 0; j < 8; ++j) m[j] = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
      if ((threadIdx.x & 16) == 0) {
#pragma unroll
        for (int j = 0; j < 8; j += 4)
          *reinterpret_cast<float4*>(&red[warp][across * 8 + j]) = make_float4(m[j], m[j + 1], m[j + 2], m[j + 3]);
      }
      __syncthreads();
      if (threadIdx.x < B) {
        float top = red[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < 8; ++w) top = fmaxf(top, red[w][threadIdx.x]);
        const int e = scale_exponent(top);
        red[0][threadIdx.x] = pow2_biased(254 - e);
        const int c = blockIdx.x * B + threadIdx.x;
        if (c < p.cols) p.s_col[static_cast<long long>(blockIdx.y) * p.cols + c] = pow2_biased(e);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) inv[j] = red[0][across * 8 + j];
    } else {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, m[j]);
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      if ((threadIdx.x & 31) == 0) red[0][warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) top = fmaxf(top, red[0][w]);
      const int e = scale_exponent(top);
      const float f = pow2_biased(254 - e);
#pragma unroll
      for (int j = 0; j < 8; ++j) inv[j] = f;
      if (threadIdx.x == 0)
        p.s_tile[(static_cast<long long>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = pow2_biased(e);
    }
    uint8_t* q = (MODE & COLUMNS) ? p.q_col : p.q_tile + static_cast<long long>(blockIdx.z) * p.q_group;
    if (n_col > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long long row = row0 + down + 16 * i;
        if (row >= p.rows) continue;
        const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
        uint2 o;
        o.x = e4m3x2(scaled(lo(w[0]), inv[0]), scaled(hi(w[0]), inv[1])) |
              (e4m3x2(scaled(lo(w[1]), inv[2]), scaled(hi(w[1]), inv[3])) << 16);
        o.y = e4m3x2(scaled(lo(w[2]), inv[4]), scaled(hi(w[2]), inv[5])) |
              (e4m3x2(scaled(lo(w[3]), inv[6]), scaled(hi(w[3]), inv[7])) << 16);
        store8(q + row * p.ldq + col, o, n_col);
      }
    }
  }
}

}  // namespace blkq
}  // namespace ocb

using namespace ocb;

// See ocb_api.h.
extern "C" int ocb_quantize_block_fp8(const void* x, void* q_row, float* s_row, void* q_col, float* s_col, void* q_tile,
                                      float* s_tile, int groups, int rows, int cols, long long ldx, long long ldq,
                                      long long x_group, long long q_group, cudaStream_t stream) {
  if (groups <= 0 || rows <= 0 || cols <= 0) return 0;
  if ((ldq % 16) != 0 || (q_group % 16) != 0) return -1;
  const void* qs[3] = {q_row, q_col, q_tile};
  for (const void* q : qs)
    if (reinterpret_cast<uintptr_t>(q) & 15) return -1;
  blkq::Params p;
  p.x = reinterpret_cast<const __nv_bfloat16*>(x);
  p.q_row = reinterpret_cast<uint8_t*>(q_row);
  p.q_col = reinterpret_cast<uint8_t*>(q_col);
  p.q_tile = reinterpret_cast<uint8_t*>(q_tile);
  p.s_row = s_row;
  p.s_col = s_col;
  p.s_tile = s_tile;
  p.rows = rows;
  p.cols = cols;
  p.ldx = ldx;
  p.ldq = ldq;
  p.x_group = x_group;
  p.q_group = q_group;
  const int vec = (ldx % 8) == 0 && (x_group % 8) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  const long long row_tiles = (static_cast<long long>(rows) + blkq::B - 1) / blkq::B;
  if (row_tiles > 65535 || groups > 65535) return -1;
  const dim3 grid((cols + blkq::B - 1) / blkq::B, static_cast<unsigned>(row_tiles), groups);
  if (q_tile != nullptr) {
    if (s_tile == nullptr || q_row != nullptr || q_col != nullptr) return -1;
    blkq::quantize_block_kernel<blkq::TILES><<<grid, blkq::THREADS, 0, stream>>>(p, vec);
  } else {
    if (groups != 1 || (q_row != nullptr && s_row == nullptr) || (q_col != nullptr && s_col == nullptr)) return -1;
    if (q_row != nullptr && q_col != nullptr) blkq::quantize_block_kernel<blkq::ROWS | blkq::COLUMNS><<<grid, blkq::THREADS, 0, stream>>>(p, vec);
    else if (q_row != nullptr) blkq::quantize_block_kernel<blkq::ROWS><<<grid, blkq::THREADS, 0, stream>>>(p, vec);
    else if (q_col != nullptr) blkq::quantize_block_kernel<blkq::COLUMNS><<<grid, blkq::THREADS, 0, stream>>>(p, vec);
    else return -1;
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}
