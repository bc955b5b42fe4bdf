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
// Memory bound: 2 bytes in, 1 byte out per orientation. 8192 x 11008: rows 55 us (4.9 TB/s), columns 51 (5.3), tiles 51 (5.3), rows
// and columns together 86 (4.2, against 106 in two passes); the measured copy rate is 6.6 TB/s.

#include "block_quant.cuh"
#include "common.cuh"
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

__device__ __forceinline__ void store8(uint8_t* dst, uint2 v, int n) {
  if (n >= 8) {
    *reinterpret_cast<uint2*>(dst) = v;
  } else {
    for (int j = 0; j < n; ++j) dst[j] = static_cast<uint8_t>((j < 4 ? v.x >> (8 * j) : v.y >> (8 * (j - 4))) & 0xffu);
  }
}

template <int MODE>
__global__ void __launch_bounds__(THREADS, MODE == (ROWS | COLUMNS) ? 3 : 4) quantize_block_kernel(const Params p, int vec) {
  __shared__ uint32_t red[8][B / 2];  // column maxima (pairs) of each warp; the tile form uses red[0][0..7]
  __shared__ float factor[B], row_scale[B];
  const int across = threadIdx.x & 15, down = threadIdx.x >> 4;
  const int warp = threadIdx.x >> 5;
  const int col = blockIdx.x * B + across * 8;
  const int n_col = min(8, p.cols - col);  // columns of this thread inside the matrix (may be <= 0)
  const long long row0 = static_cast<long long>(blockIdx.y) * B;
  const __nv_bfloat16* x = p.x + static_cast<long long>(blockIdx.z) * p.x_group;
  next_kernel_may_start();
  previous_kernel_done();
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
    for (int i = 0; i < 8; i += 2) {  // two rows share a register on their way through the half-warp
      const uint32_t a = max_abs2(max_abs2(max_abs2(max_abs2(0u, v[i].x), v[i].y), v[i].z), v[i].w);
      const uint32_t b = max_abs2(max_abs2(max_abs2(max_abs2(0u, v[i + 1].x), v[i + 1].y), v[i + 1].z), v[i + 1].w);
      uint32_t m2 = max_abs2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
      for (int o = 8; o; o >>= 1) m2 = max_abs2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float amax = h ? hi(m2) : lo(m2);
        const int e = scale_exponent(amax);
        const float inv = pow2_biased(254 - e);
        const int local = down + 16 * (i + h);
        const long long row = row0 + local;
        if (across == 0) row_scale[local] = pow2_biased(e);
        if (row < p.rows && n_col > 0)
          store8(p.q_row + row * p.ldq + col, amax == INFINITY ? e4m3x8<true>(v[i + h], inv) : e4m3x8<false>(v[i + h], inv), n_col);
      }
    }
  }

  if (MODE & (COLUMNS | TILES)) {
    uint32_t m2[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m2[0] = max_abs2(m2[0], v[i].x);
      m2[1] = max_abs2(m2[1], v[i].y);
      m2[2] = max_abs2(m2[2], v[i].z);
      m2[3] = max_abs2(m2[3], v[i].w);
    }
    float inv[8];
    bool has_inf = false;
    if (MODE & COLUMNS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) m2[j] = max_abs2(m2[j], __shfl_xor_sync(0xffffffffu, m2[j], 16));
      if ((threadIdx.x & 16) == 0) *reinterpret_cast<uint4*>(&red[warp][across * 4]) = make_uint4(m2[0], m2[1], m2[2], m2[3]);
      __syncthreads();
      if (threadIdx.x < B / 2) {
        uint32_t top = red[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < 8; ++w) top = max_abs2(top, red[w][threadIdx.x]);
        const float amax[2] = {lo(top), hi(top)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e = scale_exponent(amax[h]);
          // the reciprocal; its sign says that the column holds an infinity
          factor[2 * threadIdx.x + h] = amax[h] == INFINITY ? -pow2_biased(254 - e) : pow2_biased(254 - e);
          const int c = blockIdx.x * B + 2 * threadIdx.x + h;
          if (c < p.cols) p.s_col[static_cast<long long>(blockIdx.y) * p.cols + c] = pow2_biased(e);
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(&factor[across * 8 + j]);
        inv[j] = fabsf(f.x); inv[j + 1] = fabsf(f.y); inv[j + 2] = fabsf(f.z); inv[j + 3] = fabsf(f.w);
        has_inf |= fminf(fminf(f.x, f.y), fminf(f.z, f.w)) < 0.f;
      }
    } else {
      uint32_t top2 = max_abs2(max_abs2(m2[0], m2[1]), max_abs2(m2[2], m2[3]));
#pragma unroll
      for (int o = 16; o; o >>= 1) top2 = max_abs2(top2, __shfl_xor_sync(0xffffffffu, top2, o));
      if ((threadIdx.x & 31) == 0) red[0][warp] = top2;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) top2 = max_abs2(top2, red[0][w]);
      const float top = fmaxf(lo(top2), hi(top2));
      has_inf = top == INFINITY;
      const int e = scale_exponent(top);
#pragma unroll
      for (int j = 0; j < 8; ++j) inv[j] = pow2_biased(254 - e);
      if (threadIdx.x == 0)
        p.s_tile[(static_cast<long long>(blockIdx.z) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = pow2_biased(e);
    }
    uint8_t* q = (MODE & COLUMNS) ? p.q_col : p.q_tile + static_cast<long long>(blockIdx.z) * p.q_group;
    if (n_col > 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const long long row = row0 + down + 16 * i;
        if (row < p.rows) store8(q + row * p.ldq + col, has_inf ? e4m3x8<true>(v[i], inv) : e4m3x8<false>(v[i], inv), n_col);
      }
    }
  }
  if (MODE & ROWS) {
    __syncthreads();
    if (threadIdx.x < B && row0 + threadIdx.x < p.rows)
      p.s_row[static_cast<long long>(blockIdx.x) * p.rows + row0 + threadIdx.x] = row_scale[threadIdx.x];
  }
}

template <int MODE>
static int launch(const Params& p, int vec, dim3 grid, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = grid;
  config.blockDim = dim3(THREADS);
  config.stream = stream;
  cudaLaunchAttribute attribute = dependent_launch();
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelEx(&config, quantize_block_kernel<MODE>, p, vec) == cudaSuccess ? 0 : -4;
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
    return blkq::launch<blkq::TILES>(p, vec, grid, stream);
  }
  if (groups != 1 || (q_row != nullptr && s_row == nullptr) || (q_col != nullptr && s_col == nullptr)) return -1;
  if (q_row != nullptr && q_col != nullptr) return blkq::launch<blkq::ROWS | blkq::COLUMNS>(p, vec, grid, stream);
  if (q_row != nullptr) return blkq::launch<blkq::ROWS>(p, vec, grid, stream);
  if (q_col != nullptr) return blkq::launch<blkq::COLUMNS>(p, vec, grid, stream);
  return -1;
}
