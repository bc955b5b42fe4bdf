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
// Memory bound: 2 bytes in, 1 byte out per orientation. 8192 x 11008: rows 47 us (5.7 TB/s), columns 47, tiles 46, rows and columns
// together 61 (5.9, against 94 in two passes); the measured copy rate is 6.6 TB/s. Three things got it there from 55, 51, 51 and 86 us,
// when the issue of instructions was the bound (13 per element and orientation): scaling in packed pairs, infinities patched in afterwards
// instead of inside the cast, and a copy of the code for whole tiles that checks no edges.

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
  int row_tiles;
  int tile0, group0;  // what the launch's blockIdx.y and .z count from: neither can exceed 65535
};

// What a tile needs besides its registers.
struct Shared {
  uint32_t top[8][B / 2];  // column maxima (pairs) of each warp; the tile form uses top[0][0..7]
  uint32_t factor[B / 2];  // reciprocals of the columns' scales, in pairs; a sign says that the column holds an infinity
  float row_scale[B];
};

// FULL: the tile lies inside the matrix and its rows start on 16-byte boundaries.
template <int MODE, bool FULL>
__device__ __forceinline__ void quantize_tile(const Params& p, int vec, Shared& sh) {
  const int across = threadIdx.x & 15, down = threadIdx.x >> 4, warp = threadIdx.x >> 5;
  const int row_tile = p.tile0 + blockIdx.y, group = p.group0 + blockIdx.z;
  const int col = blockIdx.x * B + across * 8;
  const int n_col = FULL ? 8 : min(8, p.cols - col);  // columns of this thread inside the matrix (may be <= 0)
  const long long row0 = static_cast<long long>(row_tile) * B + down;
  const int n_row = FULL ? 8 : n_col <= 0 ? 0 : static_cast<int>(min(8ll, (p.rows - row0 + 15) / 16));  // rows row0 + 16 i

  uint4 v[8];
  {
    const __nv_bfloat16* src = p.x + static_cast<long long>(group) * p.x_group + row0 * p.ldx + col;
#pragma unroll
    for (int i = 0; i < 8; ++i, src += 16 * p.ldx) {
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (!FULL && i >= n_row) continue;
      if (FULL || (vec && n_col == 8)) {
        v[i] = *reinterpret_cast<const uint4*>(src);
      } else {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n_col) w[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(src)[j]) << (16 * (j & 1));
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  auto store = [&](uint8_t* dst, uint2 c) {
    if (FULL || n_col == 8) {
      *reinterpret_cast<uint2*>(dst) = c;
    } else {
      for (int j = 0; j < n_col; ++j) dst[j] = static_cast<uint8_t>((j < 4 ? c.x >> (8 * j) : c.y >> (8 * (j - 4))) & 0xffu);
    }
  };

  if (MODE & ROWS) {
    uint8_t* dst = p.q_row + row0 * p.ldq + col;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {  // two rows share a register on their way through the half-warp
      const uint32_t a = max_mag2(v[i]), b = max_mag2(v[i + 1]);
      uint32_t m2 = max_mag2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
      for (int o = 8; o; o >>= 1) m2 = max_mag2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
#pragma unroll
      for (int h = 0; h < 2; ++h, dst += 16 * p.ldq) {
        const uint32_t amax = (h ? m2 >> 16 : m2) & 0x7fffu;
        const int e = scale_exponent(amax);
        if (across == 0) sh.row_scale[down + 16 * (i + h)] = pow2_biased(e);
        uint2 c = e4m3x8(v[i + h], inverse_bf16(e) * 0x10001u);
        if (amax == BF16_INF) c = infinities_to_nan(v[i + h], c);
        if (FULL || i + h < n_row) store(dst, c);
      }
    }
  }

  if (MODE & (COLUMNS | TILES)) {
    uint4 m = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = make_uint4(max_mag2(m.x, v[i].x), max_mag2(m.y, v[i].y), max_mag2(m.z, v[i].z), max_mag2(m.w, v[i].w));
    uint4 inv;
    bool has_inf;
    if (MODE & COLUMNS) {
      m = make_uint4(max_mag2(m.x, __shfl_xor_sync(0xffffffffu, m.x, 16)), max_mag2(m.y, __shfl_xor_sync(0xffffffffu, m.y, 16)),
                     max_mag2(m.z, __shfl_xor_sync(0xffffffffu, m.z, 16)), max_mag2(m.w, __shfl_xor_sync(0xffffffffu, m.w, 16)));
      if ((threadIdx.x & 16) == 0) *reinterpret_cast<uint4*>(&sh.top[warp][across * 4]) = m;
      __syncthreads();
      if (threadIdx.x < B / 2) {
        uint32_t top = sh.top[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < 8; ++w) top = max_mag2(top, sh.top[w][threadIdx.x]);
        uint32_t pair = 0u;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t amax = (h ? top >> 16 : top) & 0x7fffu;
          const int e = scale_exponent(amax);
          pair |= (inverse_bf16(e) | (amax == BF16_INF ? 0x8000u : 0u)) << (16 * h);
          const int c = blockIdx.x * B + 2 * threadIdx.x + h;
          if (FULL || c < p.cols) p.s_col[static_cast<long long>(row_tile) * p.cols + c] = pow2_biased(e);
        }
        sh.factor[threadIdx.x] = pair;
      }
      __syncthreads();
      inv = *reinterpret_cast<const uint4*>(&sh.factor[across * 4]);
      has_inf = ((inv.x | inv.y | inv.z | inv.w) & 0x80008000u) != 0u;
      inv = make_uint4(inv.x & 0x7fff7fffu, inv.y & 0x7fff7fffu, inv.z & 0x7fff7fffu, inv.w & 0x7fff7fffu);
    } else {
      uint32_t top = max_mag2(m);
#pragma unroll
      for (int o = 16; o; o >>= 1) top = max_mag2(top, __shfl_xor_sync(0xffffffffu, top, o));
      if ((threadIdx.x & 31) == 0) sh.top[0][warp] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) top = max_mag2(top, sh.top[0][w]);
      const uint32_t amax = max(top & 0x7fffu, (top >> 16) & 0x7fffu);  // magnitudes order as their bits
      has_inf = amax == BF16_INF;
      const int e = scale_exponent(amax);
      inv.x = inv.y = inv.z = inv.w = inverse_bf16(e) * 0x10001u;
      if (threadIdx.x == 0)
        p.s_tile[(static_cast<long long>(group) * p.row_tiles + row_tile) * gridDim.x + blockIdx.x] = pow2_biased(e);
    }
    uint8_t* dst = ((MODE & COLUMNS) ? p.q_col : p.q_tile + static_cast<long long>(group) * p.q_group) + row0 * p.ldq + col;
#pragma unroll
    for (int i = 0; i < 8; ++i, dst += 16 * p.ldq) {
      uint2 c = e4m3x8(v[i], inv);
      if (has_inf) c = infinities_to_nan(v[i], c);
      if (FULL || i < n_row) store(dst, c);
    }
  }
  if (MODE & ROWS) {
    __syncthreads();
    const long long row = static_cast<long long>(row_tile) * B + threadIdx.x;
    if (threadIdx.x < B && (FULL || row < p.rows)) p.s_row[static_cast<long long>(blockIdx.x) * p.rows + row] = sh.row_scale[threadIdx.x];
  }
}

template <int MODE>
__global__ void __launch_bounds__(THREADS, MODE == (ROWS | COLUMNS) ? 3 : 4) quantize_block_kernel(const Params p, int vec) {
  __shared__ Shared sh;
  next_kernel_may_start();
  previous_kernel_done();
  const bool full = vec && (blockIdx.x + 1ll) * B <= p.cols && (p.tile0 + blockIdx.y + 1ll) * B <= p.rows;
  if (full) quantize_tile<MODE, true>(p, vec, sh);
  else quantize_tile<MODE, false>(p, vec, sh);
}

template <int MODE>
static int launch(Params p, int vec, int groups, cudaStream_t stream) {
  constexpr int MOST = 65535;  // CTAs along y and z of one launch
  cudaLaunchConfig_t config = {};
  config.blockDim = dim3(THREADS);
  config.stream = stream;
  cudaLaunchAttribute attribute = dependent_launch();
  config.attrs = &attribute;
  config.numAttrs = 1;
  for (p.group0 = 0; p.group0 < groups; p.group0 += MOST) {
    for (p.tile0 = 0; p.tile0 < p.row_tiles; p.tile0 += MOST) {
      config.gridDim = dim3((p.cols + B - 1) / B, min(p.row_tiles - p.tile0, MOST), min(groups - p.group0, MOST));
      if (cudaLaunchKernelEx(&config, quantize_block_kernel<MODE>, p, vec) != cudaSuccess) return -4;
    }
  }
  return 0;
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
  if (rows > 0x7fffffff - 512 || cols > 0x7fffffff - 512 || groups > 0x7fffffff - 65536) return -1;  // rounded up in 32 bits
  p.row_tiles = (rows + blkq::B - 1) / blkq::B;
  if (q_tile != nullptr) {
    if (s_tile == nullptr || q_row != nullptr || q_col != nullptr) return -1;
    return blkq::launch<blkq::TILES>(p, vec, groups, stream);
  }
  if (groups != 1 || (q_row != nullptr && s_row == nullptr) || (q_col != nullptr && s_col == nullptr)) return -1;
  if (q_row != nullptr && q_col != nullptr) return blkq::launch<blkq::ROWS | blkq::COLUMNS>(p, vec, groups, stream);
  if (q_row != nullptr) return blkq::launch<blkq::ROWS>(p, vec, groups, stream);
  if (q_col != nullptr) return blkq::launch<blkq::COLUMNS>(p, vec, groups, stream);
  return -1;
}
