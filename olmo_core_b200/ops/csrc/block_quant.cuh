// Arithmetic of the e4m3 quantisation with a power-of-two scale per block, shared by the quantisers and by the product that
// quantises its tokens itself.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ocb {

namespace blkq {

// Pairs of bf16 stay packed: a power of two and the product with it (of a block's element, so at most 448) are exact in bf16.

// The larger magnitudes of two pairs, NaN ignored; the signs of the result mean nothing.
__device__ __forceinline__ uint32_t max_mag2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max_mag2(const uint4& v) { return max_mag2(max_mag2(max_mag2(max_mag2(0u, v.x), v.y), v.z), v.w); }

constexpr uint32_t BF16_INF = 0x7f80u;

// Biased exponent of the scale of a block whose largest magnitude is `amax` (bits of a bf16): 448 is 1.75 * 2^8, so the exponent is
// 8 below the magnitude's, or 7 where the seven bits of its mantissa are above 0x60.
__device__ __forceinline__ int scale_exponent(uint32_t amax) {
  const int e = static_cast<int>((amax + 0x1fu) >> 7) - 8;
  return amax == 0u ? 127 : min(max(e, 1), 253);
}
__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }
// Reciprocal of that scale, as a bf16.
__device__ __forceinline__ uint32_t inverse_bf16(int e) { return static_cast<uint32_t>(254 - e) << 7; }

// Two elements times two powers of two, as e4m3.
__device__ __forceinline__ uint16_t e4m3x2(uint32_t pair, uint32_t inv) {
  uint32_t v;
  uint16_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(v) : "r"(pair), "r"(inv));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(__uint_as_float(v & 0xffff0000u)), "f"(__uint_as_float(v << 16)));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(uint32_t a, uint32_t b, uint32_t inv_a, uint32_t inv_b) {
  uint32_t r;
  asm("mov.b32 %0, {%1, %2};" : "=r"(r) : "h"(e4m3x2(a, inv_a)), "h"(e4m3x2(b, inv_b)));
  return r;
}
__device__ __forceinline__ uint2 e4m3x8(const uint4& v, const uint4& inv) {
  return make_uint2(e4m3x4(v.x, v.y, inv.x, inv.y), e4m3x4(v.z, v.w, inv.z, inv.w));
}
__device__ __forceinline__ uint2 e4m3x8(const uint4& v, uint32_t inv) { return e4m3x8(v, make_uint4(inv, inv, inv, inv)); }

// The cast saturates; where a block holds an infinity, its codes become NaN here.
static __device__ __noinline__ uint2 infinities_to_nan(uint4 v, uint2 codes) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t c[2] = {codes.x, codes.y};
  for (int j = 0; j < 8; ++j)
    if (((w[j >> 1] >> (16 * (j & 1))) & 0x7fffu) == BF16_INF) c[j >> 2] = (c[j >> 2] & ~(0xffu << (8 * (j & 3)))) | 0x7fu << (8 * (j & 3));
  return make_uint2(c[0], c[1]);
}

}  // namespace blkq
}  // namespace ocb
