// Arithmetic of the e4m3 quantisation with a power-of-two scale per block, shared by the quantisers and by the product that
// quantises its tokens itself.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ocb {

namespace blkq {

// Biased exponent of the scale of a block with the largest magnitude `amax`.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>(bits >> 23) - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return bits == 0u ? 127 : min(max(e, 1), 253);
}
__device__ __forceinline__ float pow2_biased(int e) { return __uint_as_float(static_cast<uint32_t>(e) << 23); }

// Packed magnitudes: the larger of two pairs, NaN ignored.
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("{\n\t.reg .b32 t;\n\tabs.bf16x2 t, %2;\n\tmax.bf16x2 %0, %1, t;\n\t}" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }

// Two elements (bf16 pair) times two powers of two, as e4m3. HAS_INF: the block holds an infinity, whose product with zero
// makes the NaN that the saturating cast would hide.
template <bool HAS_INF>
__device__ __forceinline__ uint32_t e4m3x2(uint32_t pair, float inv0, float inv1) {
  float a = lo(pair) * inv0, b = hi(pair) * inv1;
  if (HAS_INF) {
    a = __fmaf_rn(lo(pair), 0.f, a);
    b = __fmaf_rn(hi(pair), 0.f, b);
  }
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
template <bool HAS_INF>
__device__ __forceinline__ uint2 e4m3x8(const uint4& v, const float (&inv)[8]) {
  return make_uint2(e4m3x2<HAS_INF>(v.x, inv[0], inv[1]) | (e4m3x2<HAS_INF>(v.y, inv[2], inv[3]) << 16),
                    e4m3x2<HAS_INF>(v.z, inv[4], inv[5]) | (e4m3x2<HAS_INF>(v.w, inv[6], inv[7]) << 16));
}
template <bool HAS_INF>
__device__ __forceinline__ uint2 e4m3x8(const uint4& v, float inv) {
  return make_uint2(e4m3x2<HAS_INF>(v.x, inv, inv) | (e4m3x2<HAS_INF>(v.y, inv, inv) << 16),
                    e4m3x2<HAS_INF>(v.z, inv, inv) | (e4m3x2<HAS_INF>(v.w, inv, inv) << 16));
}

}  // namespace blkq
}  // namespace ocb
