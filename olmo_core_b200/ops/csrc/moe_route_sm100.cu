// Routing of tokens to experts, forward and gradient.
//
//   s = softmax(x) or sigmoid(x) + 1e-7       scores [E] of a token with logits x
//   r = s + bias                              what is ranked (bias: balances the load, no part of the weights)
//   value of a group of experts = sum of its two largest r; the `top_groups` best groups stay open
//   chosen = the k largest r of the open groups, the lower id first where two are equal
//   w = s[chosen], divided by its sum (normalize 1) or 2-norm (normalize 2), 0 where they are all below 2^-120;
//   counts = tokens per expert
//
// One warp per token, expert e in register e / 32 of lane e % 32: a row is read and its scores are written once, everything
// between stays in registers (and, for the groups, one row of shared memory). Tokens per expert are counted in shared memory, so
// that global atomics number one per expert and CTA.
//
// What bounds it: latency for few tokens (one: 2.6 us, 11.8 with the host), the issue of instructions for many, about 500 a token with 64
// experts and 1700 with bias and groups of 256: each of the k choices is a reduction over the whole warp for one token. 32768 tokens of
// 64 experts: 33 us (448 GB/s), of 256 in 8 groups: 88 us (798 GB/s). The gradient of 16384 x 64 takes 5.3 us, of 8191 x 256 9 us.
// Several tokens a warp, with reductions over 4 to 16 lanes, would share those instructions; that form is not built.
//
// Which experts are chosen is what exact arithmetic says, although scores are fp32: without bias and groups the ranking of the
// logits themselves decides; otherwise a token whose ranking hangs on a difference within the fp32 error (about one in a
// hundred) is ranked again in fp64.
//
// A row without any logit above -inf has scores and weights of zero. NaN ranks above every number.

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ocb_api.h"

namespace ocb {
namespace route {

constexpr unsigned FULL = 0xffffffffu;
constexpr float SIGMOID_FLOOR = 1e-7f;
// Bounds on the absolute error of an fp32 score (all are <= 1), at least twice what the operations can add up to. Softmax: a sum of
// up to 1024 terms (37 roundings on the longest path), exponentials (two steps of 2^-23) and the reciprocal: below 43 2^-24.
// Sigmoid: s (1 - s) times the exponential's relative error, and three roundings: 2^-22. The exponential is expf, not the fast one,
// whose relative error grows with |x|: small sigmoid scores, and weights made from them, would be off by |x| steps.
constexpr float SOFTMAX_ERROR = 3.8e-6f;  // 2^-18
constexpr float SIGMOID_ERROR = 4.8e-7f;  // 2^-21

struct Params {
  const void* logits;
  float* scores;       // [n][E] or null
  float* weights;      // [n][k]
  long long* experts;  // [n][k]
  int* counts;         // [E]
  const float* bias;   // [E] or null
  int n_tokens, n_experts, top_k, sigmoid, normalize, n_groups, top_groups, bf16;
  long long ld;
};

__device__ __forceinline__ float load(const void* p, long long i, int bf16) {
  return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}

// Order-preserving integer keys. 0 is below every number (even -inf) and means "not to be chosen"; NaN is the largest. The addition
// makes a positive zero of a negative one: the two are equal.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __float_as_uint(__fadd_rn(v, 0.f));
  return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long key_of(double v) {
  const unsigned long long b = __double_as_longlong(__dadd_rn(v, 0.0));
  return v != v ? ~0ull : (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(FULL, v); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
  const uint32_t hi = static_cast<uint32_t>(v >> 32);
  const uint32_t top = __reduce_max_sync(FULL, hi);
  const uint32_t low = __reduce_max_sync(FULL, hi == top ? static_cast<uint32_t>(v) : 0u);
  return (static_cast<unsigned long long>(top) << 32) | low;
}
__device__ __forceinline__ float sum_warp(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ double sum_warp(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}

// The power of two that brings the largest of a warp's scores into [1, 2), so that squares of small ones do not vanish; 0 where
// all are below 2^-120: such a norm counts as zero, because its reciprocal leaves fp32.
__device__ __forceinline__ float norm_scale(float w) {
  const uint32_t e = __reduce_max_sync(FULL, __float_as_uint(w)) >> 23;  // scores are not negative
  return e < 7u ? 0.f : __uint_as_float((254u - e) << 23);
}

// Whether two fp32 rankings as close as `hi` and `lo` may be the other way round in exact arithmetic. NaN counts as close.
__device__ __forceinline__ bool too_close(float hi, float lo, float error) {
  return !(hi - lo > 2.f * error + 2.4e-7f * fabsf(hi));
}

// The k largest keys in falling order, lower expert first among equal ones: lane j gets the j-th. With `check`, also says
// whether neighbours in that order (the first one left out included) are too close to be told apart.
template <int PL, class Key>
__device__ __forceinline__ bool pick(Key (&key)[PL], int top_k, int lane, bool check, float error, int& mine) {
  bool close = false;
  float before = 0.f;
  const int rounds = top_k + (check ? 1 : 0);
  for (int j = 0; j < rounds; ++j) {
    Key best = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < PL; ++i)
      if (key[i] > best) { best = key[i]; at = i; }
    const Key top = warp_max(best);
    if (top == 0) break;
    const uint32_t e = __reduce_min_sync(FULL, best == top ? static_cast<uint32_t>(at * 32 + lane) : 0xffffffffu);
    if (check) {
      const float v = value_of(static_cast<uint32_t>(top));
      if (j > 0) close |= too_close(before, v, error);
      before = v;
    }
    if (j < top_k && lane == j) mine = static_cast<int>(e);
#pragma unroll
    for (int i = 0; i < PL; ++i) key[i] = e == static_cast<uint32_t>(i * 32 + lane) ? static_cast<Key>(0) : key[i];
  }
  return close;
}

// Bit (first lane of a group) of the open groups. row: the ranked values of the token in shared memory. `close` as in pick().
template <class Real>
__device__ __forceinline__ uint32_t open_groups(const Real* row, const Params& p, int lane, int lanes_per_group, bool check,
                                                float error, bool& close) {
  const int size = p.n_experts / p.n_groups;
  const int g = lane / lanes_per_group, sub = lane % lanes_per_group;
  const bool valid = g < p.n_groups;
  Real a = -INFINITY, b = -INFINITY;
  bool nan = false;
  if (valid) {
    for (int j = sub; j < size; j += lanes_per_group) {
      const Real v = row[g * size + j];
      nan |= v != v;
      if (v > a) { b = a; a = v; } else if (v > b) { b = v; }
    }
  }
  for (int o = lanes_per_group >> 1; o; o >>= 1) {
    const Real oa = __shfl_xor_sync(FULL, a, o), ob = __shfl_xor_sync(FULL, b, o);
    nan |= __shfl_xor_sync(FULL, static_cast<int>(nan), o) != 0;
    const Real low = oa < a ? oa : a, high = oa < a ? a : oa;
    b = b > ob ? b : ob;
    b = b > low ? b : low;
    a = high;
  }
  const Real value = nan ? static_cast<Real>(NAN) : size > 1 ? a + b : a;
  const auto key = key_of(value);
  int ahead = 0;
  for (int o = 0; o < p.n_groups; ++o) {
    const auto other = __shfl_sync(FULL, key, o * lanes_per_group);
    ahead += other > key || (other == key && o < g);
  }
  const bool open = valid && ahead < p.top_groups;
  if (check && p.top_groups < p.n_groups) {
    const uint32_t k32 = key_of(static_cast<float>(value));
    const uint32_t least_open = __reduce_min_sync(FULL, open ? k32 : 0xffffffffu);
    const uint32_t best_shut = __reduce_max_sync(FULL, valid && !open ? k32 : 0u);
    close |= too_close(value_of(least_open), value_of(best_shut), 2.f * error);
  }
  return __ballot_sync(FULL, open && sub == 0);
}

template <int PL, bool GROUPS>
__global__ void route_kernel(const Params p, int lanes_per_group, int alone) {
  extern __shared__ double shared[];
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double* row = shared + (GROUPS ? static_cast<long long>(warp) * p.n_experts : 0);
  int* hist = reinterpret_cast<int*>(shared + (GROUPS ? static_cast<long long>(warps) * p.n_experts : 0));
  for (int e = threadIdx.x; e < p.n_experts; e += blockDim.x) hist[e] = 0;
  __syncthreads();

  int first_lane[PL];  // of the expert's group
  if (GROUPS) {
    const int size = p.n_experts / p.n_groups;
#pragma unroll
    for (int i = 0; i < PL; ++i) first_lane[i] = min((i * 32 + lane) / size, 31 / lanes_per_group) * lanes_per_group;
  }
  const bool by_logits = p.bias == nullptr;  // the ranking of the logits is the ranking of the scores

  const float error = p.sigmoid ? SIGMOID_ERROR : SOFTMAX_ERROR;
  float bias[PL];
#pragma unroll
  for (int i = 0; i < PL; ++i) bias[i] = p.bias != nullptr && i * 32 + lane < p.n_experts ? p.bias[i * 32 + lane] : 0.f;

  const long long stride = static_cast<long long>(gridDim.x) * warps;
  float next[PL];  // the next token's logits are on their way while this one is ranked
  auto fetch = [&](long long t) {
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      const int e = i * 32 + lane;
      next[i] = t < p.n_tokens && e < p.n_experts ? load(p.logits, t * p.ld + e, p.bf16) : -INFINITY;
    }
  };
  long long t = static_cast<long long>(blockIdx.x) * warps + warp;
  fetch(t);
  for (; t < p.n_tokens; t += stride) {
    float x[PL], s[PL];
    float top = -INFINITY;
    bool any = false;  // softmax: a logit above -inf, or NaN
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      x[i] = next[i];
      top = fmaxf(top, x[i]);
    }
    fetch(t + stride);
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < PL; ++i) s[i] = 1.f / (1.f + expf(-x[i])) + SIGMOID_FLOOR;
    } else {
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        s[i] = (i * 32 + lane) < p.n_experts ? expf(x[i] - top) : 0.f;
        sum += s[i];
      }
      const float inv = 1.f / sum_warp(sum);
      // NaN logits do not take part in the maximum: beside -inf alone they leave it at -inf, with a sum of NaN
#pragma unroll
      for (int i = 0; i < PL; ++i) any |= (i * 32 + lane) < p.n_experts && !(x[i] == -INFINITY);
      any = __any_sync(FULL, any);
#pragma unroll
      for (int i = 0; i < PL; ++i) s[i] = any ? s[i] * inv : 0.f;
    }
    if (p.scores != nullptr) {
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        const int e = i * 32 + lane;
        if (e < p.n_experts) p.scores[t * p.n_experts + e] = s[i];
      }
    }

    uint32_t key[PL];
    bool close = false;
    uint32_t open = FULL;
    {
      float r[PL];
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        r[i] = s[i] + bias[i];
      }
      if (GROUPS) {
        float* row32 = reinterpret_cast<float*>(row);
#pragma unroll
        for (int i = 0; i < PL; ++i)
          if (i * 32 + lane < p.n_experts) row32[i * 32 + lane] = r[i];
        __syncwarp();
        open = open_groups(row32, p, lane, lanes_per_group, true, error, close);
        __syncwarp();
      }
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        const bool in = i * 32 + lane < p.n_experts && (!GROUPS || (open >> first_lane[i]) & 1u);
        key[i] = in ? key_of(by_logits ? x[i] : r[i]) : 0u;
      }
    }
    int mine = 0;
    close |= pick(key, p.top_k, lane, !by_logits, error, mine);
    if (close) {
      double d[PL];
      if (p.sigmoid) {
#pragma unroll
        for (int i = 0; i < PL; ++i) d[i] = 1.0 / (1.0 + exp(-static_cast<double>(x[i]))) + 1e-7;
      } else {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < PL; ++i) {
          d[i] = (i * 32 + lane) < p.n_experts ? exp(static_cast<double>(x[i]) - static_cast<double>(top)) : 0.0;
          sum += d[i];
        }
        sum = sum_warp(sum);
#pragma unroll
        for (int i = 0; i < PL; ++i) d[i] = any ? d[i] / sum : 0.0;
      }
      if (p.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < PL; ++i) d[i] += static_cast<double>(bias[i]);
      }
      if (GROUPS) {
#pragma unroll
        for (int i = 0; i < PL; ++i)
          if (i * 32 + lane < p.n_experts) row[i * 32 + lane] = d[i];
        __syncwarp();
        bool unused = false;
        open = open_groups(row, p, lane, lanes_per_group, false, 0.f, unused);
        __syncwarp();
      }
      unsigned long long key64[PL];
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        const bool in = i * 32 + lane < p.n_experts && (!GROUPS || (open >> first_lane[i]) & 1u);
        key64[i] = in ? key_of(by_logits ? static_cast<double>(x[i]) : d[i]) : 0ull;
      }
      pick(key64, p.top_k, lane, false, 0.f, mine);
    }

    // lane j holds the j-th expert; its score sits in another lane's registers
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      const float v = __shfl_sync(FULL, s[i], mine & 31);
      w = (mine & ~31) == i * 32 ? v : w;
    }
    if (lane >= p.top_k) w = 0.f;
    if (p.normalize != 0) {
      const float scale = norm_scale(w), c = w * scale;
      const float total = sum_warp(p.normalize == 1 ? c : c * c);
      const float norm = p.normalize == 1 ? total : sqrtf(total);
      w = scale == 0.f ? 0.f : c / norm;
    }
    if (lane < p.top_k) {
      p.weights[t * p.top_k + lane] = w;
      p.experts[t * p.top_k + lane] = mine;
      atomicAdd(&hist[mine], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.n_experts; e += blockDim.x) {
    if (alone) p.counts[e] = hist[e];
    else if (hist[e] != 0) atomicAdd(&p.counts[e], hist[e]);
  }
}

struct GradParams {
  const float* scores;        // softmax: [n][E]
  const void* logits;         // sigmoid: [n][E], row pitch ld
  const long long* experts;   // [n][k]
  const float* d_weights;     // [n][k] or null
  const float* d_scores;      // [n][E] or null
  void* d_logits;             // [n][E], dtype of the logits
  int n_tokens, n_experts, top_k, sigmoid, normalize, bf16;
  long long ld;
};

// Gradient of a token's logits from those of its weights and scores:
//   d w / d s of the chosen: (g_j - <g, w> w_j^(p-1)) / norm with p the norm's order (1 or 2), or g_j without a norm
//   softmax: s (d - <d, s>);  sigmoid: d p (1 - p)
template <int PL>
__global__ void route_grad_kernel(const GradParams p) {
  const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (long long t = static_cast<long long>(blockIdx.x) * warps + warp; t < p.n_tokens; t += static_cast<long long>(gridDim.x) * warps) {
    float s[PL], d[PL];
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      const int e = i * 32 + lane;
      const bool in = e < p.n_experts;
      s[i] = !in ? 0.f : p.sigmoid ? load(p.logits, t * p.ld + e, p.bf16) : p.scores[t * p.n_experts + e];
      d[i] = in && p.d_scores != nullptr ? p.d_scores[t * p.n_experts + e] : 0.f;
    }
    if (p.d_weights != nullptr) {
      const int mine = lane < p.top_k ? static_cast<int>(p.experts[t * p.top_k + lane]) : 0;
      float g = lane < p.top_k ? p.d_weights[t * p.top_k + lane] : 0.f;
      if (p.normalize != 0) {
        float w = 0.f;
#pragma unroll
        for (int i = 0; i < PL; ++i) {
          const float v = __shfl_sync(FULL, s[i], mine & 31);
          w = (mine & ~31) == i * 32 ? v : w;
        }
        if (p.sigmoid) w = 1.f / (1.f + expf(-w)) + SIGMOID_FLOOR;
        if (lane >= p.top_k) w = 0.f;
        const float scale = norm_scale(w), c = w * scale;
        const float total = sum_warp(p.normalize == 1 ? c : c * c);
        const float norm = p.normalize == 1 ? total : sqrtf(total);
        const float inv = scale == 0.f ? 0.f : 1.f / norm * scale;
        const float along = sum_warp(g * (w * inv));
        g = (g - along * (p.normalize == 1 ? 1.f : w * inv)) * inv;
      }
      for (int j = 0; j < p.top_k; ++j) {
        const int e = __shfl_sync(FULL, mine, j);
        const float v = __shfl_sync(FULL, g, j);
#pragma unroll
        for (int i = 0; i < PL; ++i) d[i] += e == i * 32 + lane ? v : 0.f;
      }
    }
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < PL; ++i) {
        const float z = expf(-fabsf(s[i]));  // p (1 - p) = z / (1 + z)^2, without cancellation
        d[i] *= z / ((1.f + z) * (1.f + z));
      }
    } else {
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < PL; ++i) dot += d[i] * s[i];
      dot = sum_warp(dot);
#pragma unroll
      for (int i = 0; i < PL; ++i) d[i] = s[i] * (d[i] - dot);
    }
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      const int e = i * 32 + lane;
      if (e >= p.n_experts) continue;
      if (p.bf16) reinterpret_cast<__nv_bfloat16*>(p.d_logits)[t * p.n_experts + e] = __float2bfloat16_rn(d[i]);
      else reinterpret_cast<float*>(p.d_logits)[t * p.n_experts + e] = d[i];
    }
  }
}

static int num_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n;
}

static int launch_ok() { return cudaGetLastError() == cudaSuccess ? 0 : -4; }

static int check(int n_experts, int top_k, int normalize) {
  return n_experts > 0 && n_experts <= 1024 && top_k > 0 && top_k <= 32 && top_k <= n_experts && normalize >= 0 && normalize <= 2;
}

}  // namespace route
}  // namespace ocb

using namespace ocb;

#define OCB_PER_LANE(E, CALL)                                                                                            \
  do {                                                                                                                   \
    if ((E) <= 32) { constexpr int PL = 1; CALL; } else if ((E) <= 64) { constexpr int PL = 2; CALL; }                   \
    else if ((E) <= 128) { constexpr int PL = 4; CALL; } else if ((E) <= 256) { constexpr int PL = 8; CALL; }            \
    else if ((E) <= 512) { constexpr int PL = 16; CALL; } else { constexpr int PL = 32; CALL; }                          \
  } while (0)

// See ocb_api.h.
extern "C" int ocb_moe_route(const void* logits, float* scores, float* weights, long long* experts, int* counts,
                             const float* bias, int n_tokens, int n_experts, int top_k, int sigmoid, int normalize,
                             int n_groups, int top_groups, long long ld, int act_dtype, cudaStream_t stream) {
  if (!route::check(n_experts, top_k, normalize) || n_groups < 1 || n_groups > 32 || n_experts % n_groups != 0 ||
      top_groups < 1 || top_groups > n_groups || top_k > top_groups * (n_experts / n_groups) || counts == nullptr)
    return -1;
  if (n_tokens <= 0) return cudaMemsetAsync(counts, 0, sizeof(int) * n_experts, stream) == cudaSuccess ? 0 : -4;
  route::Params p{logits, scores, weights, experts, counts, bias, n_tokens, n_experts, top_k, sigmoid, normalize, n_groups,
                  top_groups, act_dtype == OCB_BF16, ld};
  const int sms = route::num_sms();
  if (sms <= 0) return -3;
  int lanes_per_group = 32;
  while (lanes_per_group * n_groups > 32) lanes_per_group >>= 1;
  const bool groups = n_groups > 1;
  // Large CTAs and few of them, because a CTA adds its counts to the global ones once. Few tokens: a token per warp of smaller CTAs.
  // The registers (48 a thread with 64 experts, 117 with 256 in groups) let two and one of the three and two per SM run together;
  // the others follow.
  const int warps = n_experts > 512 ? 4 : n_experts > 256 || n_tokens <= 8 ? 8 : 16;
  const long long wanted = (static_cast<long long>(n_tokens) + warps - 1) / warps;
  const long long most = static_cast<long long>(sms) * (n_experts > 128 ? 2 : 3);
  const int grid = static_cast<int>(wanted < most ? wanted : most);
  const size_t bytes = (groups ? sizeof(double) * warps * n_experts : 0) + sizeof(int) * n_experts;
  if (grid > 1 && cudaMemsetAsync(counts, 0, sizeof(int) * n_experts, stream) != cudaSuccess) return -4;
  if (groups) OCB_PER_LANE(n_experts, (route::route_kernel<PL, true><<<grid, warps * 32, bytes, stream>>>(p, lanes_per_group, grid == 1)));
  else OCB_PER_LANE(n_experts, (route::route_kernel<PL, false><<<grid, warps * 32, bytes, stream>>>(p, lanes_per_group, grid == 1)));
  return route::launch_ok();
}

extern "C" int ocb_moe_route_grad(const float* scores, const void* logits, const long long* experts, const float* d_weights,
                                  const float* d_scores, void* d_logits, int n_tokens, int n_experts, int top_k, int sigmoid,
                                  int normalize, long long ld, int act_dtype, cudaStream_t stream) {
  if (!route::check(n_experts, top_k, normalize) || (sigmoid ? logits == nullptr : scores == nullptr)) return -1;
  if (n_tokens <= 0) return 0;
  route::GradParams p{scores, logits, experts, d_weights, d_scores, d_logits, n_tokens, n_experts, top_k, sigmoid, normalize,
                      act_dtype == OCB_BF16, ld};
  const int sms = route::num_sms();
  if (sms <= 0) return -3;
  const int warps = 8;
  const long long wanted = (static_cast<long long>(n_tokens) + warps - 1) / warps;
  const int grid = static_cast<int>(wanted < sms * 8ll ? wanted : sms * 8ll);
  OCB_PER_LANE(n_experts, (route::route_grad_kernel<PL><<<grid, warps * 32, 0, stream>>>(p)));
  return route::launch_ok();
}
