// e4m3 GEMM for sm_100a whose operands carry one fp32 scale per block of 128 reduction elements:
//
//   C[m, n] (=|+=) sum_kb  sa(kb, m) * sb(kb, n) * sum_{k in block kb}  A[m, k] * B[n, k]
//
// The scales change along the reduction, so the tensor core only ever accumulates ONE block (128 elements, four K = 32
// instructions) into tensor memory; the epilogue warps read that partial tile back and add it, multiplied by its scales,
// to fp32 accumulators in registers ("promotion"). The sums over the blocks are therefore plain fp32 additions.
//
// Both operands are addressed in place, whatever their orientation: a K-major operand (reduction contiguous) arrives as
// [128 rows x 128 bytes] boxes, an MN-major one (rows of the product contiguous) as [128 k x 128 bytes] boxes, so the input
// gradient reads the forward weight's codes and the weight gradient reads row-major activations without transposed copies.
// Scales are read through strides: per row of an operand (index shift 0) or per 128 rows (shift 7).
//
// CTA layout (384 threads, three warpgroups): warp 0 = TMA producer, warp 1 = MMA issuer and tensor-memory owner, warps 2 and 3
// = scales: they run ahead of the promotion by up to eight blocks and leave each block's factors in a shared-memory ring, so
// that no promotion ever waits for a scale to come from L2; warps 4..11 = promotion and epilogue: four lane quadrants x two column halves, every thread owns
// one row and BN / 2 columns of the tile, held in registers. The first warpgroup hands registers to the other two (72 against
// 2 x 216 of the 3 x 168 at launch). All waits are bounded (common.cuh).

#include "common.cuh"
#include "ocb_api.h"
#include "tmap.h"

namespace ocb {
namespace blk {

constexpr int BM = 128;
constexpr int BKE = 128;  // reduction elements (= bytes) per stage = one scale block
constexpr int A_BYTES = BM * BKE;
constexpr int THREADS = 384;
constexpr int REGS_FEED = 72, REGS_SUM = 216;  // registers a thread after the hand-over: 72 + 2 * 216 = 3 * 168
constexpr int EPI_WARPS = 8;
constexpr int SCALE_SLOTS = 8, SCALE_BATCH = 4;  // ring of factors; blocks whose scales are fetched together
constexpr uint32_t TMEM_COLS = 512;

enum : int { EPI_BF16 = 0, EPI_F32_ACC = 1, EPI_F32 = 2 };

template <int BN>
struct Tile {
  static constexpr int STAGE_BYTES = A_BYTES + BN * BKE;
  static constexpr int STAGES = BN == 256 ? 4 : 6;
  static constexpr int ACCS = static_cast<int>(TMEM_COLS) / BN;  // partial tiles in flight between the issuer and the epilogue
  static constexpr int COLS = BN / 2;                            // columns per epilogue thread
  // a block's factors: per row and column half (sa * sb), or sa per row and sb per column
  static constexpr int FACTORS = BM + BN;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + SCALE_SLOTS * FACTORS * 4 + 1024 /*alignment slack*/ + 512 /*barriers*/;
};

struct Scales {
  const float* p;
  long long k_stride, i_stride, group_stride;  // floats between reduction blocks / rows (>> shift) / groups
  int shift;                                   // 0: one scale per row of the operand, 7: one per 128 rows
};

struct Params {
  void* C;
  long long ldc;
  int M, N, K;
  int group_m;  // rasterisation: row tiles that share a column tile while it is in L2
  int a_mn, b_mn;
  Scales sa, sb;
  const int* offsets;  // [num_groups + 1] row boundaries of the groups, or null: one product
  int num_groups;
  int* status;
};

struct TileInfo {
  int m0, m_end, n0, g;
};

struct Walker {
  const Params& p;
  int bn, tiles_m, tiles_n, tile, g, base;
  __device__ Walker(const Params& params, int bn_) : p(params), bn(bn_), g(0), base(0) {
    tiles_m = (p.M + BM - 1) / BM;
    tiles_n = (p.N + bn - 1) / bn;
    tile = blockIdx.x;
  }
  __device__ bool next(TileInfo& t) {
    if (p.offsets == nullptr) {
      if (tile >= tiles_m * tiles_n) return false;
      const int per_group = p.group_m * tiles_n;
      const int grp = tile / per_group, first_m = grp * p.group_m;
      const int gm = min(tiles_m - first_m, p.group_m);
      const int r = tile - grp * per_group;
      t.m0 = (first_m + r % gm) * BM;
      t.m_end = p.M;
      t.n0 = (r / gm) * bn;
      t.g = 0;
    } else {
      int lo, rows, tm_g;
      while (true) {
        if (g >= p.num_groups) return false;
        lo = min(max(p.offsets[g], 0), p.M);  // whatever the boundaries hold, no row outside the matrix is touched
        rows = max(min(p.offsets[g + 1], p.M) - lo, 0);
        tm_g = (rows + BM - 1) / BM;
        if (tile < base + tm_g * tiles_n) break;
        base += tm_g * tiles_n;
        ++g;
      }
      const int local = tile - base;
      t.m0 = lo + (local % tm_g) * BM;
      t.m_end = lo + rows;
      t.n0 = (local / tm_g) * bn;
      t.g = g;
    }
    tile += gridDim.x;
    return true;
  }
};

// Waits for the tensor-memory loads issued so far. The registers pass through, so that nothing that reads them can be
// scheduled ahead of the wait.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// 32 consecutive columns of one row; v holds 16 packed pairs.
template <int EPI>
__device__ __forceinline__ void store_chunk(const Params& p, long long row, int col, const uint64_t* v) {
  float f[32];
#pragma unroll
  for (int j = 0; j < 16; ++j) unpack_f32x2(v[j], f[2 * j], f[2 * j + 1]);
  if (EPI == EPI_BF16) {
    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.C) + row * p.ldc + col;
    if (col + 32 <= p.N && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint4 o;
        o.x = pack_bf16x2(f[8 * q + 0], f[8 * q + 1]);
        o.y = pack_bf16x2(f[8 * q + 2], f[8 * q + 3]);
        o.z = pack_bf16x2(f[8 * q + 4], f[8 * q + 5]);
        o.w = pack_bf16x2(f[8 * q + 6], f[8 * q + 7]);
        reinterpret_cast<uint4*>(dst)[q] = o;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col + j < p.N) dst[j] = __float2bfloat16_rn(f[j]);
    }
  } else {
    float* dst = reinterpret_cast<float*>(p.C) + row * p.ldc + col;
    if (col + 32 <= p.N && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float4 o = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
        if (EPI == EPI_F32_ACC) {
          const float4 old = reinterpret_cast<const float4*>(dst)[q];
          o.x += old.x; o.y += old.y; o.z += old.z; o.w += old.w;
        }
        reinterpret_cast<float4*>(dst)[q] = o;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col + j < p.N) dst[j] = EPI == EPI_F32_ACC ? dst[j] + f[j] : f[j];
    }
  }
}

// BCOL: the scales of B differ from row to row of B (= output column); otherwise B has one scale per 128 of its rows, which
// is one number for everything a thread owns.
template <int BN, bool BCOL, int EPI>
__global__ void __launch_bounds__(THREADS, 1)
gemm_block_fp8_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, const Params p) {
  using T = Tile<BN>;
  constexpr int STAGES = T::STAGES, ACCS = T::ACCS, COLS = T::COLS, STAGE_BYTES = T::STAGE_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* factors = reinterpret_cast<float*>(smem + STAGES * STAGE_BYTES);  // [SCALE_SLOTS][FACTORS]
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(factors + SCALE_SLOTS * T::FACTORS);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + ACCS;
  uint64_t* sfull_bar = tempty_bar + ACCS;
  uint64_t* sempty_bar = sfull_bar + SCALE_SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sempty_bar + SCALE_SLOTS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int num_kb = (p.K + BKE - 1) / BKE;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < ACCS; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], EPI_WARPS);
    }
    for (int i = 0; i < SCALE_SLOTS; ++i) {
      mbar_init(&sfull_bar[i], 2);
      mbar_init(&sempty_bar[i], EPI_WARPS);
    }
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tma_a);
    tma_prefetch_desc(&tma_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEED));
  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      Walker walker(p, BN);
      TileInfo t;
      while (ok && walker.next(t)) {
        for (int kb = 0; kb < num_kb; ++kb) {
          ok = mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer);
          if (!ok) break;
          uint8_t* sa = smem + stage * STAGE_BYTES;
          uint8_t* sb = sa + A_BYTES;
          const int k0 = kb * BKE;
          mbar_arrive_expect_tx(&full_bar[stage], STAGE_BYTES);
          // innermost coordinates are k0 (K-major) or tile origins (MN-major): multiples of 128 bytes either way; group
          // boundaries only enter the outer coordinate of a K-major A
          if (p.a_mn) tma_load_2d(sa, &tma_a, &full_bar[stage], t.m0, k0);
          else tma_load_2d(sa, &tma_a, &full_bar[stage], k0, t.m0);
          if (p.b_mn) {
#pragma unroll
            for (int j = 0; j < BN / 128; ++j)
              tma_load_3d(sb + j * (128 * BKE), &tma_b, &full_bar[stage], t.n0 + j * 128, k0, t.g);
          } else {
            tma_load_3d(sb, &tma_b, &full_bar[stage], k0, t.n0, t.g);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // let copies in flight land before shared memory goes away
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ issuer
    if (lane == 0) {
      // K-major: 8-row swizzle atoms 1024 bytes apart, K = 32 advances 32 bytes along the line. MN-major: 128-column boxes
      // 16 KB apart (leading offset), 8 k-rows per 1024 bytes, K = 32 advances 32 lines.
      constexpr uint32_t kDescHi = desc_hi_sw128(1024);
      const uint32_t idesc = make_idesc_e4m3(BM, BN) | (static_cast<uint32_t>(p.a_mn) << 15) | (static_cast<uint32_t>(p.b_mn) << 16);
      const uint32_t a_step = p.a_mn ? 256u : 2u, b_step = p.b_mn ? 256u : 2u;
      const uint32_t a_lo0 = desc_lo_sw128(smem_u32(smem), 16);
      const uint32_t b_lo0 = desc_lo_sw128(smem_u32(smem) + A_BYTES, p.b_mn ? 128 * BKE : 16);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      Walker walker(p, BN);
      TileInfo t;
      while (ok && walker.next(t)) {
        for (int kb = 0; kb < num_kb; ++kb) {
          ok = mbar_wait_bounded(&tempty_bar[acc], acc_phase ^ 1u, abort_flag, p.status, kStatusTimeoutMma) &&
               mbar_wait_bounded(&full_bar[stage], phase, abort_flag, p.status, kStatusTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * BN;
          const uint32_t a_lo = a_lo0 + stage * (STAGE_BYTES >> 4), b_lo = b_lo0 + stage * (STAGE_BYTES >> 4);
#pragma unroll
          for (uint32_t k = 0; k < BKE / 32; ++k)
            umma_ss_lean<1>(d_tmem, a_lo + k * a_step, b_lo + k * b_step, kDescHi, idesc, k != 0);
          umma_commit(&empty_bar[stage]);
          umma_commit(&tfull_bar[acc]);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          if (++acc == ACCS) { acc = 0; acc_phase ^= 1u; }
        }
      }
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------------ scales (warps 2 and 3)
    const int t64 = threadIdx.x - 64;
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    Walker walker(p, BN);
    TileInfo t;
    constexpr int PER = BCOL ? T::FACTORS / 64 : BM / 64;  // scales a thread fetches per block (and, without BCOL, two of B)
    while (ok && walker.next(t)) {
      const float* src[PER];
      long long step[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {  // factor t64 + 64 i: a row of A, or a column
        const int f = t64 + 64 * i;
        const bool is_a = i < BM / 64;
        const int at = is_a ? t.m0 + f : t.n0 + f - BM;
        const Scales& sc = is_a ? p.sa : p.sb;
        step[i] = sc.k_stride;
        src[i] = at < (is_a ? t.m_end : p.N) ? sc.p + (is_a ? 0 : t.g * sc.group_stride) + static_cast<long long>(at >> sc.shift) * sc.i_stride
                                             : nullptr;
      }
      const float* tile[2] = {nullptr, nullptr};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int col = t.n0 + h * COLS;
        if (!BCOL && col < p.N) tile[h] = p.sb.p + t.g * p.sb.group_stride + static_cast<long long>(col >> p.sb.shift) * p.sb.i_stride;
      }
      for (int kb0 = 0; ok && kb0 < num_kb; kb0 += SCALE_BATCH) {
        float v[SCALE_BATCH][PER], w[SCALE_BATCH][2];
#pragma unroll
        for (int b = 0; b < SCALE_BATCH; ++b) {
          const bool live = kb0 + b < num_kb;
#pragma unroll
          for (int i = 0; i < PER; ++i) v[b][i] = live && src[i] != nullptr ? __ldg(src[i] + (kb0 + b) * step[i]) : 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h) w[b][h] = live && tile[h] != nullptr ? __ldg(tile[h] + (kb0 + b) * p.sb.k_stride) : 0.f;
        }
#pragma unroll
        for (int b = 0; b < SCALE_BATCH; ++b) {
          if (kb0 + b >= num_kb) break;
          ok = mbar_wait_bounded(&sempty_bar[slot], phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          float* dst = factors + slot * T::FACTORS;
          if (BCOL) {
#pragma unroll
            for (int i = 0; i < PER; ++i) dst[t64 + 64 * i] = v[b][i];
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < PER; ++i) dst[h * BM + t64 + 64 * i] = v[b][i] * w[b][h];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sfull_bar[slot]);
          if (++slot == SCALE_SLOTS) { slot = 0; phase ^= 1u; }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ promotion and epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SUM));
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + half * COLS;
    // where this thread's factor sits in a slot, and where the column factors of its half start
    const float* my_factor = factors + (BCOL ? 0 : half * BM) + quad * 32 + lane;
    const float* col_factors = factors + BM + half * COLS;
    int acc = 0, slot = 0;
    uint32_t acc_phase = 0, slot_phase = 0;
    bool ok = true;
    Walker walker(p, BN);
    TileInfo t;
    while (ok && walker.next(t)) {
      uint64_t sum[COLS / 2];
#pragma unroll
      for (int j = 0; j < COLS / 2; ++j) sum[j] = 0ull;
      for (int kb = 0; kb < num_kb; ++kb) {
        ok = mbar_wait_bounded(&sfull_bar[slot], slot_phase, abort_flag, p.status, kStatusTimeoutEpilogue) &&
             mbar_wait_bounded(&tfull_bar[acc], acc_phase, abort_flag, p.status, kStatusTimeoutEpilogue);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_acc = t_row + acc * BN;
        uint32_t r[2][16];
        tmem_ld_32x16(t_acc, r[0]);
        const float s = my_factor[slot * T::FACTORS];
        const uint64_t s2 = pack_f32x2(s, s);
        const float* cf = col_factors + slot * T::FACTORS;
        tmem_ld_wait_for(r[0]);
#pragma unroll
        for (int c = 0; c < COLS / 16; ++c) {
          if (c + 1 < COLS / 16) {
            tmem_ld_32x16(t_acc + (c + 1) * 16, r[(c + 1) & 1]);
          } else {
            tc_fence_before();
            if (lane == 0) mbar_arrive(&tempty_bar[acc]);
          }
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            uint64_t f0 = s2, f1 = s2;
            if (BCOL) {
              const float4 col = *reinterpret_cast<const float4*>(cf + c * 16 + 2 * j);
              f0 = mul_f32x2(s2, pack_f32x2(col.x, col.y));
              f1 = mul_f32x2(s2, pack_f32x2(col.z, col.w));
            }
            sum[c * 8 + j] = fma_f32x2(pack_u32x2(r[c & 1][2 * j], r[c & 1][2 * j + 1]), f0, sum[c * 8 + j]);
            sum[c * 8 + j + 1] = fma_f32x2(pack_u32x2(r[c & 1][2 * j + 2], r[c & 1][2 * j + 3]), f1, sum[c * 8 + j + 1]);
          }
          if (c + 1 < COLS / 16) tmem_ld_wait_for(r[(c + 1) & 1]);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sempty_bar[slot]);
        if (++acc == ACCS) { acc = 0; acc_phase ^= 1u; }
        if (++slot == SCALE_SLOTS) { slot = 0; slot_phase ^= 1u; }
      }
      const int row = t.m0 + quad * 32 + lane, col0 = t.n0 + half * COLS;
      if (ok && row < t.m_end) {
#pragma unroll
        for (int c = 0; c < COLS / 32; ++c)
          if (col0 + c * 32 < p.N) store_chunk<EPI>(p, row, col0 + c * 32, sum + c * 16);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

static int num_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n;
}

template <int BN, bool BCOL, int EPI>
static int launch(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, long long max_tiles, cudaStream_t stream) {
  constexpr int bytes = Tile<BN>::SMEM_BYTES;
  if (cudaFuncSetAttribute(gemm_block_fp8_kernel<BN, BCOL, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return -3;
  const int sms = num_sms();
  if (sms <= 0) return -3;
  const int grid = max_tiles < sms ? static_cast<int>(max_tiles) : sms;
  gemm_block_fp8_kernel<BN, BCOL, EPI><<<grid, THREADS, bytes, stream>>>(ta, tb, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -4;
}

template <int BN, bool BCOL>
static int launch_epi(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, long long max_tiles, int epi, cudaStream_t s) {
  switch (epi) {
    case EPI_BF16: return launch<BN, BCOL, EPI_BF16>(ta, tb, p, max_tiles, s);
    case EPI_F32_ACC: return launch<BN, BCOL, EPI_F32_ACC>(ta, tb, p, max_tiles, s);
    case EPI_F32: return launch<BN, BCOL, EPI_F32>(ta, tb, p, max_tiles, s);
    default: return -1;
  }
}

static bool make_map(CUtensorMap* out, const void* ptr, bool mn, uint64_t rows, uint64_t k, uint64_t groups, long long ld,
                     long long group_bytes, int box_rows, int rank) {
  const uint64_t dims[3] = {mn ? rows : k, mn ? k : rows, groups};
  const uint64_t str[2] = {static_cast<uint64_t>(ld), static_cast<uint64_t>(group_bytes)};
  const uint32_t box[3] = {128, static_cast<uint32_t>(mn ? BKE : box_rows), 1};
  return encode_tensor_map(out, ptr, rank, dims, str, box, 1);
}

}  // namespace blk
}  // namespace ocb

using namespace ocb;

// See ocb_api.h.
extern "C" int ocb_gemm_block_fp8(const void* A, const void* B, void* C, const float* sa, const float* sb, const int* offsets,
                                  int num_groups, int M, int N, int K, long long lda, long long ldb, long long ldc,
                                  long long b_group_bytes, long long sa_k, long long sa_i, int sa_shift, long long sb_k,
                                  long long sb_i, long long sb_g, int sb_shift, int a_mn, int b_mn, int epilogue, int* status,
                                  cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || num_groups <= 0) return 0;
  if ((lda % 16) != 0 || (ldb % 16) != 0 || (b_group_bytes % 16) != 0 || (reinterpret_cast<uintptr_t>(A) & 15) ||
      (reinterpret_cast<uintptr_t>(B) & 15) || sa == nullptr || sb == nullptr)
    return -1;
  if ((sa_shift != 0 && sa_shift != 7) || (sb_shift != 0 && sb_shift != 7) || (offsets != nullptr && a_mn)) return -1;
  blk::Params p;
  p.C = C;
  p.ldc = ldc;
  p.M = M;
  p.N = N;
  p.K = K;
  p.group_m = 8;
  p.a_mn = a_mn;
  p.b_mn = b_mn;
  p.sa = {sa, sa_k, sa_i, 0, sa_shift};
  p.sb = {sb, sb_k, sb_i, sb_g, sb_shift};
  p.offsets = offsets;
  p.num_groups = num_groups;
  p.status = status;
  const int bn = 256;
  CUtensorMap ta, tb;
  if (!blk::make_map(&ta, A, a_mn != 0, M, K, 1, lda, 0, blk::BM, 2)) return -1001;
  if (!blk::make_map(&tb, B, b_mn != 0, N, K, num_groups, ldb, num_groups > 1 ? b_group_bytes : ldb, bn, 3)) return -2001;
  const long long tiles_n = (N + bn - 1) / bn;
  const long long tiles_m = (M + blk::BM - 1) / blk::BM + (offsets != nullptr ? num_groups : 0);
  const long long tiles = tiles_m * tiles_n;
  return sb_shift == 0 ? blk::launch_epi<256, true>(ta, tb, p, tiles, epilogue, stream)
                       : blk::launch_epi<256, false>(ta, tb, p, tiles, epilogue, stream);
}
