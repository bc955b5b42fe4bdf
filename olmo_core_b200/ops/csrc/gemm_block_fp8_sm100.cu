// e4m3 GEMM for sm_100a whose operands carry one power-of-two scale per block of 128 reduction elements:
//
//   C[m, n] (=|+=) sum_kb  sa(kb, m) * sb(kb, n) * sum_{k in block kb}  A[m, k] * B[n, k]
//
// The scales are applied by the tensor core (tcgen05.mma.kind::mxf8f6f4.block_scale), and the accumulator in tensor memory runs
// through the whole reduction in fp32. The instruction takes one E8M0 exponent per row and K = 32 step, a byte of a 32-bit word
// per row in tensor memory that it selects; all four steps of a block select the same byte here, so one word, and one set of
// copies into tensor memory, serves four blocks. Adding scaled partial sums in registers instead, which would allow scales of any value, was measured
// first: every block has to be read back from tensor memory, and 8192 x 11008 x 4096 took 403 us (625 us with a scale per
// column of B). This form takes 250 to 256 us, 2890 to 2960 TFLOP/s and 1.75 to 1.79 of the bf16 rate of cuBLAS, the input gradient 244 to
// 250, and the weight gradient 258 to 260. A block of a 256 x 256 tile takes 617 cycles; the instructions alone need 512, and so does shared memory (32 KB in
// and 32 KB out per SM at 128 B a cycle), which the result's way through it, 0.6 us a tile, delays further. In longer runs the power limit
// binds: 280 us at the 1.39 GHz that it leaves. Storing the result by TMA gained 3 % at K = 1024 and nothing at 4096.
//
// Both operands are addressed in place, whatever their orientation: a K-major operand (reduction contiguous) arrives as
// [rows x 128 bytes] boxes, an MN-major one (rows of the product contiguous) as [128 k x 128 bytes] boxes, so the input
// gradient reads the forward weight's codes and the weight gradient reads row-major activations without transposed copies.
// Scales are fp32 and read through strides, per row of an operand (index shift 0) or per 128 rows (shift 7); one that is no
// positive power of two becomes NaN.
//
// Two kernels: pairs of CTAs on 256 x 256 tiles for whatever fills the machine, and one CTA per 128-row tile (further down) for few
// tokens and for products of few tiles. Roles of the pair kernel's 384 threads: warp 0 = TMA producer, warp 1 = MMA issuer and
// tensor-memory owner, warps 2 and 3 = scales (they fetch those of four blocks at a time, run up to twelve blocks ahead, and lay
// the exponents out as the tensor core wants them), warps 4..11 = epilogue (four lane quadrants x two column halves; through
// shared memory, so that global accesses are whole 128-byte lines). Waits on barriers in shared memory are bounded (common.cuh).

#include <atomic>
#include <cmath>

#include "block_quant.cuh"
#include "common.cuh"
#include "ocb_api.h"
#include "tmap.h"

namespace ocb {
namespace blk {

constexpr int BM = 128;
constexpr int BKE = 128;  // reduction elements (= bytes) of one scale block
constexpr int KBS = 2;    // blocks per stage: the issuing thread's waits and commits are shared by eight MMAs
constexpr int A_BYTES = BM * BKE;
constexpr int THREADS = 384;
constexpr int EPI_WARPS = 8;
constexpr int SCALE_BATCH = 4;  // blocks whose exponents share a word
constexpr int SCALE_SLOTS = 3;  // batches in shared memory
constexpr uint32_t TMEM_COLS = 512;
constexpr int SF_BLOCK = 512;  // exponents of 128 rows for one batch

enum : int { EPI_BF16 = 0, EPI_F32_ACC = 1, EPI_F32 = 2 };

// A pair of CTAs (cta_group::2) computes a 256 x 256 tile; each stages its own 128 rows of A and half of B, so a block of the
// reduction costs an SM 32 KB of loads for four times the work of a 128 x 128 tile. The accumulator takes 256 columns; a second one
// would leave no room for the scales.
constexpr int CTAS = 2;
constexpr int BN = 256;
constexpr int B_ROWS = BN / CTAS;  // rows of B that one CTA stages
constexpr int KB_BYTES = A_BYTES + B_ROWS * BKE;
constexpr int STAGE_BYTES = KBS * KB_BYTES;  // [block][A rows, B rows]
constexpr int STAGES = 3;
constexpr int SF_BYTES = SF_BLOCK * (1 + BN / 128);
constexpr uint32_t SF_COL = BN;    // two alternating sets of scale columns: 4 of A, 4 per 128 columns of B
constexpr uint32_t SF_COLS = SF_BYTES / SF_BLOCK * 4;
constexpr int COLS = BN / 2;       // columns per epilogue thread
constexpr int STG_BYTES = 16 * 128;  // staging of one epilogue warp: 16 rows x 128 bytes
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + SCALE_SLOTS * SF_BYTES + EPI_WARPS * STG_BYTES + 1024 /*alignment slack*/ + 256;

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
  int aligned;  // C rows start on 16-byte boundaries
  Scales sa, sb;
  const int* offsets;  // [num_groups + 1] row boundaries of the groups, or null: one product
  int num_groups;
  int* status;
};

// Biased exponent of a scale; NaN's where it is no positive normal power of two.
__device__ __forceinline__ uint32_t exponent_of(float scale) {
  const uint32_t bits = __float_as_uint(scale);
  return (bits & 0x807fffffu) != 0u || bits == 0u ? 0xffu : bits >> 23;
}

struct TileInfo {
  int m0, m_end, n0, g;
};

// Walks the tiles of one pair.
struct Walker {
  static constexpr int bm = BM * CTAS, bn = BN;
  const Params& p;
  int tiles_m, tiles_n, tile, g, base;
  __device__ Walker(const Params& params) : p(params), g(0), base(0) {
    tiles_m = (p.M + bm - 1) / bm;
    tiles_n = (p.N + bn - 1) / bn;
    tile = blockIdx.x / CTAS;
  }
  __device__ bool next(TileInfo& t) {
    if (p.offsets == nullptr) {
      if (tile >= tiles_m * tiles_n) return false;
      const int per_group = p.group_m * tiles_n;
      const int grp = tile / per_group, first_m = grp * p.group_m;
      const int gm = min(tiles_m - first_m, p.group_m);
      const int r = tile - grp * per_group;
      t.m0 = (first_m + r % gm) * bm;
      t.m_end = p.M;
      t.n0 = (r / gm) * bn;
      t.g = 0;
    } else {
      int lo, rows, tm_g;
      while (true) {
        if (g >= p.num_groups) return false;
        lo = min(max(p.offsets[g], 0), p.M);  // whatever the boundaries hold, no row outside the matrix is touched
        rows = max(min(p.offsets[g + 1], p.M) - lo, 0);
        tm_g = (rows + bm - 1) / bm;
        if (tile < base + tm_g * tiles_n) break;
        base += tm_g * tiles_n;
        ++g;
      }
      const int local = tile - base;
      t.m0 = lo + (local % tm_g) * bm;
      t.m_end = lo + rows;
      t.n0 = (local / tm_g) * bn;
      t.g = g;
    }
    tile += gridDim.x / CTAS;
    return true;
  }
};

// A waiting thread asks to be suspended (for up to 20 us) before it starts to look at the clock.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t"
      "}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
      : "memory");
  if (ok) return true;
  return mbar_wait_bounded(bar, parity, abort_flag, status, code);
}

// ---- CTA pairs ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_cta(uint32_t smem_addr, uint32_t cta_rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(cta_rank));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrive on an mbarrier of any CTA of the cluster (address from map_to_cta).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Tiled loads of one CTA of a pair into its own shared memory; the bytes count on a barrier that may be the other CTA's.
__device__ __forceinline__ void pair_load_2d(void* smem_dst, const CUtensorMap* desc, uint32_t pair_bar, int32_t c0, int32_t c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(desc)), "r"(pair_bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void pair_load_3d(void* smem_dst, const CUtensorMap* desc, uint32_t pair_bar, int32_t c0, int32_t c1,
                                             int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(desc)), "r"(pair_bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
// D (+)= (A * SFA) (B * SFB)^T for K = 32 with E8M0 scales in tensor memory, by one CTA or a pair (GROUP); issued by the one thread (of a pair: of the leader)
// whose `issue` is set.
template <int GROUP>
__device__ __forceinline__ void umma(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t tsfa,
                                     uint32_t tsfb, uint32_t accumulate, uint32_t issue) {
  if (GROUP == 1) {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.b32 q, %8, 0;\n\t"
        ".reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], da, db, %4, [%5], [%6], p;\n\t"
        "}\n" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(tsfa), "r"(tsfb), "r"(accumulate), "r"(issue)
        : "memory");
  } else {
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.b32 q, %8, 0;\n\t"
        ".reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %7, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], da, db, %4, [%5], [%6], p;\n\t"
        "}\n" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(tsfa), "r"(tsfb), "r"(accumulate), "r"(issue)
        : "memory");
  }
}
// 32 rows x 16 bytes of scales from shared memory into 4 columns, replicated to the four lane quadrants; of a pair, each CTA
// copies from its own shared memory into its own tensor memory.
template <int GROUP>
__device__ __forceinline__ void sf_copy(uint32_t tmem_dst, uint32_t smem_src) {
  // no swizzle, 8-row x 16-byte core matrices every 128 bytes
  const uint64_t desc = static_cast<uint64_t>((smem_src >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128u >> 4) << 32) | (1ull << 46);
  if (GROUP == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem_dst), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem_dst), "l"(desc) : "memory");
}
// `bar` (and the other CTA's at the same offset) observes the completion of the MMAs issued so far.
template <int GROUP>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (GROUP == 1) {
    umma_commit(bar);
  } else {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
  }
}

// Waits for the tensor-memory loads issued so far. The registers pass through, so that nothing that reads them can be
// scheduled ahead of the wait.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// ---- epilogue staging ------------------------------------------------------------------------------------------------
// 16-byte slot `chunk` (0..7) of staged row `row` (0..15); the XOR keeps both the row-per-thread and the 8-lanes-per-row
// access patterns free of bank conflicts.
__device__ __forceinline__ uint4* stg_slot(uint8_t* stg, int row, int chunk) {
  return reinterpret_cast<uint4*>(stg + row * 128 + ((chunk ^ (row & 7)) << 4));
}
// Moves a staged block to global memory, 8 lanes per 128-byte row; `bytes` of every row are inside the matrix. Rows that do not
// start on 16-byte boundaries go element by element, a row at a time.
template <int EPI>
__device__ __forceinline__ void stg_store(uint8_t* stg, uint8_t* dst0, long long ld_bytes, int rows, int bytes, bool aligned, int lane) {
  if (!aligned) {
    constexpr int ES = EPI == EPI_BF16 ? 2 : 4;
#pragma unroll 4
    for (int rr = 0; rr < min(rows, 16); ++rr) {
#pragma unroll
      for (int j = 0; j < 4 / ES; ++j) {
        const int at = (lane + 32 * j) * ES;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(stg_slot(stg, rr, at >> 4)) + (at & 15);
        uint8_t* dst = dst0 + rr * ld_bytes + at;
        if (at >= bytes) continue;
        if (EPI == EPI_BF16) *reinterpret_cast<uint16_t*>(dst) = *reinterpret_cast<const uint16_t*>(src);
        else if (EPI == EPI_F32) *reinterpret_cast<float*>(dst) = *reinterpret_cast<const float*>(src);
        else *reinterpret_cast<float*>(dst) += *reinterpret_cast<const float*>(src);
      }
    }
    return;
  }
  const int cc = (lane & 7) * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = i * 4 + (lane >> 3);
    if (rr >= rows || cc >= bytes) continue;
    const uint4 v = *stg_slot(stg, rr, lane & 7);
    uint8_t* dst = dst0 + rr * ld_bytes + cc;
    if (EPI == EPI_F32_ACC) {
      const float f[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
      if (cc + 16 <= bytes) {  // one addition per element, performed in L2
        asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(dst), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3])
                     : "memory");
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (cc + 4 * j < bytes) atomicAdd(reinterpret_cast<float*>(dst) + j, f[j]);
      }
    } else if (cc + 16 <= bytes) {
      *reinterpret_cast<uint4*>(dst) = v;
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 8; ++j)  // 2-byte pieces serve both element sizes
        if (cc + 2 * j < bytes) reinterpret_cast<uint16_t*>(dst)[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

template <int EPI>
__global__ void __launch_bounds__(THREADS, 1)
gemm_block_fp8_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_smem = smem + STAGES * STAGE_BYTES;
  uint8_t* stg_smem = sf_smem + SCALE_SLOTS * SF_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(stg_smem + EPI_WARPS * STG_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 1;
  uint64_t* sfull_bar = tempty_bar + 1;
  uint64_t* sempty_bar = sfull_bar + SCALE_SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sempty_bar + SCALE_SLOTS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int num_kb = (p.K + BKE - 1) / BKE;
  const uint32_t cta = cluster_ctarank();  // 0 = leader of the pair

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < SCALE_SLOTS; ++i) {
      mbar_init(&sfull_bar[i], 2 * CTAS);  // the scale warps of both CTAs
      mbar_init(&sempty_bar[i], 1);
    }
    mbar_init(tfull_bar, 1);
    mbar_init(tempty_bar, EPI_WARPS * CTAS);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tma_a);
    tma_prefetch_desc(&tma_b);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  previous_kernel_done();
  tc_fence_before();
  __syncthreads();
  next_kernel_may_start();  // after this CTA has its tensor memory: one of the next kernel never waits for it with that in hand
  cluster_sync_all();  // the other CTA's barriers are initialised before anything is signalled across
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      Walker walker(p);
      TileInfo t;
      while (ok && walker.next(t)) {
        const int m0 = t.m0 + static_cast<int>(cta) * BM, n0 = t.n0 + static_cast<int>(cta) * B_ROWS;
        for (int kb = 0; kb < num_kb; kb += KBS) {
          ok = wait_for(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer);
          if (!ok) break;
          const int blocks = min(KBS, num_kb - kb);
          if (cta == 0) mbar_arrive_expect_tx(&full_bar[stage], CTAS * KB_BYTES * blocks);
          const uint32_t pair_bar = map_to_cta(smem_u32(&full_bar[stage]), 0);
          for (int j = 0; j < blocks; ++j) {
            uint8_t* sa = smem + stage * STAGE_BYTES + j * KB_BYTES;
            uint8_t* sb = sa + A_BYTES;
            const int k0 = (kb + j) * BKE;
            // innermost coordinates are k0 (K-major) or tile origins (MN-major): multiples of 128 bytes either way; group
            // boundaries only enter the outer coordinate of a K-major A
            if (p.a_mn) pair_load_2d(sa, &tma_a, pair_bar, m0, k0);
            else pair_load_2d(sa, &tma_a, pair_bar, k0, m0);
            if (p.b_mn) pair_load_3d(sb, &tma_b, pair_bar, n0, k0, t.g);
            else pair_load_3d(sb, &tma_b, pair_bar, k0, n0, t.g);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      if (!ok) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // let copies in flight land before shared memory goes away
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ issuer (the leader's)
    // The whole warp walks the loop, so that descriptors can live in uniform registers; one lane issues.
    if (cta == 0) {
      const uint32_t issue = lane == 0;
      // K-major: 8-row swizzle atoms 1024 bytes apart, K = 32 advances 32 bytes along the line. MN-major: one 128-column box,
      // 8 k-rows per 1024 bytes, K = 32 advances 32 lines.
      constexpr uint32_t kDescHi = desc_hi_sw128(1024);
      // kind::mxf8f6f4: e4m3 A and B, majors at bits 15 and 16, N >> 3 at 17, E8M0 scales (23), M >> 4 at 24; the byte that
      // holds the exponents at 29 (A) and 4 (B)
      const uint32_t idesc = (static_cast<uint32_t>(p.a_mn) << 15) | (static_cast<uint32_t>(p.b_mn) << 16) |
                             (static_cast<uint32_t>(BN >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(BM * CTAS >> 4) << 24);
      const uint32_t a_step = p.a_mn ? 256u : 2u, b_step = p.b_mn ? 256u : 2u;
      const uint32_t a_lo0 = desc_lo_sw128(smem_u32(smem), 16);
      const uint32_t b_lo0 = desc_lo_sw128(smem_u32(smem) + A_BYTES, 16);
      const uint32_t sf0 = smem_u32(sf_smem);
      int stage = 0, slot = 0;
      uint32_t phase = 0, acc_phase = 0, slot_phase = 0;
      // the two sets of scale columns take turns
      uint32_t tsfa = tmem_base + SF_COL;
      const uint32_t sf_flip = tsfa ^ (tsfa + SF_COLS);
      bool ok = true;
      Walker walker(p);
      TileInfo t;
      while (ok && walker.next(t)) {
        ok = wait_for(tempty_bar, acc_phase ^ 1u, abort_flag, p.status, kStatusTimeoutMma);
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < num_kb; kb += KBS) {
          const bool first_of_batch = (kb & (SCALE_BATCH - 1)) == 0;
          if (first_of_batch) {  // copies and MMAs of one thread execute in issue order
            ok = wait_for(&sfull_bar[slot], slot_phase, abort_flag, p.status, kStatusTimeoutMma);
            if (!ok) break;
            tc_fence_after();
            const uint32_t ss = sf0 + slot * SF_BYTES;
            if (issue) {
              sf_copy<CTAS>(tsfa, ss);
#pragma unroll
              for (uint32_t b = 0; b < BN / 128; ++b) sf_copy<CTAS>(tsfa + 4 + 4 * b, ss + SF_BLOCK * (1 + b));
            }
          }
          ok = wait_for(&full_bar[stage], phase, abort_flag, p.status, kStatusTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a_lo = a_lo0 + stage * (STAGE_BYTES >> 4), b_lo = b_lo0 + stage * (STAGE_BYTES >> 4);
          const uint32_t byte0 = first_of_batch ? 0u : 2u;
          uint32_t id = idesc + byte0 * ((1u << 29) | (1u << 4)), ta = tsfa + (byte0 << 30), tb = ta + 4;
#pragma unroll
          for (uint32_t k = 0; k < BKE / 32; ++k)
            umma<CTAS>(tmem_base, a_lo + k * a_step, b_lo + k * b_step, kDescHi, id, ta, tb, (kb | static_cast<int>(k)) != 0, issue);
          if (kb + 1 < num_kb) {
            id += (1u << 29) | (1u << 4);
            ta += 1u << 30;
            tb += 1u << 30;
#pragma unroll
            for (uint32_t k = 0; k < BKE / 32; ++k)
              umma<CTAS>(tmem_base, a_lo + (KB_BYTES >> 4) + k * a_step, b_lo + (KB_BYTES >> 4) + k * b_step, kDescHi, id, ta, tb, 1u, issue);
          }
          if (issue) commit<CTAS>(&empty_bar[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          if (!first_of_batch || kb + KBS >= num_kb) {
            if (issue) commit<CTAS>(&sempty_bar[slot]);
            tsfa ^= sf_flip;
            if (++slot == SCALE_SLOTS) { slot = 0; slot_phase ^= 1u; }
          }
        }
        if (ok && issue) commit<CTAS>(tfull_bar);
        acc_phase ^= 1u;
      }
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------------ scales (warps 2 and 3)
    const int t64 = threadIdx.x - 64;
    constexpr int PER = (BM + BN) / 64;  // rows whose scales a thread carries: t64 + 64 i of A, then of B
    const uint32_t sfull_leader = map_to_cta(smem_u32(sfull_bar), 0);
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    Walker walker(p);
    TileInfo t;
    while (ok && walker.next(t)) {
      const float* src[PER];
      long long step[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int f = t64 + 64 * i;
        const bool is_a = i < BM / 64;
        const int at = is_a ? t.m0 + static_cast<int>(cta) * BM + f : t.n0 + f - BM;
        const Scales& sc = is_a ? p.sa : p.sb;
        step[i] = sc.k_stride;
        src[i] = at < (is_a ? t.m_end : p.N)
                     ? sc.p + (is_a ? 0 : t.g * sc.group_stride) + static_cast<long long>(at >> sc.shift) * sc.i_stride
                     : nullptr;
      }
      float next[SCALE_BATCH][PER];
      auto fetch = [&](int kb0) {
#pragma unroll
        for (int b = 0; b < SCALE_BATCH; ++b)
#pragma unroll
          for (int i = 0; i < PER; ++i)  // rows outside the matrix: any valid scale, their products are not stored
            next[b][i] = kb0 + b < num_kb && src[i] != nullptr ? src[i][(kb0 + b) * step[i]] : 1.f;
      };
      fetch(0);
      for (int kb0 = 0; kb0 < num_kb; kb0 += SCALE_BATCH) {
        uint32_t words[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          words[i] = 0u;
#pragma unroll
          for (int b = 0; b < SCALE_BATCH; ++b) words[i] |= exponent_of(next[b][i]) << (8 * b);
        }
        fetch(kb0 + SCALE_BATCH);  // on its way while this batch waits for its slot
        ok = wait_for(&sempty_bar[slot], phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        uint32_t* dst = reinterpret_cast<uint32_t*>(sf_smem + slot * SF_BYTES);
#pragma unroll
        for (int i = 0; i < PER; ++i) {  // row r of a 128-row block: 32-bit word 4 (r % 32) + r / 32 of its 512 bytes
          const int f = t64 + 64 * i;
          dst[(f >> 7) * (SF_BLOCK / 4) + (f & 31) * 4 + ((f >> 5) & 3)] = words[i];
        }
        fence_proxy_async_smem();  // the tensor core's copy reads what the threads wrote
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(sfull_leader + slot * 8);
        if (++slot == SCALE_SLOTS) { slot = 0; phase ^= 1u; }
      }
    }
  } else {
    // ------------------------------------------------------------------ epilogue
    const int quad = warp & 3, half = (warp - 4) >> 2;
    uint8_t* stg = stg_smem + (warp - 4) * STG_BYTES;
    const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + half * COLS;
    const uint32_t tempty_leader = map_to_cta(smem_u32(tempty_bar), 0);
    uint32_t acc_phase = 0;
    bool ok = true;
    Walker walker(p);
    TileInfo t;
    while (ok && walker.next(t)) {
      ok = wait_for(tfull_bar, acc_phase, abort_flag, p.status, kStatusTimeoutEpilogue);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      uint32_t r[COLS / 32][32];
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) tmem_ld_32x32(t_row + c * 32, r[c]);
#pragma unroll
      for (int c = 0; c < COLS / 32; ++c) tmem_ld_wait_for(r[c]);
      tc_fence_before();  // the accumulator is in registers: the issuer may start the next tile
      if (lane == 0) mbar_arrive_cluster(tempty_leader);
      acc_phase ^= 1u;
      const int row0 = t.m0 + static_cast<int>(cta) * BM + quad * 32, col0 = t.n0 + half * COLS;
      const int rows = min(32, t.m_end - row0);
      if (rows <= 0) continue;
      constexpr int ES = EPI == EPI_BF16 ? 2 : 4, CHUNK = 128 / ES;  // columns of a staged block
#pragma unroll
      for (int c = 0; c < COLS / CHUNK; ++c) {
        const int bytes = min(128, (p.N - (col0 + c * CHUNK)) * ES);
        if (bytes <= 0) break;
        uint4 o[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (EPI == EPI_BF16) {
            const uint32_t* s = &r[2 * c + (q >> 2)][(q & 3) * 8];
            o[q].x = pack_bf16x2(__uint_as_float(s[0]), __uint_as_float(s[1]));
            o[q].y = pack_bf16x2(__uint_as_float(s[2]), __uint_as_float(s[3]));
            o[q].z = pack_bf16x2(__uint_as_float(s[4]), __uint_as_float(s[5]));
            o[q].w = pack_bf16x2(__uint_as_float(s[6]), __uint_as_float(s[7]));
          } else {
            const uint32_t* s = &r[c][q * 4];
            o[q] = make_uint4(s[0], s[1], s[2], s[3]);
          }
        }
        uint8_t* dst = reinterpret_cast<uint8_t*>(p.C) + (static_cast<long long>(row0) * p.ldc + col0 + c * CHUNK) * ES;
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // sixteen rows at a time
          __syncwarp();
          if ((lane >> 4) == h) {
#pragma unroll
            for (int q = 0; q < 8; ++q) *stg_slot(stg, lane & 15, q) = o[q];
          }
          __syncwarp();
          stg_store<EPI>(stg, dst + h * 16 * p.ldc * ES, p.ldc * ES, rows - 16 * h, bytes, p.aligned != 0, lane);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // nothing of the other CTA signals into this one's shared memory any more
  if (warp == 1) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
  }
}

// ---- small products --------------------------------------------------------------------------------------------------
// One CTA per 128 x BN tile and reduction part. Few tokens against a weight: the weight's rows take the 128-row side and the
// tokens the BN side (SWAP: D is C transposed), so a tile is no larger than it has to be and every SM streams weights. The
// reduction is split over the CTAs of a cluster; each leaves its fp32 part in its own shared memory, and the CTAs then add the
// parts in rank order, each for its share of the rows of C (distributed shared memory: no workspace, no atomics, the same bits
// every time). Groups (SWAP only): a CTA finds its group and its tokens from the device-side boundaries.
//
// FUSED (SWAP, up to 16 tokens a tile): the tokens arrive in bf16, and the warps of the epilogue, which have nothing else to do
// before the end, quantise them straight into the stages beside the weight's codes. Every CTA does that for its part of the
// reduction, out of L2; in exchange there is no quantiser launch in front (one token against 4096 x 11008, with the host: 18.4 us
// with the launch, 14.4 without; two scale warps in place of the epilogue's took 16.8).
//
// What bounds it: the weight's bytes (one token against 4096 x 11008: 12.5 us, 3.6 TB/s, against 6.9 us at the measured copy
// rate), and about 4.4 us in which barriers, tensor memory and tensor maps are set up, the first loads arrive, and the parts are
// added. 64 experts of 1024 x 2048 for 128 random rows, which reach 50 of them: 21.4 us, 4.9 TB/s.
constexpr int SMALL_THREADS = 256;  // warps as above, with one epilogue warpgroup

// MANY: three CTAs per SM with a short ring each, instead of two with a deeper one (see fuller_with_three()).
template <int BN, bool MANY>
struct SmallTile {
  static constexpr int CTAS = MANY ? 3 : 2;
  static constexpr int KB_BYTES = A_BYTES + BN * BKE;
  static constexpr int STAGES = MANY || BN >= 128 ? 3 : BN >= 64 ? 4 : BN >= 32 ? 5 : 6;
  static constexpr uint32_t TMEM = BN >= 128 ? 256 : BN >= 64 ? 128 : BN >= 32 ? 64 : 32;  // BN + 16 scale columns
  static constexpr int SF_BYTES = 2 * SF_BLOCK;
  static constexpr int SMEM_BYTES = STAGES * KB_BYTES + SCALE_SLOTS * SF_BYTES + 1024 + 256;
  // the fp32 part reuses the stages: [BN][128] (SWAP) or [128][BN + 4]
  static_assert(STAGES * KB_BYTES >= 128 * (BN + 4) * 4, "the parts do not fit");
  static_assert(CTAS * (SMEM_BYTES + 1024) <= 228 * 1024, "the CTAs of an SM do not fit");
};

struct SmallParams {
  void* C;
  long long ldc;
  int M, N, K;   // rows of the 128-row side (of one group), rows of the BN side (all groups), reduction
  int a_mn, b_mn, epi, vector;  // vector: C rows start on 16-byte boundaries
  int parts, kb_per_part;
  Scales sa, sb;
  const __nv_bfloat16* x;  // FUSED: the BN side [N][K]
  long long ldx;
  int x_vector;  // its rows start on 16-byte boundaries
  const int* offsets;
  int num_groups;
  int* status;
};

// Eight elements of a row of x, zeros outside.
__device__ __forceinline__ uint4 load_x8(const SmallParams& p, const __nv_bfloat16* row, int k) {
  if (row == nullptr || k >= p.K) return make_uint4(0u, 0u, 0u, 0u);
  if (p.x_vector && k + 8 <= p.K) return *reinterpret_cast<const uint4*>(row + k);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k + j < p.K) w[j >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(row)[k + j]) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float4 load_cluster_f4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}

template <int BN, bool SWAP, bool FUSED, bool MANY>
__global__ void __launch_bounds__(SMALL_THREADS, (SmallTile<BN, MANY>::CTAS))
gemm_block_fp8_small_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b, const SmallParams p) {
  using T = SmallTile<BN, MANY>;
  constexpr int STAGES = T::STAGES;
  static_assert(!FUSED || (SWAP && BN == 16), "eight threads per token cover sixteen tokens");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sf_smem = smem + STAGES * T::KB_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(sf_smem + SCALE_SLOTS * T::SF_BYTES);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* sfull_bar = empty_bar + STAGES;
  uint64_t* sempty_bar = sfull_bar + SCALE_SLOTS;
  uint64_t* done_bar = sempty_bar + SCALE_SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* tile_info = reinterpret_cast<int*>(tmem_slot + 2);  // group, first row and end of the BN side

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = blockIdx.x % p.parts, tile = blockIdx.x / p.parts;
  const int tiles_a = (p.M + BM - 1) / BM;
  const int a_tile = tile % tiles_a, b_tile = tile / tiles_a;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], FUSED ? 5 : 1);  // the weight's bytes, and the four warps that write the tokens' codes
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < SCALE_SLOTS; ++i) {
      mbar_init(&sfull_bar[i], FUSED ? 6 : 2);
      mbar_init(&sempty_bar[i], 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tma_a);
    tma_prefetch_desc(&tma_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, T::TMEM);
    tmem_relinquish();
  }
  previous_kernel_done();
  if (warp == 2) {
    int g = 0, b0 = b_tile * BN, b_end = p.N;
    if (p.offsets != nullptr) {  // which group does the b_tile-th tile of the BN side belong to?
      int before = 0;
      g = -1;
      for (int base = 0; base < p.num_groups && g < 0; base += 32) {
        int lo = 0, rows = 0;
        if (base + lane < p.num_groups) {
          lo = min(max(p.offsets[base + lane], 0), p.N);
          rows = max(min(p.offsets[base + lane + 1], p.N) - lo, 0);
        }
        const int tiles = (rows + BN - 1) / BN;
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, b_tile < before + upto);
        if (hit != 0u) {
          const int l = __ffs(hit) - 1;
          g = base + l;
          const int first = before + __shfl_sync(0xffffffffu, upto - tiles, l);
          b0 = __shfl_sync(0xffffffffu, lo, l) + (b_tile - first) * BN;
          b_end = __shfl_sync(0xffffffffu, lo + rows, l);
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    if (lane == 0) {
      tile_info[0] = g;
      tile_info[1] = b0;
      tile_info[2] = b_end;
    }
  }
  tc_fence_before();
  __syncthreads();
  next_kernel_may_start();  // after this CTA has its tensor memory
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int g = tile_info[0], b0 = tile_info[1], b_end = tile_info[2];
  const int a0 = a_tile * BM;
  const int num_kb = (p.K + BKE - 1) / BKE;
  const int kb_first = part * p.kb_per_part;
  const int kbs = g < 0 ? 0 : max(min(p.kb_per_part, num_kb - kb_first), 0);  // a tile nobody needs: no blocks, nothing stored
  bool ok = true;

  if (warp == 0) {
    // ------------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = 0; kb < kbs; ++kb) {
        ok = wait_for(&empty_bar[stage], phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer);
        if (!ok) break;
        uint8_t* sa = smem + stage * T::KB_BYTES;
        uint8_t* sb = sa + A_BYTES;
        const int k0 = (kb_first + kb) * BKE;
        const int ga = SWAP ? g : 0, gb = SWAP ? 0 : g;
        mbar_arrive_expect_tx(&full_bar[stage], FUSED ? A_BYTES : T::KB_BYTES);
        // innermost coordinates: k0 (K-major) or a0 / b0 of an ungrouped operand (MN-major), multiples of 128 bytes
        if (p.a_mn) tma_load_3d(sa, &tma_a, &full_bar[stage], a0, k0, ga);
        else tma_load_3d(sa, &tma_a, &full_bar[stage], k0, a0, ga);
        if (!FUSED && p.b_mn) tma_load_3d(sb, &tma_b, &full_bar[stage], b0, k0, gb);
        else if (!FUSED) tma_load_3d(sb, &tma_b, &full_bar[stage], k0, b0, gb);
        if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      }
      if (!ok) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // let copies in flight land before shared memory is used again
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ issuer
    const uint32_t issue = lane == 0;
    constexpr uint32_t kDescHi = desc_hi_sw128(1024);
    const uint32_t idesc = (static_cast<uint32_t>(p.a_mn) << 15) | (static_cast<uint32_t>(p.b_mn) << 16) |
                           (static_cast<uint32_t>(BN >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(BM >> 4) << 24);
    const uint32_t a_step = p.a_mn ? 256u : 2u, b_step = p.b_mn ? 256u : 2u;
    const uint32_t a_lo0 = desc_lo_sw128(smem_u32(smem), 16);
    const uint32_t b_lo0 = desc_lo_sw128(smem_u32(smem) + A_BYTES, 16);
    const uint32_t sf0 = smem_u32(sf_smem);
    int stage = 0, slot = 0;
    uint32_t phase = 0, slot_phase = 0;
    uint32_t tsfa = tmem_base + BN;
    const uint32_t sf_flip = tsfa ^ (tsfa + 8);
    for (int kb = 0; kb < kbs; ++kb) {
      const uint32_t in_batch = static_cast<uint32_t>(kb) & (SCALE_BATCH - 1);
      if (in_batch == 0) {
        ok = wait_for(&sfull_bar[slot], slot_phase, abort_flag, p.status, kStatusTimeoutMma);
        if (!ok) break;
        tc_fence_after();
        if (issue) {
          sf_copy<1>(tsfa, sf0 + slot * T::SF_BYTES);
          sf_copy<1>(tsfa + 4, sf0 + slot * T::SF_BYTES + SF_BLOCK);
        }
      }
      ok = wait_for(&full_bar[stage], phase, abort_flag, p.status, kStatusTimeoutMma);
      if (!ok) break;
      tc_fence_after();
      const uint32_t a_lo = a_lo0 + stage * (T::KB_BYTES >> 4), b_lo = b_lo0 + stage * (T::KB_BYTES >> 4);
      const uint32_t id = idesc + in_batch * ((1u << 29) | (1u << 4)), ta = tsfa + (in_batch << 30), tb = ta + 4;
#pragma unroll
      for (uint32_t k = 0; k < BKE / 32; ++k)
        umma<1>(tmem_base, a_lo + k * a_step, b_lo + k * b_step, kDescHi, id, ta, tb, (kb | static_cast<int>(k)) != 0, issue);
      if (issue) commit<1>(&empty_bar[stage]);
      if (++stage == STAGES) { stage = 0; phase ^= 1u; }
      if (in_batch == SCALE_BATCH - 1 || kb + 1 == kbs) {
        if (issue) commit<1>(&sempty_bar[slot]);
        tsfa ^= sf_flip;
        if (++slot == SCALE_SLOTS) { slot = 0; slot_phase ^= 1u; }
      }
    }
    if (ok && issue && kbs > 0) commit<1>(done_bar);
  } else if (warp < 4) {
    // ------------------------------------------------------------------ scales
    const int t64 = threadIdx.x - 64;
    constexpr int PER = 2 + (FUSED ? 0 : (BN + 63) / 64);
    const float* src[PER];
    long long step[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const bool is_a = i < 2;
      const int f = is_a ? t64 + 64 * i : t64 + 64 * (i - 2);
      const int at = (is_a ? a0 : b0) + f;
      const Scales& sc = is_a ? p.sa : p.sb;
      step[i] = sc.k_stride;
      const bool in = is_a ? at < p.M : f < BN && at < b_end;
      src[i] = in ? sc.p + g * sc.group_stride + static_cast<long long>(at >> sc.shift) * sc.i_stride + kb_first * sc.k_stride : nullptr;
    }
    int slot = 0;
    uint32_t phase = 0;
    float next[SCALE_BATCH][PER];
    auto fetch = [&](int kb0) {
#pragma unroll
      for (int b = 0; b < SCALE_BATCH; ++b)
#pragma unroll
        for (int i = 0; i < PER; ++i) next[b][i] = kb0 + b < kbs && src[i] != nullptr ? src[i][(kb0 + b) * step[i]] : 1.f;
    };
    fetch(0);
    for (int kb0 = 0; kb0 < kbs; kb0 += SCALE_BATCH) {
      uint32_t words[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        words[i] = 0u;
#pragma unroll
        for (int b = 0; b < SCALE_BATCH; ++b) words[i] |= exponent_of(next[b][i]) << (8 * b);
      }
      fetch(kb0 + SCALE_BATCH);
      ok = wait_for(&sempty_bar[slot], phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint32_t* dst = reinterpret_cast<uint32_t*>(sf_smem + slot * T::SF_BYTES);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int f = i < 2 ? t64 + 64 * i : t64 + 64 * (i - 2);
        dst[(i < 2 ? 0 : SF_BLOCK / 4) + (f & 31) * 4 + ((f >> 5) & 3)] = words[i];
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sfull_bar[slot]);
      if (++slot == SCALE_SLOTS) { slot = 0; phase ^= 1u; }
    }
  } else {
    // ------------------------------------------------------------------ this CTA's part into shared memory
    const int quad = warp & 3;
    if (FUSED) {
      // First the tokens: eight threads share one, sixteen elements of a block each.
      const int token = (threadIdx.x - 128) >> 3, piece = threadIdx.x & 7;
      const __nv_bfloat16* x_row = b0 + token < b_end ? p.x + (b0 + token) * p.ldx : nullptr;
      const bool any = __any_sync(0xffffffffu, x_row != nullptr);  // a warp without tokens only keeps the barriers going
      uint4 next[SCALE_BATCH][2];
      auto fetch = [&](int kb0) {
#pragma unroll
        for (int b = 0; b < SCALE_BATCH; ++b)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            next[b][q] = load_x8(p, kb0 + b < kbs ? x_row : nullptr, (kb_first + kb0 + b) * BKE + piece * 16 + q * 8);
      };
      int slot = 0, stage = 0;
      uint32_t phase = 0, stage_phase = 0;
      fetch(0);
      for (int kb0 = 0; kb0 < kbs && ok; kb0 += SCALE_BATCH) {
        uint4 codes[SCALE_BATCH];
        uint32_t word = 0u;
        if (any) {
#pragma unroll
          for (int b = 0; b < SCALE_BATCH; ++b) {
            const uint4 lo = next[b][0], hi = next[b][1];
            uint32_t m2 = blkq::max_mag2(blkq::max_mag2(lo), blkq::max_mag2(hi));
#pragma unroll
            for (int o = 4; o; o >>= 1) m2 = blkq::max_mag2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
            const uint32_t amax = max(m2 & 0x7fffu, (m2 >> 16) & 0x7fffu);
            const int e = blkq::scale_exponent(amax);
            const uint32_t inv = blkq::inverse_bf16(e) * 0x10001u;
            uint2 c0 = blkq::e4m3x8(lo, inv), c1 = blkq::e4m3x8(hi, inv);
            if (amax == blkq::BF16_INF) {
              c0 = blkq::infinities_to_nan(lo, c0);
              c1 = blkq::infinities_to_nan(hi, c1);
            }
            codes[b] = make_uint4(c0.x, c0.y, c1.x, c1.y);
            word |= static_cast<uint32_t>(e) << (8 * b);
          }
          fetch(kb0 + SCALE_BATCH);
        }
        ok = wait_for(&sempty_bar[slot], phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (any && piece == 0) reinterpret_cast<uint32_t*>(sf_smem + slot * T::SF_BYTES + SF_BLOCK)[token * 4] = word;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sfull_bar[slot]);
        if (++slot == SCALE_SLOTS) { slot = 0; phase ^= 1u; }
#pragma unroll
        for (int b = 0; b < SCALE_BATCH; ++b) {
          if (kb0 + b >= kbs) break;
          ok = wait_for(&empty_bar[stage], stage_phase ^ 1u, abort_flag, p.status, kStatusTimeoutProducer);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (any)  // the 128-byte swizzle: 16-byte piece c of row r sits at c ^ (r % 8)
            *reinterpret_cast<uint4*>(smem + stage * T::KB_BYTES + A_BYTES + token * 128 + ((piece ^ (token & 7)) << 4)) = codes[b];
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full_bar[stage]);
          if (++stage == STAGES) { stage = 0; stage_phase ^= 1u; }
        }
      }
    }
    if (kbs > 0 && ok) {
      ok = wait_for(done_bar, 0, abort_flag, p.status, kStatusTimeoutEpilogue);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    // every load into the stages has been consumed by an MMA that is complete: their memory is free
    float* out = reinterpret_cast<float*>(smem);
    const int row = quad * 32 + lane;
#pragma unroll
    for (int c = 0; c < BN / 16; ++c) {
      uint32_t r[16];
      if (kbs > 0 && ok) {
        tmem_ld_32x16(tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + c * 16, r);
        tmem_ld_wait_for(r);
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) r[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (SWAP) {
          out[(c * 16 + j) * 128 + row] = __uint_as_float(r[j]);
        } else if ((j & 3) == 0) {
          *reinterpret_cast<uint4*>(out + row * (BN + 4) + c * 16 + j) = make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (p.parts > 1) cluster_sync_all();  // all parts are in place
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, T::TMEM);
  }

  // Sum of the parts, in rank order. A row of C has `inner` columns here; rank `part` takes rows part, part + parts, ...
  constexpr int INNER = SWAP ? 128 : BN, PITCH = SWAP ? 128 : BN + 4;
  const int c_row0 = SWAP ? b0 : a0, c_col0 = SWAP ? a0 : b0;
  const int rows = SWAP ? min(BN, b_end - b0) : min(128, p.M - a0);
  const int cols = SWAP ? min(128, p.M - a0) : min(BN, b_end - b0);
  if (g >= 0 && *abort_flag == 0) {
    const uint32_t mine = smem_u32(smem);
    constexpr int PER_ROW = INNER / 4, ROWS_AT_ONCE = SMALL_THREADS / PER_ROW;
    const int q = threadIdx.x % PER_ROW;
    for (int i = part + (threadIdx.x / PER_ROW) * p.parts; i < rows; i += ROWS_AT_ONCE * p.parts) {
      const uint32_t at = mine + static_cast<uint32_t>(i * PITCH + 4 * q) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = 0; r < p.parts; ++r) {
        const float4 x = p.parts > 1 ? load_cluster_f4(map_to_cta(at, r)) : *reinterpret_cast<const float4*>(smem + (i * PITCH + 4 * q) * 4);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
      }
      const float f[4] = {v.x, v.y, v.z, v.w};
      const long long first = static_cast<long long>(c_row0 + i) * p.ldc + c_col0 + 4 * q;
      const int n = cols - 4 * q;
      if (n <= 0) continue;
      if (p.epi == EPI_BF16) {
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.C) + first;
        if (p.vector && n >= 4) {
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < n) dst[j] = __float2bfloat16_rn(f[j]);
        }
      } else {
        float* dst = reinterpret_cast<float*>(p.C) + first;
        const bool add = p.epi == EPI_F32_ACC;
        if (p.vector && n >= 4) {
          float4 old = add ? *reinterpret_cast<const float4*>(dst) : make_float4(0.f, 0.f, 0.f, 0.f);
          if (add) { v.x += old.x; v.y += old.y; v.z += old.z; v.w += old.w; }
          *reinterpret_cast<float4*>(dst) = v;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < n) dst[j] = add ? dst[j] + f[j] : f[j];
        }
      }
    }
  }
  if (p.parts > 1) cluster_sync_all();  // the other CTAs have read this one's part
}

// Properties of a device and settings of a kernel on it are looked up once per device.
static int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess ? dev : -1;
}
static int num_sms(int dev) {
  static std::atomic<int> known[64];
  if (dev < 0) return 0;
  int n = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}
template <class Kernel>
static bool allow_smem(Kernel kernel, int bytes, std::atomic<uint64_t>& done, int dev) {
  const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
  if ((done.load(std::memory_order_relaxed) & bit) != 0) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

template <int EPI>
static int launch(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, long long max_tiles, int dev, cudaStream_t stream) {
  constexpr int bytes = SMEM_BYTES;
  auto kernel = gemm_block_fp8_kernel<EPI>;
  static std::atomic<uint64_t> done;
  if (!allow_smem(kernel, bytes, done, dev)) return -3;
  const int units = num_sms(dev) / CTAS;
  if (units <= 0) return -3;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(max_tiles < units ? max_tiles : units) * CTAS);
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attributes[2] = {dependent_launch(), {}};
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = CTAS;
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, kernel, ta, tb, p) == cudaSuccess ? 0 : -4;
}

static int launch_epi(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, long long max_tiles, int epi, int dev, cudaStream_t s) {
  switch (epi) {
    case EPI_BF16: return launch<EPI_BF16>(ta, tb, p, max_tiles, dev, s);
    case EPI_F32_ACC: return launch<EPI_F32_ACC>(ta, tb, p, max_tiles, dev, s);
    case EPI_F32: return launch<EPI_F32>(ta, tb, p, max_tiles, dev, s);
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

template <int BN, bool SWAP, bool FUSED = false, bool MANY = false>
static int launch_small(const CUtensorMap& ta, const CUtensorMap& tb, const SmallParams& p, long long tiles, int dev, cudaStream_t stream) {
  constexpr int bytes = SmallTile<BN, MANY>::SMEM_BYTES;
  auto kernel = gemm_block_fp8_small_kernel<BN, SWAP, FUSED, MANY>;
  static std::atomic<uint64_t> done;
  if (!allow_smem(kernel, bytes, done, dev)) return -3;
  if (tiles * p.parts > 0x7fffffffll) return -1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(tiles * p.parts));
  config.blockDim = dim3(SMALL_THREADS);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attributes[2] = {dependent_launch(), {}};
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = p.parts;
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  config.attrs = attributes;
  config.numAttrs = 2;
  return cudaLaunchKernelEx(&config, kernel, ta, tb, p) == cudaSuccess ? 0 : -4;
}

struct Product {
  const void *A, *B;  // A null: its rows are x (bf16), quantised on the way
  const __nv_bfloat16* x;
  long long ldx;
  void* C;
  int M, N, K, groups;
  long long lda, ldb, ldc, b_group_bytes;
  Scales sa, sb;
  int a_mn, b_mn, epi;
  const int* offsets;
  int* status;
};

static int run_pair(const Product& x, int dev, cudaStream_t stream) {
  Params p;
  p.C = x.C;
  p.ldc = x.ldc;
  p.M = x.M;
  p.N = x.N;
  p.K = x.K;
  p.group_m = 8;
  p.a_mn = x.a_mn;
  p.b_mn = x.b_mn;
  p.aligned = (reinterpret_cast<uintptr_t>(x.C) & 15) == 0 && (x.ldc * (x.epi == EPI_BF16 ? 2 : 4)) % 16 == 0;
  p.sa = x.sa;
  p.sb = x.sb;
  p.offsets = x.offsets;
  p.num_groups = x.groups;
  p.status = x.status;
  CUtensorMap ta, tb;
  if (!make_map(&ta, x.A, x.a_mn != 0, x.M, x.K, 1, x.lda, 0, BM, 2)) return -1001;
  if (!make_map(&tb, x.B, x.b_mn != 0, x.N, x.K, x.groups, x.ldb, x.groups > 1 ? x.b_group_bytes : x.ldb, B_ROWS, 3)) return -2001;
  const long long tiles_m = (x.M + BM * CTAS - 1) / (BM * CTAS) + (x.offsets != nullptr ? x.groups : 0);
  return launch_epi(ta, tb, p, tiles_m * ((x.N + BN - 1) / BN), x.epi, dev, stream);
}

// Whether `tiles` CTAs fill the SMs in fewer rounds at three per SM than at two. For groups `tiles` is what rows that fall on them at
// random are expected to reach; how many there are is known on the device alone. With as many as there can be three per SM cost a little:
// 64 groups of two rows each, 512 tiles: 38.9 us against 36.9 (product alone, cold L2). Up to 16 rows against weights of 64 experts, two and
// three per SM: 424 tiles of 16 blocks 28.5 and 22.1 us, of 8 blocks 31.0 and 24.8 (848 tiles), 384 of 32 blocks 47.3 and 36.5; but 504 of 16
// blocks 31.2 and 32.9, 512 of 32 blocks 49.7 and 58.3 (two rounds either way, and the second is emptier with three).
static bool fuller_with_three(double tiles, int sms) { return std::ceil(tiles / (3 * sms)) < std::ceil(tiles / (2 * sms)); }

// swap: the rows of B take the 128-row side and the rows of A the side of bn. many: see SmallTile, for bn = 16.
static int run_small(const Product& x, bool swap, int bn, int parts, bool many, int dev, cudaStream_t stream) {
  SmallParams p;
  p.C = x.C;
  p.ldc = x.ldc;
  p.M = swap ? x.N : x.M;
  p.N = swap ? x.M : x.N;
  p.K = x.K;
  p.a_mn = swap ? x.b_mn : x.a_mn;
  p.b_mn = swap ? x.a_mn : x.b_mn;
  p.epi = x.epi;
  p.vector = (reinterpret_cast<uintptr_t>(x.C) & 15) == 0 && (x.ldc * (x.epi == EPI_BF16 ? 2 : 4)) % 16 == 0;
  p.parts = parts;
  p.kb_per_part = ((x.K + BKE - 1) / BKE + parts - 1) / parts;
  p.sa = swap ? x.sb : x.sa;
  p.sb = swap ? x.sa : x.sb;
  p.offsets = x.offsets;
  p.num_groups = x.groups;
  p.status = x.status;
  const long long group_bytes = x.groups > 1 ? x.b_group_bytes : x.ldb;
  const int rows_a = swap ? bn : BM, rows_b = swap ? BM : bn;
  p.x = x.x;
  p.ldx = x.ldx;
  p.x_vector = x.ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x.x) & 15) == 0;
  CUtensorMap ma, mb;
  if (x.A != nullptr && !make_map(&ma, x.A, x.a_mn != 0, x.M, x.K, 1, x.lda, x.lda, rows_a, 3)) return -1001;
  if (!make_map(&mb, x.B, x.b_mn != 0, x.N, x.K, x.groups, x.ldb, group_bytes, rows_b, 3)) return -2001;
  if (x.A == nullptr) ma = mb;  // not used
  const CUtensorMap &ta = swap ? mb : ma, &tb = swap ? ma : mb;
  long long b_tiles = (p.N + bn - 1) / bn;
  // every group can end inside a tile; a group without rows has none
  if (x.offsets != nullptr) b_tiles = p.N / bn + (x.groups < p.N ? x.groups : p.N);
  const long long tiles = b_tiles * ((p.M + BM - 1) / BM);
  if (x.A == nullptr)
    return many ? launch_small<16, true, true, true>(ta, tb, p, tiles, dev, stream) : launch_small<16, true, true>(ta, tb, p, tiles, dev, stream);
  if (swap) {
    switch (bn) {
      case 16: if (many) return launch_small<16, true, false, true>(ta, tb, p, tiles, dev, stream);
               return launch_small<16, true>(ta, tb, p, tiles, dev, stream);
      case 32: return launch_small<32, true>(ta, tb, p, tiles, dev, stream);
      case 64: return launch_small<64, true>(ta, tb, p, tiles, dev, stream);
      default: return launch_small<128, true>(ta, tb, p, tiles, dev, stream);
    }
  }
  return launch_small<128, false>(ta, tb, p, tiles, dev, stream);
}

// How many parts the reduction of `tiles` small tiles is cut into: what leaves the busiest SM the fewest blocks to work through,
// while all CTAs are resident (two per SM) and a part is two blocks at least. Of equally good ones the fewest; where weights are
// streamed for few tokens (`stream`) the most, because two CTAs hide each other's latencies (1 x 4096 x 11008: 17.2 us in 4 parts,
// 12.9 in 8).
static int split(long long tiles, long long kb, int sms, bool stream) {
  int best = 1;
  long long least = 0;
  for (int parts = 1; parts <= 8; ++parts) {
    if (parts > 1 && (tiles * parts > 2 * sms || kb < 2 * parts)) break;
    const long long load = ((tiles * parts + sms - 1) / sms) * ((kb + parts - 1) / parts);
    if (parts == 1 || load < least || (stream && load == least)) {
      best = parts;
      least = load;
    }
  }
  return best;
}

// Which kernel. The pair kernel does four times the work of a 128 x 128 tile per block on two SMs and is as fast per block, so it
// takes whatever fills a fair part of the 74 pairs; the 128-row kernel takes few tokens (weights on the wide side), and products
// of so few tiles that cutting the reduction gains more. Microseconds, measured back to back on random operands:
//   pair:             5 + 0.43 per block and wave of 256 x 256 tiles   (1024 x 4096 x 4096: 18.8, 2048 x 2048 x 2048: 13.2)
//   128-row, 128 wide 5.5 + 0.5 per block and wave of 128 x 128 tiles  (38.1 and 25.3), 0.7 more for a cut reduction
// The BN side of the small kernel for groups of `mean` rows (or so many rows without groups). 64 groups of 1024 x 2048 with rows at random,
// microseconds (in timer steps of 2) of the product alone from cold L2, for 16, 32, 64 and 128 columns and for pairs of CTAs, which run()
// takes above 128:
//   mean   8:  37   37   39   41   45        mean  48:  68   51   41   43   47        mean 128:   -   88   66   55   49
//   mean  16:  43   39   39   41   45        mean  64:   -   59   47   43   47        mean 160:   -    -   76   66   49
//   mean  32:  55   45   41   41   45        mean  96:   -   72   55   47   49        mean 256:   -    -  100   80   59
static int small_width(long long mean, bool grouped) {
  if (grouped) return mean <= 8 ? 16 : mean <= 16 ? 32 : mean <= 48 ? 64 : 128;
  return mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : 128;
}
// Whether the rows of A (M of them in `groups` groups) are quantised inside the product.
static bool fused(int M, int groups, bool grouped) { return small_width(grouped ? M / groups : M, grouped) == 16; }

static int run(const Product& x, cudaStream_t stream) {
  const int dev = current_device(), sms = num_sms(dev);
  if (sms <= 0) return -3;
  const long long kb = (x.K + BKE - 1) / BKE;
  const long long tiles_n = (x.N + 127) / 128;
  if (x.offsets != nullptr) {
    const long long mean = x.M / x.groups;  // rows of a group
    if (mean > 128) return run_pair(x, dev, stream);
    const int bn = small_width(mean, true);
    const long long used = x.groups < x.M ? x.groups : x.M;
    const int parts = split(used * tiles_n, kb, sms, true);
    // rows that fall on the groups evenly at random leave some without any
    const double some = x.groups * (1.0 - std::exp(-static_cast<double>(x.M) / x.groups));
    return run_small(x, true, bn, parts, parts == 1 && bn == 16 && fuller_with_three(some * tiles_n, sms), dev, stream);
  }
  if (x.M <= 128 && !x.a_mn) {
    const int bn = small_width(x.M, false);
    const int parts = split(tiles_n, kb, sms, true);
    return run_small(x, true, bn, parts, parts == 1 && bn == 16 && fuller_with_three(static_cast<double>(tiles_n), sms), dev, stream);
  }
  const long long pair_tiles = static_cast<long long>((x.M + 255) / 256) * ((x.N + 255) / 256);
  const long long small_tiles = static_cast<long long>((x.M + 127) / 128) * tiles_n;
  const int parts = split(small_tiles, kb, sms, false), pairs = sms / 2;
  const double pair_us = 5.0 + 0.43 * static_cast<double>(kb * ((pair_tiles + pairs - 1) / pairs));
  const double small_us = 5.5 + 0.5 * static_cast<double>(((kb + parts - 1) / parts) * ((small_tiles * parts + sms - 1) / sms)) + (parts > 1 ? 0.7 : 0.0);
  return small_us < pair_us ? run_small(x, false, 128, parts, false, dev, stream) : run_pair(x, dev, stream);
}

}  // namespace blk
}  // namespace ocb

using namespace ocb;

static int gemm_block_fp8(const void* A, const void* x, long long ldx, const void* B, void* C, const float* sa, const float* sb,
                          const int* offsets, int num_groups, int M, int N, int K, long long lda, long long ldb, long long ldc,
                          long long b_group_bytes, long long sa_k, long long sa_i, int sa_shift, long long sb_k, long long sb_i,
                          long long sb_g, int sb_shift, int a_mn, int b_mn, int epilogue, int* status, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || K <= 0 || num_groups <= 0) return 0;
  if ((lda % 16) != 0 || (ldb % 16) != 0 || (b_group_bytes % 16) != 0 || (reinterpret_cast<uintptr_t>(A) & 15) ||
      (reinterpret_cast<uintptr_t>(B) & 15) || (A != nullptr && sa == nullptr) || sb == nullptr)
    return -1;
  // sizes are rounded up to tiles in 32 bits
  if (M > 0x7fffffff - 512 || N > 0x7fffffff - 512 || K > 0x7fffffff - 512) return -1;
  if ((sa_shift != 0 && sa_shift != 7) || (sb_shift != 0 && sb_shift != 7) || (offsets != nullptr && a_mn)) return -1;
  if (epilogue < blk::EPI_BF16 || epilogue > blk::EPI_F32) return -1;
  blk::Product p;
  p.A = A;
  p.B = B;
  p.x = reinterpret_cast<const __nv_bfloat16*>(x);
  p.ldx = ldx;
  p.C = C;
  p.M = M;
  p.N = N;
  p.K = K;
  p.groups = num_groups;
  p.lda = lda;
  p.ldb = ldb;
  p.ldc = ldc;
  p.b_group_bytes = b_group_bytes;
  p.sa = {sa, sa_k, sa_i, 0, sa_shift};
  p.sb = {sb, sb_k, sb_i, sb_g, sb_shift};
  p.a_mn = a_mn;
  p.b_mn = b_mn;
  p.epi = epilogue;
  p.offsets = offsets;
  p.status = status;
  return blk::run(p, stream);
}

// See ocb_api.h.
extern "C" int ocb_gemm_block_fp8(const void* A, const void* B, void* C, const float* sa, const float* sb, const int* offsets,
                                  int num_groups, int M, int N, int K, long long lda, long long ldb, long long ldc,
                                  long long b_group_bytes, long long sa_k, long long sa_i, int sa_shift, long long sb_k,
                                  long long sb_i, long long sb_g, int sb_shift, int a_mn, int b_mn, int epilogue, int* status,
                                  cudaStream_t stream) {
  if (A == nullptr) return -1;
  return gemm_block_fp8(A, nullptr, 0, B, C, sa, sb, offsets, num_groups, M, N, K, lda, ldb, ldc, b_group_bytes, sa_k, sa_i,
                        sa_shift, sb_k, sb_i, sb_g, sb_shift, a_mn, b_mn, epilogue, status, stream);
}

extern "C" int ocb_linear_block_fp8_fused(int M, int num_groups, int grouped) { return blk::fused(M, num_groups < 1 ? 1 : num_groups, grouped != 0); }

// See ocb_api.h.
extern "C" int ocb_linear_block_fp8(const void* x, long long ldx, void* q_row, float* s_row, void* q_col, float* s_col,
                                    long long ldq, const void* W, const float* sw, const int* offsets, int num_groups, void* C,
                                    int M, int N, int K, long long ldw, long long w_group_bytes, long long sw_k, long long sw_i,
                                    long long sw_g, int w_mn, long long ldc, int epilogue, int* status, cudaStream_t stream) {
  const bool inside = q_row == nullptr;
  if (inside && !blk::fused(M, num_groups < 1 ? 1 : num_groups, offsets != nullptr)) return -1;
  if (!inside || q_col != nullptr) {
    const int rc = ocb_quantize_block_fp8(x, q_row, s_row, q_col, s_col, nullptr, nullptr, 1, M, K, ldx, ldq, 0, 0, stream);
    if (rc != 0) return rc;
  }
  return gemm_block_fp8(q_row, x, ldx, W, C, s_row, sw, offsets, num_groups, M, N, K, inside ? 0 : ldq, ldw, ldc, w_group_bytes,
                        M, 1, 0, sw_k, sw_i, sw_g, 7, 0, w_mn, epilogue, status, stream);
}
