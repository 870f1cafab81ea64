// 8-bit GEMM with one scale per block of 128 along K, on the 5th-generation tensor cores.
//
//   D[m, n] = epilogue( sum_b sA[b, m] sB[b, n] sum_{k in block b} A[m, k] B[n, k] )
//
// A (M, K) and B (N, K) are e4m3 or e5m2, both K-major, rows padded to 16 bytes. sA has one scale per
// row and K block (or per 128 rows), sB one per 128 rows (weights) or one per row (weight gradients).
//
// CTA = 4 control warps (two idle) + 8 epilogue warps, one CTA per SM, persistent over output tiles of
// 128 x 128, or 256 x 256 by a pair of CTAs (cta_group::2: each CTA holds its 128 rows of A and half of
// B in its shared memory and its 128 rows of the products in its TMEM; the even CTA issues the MMAs):
//   warp 0     TMA producer: 128-byte wide tiles of A and B into a ring of shared-memory stages.
//   warp 1     MMA issuer: four K = 32 steps of tcgen05.mma (kind::f8f6f4) per K block into one of the
//              TMEM units, which holds the products of that K block alone. One thread issues everything,
//              so its instructions count: descriptors advance by additions.
//   warps 4..  epilogue: read a unit with tcgen05.ld, multiply by the scales and add in fp32 registers
//              (a warp owns 32 rows x BN / 2 columns) while the tensor core fills the other units. A lane
//              fetches its row's scale two K blocks ahead; with a scale per row of B also its share
//              of the warp's column scales, which the lanes pass on through a small double-buffered strip
//              of shared memory that belongs to the warp alone.
//              After the last block the warp applies bias, GELU, LayerScale and residual, rounds into 128-byte
//              swizzled rows of shared memory and leaves the stores (or, to accumulate, the additions) to TMA
//              while it goes on with the next tile; the residual came into the same rows by TMA during the K
//              loop. Odd widths and a few combinations take a second form, which turns the sums through
//              shared memory so that four lanes hold 16 columns of one row.
// What bounds it: the additions. 128 x 256 sums a K block and CTA are 256 FMA cycles of the SM at best, with a
// scale per column twice that, against 512 cycles of MMA; with both emptied of arithmetic the same pipeline runs
// at 2590 TFLOP/s. Measured (ten launches from a graph, bf16 out): 8192^3 2000 TFLOP/s with scales per weight block, 1330
// with a scale per row of both; 16384 x 1280 x 5120 (M x N x K) 128 us (1680 TFLOP/s), with a residual 137 us (228 us when
// the lanes fetched it), 16384 x 5120 x 1280 128 us, with GELU 230 us, with its pre-activation as well 246 us; 5120 x 1280 x
// 16384 with row scales to fp32 192 us, added to a gradient 258 us.
// Tried and slower: sums by packed f32x2 FMAs (1620 at 8192^3), 16 epilogue warps of 64 columns (1315), stores by
// the lanes instead of TMA (16384 x 5120 x 1280: 155 us).
// The scales are applied in fp32 outside the tensor core, so they may be any finite fp32 numbers, and no sum
// longer than 128 products is left to the tensor core's own accumulation. A term is sum (sa sb) with a scale per block of
// B and (sum sa) sb with one per row. Where the bracket may be past fp32's range though the term is not, the row is summed
// in units of up to 2^40 (in place, in branches that other rows never take: 2 to 5 % of the time of the calls above for the
// tests, against 10 to 50 % for longer arithmetic beside or inside the loop over K). Of the other end: products of scales
// below 2^-149 count as zero, which leaves out less than 2^-125 a block (2^-111 with two e5m2 operands).
//
// All waits are bounded (see common.cuh); on a timeout the kernel records an error code, drains the
// copies and MMAs it issued, frees its tensor memory and returns.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <atomic>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "block_ops.h"
#include "common.cuh"
#include "errors.h"
#include "gemm_common.cuh"

namespace mia {

constexpr int kF8K = 128;         // K block: bytes of a swizzled row, and the scales' block
constexpr int kF8EpiWarps = 8;
constexpr int kF8FirstEpi = 4;    // warps 0..3: producer, MMA issuer, two idle
constexpr int kF8Threads = 32 * (kF8FirstEpi + kF8EpiWarps);
constexpr int kF8ATile = 128 * kF8K;

struct Fp8Operands {
  const float* sa;
  int64_t sa_ld;
  int sa_shift;  // 0: a scale per row, 7: per 128 rows
  const float* sb;
  int64_t sb_ld;
  int a_format, b_format;  // 0 = e4m3, 1 = e5m2
  // A scale per row of B: scales of A from this power of two on may carry their product with a sum past the range.
  // 128 products are below 2^25, 2^32 or 2^39 for none, one or two e5m2 operands.
  int safe_exponent;
  float safe_scale;
};

template <int CG, int BN, int STAGES>
struct F8Smem {
  static constexpr int kBTile = BN / CG * kF8K;
  static constexpr int kStage = kF8ATile + kBTile;
  static constexpr int kScales = kF8EpiWarps * 2 * (BN / 2) * 4;  // two strips for each epilogue warp
  // Staging of the stores: BN / 128 boxes of 32 rows x 128 bytes for each epilogue warp.
  static constexpr int kWarpStaging = BN / 128 * 4096;
  static constexpr int kStaging = kF8EpiWarps * kWarpStaging;
  static constexpr int kBytes = STAGES * kStage + kStaging + kScales + 1024 /*align*/ + 256 /*barriers*/;
};

// One lane of a converged warp. Unlike a test of the lane index, the compiler knows that a single thread
// passes it, and keeps the operands of the TMA and tcgen05 instructions behind it in uniform registers:
// the four MMAs of a K block then issue in their execution time instead of about 140 cycles each.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

// A load that stays where it is written: the compiler would move a plain one down to its first use, behind
// the waits it is meant to overlap.
__device__ __forceinline__ float load_now(const float* p) {
  float v;
  asm volatile("ld.global.nc.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}

// A staged box to global memory (clipped at the tensor's edges), stored or added; bulk groups belong to
// the thread that issues them.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void tma_add_2d(const CUtensorMap* map, const void* src, int c0, int c1) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// 16 lanes x 32 columns: thread t receives, of every eight columns g, columns 2 (t % 4) and + 1 of row t / 4
// in r[4 g], r[4 g + 1] and of row t / 4 + 8 in r[4 g + 2], r[4 g + 3].
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld_32x32b_x32(taddr, r); }
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) { tmem_ld_wait_regs(r); }
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) { tmem_ld_wait_regs16(r); }

// Whether `bar` has completed phase `parity`, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// mbar_wait for a whole warp: one lane polls, a shuffle gives the others its answer, and __syncwarp what the
// barrier ordered: a shuffle alone orders no memory. Polling with all lanes costs 32 barrier operations a
// try, and lanes that see the barrier complete in different tries would have to be brought together before the
// warp-wide TMEM loads that follow.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err,
                                               int code) {
  int ok = 0;
  if (threadIdx.x % 32 == 0) ok = mbar_wait(bar, parity, abort_flag, err, code) ? 1 : 0;
  ok = __shfl_sync(0xffffffffu, ok, 0);
  __syncwarp();
  return ok != 0;
}

// One K block: four steps of 32, the first of which overwrites D. A step of 32 bytes along the swizzled rows
// adds 2 to the address field of either descriptor.
#define MIA_MMA_F8_BLOCK(GROUP)                                                          \
  asm volatile(                                                                          \
      "{\n\t.reg .pred f, t;\n\t.reg .b64 a, b;\n\t"                                     \
      "setp.ne.b32 f, 0, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"                                 \
      "tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], %1, %2, %3, f;\n\t"           \
      "add.s64 a, %1, 2;\n\tadd.s64 b, %2, 2;\n\t"                                       \
      "tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], a, b, %3, t;\n\t"             \
      "add.s64 a, %1, 4;\n\tadd.s64 b, %2, 4;\n\t"                                       \
      "tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], a, b, %3, t;\n\t"             \
      "add.s64 a, %1, 6;\n\tadd.s64 b, %2, 6;\n\t"                                       \
      "tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], a, b, %3, t;\n\t}" ::"r"(d_tmem), \
      "l"(a_desc), "l"(b_desc), "r"(idesc))

template <int CG>
__device__ __forceinline__ void tc_mma_f8_block(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc) {
  if constexpr (CG == 2) MIA_MMA_F8_BLOCK("2");
  else MIA_MMA_F8_BLOCK("1");
}

// Larger units for the sums of rows whose scales would carry a term past fp32's range on the way to a product that lies
// in it: as large as that row needs, up to 2^40. More is not needed: a sum is zero or at least 2^-32 (e5m2) in size, so that
// what is past the range in those units is past it in the result.
constexpr int kF8HalfUnits = 20;
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// e with |v| < 2^e (infinities and NaN: 2^128)
__device__ __forceinline__ int exponent_above(float v) { return min((int)(__float_as_uint(v) >> 23 & 255), 254) - 126; }

// 128 accumulators a thread (BN = 256) need more than the 168 registers that 384 threads can start with:
// the four control warps hand theirs down. 128 * 40 + 256 * 232 = 384 * 168.
constexpr int kF8LaunchRegs = 168, kF8ControlRegs = 40, kF8EpilogueRegs = 232;
static_assert(128 * kF8ControlRegs + 32 * kF8EpiWarps * kF8EpilogueRegs <= kF8Threads * kF8LaunchRegs, "register split");

// Four columns n .. n + 3 of row m: bias, GELU (keeping the pre-activation), LayerScale, residual,
// accumulation, store. `vec`: N % 4 == 0 and all four columns exist.
__device__ __forceinline__ void fp8_store4(const GemmParams& p, int64_t m, int n, float4 acc, bool vec) {
  float v[4] = {acc.x, acc.y, acc.z, acc.w};
  const int64_t at = m * p.N + n;
  const int count = vec ? 4 : min(4, p.N - n);
  auto vec_f32 = [&](const float* src, float (&o)[4]) {
    if (vec) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(src));
      o[0] = f.x; o[1] = f.y; o[2] = f.z; o[3] = f.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = j < count ? src[j] : 0.f;
    }
  };
  auto load_bf16 = [&](const __nv_bfloat16* src, float (&o)[4]) {
    if (vec) {
      const uint2 u = *reinterpret_cast<const uint2*>(src);
      o[0] = bf16_lo(u.x); o[1] = bf16_hi(u.x); o[2] = bf16_lo(u.y); o[3] = bf16_hi(u.y);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = j < count ? __bfloat162float(src[j]) : 0.f;
    }
  };
  auto store_bf16 = [&](__nv_bfloat16* dst) {
    if (vec) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < count) dst[j] = __float2bfloat16_rn(v[j]);
    }
  };
  float t[4];
  if (p.bias != nullptr) {
    vec_f32(p.bias + n, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += t[j];
  }
  if (p.act == kActGelu) {
    if (p.aux_out != nullptr) store_bf16(p.aux_out + at);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = gelu_erf(v[j]);
  }
  if (p.gamma != nullptr) {
    vec_f32(p.gamma + n, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= t[j];
  }
  if (p.residual != nullptr) {
    load_bf16(p.residual + at, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += t[j];
  }
  if (p.d_fp32) {
    float* dst = reinterpret_cast<float*>(p.D) + at;
    if (vec) {
      float4* d4 = reinterpret_cast<float4*>(dst);
      if (p.accumulate) {
        const float4 old = *d4;
        v[0] += old.x; v[1] += old.y; v[2] += old.z; v[3] += old.w;
      }
      *d4 = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < count) dst[j] = p.accumulate ? dst[j] + v[j] : v[j];
    }
  } else {
    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p.D) + at;
    if (p.accumulate) {
      load_bf16(dst, t);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += t[j];
    }
    store_bf16(dst);
  }
}

template <int CG, int BN, int HALVES, int STAGES, bool SB_ROW, bool FULL>
__global__ void __launch_bounds__(kF8Threads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmAux,
                    const __grid_constant__ CUtensorMap tmRes,
                    const GemmParams p, const Fp8Operands o) {
  using L = F8Smem<CG, BN, STAGES>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smA = smem;
  uint8_t* smB = smem + STAGES * kF8ATile;
  uint8_t* smT = smem + STAGES * L::kStage;
  float* smS = reinterpret_cast<float*>(smT + L::kStaging);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smT + L::kStaging + L::kScales);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;  // [kUnits]
  uint64_t* tempty_bar = tfull_bar + 4;      // [kUnits]
  uint64_t* drain_bar = tempty_bar + 4;      // [1]
  uint64_t* res_bar = drain_bar + 1;         // [kF8EpiWarps]
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(res_bar + kF8EpiWarps);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int rank = CG == 2 ? (int)cluster_ctarank() : 0;
  const int worker = blockIdx.x / CG, workers = gridDim.x / CG;
  constexpr int kUnitCols = BN / HALVES;
  constexpr int kUnits = 512 / kUnitCols < 4 ? 512 / kUnitCols : 4;
  constexpr uint32_t kTmemCols = kUnits * kUnitCols;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);   // the even CTA's producer announces the bytes of the pair
      mbar_init(&empty_bar[s], 1);  // one commit of the MMA issuer, to both CTAs
    }
    for (int a = 0; a < kUnits; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], CG * kF8EpiWarps / HALVES);  // the unit's epilogue warps of the pair, on the even CTA
    }
    mbar_init(drain_bar, 1);
    for (int w = 0; w < kF8EpiWarps; ++w) mbar_init(&res_bar[w], 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(tmem_base_slot, kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_base_slot, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  // Work unit -> output tile (m fastest, so that concurrent CTAs share tiles of B) and its K blocks.
  const int total_k = (p.K + kF8K - 1) / kF8K;
  struct Unit {
    int m0, n0, kb0, num_k;
  };
  auto work_unit = [&](int index) {
    const int tiles = p.num_m_tiles * p.num_n_tiles, tile = index % tiles;
    const int kb0 = index / tiles * p.k_blocks_per_split;
    return Unit{tile % p.num_m_tiles * (128 * CG), tile / p.num_m_tiles * BN, kb0, min(p.k_blocks_per_split, total_k - kb0)};
  };

  if (warp < kF8FirstEpi) {
    if constexpr (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kF8ControlRegs));
    if (warp == 0 && elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      bool ok = true;
      for (int tile = worker; tile < p.num_tiles && ok; tile += workers) {
        const Unit u = work_unit(tile);
        const int m0 = u.m0 + 128 * rank, n0 = u.n0 + BN / CG * rank;
        for (int kb = u.kb0; kb < u.kb0 + u.num_k; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.err, kErrFp8ProducerWait)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], CG * L::kStage);
          if constexpr (CG == 2) {
            tma_load_2d_pair(smA + stage * kF8ATile, &tmA, &full_bar[stage], kb * kF8K, m0);
            tma_load_2d_pair(smB + stage * L::kBTile, &tmB, &full_bar[stage], kb * kF8K, n0);
          } else {
            tma_load_2d(smA + stage * kF8ATile, &tmA, &full_bar[stage], kb * kF8K, m0);
            tma_load_2d(smB + stage * L::kBTile, &tmB, &full_bar[stage], kb * kF8K, n0);
          }
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && rank == 0) {  // let the copies in flight land before this CTA's shared memory goes away
        int s = stage, ph = phase;
        for (int i = 0; i < STAGES && i < issued; ++i) {
          if (--s < 0) {
            s = STAGES - 1;
            ph ^= 1;
          }
          mbar_wait(&full_bar[s], ph, nullptr, nullptr, 0);
        }
      }
    } else if (warp == 1 && rank == 0 && elect_one()) {
      const uint32_t idesc = make_idesc_f8(128 * CG, kUnitCols, o.a_format, o.b_format);
      const uint64_t a_desc0 = make_sdesc_sw128(smem_u32(smA), 16, 1024);
      const uint64_t b_desc0 = make_sdesc_sw128(smem_u32(smB), 16, 1024);
      uint64_t a_desc = a_desc0, b_desc = b_desc0;
      uint32_t d_tmem = tmem_base;
      int stage = 0;
      uint32_t phase = 0;
      int unit = 0;
      uint32_t unit_phase = 0;
      bool ok = true;
      bool any_mma = false;
      for (int tile = worker; tile < p.num_tiles && ok; tile += workers) {
        const int num_k = work_unit(tile).num_k;
        for (int kb = 0; kb < num_k && ok; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, abort_flag, p.err, kErrFp8MmaWait)) {
            ok = false;
            break;
          }
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            if (!mbar_wait(&tempty_bar[unit], unit_phase ^ 1, abort_flag, p.err, kErrFp8MmaWait)) {
              ok = false;
              break;
            }
            tc_fence_after();
            tc_mma_f8_block<CG>(d_tmem, a_desc, b_desc + h * ((kUnitCols / CG * kF8K) >> 4), idesc);
            any_mma = true;
            if constexpr (CG == 2) tc_commit_pair_both(&tfull_bar[unit]);
            else tc_commit(&tfull_bar[unit]);
            d_tmem += kUnitCols;
            if (++unit == kUnits) {
              unit = 0;
              unit_phase ^= 1;
              d_tmem = tmem_base;
            }
          }
          if (!ok) break;
          if constexpr (CG == 2) tc_commit_pair_both(&empty_bar[stage]);
          else tc_commit(&empty_bar[stage]);
          a_desc += kF8ATile >> 4;
          b_desc += L::kBTile >> 4;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
            a_desc = a_desc0;
            b_desc = b_desc0;
          }
        }
      }
      if (!ok && any_mma) {
        if constexpr (CG == 2) tc_commit_pair_both(drain_bar);
        else tc_commit(drain_bar);
        mbar_wait(drain_bar, 0, nullptr, nullptr, 0);
      }
    }
  } else {
    if constexpr (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kF8EpilogueRegs));
    const int lane_group = warp % 4;                // TMEM lanes 32 * lane_group .. + 31
    const int part = (warp - kF8FirstEpi) / 4;
    constexpr int kCols = BN / 2;
    // How a warp's 32 rows x kCols columns lie in its registers. With a scale per block: lane = row, 32 columns
    // a load, so that a thread multiplies everything by one number. With a scale per column that layout would
    // read kCols scales a thread from shared memory (at 128 bytes a cycle the whole SM twice the time of the
    // MMAs), so a load brings 16 rows x 32 columns instead: a thread has two columns of every eight, in four rows.
    constexpr int kWidth = SB_ROW ? 16 : 32;  // registers a load fills: two loads in flight fit beside the sums
    constexpr int kChunks = kCols / kWidth;
    constexpr int kRowsT = SB_ROW ? 4 : 1;    // rows a thread holds: 8 i + lane / 4, or its lane
    const int row_t = SB_ROW ? lane / 4 : lane;
    auto row_of = [](int j) { return SB_ROW ? (j >> 1 & 1) + 2 * (j >> 4 & 1) : 0; };  // of register j: which of kRowsT
    auto chunk_at = [](int c) { return SB_ROW ? (c / 2) * 32 + ((uint32_t)(c % 2 * 16) << 16) : c * 32; };  // TMEM offset
    constexpr int kLaneCols = kCols / 32;
    // One unit: the warps' halves are its two column ranges. Two units (a 256-wide tile of a pair): unit h
    // holds columns 64 h .. + 63 of the even CTA's 128 rows of B, then the same of the odd CTA's.
    const int half = HALVES == 2 ? part : 0;
    const int t_col = HALVES == 2 ? 0 : part * kCols;
    const int n_col = HALVES == 2 ? half * 64 : part * kCols;
    auto column = [](int c) { return HALVES == 2 && c >= 64 ? c + 64 : c; };  // of the warp's kCols
    float* strip = smS + (warp - kF8FirstEpi) * 2 * kCols;
    uint8_t* const staging = smT + (warp - kF8FirstEpi) * L::kWarpStaging;
    int unit = half;
    uint32_t unit_phase = 0;
    bool ok = true, ready = false;
    constexpr int kBoxes = L::kWarpStaging / 4096;  // of 32 rows x 64 bf16 columns
    uint64_t* const my_res = &res_bar[warp - kF8FirstEpi];
    uint32_t res_phase = 0;
    bool res_pending = false;
    // The largest scales of a tile's blocks of B (kSb of them, see below), spread over the lanes.
    constexpr int kSb = SB_ROW ? kLaneCols : HALVES;
    float b_tile[kSb];
    auto fetch_b_tile = [&](int index) {
      if (index >= p.num_tiles) return;
      const Unit v = work_unit(index);
#pragma unroll
      for (int i = 0; i < kSb; ++i) {
        const float* const from = o.sb + v.kb0 * o.sb_ld + (min(v.n0 + n_col + 128 * i, p.N - 1) >> 7);
        b_tile[i] = load_now(from + min(lane, v.num_k - 1) * o.sb_ld);
        for (int kb = lane + 32; kb < v.num_k; kb += 32) b_tile[i] = fmaxf(fabsf(b_tile[i]), fabsf(load_now(from + kb * o.sb_ld)));
      }
    };
    if (!SB_ROW) fetch_b_tile(worker);
    for (int tile = worker; tile < p.num_tiles && ok; tile += workers) {
      const Unit u = work_unit(tile);
      const int num_k = u.num_k;
      const int m_warp = u.m0 + 128 * rank + lane_group * 32;
      const int n0 = u.n0 + n_col;
      const uint32_t t_row = tmem_base + ((uint32_t)(lane_group * 32) << 16) + t_col;
      float sum[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j) sum[j] = 0.f;
      // Scales: this row's, and of B either one per block the warp's columns lie in (one, or two with HALVES
      // == 2) or, with a scale per row of B, those of columns n0 + column(32 i) + lane. Rows and columns past
      // the edge fetch the last one: their sums are never stored.
      const float* sa = o.sa + u.kb0 * o.sa_ld;
      int sa_at[kRowsT];
#pragma unroll
      for (int i = 0; i < kRowsT; ++i) sa_at[i] = min(m_warp + row_t + 8 * i, p.M - 1) >> o.sa_shift;
      const float* sb = o.sb + u.kb0 * o.sb_ld;
      int sb_at[kSb];
#pragma unroll
      for (int i = 0; i < kSb; ++i)
        sb_at[i] = SB_ROW ? min(n0 + column(32 * i) + lane, p.N - 1) : min(n0 + 128 * i, p.N - 1) >> 7;
      float sa_ahead[2][kRowsT], sb_ahead[2][kSb];  // of K blocks kb and kb + 1
#pragma unroll
      for (int d = 0; d < 2; ++d) {
#pragma unroll
        for (int i = 0; i < kRowsT; ++i) sa_ahead[d][i] = load_now(sa + sa_at[i]);
#pragma unroll
        for (int i = 0; i < kSb; ++i) sb_ahead[d][i] = load_now(sb + sb_at[i]);
        if (d + 1 < num_k) {
          sa += o.sa_ld;
          sb += o.sb_ld;
        }
      }
      // The rows' units. With a scale per row of B: 1 / down, above 1 only while a block with a large row scale is added
      // (back in units of 1 a sum overflows where the result would). Else 1 / down^2 for the whole tile, half of it for
      // either scale, so that no scale of the quantiser (2^-126 and more) is lost. Either way a row with such a block keeps
      // nothing below 2^-109. `large`: some row of the warp has them.
      float down[kRowsT];
#pragma unroll
      for (int i = 0; i < kRowsT; ++i) down[i] = 1.f;
      bool large = false;
      if (!SB_ROW) {
        // The product of two scales can be past the range only if one of B is above 1 (weights beyond 448): then
        // the rows' own products decide. B's scales of this tile came a tile ahead.
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kSb; ++i) top = fmaxf(top, fabsf(b_tile[i]));
        large = __any_sync(0xffffffffu, top >= 1.f);
        if (large) {
          int most = 128;  // above the exponents of every product
          for (int kb = 0; kb < num_k; ++kb) {
            const int ea = exponent_above(o.sa[(u.kb0 + kb) * o.sa_ld + sa_at[0]]);
#pragma unroll
            for (int i = 0; i < kSb; ++i)
              most = max(most, ea + exponent_above(o.sb[(u.kb0 + kb) * o.sb_ld + sb_at[i]]));
          }
          down[0] = power_of_two(-min((most - 127) / 2, kF8HalfUnits));
        }
      }
      if (!FULL && p.residual != nullptr) {
        // this warp's part of the residual, into the staging rows its outputs will leave from; outside the K loop,
        // where the test alone cost the calls without a residual a tenth of their time
        if (elect_one()) {
          bulk_wait_read();  // the last tile's stores have read them
          mbar_arrive_expect_tx(my_res, kBoxes * 4096);
#pragma unroll
          for (int box = 0; box < kBoxes; ++box)
            tma_load_2d(staging + box * 4096, &tmRes, my_res, n0 + column(box * 64), m_warp);
        }
        __syncwarp();
        res_pending = true;
      }
      // Whether a row's scale of the coming block is large enough to carry its product with a sum past the range.
      auto large_rows = [&] {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < kRowsT; ++i) top = fmaxf(top, fabsf(sa_ahead[0][i]));
        return top >= o.safe_scale;
      };
      // The usual block with a scale per row of B: its unit is known to be full, and its row scales not to be large. One
      // branch for both tests: a second one in this loop costs a tenth of the time.
      bool usual = false;
      for (int kb = 0; kb < num_k; ++kb) {
        if (SB_ROW ? !usual : !ready) {
          if (!ready && !mbar_wait_warp(&tfull_bar[unit], unit_phase, abort_flag, p.err, kErrFp8EpilogueWait)) {
            ok = false;
            break;
          }
          if (SB_ROW) large = large || __any_sync(0xffffffffu, large_rows());
          if (SB_ROW && large) {  // in place, so that the loop below keeps its registers
#pragma unroll
            for (int i = 0; i < kRowsT; ++i) {
              const float unit = power_of_two(-max(exponent_above(sa_ahead[0][i]) - o.safe_exponent, 0));
              const float f = unit / down[i];
              down[i] = unit;
#pragma unroll
              for (int j = 0; j < kCols; ++j)
                if (row_of(j) == i) sum[j] *= f;
              sa_ahead[0][i] *= down[i];
            }
          }
        }
        tc_fence_after();
        uint32_t r[2][kWidth];  // the next columns are on their way while these are added
        const uint32_t t_unit = t_row + unit * kUnitCols;
        tmem_load(t_unit, r[0]);
        // behind the first load: this block's scales into place, those of two blocks on under way
        float s1[SB_ROW ? kRowsT : kSb];
        float* const sbv = strip + (kb & 1) * kCols;
        if (SB_ROW) {
#pragma unroll
          for (int i = 0; i < kRowsT; ++i) s1[i] = sa_ahead[0][i];
          // the strip of two K blocks ago: every lane has passed the barrier after reading it
#pragma unroll
          for (int i = 0; i < kSb; ++i) sbv[lane + 32 * i] = sb_ahead[0][i];
          __syncwarp();
        } else {
#pragma unroll
          for (int i = 0; i < kSb; ++i) {
            const float s = (sa_ahead[0][0] * down[0]) * (sb_ahead[0][i] * down[0]);
            s1[i] = fabsf(s) > FLT_MAX ? copysignf(FLT_MAX, s) : s;  // a zero sum stays zero, and NaN NaN
          }
        }
#pragma unroll
        for (int i = 0; i < kRowsT; ++i) {
          sa_ahead[0][i] = sa_ahead[1][i];
          sa_ahead[1][i] = load_now(sa + sa_at[i]);
        }
#pragma unroll
        for (int i = 0; i < kSb; ++i) {
          sb_ahead[0][i] = sb_ahead[1][i];
          sb_ahead[1][i] = load_now(sb + sb_at[i]);
        }
        if (kb + 3 < num_k) {
          sa += o.sa_ld;
          sb += o.sb_ld;
        }
        int next = unit + HALVES;
        const uint32_t next_phase = next >= kUnits ? unit_phase ^ 1 : unit_phase;
        next = next >= kUnits ? next - kUnits : next;
        int seen = 0;
        float2 bs[2][4];  // scales of this thread's columns of 32, fetched one step ahead as well
        const float2* const my_scales = reinterpret_cast<const float2*>(sbv) + (lane & 3);
        if (SB_ROW) {
#pragma unroll
          for (int g = 0; g < 4; ++g) bs[0][g] = my_scales[g * 4];
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          uint32_t(&now)[kWidth] = r[c & 1];
          tmem_wait(now);
          if (c + 1 < kChunks) {
            tmem_load(t_unit + chunk_at(c + 1), r[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (CG == 2) mbar_arrive_cluster(&tempty_bar[unit], 0);
              else mbar_arrive(&tempty_bar[unit]);
              seen = mbar_test(&tfull_bar[next], next_phase) ? 1 : 0;  // answered while the last columns are added
            }
          }
          float* const x = sum + c * kWidth;
          if (SB_ROW) {
            if (c % 2 == 0 && c + 2 < kChunks) {
#pragma unroll
              for (int g = 0; g < 4; ++g) bs[(c / 2 + 1) & 1][g] = my_scales[(c / 2 + 1) * 16 + g * 4];
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float2 b = bs[(c / 2) & 1][g];
              const float lo = s1[(c % 2 * 2) % kRowsT], hi = s1[(c % 2 * 2 + 1) % kRowsT];
              x[4 * g] = fmaf(__uint_as_float(now[(4 * g) % kWidth]) * lo, b.x, x[4 * g]);
              x[4 * g + 1] = fmaf(__uint_as_float(now[(4 * g + 1) % kWidth]) * lo, b.y, x[4 * g + 1]);
              x[4 * g + 2] = fmaf(__uint_as_float(now[(4 * g + 2) % kWidth]) * hi, b.x, x[4 * g + 2]);
              x[4 * g + 3] = fmaf(__uint_as_float(now[(4 * g + 3) % kWidth]) * hi, b.y, x[4 * g + 3]);
            }
          } else {
#pragma unroll
            for (int q = 0; q < kWidth; ++q)
              x[q] = fmaf(__uint_as_float(now[q]), s1[!SB_ROW && kSb == 2 ? c * kWidth / 64 : 0], x[q]);
          }
        }
        if (SB_ROW) {
          const int news = __reduce_or_sync(0xffffffffu, seen | (large_rows() ? 2 : 0));
          __syncwarp();  // as in mbar_wait_warp
          ready = (news & 1) != 0;
          usual = news == 1 && !large;
        } else {
          ready = __shfl_sync(0xffffffffu, seen, 0) != 0;
          __syncwarp();  // as in mbar_wait_warp
        }
        unit = next;
        unit_phase = next_phase;
      }
      if (!ok) break;
      if (!SB_ROW) fetch_b_tile(tile + workers);
      if (large) {
#pragma unroll
        for (int j = 0; j < kCols; ++j) sum[j] *= 1.f / (SB_ROW ? down[row_of(j)] : down[0] * down[0]);
      }
      if constexpr (!FULL) {
        // sum = op(sum, vec[n]) for a vector over the columns
        auto per_column = [&](const float* vec, auto op) {
          if (SB_ROW) {
#pragma unroll
            for (int g = 0; g < kCols / 8; ++g) {  // eight columns: registers 32 (g / 4) + 4 (g % 4) .. + 3, and 16 on
              const int n = n0 + column(g * 8) + (lane & 3) * 2;
              const float2 v = n < p.N ? __ldg(reinterpret_cast<const float2*>(vec + n)) : make_float2(0.f, 0.f);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float* x = sum + g / 4 * 32 + i / 2 * 16 + g % 4 * 4 + i % 2 * 2;
                op(x[0], v.x);
                op(x[1], v.y);
              }
            }
          } else {
#pragma unroll
            for (int c = 0; c < kCols; c += 4) {
              const int n = n0 + column(c);
              const float4 v = n < p.N ? __ldg(reinterpret_cast<const float4*>(vec + n)) : make_float4(0.f, 0.f, 0.f, 0.f);
              op(sum[c], v.x);
              op(sum[c + 1], v.y);
              op(sum[c + 2], v.z);
              op(sum[c + 3], v.w);
            }
          }
        };
        if (p.bias != nullptr) per_column(p.bias, [](float& x, float v) { x += v; });
        // Boxes of 64 bf16 or 32 fp32 columns into 128-byte rows whose 16-byte pieces are XOR-swizzled with the
        // row's low three bits, as the tensor maps expect, from column `first` of the warp's on.
        auto stage = [&](const CUtensorMap* map, int first, auto wide, bool add) {
          constexpr bool kF32 = decltype(wide)::value;
          constexpr int kBoxCols = kF32 ? 32 : 64;
          if (elect_one()) bulk_wait_read();  // the staging rows are free again
          __syncwarp();
#pragma unroll
          for (int box = 0; box < kBoxes; ++box) {
            uint8_t* const at = staging + box * 4096;
            const float* const src = sum + first + box * kBoxCols;
            if constexpr (SB_ROW) {
#pragma unroll
              for (int g = 0; g < kBoxCols / 8; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int row = i * 8 + lane / 4;
                  const float* x = src + g / 4 * 32 + i / 2 * 16 + g % 4 * 4 + i % 2 * 2;
                  if constexpr (kF32)
                    *reinterpret_cast<float2*>(at + row * 128 + (((2 * g + (lane & 3) / 2) ^ (row & 7)) << 4) +
                                               (lane & 1) * 8) = make_float2(x[0], x[1]);
                  else
                    *reinterpret_cast<uint32_t*>(at + row * 128 + ((g ^ (row & 7)) << 4) + (lane & 3) * 4) =
                        pack_bf16x2(x[0], x[1]);
                }
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                uint4 u;
                if constexpr (kF32) {
                  const float* x = src + j * 4;
                  u = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
                } else {
                  const float* x = src + j * 8;
                  u = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                 pack_bf16x2(x[6], x[7]));
                }
                *reinterpret_cast<uint4*>(at + lane * 128 + ((j ^ (lane & 7)) << 4)) = u;
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (elect_one()) {
#pragma unroll
            for (int box = 0; box < kBoxes; ++box) {
              const int n = n0 + column(first + box * kBoxCols);
              if (n < p.N && m_warp < p.M) {
                if (add) tma_add_2d(map, staging + box * 4096, n, m_warp);
                else tma_store_2d(map, staging + box * 4096, n, m_warp);
              }
            }
            bulk_commit();
          }
        };
        if (p.act == kActGelu) {
          if (p.aux_out != nullptr) stage(&tmAux, 0, std::false_type{}, false);
#pragma unroll
          for (int c = 0; c < kCols; ++c) sum[c] = gelu_erf(sum[c]);
        }
        if (p.gamma != nullptr) per_column(p.gamma, [](float& x, float v) { x *= v; });
        if (p.residual != nullptr) {
          res_pending = false;
          if (!mbar_wait_warp(my_res, res_phase, abort_flag, p.err, kErrFp8EpilogueWait)) {
            res_pending = true;
            ok = false;
            break;
          }
          res_phase ^= 1;
#pragma unroll
          for (int box = 0; box < kBoxes; ++box) {
            const uint8_t* const at = staging + box * 4096;
            float* const x0 = sum + box * 64;
            if constexpr (SB_ROW) {
#pragma unroll
              for (int g = 0; g < 8; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int row = i * 8 + lane / 4;
                  float* x = x0 + g / 4 * 32 + i / 2 * 16 + g % 4 * 4 + i % 2 * 2;
                  const uint32_t u = *reinterpret_cast<const uint32_t*>(at + row * 128 + ((g ^ (row & 7)) << 4) + (lane & 3) * 4);
                  x[0] += bf16_lo(u);
                  x[1] += bf16_hi(u);
                }
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const uint4 u = *reinterpret_cast<const uint4*>(at + lane * 128 + ((j ^ (lane & 7)) << 4));
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                  x0[j * 8 + 2 * h] += bf16_lo(w[h]);
                  x0[j * 8 + 2 * h + 1] += bf16_hi(w[h]);
                }
              }
            }
          }
          __syncwarp();
        }
        if (p.d_fp32) {
          const bool add = p.accumulate != 0 || p.splits > 1;
          stage(&tmD, 0, std::true_type{}, add);
          stage(&tmD, kCols / 2, std::true_type{}, add);
        } else {
          stage(&tmD, 0, std::false_type{}, false);
        }
      } else {
        // 16 columns at a time as 64-byte rows, their 16-byte pieces XOR-swizzled so that no access meets a bank
        // conflict; then lane = (row of eight, four columns)
        const bool n_vec = p.N % 4 == 0;
        const int row0 = m_warp + lane / 4, rows_left = p.M - row0;
        const float4* const take =
            reinterpret_cast<const float4*>(staging) + (lane / 4) * 4 + ((lane & 3) ^ ((lane >> 3) & 3));
        const int n_lane = n0 + (lane & 3) * 4;
#pragma unroll
        for (int c = 0; c < kCols / 16; ++c) {
          __syncwarp();
          if constexpr (SB_ROW) {
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int row = i * 8 + lane / 4;
                const float* x = sum + c / 2 * 32 + i / 2 * 16 + (c % 2 * 2 + g) * 4 + i % 2 * 2;
                *reinterpret_cast<float2*>(staging + row * 64 + (((2 * g + (lane & 3) / 2) ^ ((row >> 1) & 3)) << 4) +
                                           (lane & 1) * 8) = make_float2(x[0], x[1]);
              }
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float* x = sum + c * 16 + 4 * q;
              reinterpret_cast<float4*>(staging)[lane * 4 + (q ^ ((lane >> 1) & 3))] = make_float4(x[0], x[1], x[2], x[3]);
            }
          }
          __syncwarp();
          float4 v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) v[q] = take[q * 32];
          const int n = n_lane + column(c * 16);
          if (n >= p.N) continue;
#pragma unroll 1
          for (int q = 0; q < 4; ++q)
            if (8 * q < rows_left) fp8_store4(p, row0 + 8 * q, n, q == 0 ? v[0] : q == 1 ? v[1] : q == 2 ? v[2] : v[3], n_vec);
        }
      }
    }
    if (!FULL && elect_one()) {
      if (res_pending) mbar_wait(my_res, res_phase, nullptr, nullptr, 0);  // given up on: let it land all the same
      bulk_wait_all();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // the peer no longer reads this CTA's shared memory or signals its barriers
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, kTmemCols);
    else tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------ host

template <int CG, int BN, int HALVES, int STAGES, bool SB_ROW, bool FULL>
static void launch_fp8(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& td,
                       const CUtensorMap& taux, const CUtensorMap& tres, GemmParams& p, const Fp8Operands& o, bool may_split,
                       int device, cudaStream_t stream) {
  using L = F8Smem<CG, BN, STAGES>;
  auto kern = fp8_gemm_kernel<CG, BN, HALVES, STAGES, SB_ROW, FULL>;
  static std::atomic<bool> configured[64] = {};
  if (!configured[device].load(std::memory_order_acquire)) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
    cudaFuncAttributes attr;
    C10_CUDA_CHECK(cudaFuncGetAttributes(&attr, kern));
    // the epilogue warps' larger share comes out of the block's own registers: with fewer they would wait for good
    TORCH_CHECK(BN < 256 || attr.numRegs >= kF8LaunchRegs, "fp8_gemm: built with ", attr.numRegs, " registers a thread, ",
                kF8LaunchRegs, " needed");
    configured[device].store(true, std::memory_order_release);
  }
  p.num_m_tiles = (p.M + 128 * CG - 1) / (128 * CG);
  p.num_n_tiles = (p.N + BN - 1) / BN;
  TORCH_CHECK((int64_t)p.num_m_tiles * p.num_n_tiles < (1ll << 30), "fp8_gemm: output too large");
  const int tiles = p.num_m_tiles * p.num_n_tiles, num_k = (p.K + kF8K - 1) / kF8K, workers = sm_count(device) / CG;
  // Two halves of K where the last wave of whole tiles would leave many SMs idle (weight gradients: a long K and
  // few tiles). Both halves are added to a cleared fp32 output; a sum of two does not depend on their order. Measured
  // at 5120 x 1280 x 16384 (100 tiles of 256 x 256 for 74 pairs): 217 -> 187 us when it came, 192 us now.
  auto waves = [&](int units) { return (units + workers - 1) / workers; };
  p.splits = may_split && num_k >= 16 && 0.85 * 2 * waves(tiles) >= waves(2 * tiles) ? 2 : 1;
  p.k_blocks_per_split = (num_k + p.splits - 1) / p.splits;
  p.num_tiles = tiles * p.splits;
  if (p.splits > 1) C10_CUDA_CHECK(cudaMemsetAsync(p.D, 0, (size_t)p.M * p.N * sizeof(float), stream));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CG * std::min(p.num_tiles, workers), 1, 1);
  cfg.blockDim = dim3(kF8Threads, 1, 1);
  cfg.dynamicSmemBytes = L::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 2 ? 1 : 0;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, ta, tb, td, taux, tres, p, o));
}

// Tile shape: the share of the SMs' time that goes into real output (waves of tiles over the SMs, rows and
// columns past the edge) counts for each shape, and a 256 x 256 tile runs about 1.4 times the rate of four
// 128 x 128 ones. Measured, 256 against 128, bf16 out, scales per weight block: 16384 x 1280 x 5120 (M x N
// x K) 128 / 217 us, 16384 x 5120 x 1280 129 / 156 us, 2048 x 4096 x 1024 16.6 / 19.2 us; with half of the
// SMs idle 2048 x 1024 x 4096 21.0 / 15.4 us, 1029 x 640 x 1712 13.1 / 10.4 us.
enum Fp8Tile : int { kTile128 = 0, kTile256 = 1 };

// -1: by the rule below; otherwise every call takes this tile (`set_fp8_tile`, tests and measurements).
static std::atomic<int> g_fp8_tile{-1};

int64_t set_fp8_tile(int64_t tile) {
  TORCH_CHECK(tile >= -1 && tile <= kTile256, "set_fp8_tile: -1 (automatic), 0 or 1");
  return g_fp8_tile.exchange((int)tile);
}

static int choose_tile(int64_t M, int64_t N, int sms) {
  const int forced = g_fp8_tile.load(std::memory_order_relaxed);
  if (forced >= 0) return forced;
  auto eff = [&](int cg, int bn) {
    const int64_t tiles = (M + 128 * cg - 1) / (128 * cg) * ((N + bn - 1) / bn);
    const int64_t workers = sms / cg, waves = (tiles + workers - 1) / workers;
    return (double)M * N / ((double)waves * workers * 128 * cg * bn);
  };
  return M > 128 && eff(2, 256) >= 0.7 * eff(1, 128) ? kTile256 : kTile128;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// a (M, ceil16(K)) and b (N, ceil16(K)) 8-bit, `k` the summed extent; a_scale (ceil(K / 128), M or
// ceil(M / 128)) and b_scale (ceil(K / 128), N or ceil(N / 128)) fp32 with unit inner stride.
void fp8_gemm(torch::Tensor a, torch::Tensor a_scale, bool a_block, torch::Tensor b, torch::Tensor b_scale, bool b_block,
              int64_t k, torch::Tensor d, c10::optional<torch::Tensor> bias, c10::optional<torch::Tensor> residual,
              c10::optional<torch::Tensor> gamma, c10::optional<torch::Tensor> aux_out, int64_t act, bool accumulate) {
  TORCH_CHECK(a.is_cuda() && b.device() == a.device() && d.device() == a.device() && a_scale.device() == a.device() &&
                  b_scale.device() == a.device(),
              "fp8_gemm: CUDA tensors of one device expected");
  auto format = [](const torch::Tensor& t) {
    if (t.scalar_type() == at::kFloat8_e4m3fn) return 0;
    TORCH_CHECK(t.scalar_type() == at::kFloat8_e5m2, "fp8_gemm: e4m3fn or e5m2 operands expected");
    return 1;
  };
  Fp8Operands o{};
  o.a_format = format(a);
  o.b_format = format(b);
  o.safe_exponent = 102 - 7 * (o.a_format + o.b_format);
  o.safe_scale = std::ldexp(1.f, o.safe_exponent);
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && d.dim() == 2 && a.stride(1) == 1 && b.stride(1) == 1 && d.is_contiguous(),
              "fp8_gemm: row-major 2-D operands expected");
  const int64_t M = a.size(0), N = b.size(0);
  TORCH_CHECK(k > 0 && a.size(1) >= k && b.size(1) >= k && a.stride(0) % 16 == 0 && b.stride(0) % 16 == 0 &&
                  a.stride(0) >= k && b.stride(0) >= k,
              "fp8_gemm: operand rows must hold K = ", k, " elements at a stride that is a multiple of 16");
  TORCH_CHECK(M <= INT32_MAX && N <= INT32_MAX && k <= INT32_MAX, "fp8_gemm: extent too large");
  TORCH_CHECK(d.size(0) == M && d.size(1) == N && (d.scalar_type() == at::kBFloat16 || d.scalar_type() == at::kFloat),
              "fp8_gemm: output must be bf16 or fp32 (M, N)");
  TORCH_CHECK(aligned16(a.data_ptr()) && aligned16(b.data_ptr()) && aligned16(d.data_ptr()),
              "fp8_gemm: 16-byte aligned base addresses expected");
  const int64_t kb = (k + kF8K - 1) / kF8K;
  auto check_scale = [&](const torch::Tensor& s, int64_t rows, bool block, const char* name) {
    TORCH_CHECK(s.scalar_type() == at::kFloat && s.dim() == 2 && s.size(0) == kb &&
                    s.size(1) == (block ? (rows + 127) / 128 : rows) && (s.stride(1) == 1 || s.size(1) <= 1),
                "fp8_gemm: ", name, " must be fp32 (K blocks, rows or blocks of 128 rows)");
  };
  check_scale(a_scale, M, a_block, "a_scale");
  check_scale(b_scale, N, b_block, "b_scale");
  o.sa = a_scale.data_ptr<float>();
  o.sa_ld = a_scale.stride(0);
  o.sa_shift = a_block ? 7 : 0;
  o.sb = b_scale.data_ptr<float>();
  o.sb_ld = b_scale.stride(0);
  if (M == 0 || N == 0) return;
  c10::cuda::CUDAGuard guard(a.device());
  const int device = a.get_device();
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  GemmParams p{};
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)k;
  p.D = d.data_ptr();
  p.d_fp32 = d.scalar_type() == at::kFloat;
  p.act = (int)act;
  p.accumulate = accumulate ? 1 : 0;
  p.err = error_word(device);
  auto check_vec = [&](const c10::optional<torch::Tensor>& t, const char* name) -> const float* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == a.device() && t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == N &&
                    aligned16(t->data_ptr()),
                "fp8_gemm: ", name, " must be a contiguous, aligned fp32 vector of length N");
    return t->data_ptr<float>();
  };
  auto check_mat = [&](const c10::optional<torch::Tensor>& t, const char* name) -> __nv_bfloat16* {
    if (!t.has_value()) return nullptr;
    TORCH_CHECK(t->device() == a.device() && t->scalar_type() == at::kBFloat16 && t->is_contiguous() && t->dim() == 2 &&
                    t->size(0) == M && t->size(1) == N && aligned16(t->data_ptr()),
                "fp8_gemm: ", name, " must be a contiguous, aligned bf16 (M, N) matrix");
    return reinterpret_cast<__nv_bfloat16*>(t->data_ptr());
  };
  p.bias = check_vec(bias, "bias");
  p.gamma = check_vec(gamma, "gamma");
  p.residual = check_mat(residual, "residual");
  p.aux_out = check_mat(aux_out, "aux_out");
  TORCH_CHECK(act == kActNone || act == kActGelu, "fp8_gemm: act must be none or GELU");
  const int tile = choose_tile(M, N, sm_count(device));
  const CUtensorMap ta = make_u8_map(a.data_ptr(), k, M, a.stride(0), kF8K, 128);
  const CUtensorMap tb = make_u8_map(b.data_ptr(), k, N, b.stride(0), kF8K, 128);
  // TMA moves rows of a multiple of 16 bytes and adds in fp32 only; the pre-activation and the residual would
  // want the staging rows at the same time.
  const bool bf16_rows = !p.d_fp32 || p.aux_out != nullptr || p.residual != nullptr;
  const bool full = N % (bf16_rows ? 8 : 4) != 0 || (accumulate && !p.d_fp32) ||
                    (p.aux_out != nullptr && p.residual != nullptr);
  CUtensorMap td = ta, taux = ta, tres = ta;
  if (!full) {
    td = make_store_map(d.data_ptr(), N, M, p.d_fp32);
    if (p.aux_out != nullptr) taux = make_store_map(p.aux_out, N, M, false);
    if (p.residual != nullptr) tres = make_store_map(p.residual, N, M, false);
  }
  const bool may_split = !full && p.d_fp32 && !accumulate && act == kActNone && p.bias == nullptr &&
                         p.gamma == nullptr && p.residual == nullptr;
  auto run = [&](auto row, auto rest) {
    constexpr bool kRow = decltype(row)::value, kFull = decltype(rest)::value;
    if (tile == kTile256) launch_fp8<2, 256, 2, 4, kRow, kFull>(ta, tb, td, taux, tres, p, o, may_split, device, stream);
    else launch_fp8<1, 128, 1, 5, kRow, kFull>(ta, tb, td, taux, tres, p, o, may_split, device, stream);
  };
  if (b_block) full ? run(std::false_type{}, std::true_type{}) : run(std::false_type{}, std::false_type{});
  else full ? run(std::true_type{}, std::true_type{}) : run(std::true_type{}, std::false_type{});
}

}  // namespace mia
