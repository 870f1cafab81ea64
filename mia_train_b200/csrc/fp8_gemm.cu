// 8-bit GEMM with one scale per block of 128 along K, on the 5th-generation tensor cores.
//
//   D[m, n] = epilogue( sum_b sA[b, m] sB[b, n] sum_{k in block b} A[m, k] B[n, k] )
//
// A (M, K) and B (N, K) are e4m3 or e5m2, both K-major, rows padded to 16 bytes. sA has one scale per
// row and K block (or per 128 rows), sB one per 128 rows (weights) or one per row (weight gradients).
//
// CTA = 4 control warps (two idle) + 8 epilogue warps, one CTA per SM, persistent over 128 x 128 tiles:
//   warp 0     TMA producer: 128 x 128-byte tiles of A and B into a ring of shared-memory stages.
//   warp 1     MMA issuer: four K = 32 steps of tcgen05.mma (kind::f8f6f4) per K block into one of two
//              TMEM accumulators, which holds the products of that K block alone.
//   warps 4..  epilogue: read each K block's products with tcgen05.ld, multiply by the scales and add in
//              fp32 registers (a warp owns 32 rows x 64 columns), while the tensor core fills the other
//              accumulator; after the last block bias / GELU / LayerScale / residual / accumulate and
//              the stores (`epilogue_chunk`). A lane prefetches its row's scale of the next K block; with
//              a scale per row of B also its share of the warp's column scales, which the lanes pass on
//              through a small double-buffered strip of shared memory that belongs to the warp alone.
// The scales are applied in fp32 outside the tensor core, so they may be any fp32 numbers, and no sum
// longer than 128 products is left to the tensor core's own accumulation.
//
// All waits are bounded (see common.cuh); on a timeout the kernel records an error code, drains the
// copies and MMAs it issued, frees its tensor memory and returns.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cfloat>

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
};

template <int BN, int STAGES>
struct F8Smem {
  static constexpr int kBTile = BN * kF8K;
  static constexpr int kStage = kF8ATile + kBTile;
  static constexpr int kScales = 2 * 4 * BN * 4;  // two strips of BN / 2 floats for each epilogue warp
  static constexpr int kBytes = STAGES * kStage + kScales + 1024 /*align*/ + 256 /*barriers*/;
};

__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t pack_u32x2(uint32_t a, uint32_t b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// mbar_wait by a whole warp. The lanes poll the barrier one by one and may see it complete in different
// polls; the vote brings them together again before the warp-wide TMEM loads that follow.
__device__ __forceinline__ bool mbar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err,
                                               int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code));
}

template <int BN, int STAGES, bool SB_ROW>
__global__ void __launch_bounds__(kF8Threads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const GemmParams p, const Fp8Operands o) {
  using L = F8Smem<BN, STAGES>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smA = smem;
  uint8_t* smB = smem + STAGES * kF8ATile;
  float* smS = reinterpret_cast<float*>(smem + STAGES * L::kStage);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * L::kStage + L::kScales);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;           // [2]
  uint64_t* tempty_bar = tfull_bar + 2;               // [2]
  uint64_t* drain_bar = tempty_bar + 2;               // [1]
  uint32_t* tmem_base_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_base_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  constexpr uint32_t kTmemCols = 2 * BN;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], kF8EpiWarps);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(tmem_base_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  const int num_k = (p.K + kF8K - 1) / kF8K;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < p.num_tiles && ok; tile += gridDim.x) {
        const int m0 = (tile % p.num_m_tiles) * 128, n0 = (tile / p.num_m_tiles) * BN;
        for (int kb = 0; kb < num_k; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag, p.err, kErrFp8ProducerWait)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full_bar[stage], L::kStage);
          tma_load_2d(smA + stage * kF8ATile, &tmA, &full_bar[stage], kb * kF8K, m0);
          tma_load_2d(smB + stage * L::kBTile, &tmB, &full_bar[stage], kb * kF8K, n0);
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) {
        int s = stage, ph = phase;
        for (int i = 0; i < STAGES && i < issued; ++i) {
          if (--s < 0) {
            s = STAGES - 1;
            ph ^= 1;
          }
          mbar_wait(&full_bar[s], ph, nullptr, nullptr, 0);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_f8(128, BN, o.a_format, o.b_format);
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      bool any_mma = false;
      for (int tile = blockIdx.x; tile < p.num_tiles && ok; tile += gridDim.x) {
        for (int kb = 0; kb < num_k; ++kb) {
          if (!mbar_wait(&tempty_bar[acc], acc_phase ^ 1, abort_flag, p.err, kErrFp8MmaWait) ||
              !mbar_wait(&full_bar[stage], phase, abort_flag, p.err, kErrFp8MmaWait)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * BN;
          const uint32_t a_base = smem_u32(smA + stage * kF8ATile);
          const uint32_t b_base = smem_u32(smB + stage * L::kBTile);
#pragma unroll
          for (int k = 0; k < kF8K / 32; ++k)
            tc_mma_f8(d_tmem, make_sdesc_sw128(a_base + k * 32, 16, 1024), make_sdesc_sw128(b_base + k * 32, 16, 1024),
                      idesc, k > 0 ? 1u : 0u);
          any_mma = true;
          tc_commit(&empty_bar[stage]);
          tc_commit(&tfull_bar[acc]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
          acc ^= 1;
          if (acc == 0) acc_phase ^= 1;
        }
      }
      if (!ok && any_mma) {
        tc_commit(drain_bar);
        mbar_wait(drain_bar, 0, nullptr, nullptr, 0);
      }
    }
  } else if (warp >= kF8FirstEpi) {
    const int lane_group = warp % 4;                     // TMEM lanes 32 * lane_group .. + 31
    const int col_part = (warp - kF8FirstEpi) / 4;       // half of the tile's columns
    constexpr int kCols = BN / 2;
    constexpr int kChunks = kCols / 32;
    constexpr int kLaneCols = kCols / 32;
    float* strip = smS + (warp - kF8FirstEpi) * 2 * kCols;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < p.num_tiles && ok; tile += gridDim.x) {
      const int m = (tile % p.num_m_tiles) * 128 + lane_group * 32 + lane;
      const int n0 = (tile / p.num_m_tiles) * BN + col_part * kCols;
      const uint32_t t_row = tmem_base + ((uint32_t)(lane_group * 32) << 16) + col_part * kCols;
      uint64_t sum[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) sum[j] = 0;
      const bool live = m < p.M;
      const float* sa = o.sa + (live ? (m >> o.sa_shift) : 0);
      // SB_ROW: this lane fetches the scales of columns n0 + lane + 32 i
      const float* sb = o.sb + (SB_ROW ? n0 + lane : min(n0, p.N - 1) >> 7);
      float sa_next = live ? __ldg(sa) : 0.f;
      float sb_next[kLaneCols];
#pragma unroll
      for (int i = 0; i < kLaneCols; ++i)
        sb_next[i] = SB_ROW ? (n0 + lane + 32 * i < p.N ? __ldg(sb + 32 * i) : 0.f) : (i == 0 ? __ldg(sb) : 0.f);
      for (int kb = 0; kb < num_k; ++kb) {
        const float sa_now = sa_next, sb_now = sb_next[0];
        const float* sbv = strip + (kb & 1) * kCols;
        if (SB_ROW) {
          // the strip of two K blocks ago: every lane has passed the barrier after reading it
#pragma unroll
          for (int i = 0; i < kLaneCols; ++i) strip[(kb & 1) * kCols + lane + 32 * i] = sb_next[i];
          __syncwarp();
        }
        if (kb + 1 < num_k) {
          if (live) sa_next = __ldg(sa + (kb + 1) * o.sa_ld);
#pragma unroll
          for (int i = 0; i < kLaneCols; ++i)
            if (SB_ROW ? n0 + lane + 32 * i < p.N : i == 0) sb_next[i] = __ldg(sb + (kb + 1) * o.sb_ld + 32 * i);
        }
        if (!mbar_wait_warp(&tfull_bar[acc], acc_phase, abort_flag, p.err, kErrFp8EpilogueWait)) {
          ok = false;
          break;
        }
        tc_fence_after();
        float s = sa_now;
        if (!SB_ROW) {
          s = sa_now * sb_now;
          s = s > FLT_MAX ? FLT_MAX : s;  // two huge scales over a zero product stay zero; NaN stays NaN
        }
        const uint64_t s2 = pack_f32x2(s, s);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(t_row + acc * BN + c * 32, r);
          tmem_ld_wait_regs(r);
          if (c == kChunks - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty_bar[acc]);
          }
          if (SB_ROW) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const float4 b = reinterpret_cast<const float4*>(sbv)[c * 8 + q];
              uint64_t& x = sum[c * 16 + 2 * q];
              uint64_t& y = sum[c * 16 + 2 * q + 1];
              x = fma_f32x2(mul_f32x2(pack_u32x2(r[4 * q], r[4 * q + 1]), s2), pack_f32x2(b.x, b.y), x);
              y = fma_f32x2(mul_f32x2(pack_u32x2(r[4 * q + 2], r[4 * q + 3]), s2), pack_f32x2(b.z, b.w), y);
            }
          } else {
#pragma unroll
            for (int q = 0; q < 16; ++q)
              sum[c * 16 + q] = fma_f32x2(pack_u32x2(r[2 * q], r[2 * q + 1]), s2, sum[c * 16 + q]);
          }
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      if (!ok) break;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        uint32_t r[32];
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          r[2 * q] = (uint32_t)sum[c * 16 + q];
          r[2 * q + 1] = (uint32_t)(sum[c * 16 + q] >> 32);
        }
        epilogue_chunk<kEpiAll>(p, m, n0 + c * 32, r);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ------------------------------------------------------------------------------------------ host

template <int BN, int STAGES, bool SB_ROW>
static void launch_fp8(const CUtensorMap& ta, const CUtensorMap& tb, GemmParams& p, const Fp8Operands& o, int device,
                       cudaStream_t stream) {
  using L = F8Smem<BN, STAGES>;
  auto kern = fp8_gemm_kernel<BN, STAGES, SB_ROW>;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes));
  p.num_m_tiles = (p.M + 127) / 128;
  p.num_n_tiles = (p.N + BN - 1) / BN;
  p.num_tiles = p.num_m_tiles * p.num_n_tiles;
  kern<<<std::min(p.num_tiles, sm_count(device)), kF8Threads, L::kBytes, stream>>>(ta, tb, p, o);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
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
  p.splits = 1;
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
  const CUtensorMap ta = make_u8_map(a.data_ptr(), k, M, a.stride(0), kF8K, 128);
  const CUtensorMap tb = make_u8_map(b.data_ptr(), k, N, b.stride(0), kF8K, 128);
  if (b_block) launch_fp8<128, 6, false>(ta, tb, p, o, device, stream);
  else launch_fp8<128, 6, true>(ta, tb, p, o, device, stream);
}

}  // namespace mia
