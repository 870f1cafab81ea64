// Quantisation of a matrix to 8-bit floating point with one power-of-two scale per block.
//
//   s = the smallest power of two >= 2^-126 with max_block |v| / s <= 448 (e4m3) or 57344 (e5m2)
//   q = v / s rounded to the nearest 8-bit value, ties to even
//
// Both limits are 1.75 times a power of two, so the exponent of s follows from the bits of the
// block's largest magnitude, and the division is exact: the only rounding is the one to 8 bits. A
// block that holds an infinity or a NaN gets the scale NaN, which reaches every product it takes part
// in (e4m3 has no infinity to carry).
//
// One CTA takes a 128 x 128 tile of v, read once, and writes what the caller asked for:
//   rows    q (R, C) with 1 x 128 blocks
//   cols    q^T (C, R) with blocks of 128 along the rows of v: the K-major operand of a product
//           summed over the rows (weight gradients)
//   block   q and/or q^T with one scale for the whole tile (weights: both directions share it)
//   sums    column sums of the tile, for the bias gradient
// v = x, or x * gelu'(aux) * gamma (the gradient behind an activation and a per-column scale).
// Thread (tx, ty) holds rows 8 ty .. 8 ty + 7 of columns 8 tx .. 8 tx + 7, so that it owns eight
// consecutive bytes of both q and q^T; q^T goes through shared memory in 8-byte units, XOR-swizzled
// by tx so that neither side meets a bank conflict, and leaves as 16-byte stores.
// Instructions, not bytes, are scarce (ncu: 15 a value for q alone in a first version that kept fp32
// values): bf16 input stays packed, its magnitudes are compared two at a time as 16-bit integers (their
// order as numbers, NaN above infinity above the rest), and rows are reduced in pairs. Measured: 16384 x
// 5120 bf16 to q 51 us (4.97 TB/s of all bytes read and written), to q^T 48 us, to both 68 us, with column
// sums 83 us; 5120 x 1280 fp32 with one scale a tile to both 15 us.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>
#include <torch/extension.h>

#include <type_traits>

#include "block_ops.h"
#include "common.cuh"
#include "vec8.cuh"

namespace mia {

constexpr int kQBlk = 128;

struct QuantParams {
  const void* x;  // (R, C) row stride x_ld
  int64_t x_ld;
  const __nv_bfloat16* aux;  // (R, C) contiguous, or nullptr: no gelu'
  const float* gamma;        // (C), or nullptr
  int64_t R;
  int64_t C;
  uint8_t* q;  // (R, q_ld)
  int64_t q_ld;
  float* q_scale;  // 1 x 128: [c / 128][r], row stride q_scale_ld; block: [c / 128][r / 128]
  int64_t q_scale_ld;
  uint8_t* qt;  // (C, qt_ld)
  int64_t qt_ld;
  float* qt_scale;  // 1 x 128: [r / 128][c]; block: [r / 128][c / 128]
  int64_t qt_scale_ld;
  float* sums;  // (ceil(R / 128), C)
  int col_tiles;
};

// Scale for a block whose largest |v| has the given fp32 bits, and its reciprocal. A mantissa above 1.75
// carries into the exponent.
template <bool E5M2>
__device__ __forceinline__ void pow2_scale(uint32_t amax_bits, float& scale, float& inv) {
  const int e = max((int)((amax_bits + 0x1FFFFFu) >> 23) - (E5M2 ? 15 : 8), 1);
  const bool finite = amax_bits < 0x7F800000u;
  scale = __uint_as_float(finite ? (uint32_t)e << 23 : 0x7FC00000u);
  inv = __uint_as_float(finite ? (uint32_t)(254 - e) << 23 : 0x7FC00000u);
}

template <bool E5M2>
__device__ __forceinline__ uint32_t cvt4(float a, float b, float c, float d) {
  constexpr __nv_fp8_interpretation_t f = E5M2 ? __NV_E5M2 : __NV_E4M3;
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, f);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, f);
  return lo | hi << 16;
}

// A thread's 8 x 8 values: fp32 in general.
template <typename T, bool PACKED>
struct QuantTile {
  float v[8][8];
  __device__ __forceinline__ float get(int i, int j) const { return v[i][j]; }
  __device__ __forceinline__ void load(const T* src, int64_t ld, int rows, int cols, bool vec) {
    if (vec) {
      Raw8<T> raw[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[i] = i < rows ? load_raw8(src + i * ld) : Raw8<T>{};
#pragma unroll
      for (int i = 0; i < 8; ++i) unpack8(raw[i], v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = (i < rows && j < cols) ? to_f32(src[i * ld + j]) : 0.f;
    }
  }
  static __device__ __forceinline__ uint32_t mag(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }
  // fp32 bits of the largest magnitude of row i over the 16 threads of the row
  __device__ __forceinline__ void row_max(uint32_t (&m)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) m[i] = max(m[i], mag(v[i][j]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m[i] = max(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
    }
  }
  // of column j over the warp's 16 rows
  __device__ __forceinline__ void col_max(uint32_t (&m)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m[j] = max(m[j], mag(v[i][j]));
      m[j] = max(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
    }
  }
};

// bf16 pairs as they come.
template <>
struct QuantTile<__nv_bfloat16, true> {
  uint32_t w[8][4];
  __device__ __forceinline__ float get(int i, int j) const { return j & 1 ? bf16_hi(w[i][j / 2]) : bf16_lo(w[i][j / 2]); }
  __device__ __forceinline__ void load(const __nv_bfloat16* src, int64_t ld, int rows, int cols, bool vec) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (vec) {
        if (i < rows) u = *reinterpret_cast<const uint4*>(src + i * ld);
      } else if (i < rows) {
        const uint16_t* e = reinterpret_cast<const uint16_t*>(src + i * ld);
        uint32_t t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          t[k] = (2 * k < cols ? e[2 * k] : 0u) | (2 * k + 1 < cols ? (uint32_t)e[2 * k + 1] << 16 : 0u);
        u = make_uint4(t[0], t[1], t[2], t[3]);
      }
      w[i][0] = u.x; w[i][1] = u.y; w[i][2] = u.z; w[i][3] = u.w;
    }
  }
  __device__ __forceinline__ uint32_t mag2(int i, int k) const { return w[i][k] & 0x7FFF7FFFu; }
  __device__ __forceinline__ void row_max(uint32_t (&m)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const uint32_t a = __vmaxu2(__vmaxu2(mag2(i, 0), mag2(i, 1)), __vmaxu2(mag2(i, 2), mag2(i, 3)));
      const uint32_t b = __vmaxu2(__vmaxu2(mag2(i + 1, 0), mag2(i + 1, 1)), __vmaxu2(mag2(i + 1, 2), mag2(i + 1, 3)));
      uint32_t two = __vmaxu2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));  // row i low, row i + 1 high
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, o));
      m[i] = two << 16;
      m[i + 1] = two & 0xFFFF0000u;
    }
  }
  __device__ __forceinline__ void col_max(uint32_t (&m)[8]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t two = mag2(0, k);
#pragma unroll
      for (int i = 1; i < 8; ++i) two = __vmaxu2(two, mag2(i, k));
      two = __vmaxu2(two, __shfl_xor_sync(0xffffffffu, two, 16));
      m[2 * k] = two << 16;
      m[2 * k + 1] = two & 0xFFFF0000u;
    }
  }
};

enum QuantMode : int { kQuantRows = 1, kQuantCols = 2, kQuantBlock = 4, kQuantSums = 8 };

template <typename T, int MODE, bool AUX, bool E5M2>
__global__ void __launch_bounds__(256, sizeof(T) == 2 && !AUX ? 3 : 2) quant_kernel(const QuantParams p) {
  constexpr bool kBlock = (MODE & kQuantBlock) != 0;
  constexpr bool kRows = (MODE & kQuantRows) != 0;
  constexpr bool kCols = (MODE & kQuantCols) != 0;
  constexpr bool kSums = (MODE & kQuantSums) != 0;
  __shared__ __align__(16) uint32_t col_red[8][kQBlk];
  __shared__ __align__(16) float col_inv[kQBlk];
  __shared__ __align__(16) uint2 tile[kCols ? kQBlk * 16 : 1];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int tx = tid % 16, ty = tid / 16;
  const int64_t rb = blockIdx.x / p.col_tiles, cb = blockIdx.x % p.col_tiles;
  const int64_t r0 = rb * kQBlk + ty * 8, c0 = cb * kQBlk + tx * 8;
  const int rows = (int)min((int64_t)8, p.R - r0), cols = (int)min((int64_t)8, p.C - c0);  // may be negative: none
  QuantTile<T, std::is_same_v<T, __nv_bfloat16> && !AUX> t;
  const bool vec = cols == 8 && p.x_ld % 8 == 0 && (reinterpret_cast<uintptr_t>(p.x) & 15) == 0;
  t.load(reinterpret_cast<const T*>(p.x) + r0 * p.x_ld + c0, p.x_ld, rows, cols, vec);
  if constexpr (AUX) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i < rows && j < cols) {
          if (p.aux != nullptr) t.v[i][j] *= gelu_erf_grad(__bfloat162float(p.aux[(r0 + i) * p.C + c0 + j]));
          if (p.gamma != nullptr) t.v[i][j] *= p.gamma[c0 + j];
        }
  }

  float blk_inv = 0.f;
  if constexpr (kBlock) {
    uint32_t m8[8];
    t.col_max(m8);
    uint32_t m = m8[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = max(m, m8[j]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) col_red[0][warp] = m;
    __syncthreads();
    m = col_red[0][0];
#pragma unroll
    for (int k = 1; k < 8; ++k) m = max(m, col_red[0][k]);
    float blk_scale;
    pow2_scale<E5M2>(m, blk_scale, blk_inv);
    if (tid == 0) {
      if (kRows) p.q_scale[cb * p.q_scale_ld + rb] = blk_scale;
      if (kCols) p.qt_scale[rb * p.qt_scale_ld + cb] = blk_scale;
    }
  } else if constexpr (kCols) {
    uint32_t m[8];
    t.col_max(m);
    if (lane < 16) {
      *reinterpret_cast<uint4*>(&col_red[warp][tx * 8]) = make_uint4(m[0], m[1], m[2], m[3]);
      *reinterpret_cast<uint4*>(&col_red[warp][tx * 8 + 4]) = make_uint4(m[4], m[5], m[6], m[7]);
    }
  }
  if constexpr (kRows) {
    float inv[8], scale[8];
    if constexpr (!kBlock) {
      uint32_t m[8];
      t.row_max(m);
#pragma unroll
      for (int i = 0; i < 8; ++i) pow2_scale<E5M2>(m[i], scale[i], inv[i]);
      if (tx < 8 && tx < rows) {  // lane tx of a row group writes the scale of row tx: eight in one sector
        float mine = scale[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mine = tx == i ? scale[i] : mine;
        p.q_scale[cb * p.q_scale_ld + r0 + tx] = mine;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float k = kBlock ? blk_inv : inv[i];
      if (i < rows && c0 < p.q_ld)
        *reinterpret_cast<uint2*>(p.q + (r0 + i) * p.q_ld + c0) =
            make_uint2(cvt4<E5M2>(t.get(i, 0) * k, t.get(i, 1) * k, t.get(i, 2) * k, t.get(i, 3) * k),
                       cvt4<E5M2>(t.get(i, 4) * k, t.get(i, 5) * k, t.get(i, 6) * k, t.get(i, 7) * k));
    }
  }
  if constexpr (kCols) {
    if constexpr (!kBlock) {
      __syncthreads();
      if (tid < kQBlk) {
        uint32_t m = col_red[0][tid];
#pragma unroll
        for (int k = 1; k < 8; ++k) m = max(m, col_red[k][tid]);
        float s, inv;
        pow2_scale<E5M2>(m, s, inv);
        col_inv[tid] = inv;
        if (cb * kQBlk + tid < p.C) p.qt_scale[rb * p.qt_scale_ld + cb * kQBlk + tid] = s;
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float k = kBlock ? blk_inv : col_inv[tx * 8 + j];
      tile[(tx * 8 + j) * 16 + (ty ^ tx)] =
          make_uint2(cvt4<E5M2>(t.get(0, j) * k, t.get(1, j) * k, t.get(2, j) * k, t.get(3, j) * k),
                     cvt4<E5M2>(t.get(4, j) * k, t.get(5, j) * k, t.get(6, j) * k, t.get(7, j) * k));
    }
    __syncthreads();
    const int64_t t0 = rb * kQBlk;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int c = it * 32 + tid / 8, seg = tid % 8;  // column of v, 16-byte segment of its 128 rows
      const int f = c / 8;
      const uint2 a = tile[c * 16 + ((2 * seg) ^ f)], b = tile[c * 16 + ((2 * seg + 1) ^ f)];
      if (cb * kQBlk + c < p.C && t0 + seg * 16 < p.qt_ld)
        *reinterpret_cast<uint4*>(p.qt + (cb * kQBlk + c) * p.qt_ld + t0 + seg * 16) = make_uint4(a.x, a.y, b.x, b.y);
    }
  }
  if constexpr (kSums) {
    __syncthreads();  // col_red is free again
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float a = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) a += t.get(i, j);
      a += __shfl_xor_sync(0xffffffffu, a, 16);
      if (lane < 16) col_red[warp][tx * 8 + j] = __float_as_uint(a);
    }
    __syncthreads();
    if (tid < kQBlk && cb * kQBlk + tid < p.C) {
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) a += __uint_as_float(col_red[k][tid]);
      p.sums[rb * p.C + cb * kQBlk + tid] = a;
    }
  }
}

// out[c] (+)= sum_k parts[k][c] in a fixed order; 32 columns x 8 slices of k a CTA.
__global__ void __launch_bounds__(256) quant_sums_kernel(const float* __restrict__ parts, int64_t n, int64_t C, float* out,
                                                         int accumulate) {
  __shared__ float red[8][32];
  const int lane = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float a = 0.f;
  if (c < C)
    for (int64_t k = slice; k < n; k += 8) a += parts[k * C + c];
  red[slice][lane] = a;
  __syncthreads();
  if (slice == 0 && c < C) {
#pragma unroll
    for (int k = 1; k < 8; ++k) a += red[k][lane];
    out[c] = accumulate ? out[c] + a : a;
  }
}

// The combinations that exist: 1 x 128 blocks either way or both, for e4m3 with the column sums of a gradient as
// well; 128 x 128 blocks of a weight, alone or both ways; the factors of a gradient (AUX) are bf16 and e4m3.
template <typename T, bool AUX, bool E5M2>
static bool launch_quant(const QuantParams& p, int mode, unsigned blocks, cudaStream_t stream) {
#define MIA_QUANT_CASE(M) \
  case M: quant_kernel<T, M, AUX, E5M2><<<blocks, 256, 0, stream>>>(p); return true;
  switch (mode) {
    MIA_QUANT_CASE(kQuantRows)
    MIA_QUANT_CASE(kQuantCols)
    MIA_QUANT_CASE(kQuantRows | kQuantCols)
  }
  if constexpr (!E5M2) {
    switch (mode) {
      MIA_QUANT_CASE(kQuantSums)
      MIA_QUANT_CASE(kQuantRows | kQuantSums)
      MIA_QUANT_CASE(kQuantCols | kQuantSums)
      MIA_QUANT_CASE(kQuantRows | kQuantCols | kQuantSums)
    }
  }
  if constexpr (!AUX) {
    switch (mode) {
      MIA_QUANT_CASE(kQuantBlock | kQuantRows)
      MIA_QUANT_CASE(kQuantBlock | kQuantRows | kQuantCols)
    }
  }
#undef MIA_QUANT_CASE
  return false;
}

static void check_fp8(const torch::Tensor& q, const torch::Tensor& scale, int64_t rows, int64_t cols, int64_t scale_cols,
                      const torch::Tensor& like, bool e5m2) {
  TORCH_CHECK(q.device() == like.device() && q.dim() == 2 && q.is_contiguous() && q.size(0) == rows &&
                  q.size(1) % 16 == 0 && q.size(1) >= cols && q.size(1) - cols < 16 &&
                  q.scalar_type() == (e5m2 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn) &&
                  (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15) == 0,
              "fp8_quantize: 8-bit output must be contiguous, 16-byte aligned, its rows padded to 16 columns");
  TORCH_CHECK(scale.device() == like.device() && scale.scalar_type() == at::kFloat && scale.dim() == 2 &&
                  scale.size(0) == (cols + kQBlk - 1) / kQBlk && scale.size(1) == scale_cols && scale.stride(1) == 1,
              "fp8_quantize: scale must be fp32 (blocks of columns, rows or blocks of rows)");
}

// x (R, C) row-major (any row stride). Each output is optional; `block` picks 128 x 128 scales.
// `sums` (C) fp32 receives (or, with `accumulate`, is added) the column sums of v.
void fp8_quantize(torch::Tensor x, c10::optional<torch::Tensor> aux, c10::optional<torch::Tensor> gamma, bool block,
                  bool e5m2, c10::optional<torch::Tensor> q, c10::optional<torch::Tensor> q_scale,
                  c10::optional<torch::Tensor> qt, c10::optional<torch::Tensor> qt_scale,
                  c10::optional<torch::Tensor> sums, bool accumulate) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && (x.stride(1) == 1 || x.size(1) <= 1), "fp8_quantize: row-major CUDA matrix expected");
  QuantParams p{};
  p.x = x.data_ptr();
  p.x_ld = x.stride(0);
  p.R = x.size(0);
  p.C = x.size(1);
  const int64_t rb = (p.R + kQBlk - 1) / kQBlk, cb = (p.C + kQBlk - 1) / kQBlk;
  int mode = block ? kQuantBlock : 0;
  TORCH_CHECK(q.has_value() == q_scale.has_value() && qt.has_value() == qt_scale.has_value(),
              "fp8_quantize: values and scales come together");
  if (q.has_value()) {
    check_fp8(*q, *q_scale, p.R, p.C, block ? rb : p.R, x, e5m2);
    p.q = reinterpret_cast<uint8_t*>(q->data_ptr());
    p.q_ld = q->size(1);
    p.q_scale = q_scale->data_ptr<float>();
    p.q_scale_ld = q_scale->stride(0);
    mode |= kQuantRows;
  }
  if (qt.has_value()) {
    check_fp8(*qt, *qt_scale, p.C, p.R, block ? cb : p.C, x, e5m2);
    p.qt = reinterpret_cast<uint8_t*>(qt->data_ptr());
    p.qt_ld = qt->size(1);
    p.qt_scale = qt_scale->data_ptr<float>();
    p.qt_scale_ld = qt_scale->stride(0);
    mode |= kQuantCols;
  }
  if (aux.has_value()) {
    TORCH_CHECK(aux->device() == x.device() && aux->scalar_type() == at::kBFloat16 && aux->is_contiguous() &&
                    aux->numel() == p.R * p.C,
                "fp8_quantize: aux must be a contiguous bf16 matrix of x's shape");
    p.aux = reinterpret_cast<const __nv_bfloat16*>(aux->data_ptr());
  }
  if (gamma.has_value()) {
    TORCH_CHECK(gamma->device() == x.device() && gamma->scalar_type() == at::kFloat && gamma->is_contiguous() &&
                    gamma->numel() == p.C,
                "fp8_quantize: gamma must be a contiguous fp32 vector of x's width");
    p.gamma = gamma->data_ptr<float>();
  }
  c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  torch::Tensor parts;
  if (sums.has_value()) {
    TORCH_CHECK(sums->device() == x.device() && sums->scalar_type() == at::kFloat && sums->is_contiguous() &&
                    sums->numel() == p.C,
                "fp8_quantize: sums must be a contiguous fp32 vector of x's width");
    parts = torch::empty({rb, p.C}, x.options().dtype(at::kFloat));
    p.sums = parts.data_ptr<float>();
    mode |= kQuantSums;
  }
  if (p.C == 0 || mode == 0) return;
  if (p.R > 0) {
    TORCH_CHECK(rb * cb <= INT32_MAX, "fp8_quantize: matrix too large");
    p.col_tiles = (int)cb;
    const bool extra = p.aux != nullptr || p.gamma != nullptr;
    const unsigned blocks = (unsigned)(rb * cb);
    auto run = [&](auto type) {
      using T = decltype(type);
      if (extra) {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) return !e5m2 && launch_quant<T, true, false>(p, mode, blocks, stream);
        return false;
      }
      return e5m2 ? launch_quant<T, false, true>(p, mode, blocks, stream) : launch_quant<T, false, false>(p, mode, blocks, stream);
    };
    bool ran = false;
    if (x.scalar_type() == at::kBFloat16) ran = run(__nv_bfloat16{});
    else if (x.scalar_type() == at::kHalf) ran = run(__half{});
    else if (x.scalar_type() == at::kFloat) ran = run(float{});
    else TORCH_CHECK(false, "fp8_quantize: bf16, fp16 or fp32 expected");
    TORCH_CHECK(ran, "fp8_quantize: unsupported combination of type, format, factors and outputs (", mode, ")");
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  if (sums.has_value()) {
    quant_sums_kernel<<<(unsigned)((p.C + 31) / 32), 256, 0, stream>>>(p.sums, rb, p.C, sums->data_ptr<float>(),
                                                                       accumulate ? 1 : 0);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

}  // namespace mia
