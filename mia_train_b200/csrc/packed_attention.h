// Packed-sequence attention: what its row kernels (packed_attention.cu) and tile kernels share.
#pragma once

#include "sequence_kernels.h"
#include "vec8.cuh"

namespace mia {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------------------- one row, one warp
// The formulas with nothing around them: a warp owns a row, takes 32 partners at a time (a lane forms the products
// of one of them), then every lane sums its channels lane, lane + 32, ... over the 32. Only rows inside the mask are
// read, so that nothing from another sequence can reach the result, whatever it holds.

constexpr int kRowScratch = 256;  // floats of shared memory per warp: two rows of up to 128 channels

template <typename T>
__device__ __forceinline__ void stage_row(float* dst, const T* src, int D, int lane) {
  for (int c = lane; c < D; c += 32) dst[c] = to_f32(src[c]);
}

template <typename T>
__device__ __forceinline__ float dot_row(const float* a, const T* b, int D) {
  float s = 0.f;
  for (int c = 0; c < D; c += 8) {
    float v[8];
    unpack8<T>(load_raw8<T>(b + c), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(a[c + e], v[e], s);
  }
  return s;
}

// What a row's sums give, and its lse. A sum of weights of 0 is a row that sees no key (zeros, and an lse of +inf, with
// which every later exp2(s - lse) is 0) or one whose scores are all -inf (NaN, as 0 / 0).
__device__ __forceinline__ float row_value(bool sees, float value, float sum) {
  return sum != 0.f ? value / sum : sees ? NAN : 0.f;
}
__device__ __forceinline__ float row_lse(bool sees, float m, float sum) {
  return sum != 0.f ? m + log2f(sum) : sees ? NAN : INFINITY;
}

// o_i = sum_j p_ij v_j with p the softmax of scale q_i . k_j, by running maximum and sum. lse is m + log2(l) in units
// of log2.
template <typename T>
__device__ void forward_row(const T* q, const T* k, const T* v, int64_t k_row, int64_t v_row, int lo, int hi, int D,
                            float scale_log2, float* scratch, int lane, float (&o)[4], float& lse) {
  stage_row(scratch, q, D, lane);
  __syncwarp();
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = 0.f;
  for (int j0 = lo; j0 < hi; j0 += 32) {
    const int j = j0 + lane;
    const float s = j < hi ? dot_row<T>(scratch, k + j * k_row, D) * scale_log2 : -INFINITY;
    float top = s;
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float m_new = fmaxf(m, top);
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float fade = exp2f(m - ref);
    const float p = j < hi ? exp2f(s - ref) : 0.f;
    l = l * fade + p;  // each lane sums its own keys
    m = m_new;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] *= fade;
    const int n = min(32, hi - j0);
    for (int jj = 0; jj < n; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, p, jj);
      const T* row = v + (j0 + jj) * v_row;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < D) o[i] = fmaf(pj, to_f32(row[lane + 32 * i]), o[i]);
    }
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
  const float inv = row_value(hi > lo, 1.f, l);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] *= inv;
  lse = row_lse(hi > lo, m, l);
  __syncwarp();
}

// dq_i = scale sum_j p_ij (do_i . v_j - delta_i) k_j
template <typename T>
__device__ void dq_row(const T* q, const T* dout, const T* k, const T* v, int64_t k_row, int64_t v_row, int lo, int hi,
                       int D, float scale, float lse, float delta, float* scratch, int lane, float (&dq)[4]) {
  stage_row(scratch, q, D, lane);
  stage_row(scratch + 128, dout, D, lane);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) dq[i] = 0.f;
  for (int j0 = lo; j0 < hi; j0 += 32) {
    const int j = j0 + lane;
    float ds = 0.f;
    if (j < hi) {
      const float p = exp2f(dot_row<T>(scratch, k + j * k_row, D) * (scale * kLog2e) - lse);
      ds = p * (dot_row<T>(scratch + 128, v + j * v_row, D) - delta);
    }
    const int n = min(32, hi - j0);
    for (int jj = 0; jj < n; ++jj) {
      const float d = __shfl_sync(0xffffffffu, ds, jj);
      const T* row = k + (j0 + jj) * k_row;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < D) dq[i] = fmaf(d, to_f32(row[lane + 32 * i]), dq[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) dq[i] *= scale;
  __syncwarp();
}

// dv_j += sum_i p_ij do_i, dk_j += scale sum_i p_ij (do_i . v_j - delta_i) q_i over the queries of one head
template <typename T>
__device__ void dkv_row(const T* k, const T* v, const T* q, const T* dout, int64_t q_row, int64_t do_row, int lo,
                        int hi, int D, float scale, const float* lse, const float* delta, float* scratch, int lane,
                        float (&dk)[4], float (&dv)[4]) {
  stage_row(scratch, k, D, lane);
  stage_row(scratch + 128, v, D, lane);
  __syncwarp();
  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    float p = 0.f, ds = 0.f;
    if (i < hi) {
      p = exp2f(dot_row<T>(scratch, q + i * q_row, D) * (scale * kLog2e) - lse[i]);
      ds = p * (dot_row<T>(scratch + 128, dout + i * do_row, D) - delta[i]) * scale;
    }
    const int n = min(32, hi - i0);
    for (int ii = 0; ii < n; ++ii) {
      const float pi = __shfl_sync(0xffffffffu, p, ii), di = __shfl_sync(0xffffffffu, ds, ii);
      const T *qr = q + (i0 + ii) * q_row, *dr = dout + (i0 + ii) * do_row;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 32 * c < D) {
          dv[c] = fmaf(pi, to_f32(dr[lane + 32 * c]), dv[c]);
          dk[c] = fmaf(di, to_f32(qr[lane + 32 * c]), dk[c]);
        }
    }
  }
  __syncwarp();
}

// store_row, and in `low` (which may be null) what rounding took away
template <typename T>
__device__ __forceinline__ void store_row_low(T* dst, T* low, const float (&x)[4], int D, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < D) {
      const T y = from_f32<T>(x[i]);
      dst[lane + 32 * i] = y;
      if (low != nullptr) low[lane + 32 * i] = from_f32<T>(x[i] - to_f32(y));
    }
}

template <typename T>
__device__ __forceinline__ void store_row(T* dst, const float (&x)[4], int D, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 32 * i < D) dst[lane + 32 * i] = from_f32<T>(x[i]);
}

}  // namespace mia
