// Softmax attention over sequences of different lengths laid end to end, forward and backward.
//
//   o_i = sum_j p_ij v_j,  p_i = softmax over the keys j in [lo_i, hi_i) of scale q_i . k_j
//   delta_i = do_i . o_i,  dS_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i p_ij do_i
//
// q (Tq, Hq, D), k and v (Tk, Hk, D); a key head serves Hq / Hk query heads, whose contributions to dk and dv add up.
// The mask is a pair of bounds per query (and, for dk and dv, per key), made once for a batch's lengths; rows that
// see nothing give zeros. This file holds the kernels with a warp per row, which run every head size and type.
#include <type_traits>

#include "packed_attention.h"

namespace mia {
namespace {

constexpr int kWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) packed_fwd_rows_kernel(PackedProblem P, T* __restrict__ o,
                                                               float* __restrict__ lse) {
  __shared__ float scratch[kWarps][kRowScratch];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t at = (int64_t)blockIdx.x * kWarps + warp;
  if (at >= (int64_t)P.Tq * P.Hq) return;
  const int i = (int)(at / P.Hq), h = (int)(at % P.Hq), g = h / P.group;
  const int2 b = P.q_bounds[i];
  float acc[4], stat;
  forward_row<T>((const T*)P.q + i * P.qs.row + h * P.qs.head, (const T*)P.k + g * P.ks.head,
                 (const T*)P.v + g * P.vs.head, P.ks.row, P.vs.row, b.x, b.y, P.D, P.scale * kLog2e, scratch[warp], lane,
                 acc, stat);
  store_row<T>(o + at * P.D, acc, P.D, lane);
  if (lane == 0) lse[(int64_t)h * P.lse_stride + i] = stat;
}

// delta_i = do_i . o_i, a warp per row
template <typename T>
__global__ void __launch_bounds__(256) packed_delta_kernel(const T* __restrict__ o, const T* __restrict__ dout, HeadRows ds,
                                                    int Tq, int Hq, int D, int stride, float* __restrict__ delta) {
  const int lane = threadIdx.x % 32;
  const int64_t at = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (at >= (int64_t)Tq * Hq) return;
  const int i = (int)(at / Hq), h = (int)(at % Hq);
  const T *a = o + at * D, *b = dout + i * ds.row + h * ds.head;
  float s = 0.f;
  for (int c = lane; c < D; c += 32) s = fmaf(to_f32(a[c]), to_f32(b[c]), s);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
  if (lane == 0) delta[(int64_t)h * stride + i] = s;
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) packed_dq_rows_kernel(PackedProblem P, const T* __restrict__ dout, HeadRows ds,
                                                              const float* __restrict__ lse,
                                                              const float* __restrict__ delta, T* __restrict__ dq) {
  __shared__ float scratch[kWarps][kRowScratch];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t at = (int64_t)blockIdx.x * kWarps + warp;
  if (at >= (int64_t)P.Tq * P.Hq) return;
  const int i = (int)(at / P.Hq), h = (int)(at % P.Hq), g = h / P.group;
  const int2 b = P.q_bounds[i];
  const int64_t stat = (int64_t)h * P.lse_stride + i;
  float acc[4];
  dq_row<T>((const T*)P.q + i * P.qs.row + h * P.qs.head, dout + i * ds.row + h * ds.head,
            (const T*)P.k + g * P.ks.head, (const T*)P.v + g * P.vs.head, P.ks.row, P.vs.row, b.x, b.y, P.D, P.scale,
            lse[stat], delta[stat], scratch[warp], lane, acc);
  store_row<T>(dq + at * P.D, acc, P.D, lane);
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) packed_dkv_rows_kernel(PackedProblem P, const T* __restrict__ dout, HeadRows ds,
                                                               const float* __restrict__ lse,
                                                               const float* __restrict__ delta, T* __restrict__ dk,
                                                               T* __restrict__ dv) {
  __shared__ float scratch[kWarps][kRowScratch];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t at = (int64_t)blockIdx.x * kWarps + warp;
  if (at >= (int64_t)P.Tk * P.Hk) return;
  const int j = (int)(at / P.Hk), g = (int)(at % P.Hk);
  const int2 b = P.k_bounds[j];
  float a[4] = {0.f, 0.f, 0.f, 0.f}, c[4] = {0.f, 0.f, 0.f, 0.f};
  for (int h = g * P.group; h < (g + 1) * P.group; ++h)
    dkv_row<T>((const T*)P.k + j * P.ks.row + g * P.ks.head, (const T*)P.v + j * P.vs.row + g * P.vs.head,
               (const T*)P.q + h * P.qs.head, dout + h * ds.head, P.qs.row, ds.row, b.x, b.y, P.D, P.scale,
               lse + (int64_t)h * P.lse_stride, delta + (int64_t)h * P.lse_stride, scratch[warp], lane, a, c);
  store_row<T>(dk + at * P.D, a, P.D, lane);
  store_row<T>(dv + at * P.D, c, P.D, lane);
}

unsigned grid_of(int64_t items, int per) { return (unsigned)((items + per - 1) / per); }

template <typename F>
void by_type(SequenceType type, F&& f) {
  if (type == kSeqBf16) f((__nv_bfloat16*)nullptr);
  else if (type == kSeqF16) f((__half*)nullptr);
  else f((float*)nullptr);
}

}  // namespace

cudaError_t packed_fwd_rows(const PackedProblem& P, void* o, float* lse, cudaStream_t stream) {
  by_type(P.type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    packed_fwd_rows_kernel<T><<<grid_of((int64_t)P.Tq * P.Hq, kWarps), kWarps * 32, 0, stream>>>(P, (T*)o, lse);
  });
  return cudaGetLastError();
}

cudaError_t packed_bwd_rows(const PackedProblem& P, const void* o, const void* dout, HeadRows ds, const float* lse,
                            float* delta, void* dq, void* dk, void* dv, cudaStream_t stream) {
  by_type(P.type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const T* go = (const T*)dout;
    if (P.Tq > 0) {
      packed_delta_kernel<T><<<grid_of((int64_t)P.Tq * P.Hq, 8), 256, 0, stream>>>((const T*)o, go, ds, P.Tq, P.Hq, P.D,
                                                                                  P.lse_stride, delta);
      packed_dq_rows_kernel<T><<<grid_of((int64_t)P.Tq * P.Hq, kWarps), kWarps * 32, 0, stream>>>(P, go, ds, lse, delta,
                                                                                                 (T*)dq);
    }
    if (P.Tk > 0)
      packed_dkv_rows_kernel<T><<<grid_of((int64_t)P.Tk * P.Hk, kWarps), kWarps * 32, 0, stream>>>(
          P, go, ds, lse, delta, (T*)dk, (T*)dv);
  });
  return cudaGetLastError();
}

}  // namespace mia
