// Softmax attention over sequences of different lengths laid end to end, forward and backward.
//
//   o_i = sum_j p_ij v_j,  p_i = softmax over the keys j in [lo_i, hi_i) of scale q_i . k_j
//   delta_i = do_i . o_i,  dS_ij = p_ij (do_i . v_j - delta_i)
//   dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i p_ij do_i
//
// q (Tq, Hq, D), k and v (Tk, Hk, D); a key head serves Hq / Hk query heads, whose contributions to dk and dv add up.
// The mask is a pair of bounds per query (and, for dk and dv, per key), made once for a batch's lengths; rows that
// see nothing give zeros. This file holds the kernels with a warp per row, which run every head size and type, and the
// forward kernel for few queries over many keys.
#include <algorithm>
#include <type_traits>

#include "packed_attention.h"
#include "sequence_types.cuh"

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
  store_row_low<T>(o + at * P.D, P.o_low != nullptr ? (T*)P.o_low + at * P.D : nullptr, acc, P.D, lane);
  if (lane == 0) lse[(int64_t)h * P.lse_stride + i] = stat;
}

// delta_i = do_i . o_i, a warp per row
template <typename T>
__global__ void __launch_bounds__(256) packed_delta_kernel(const T* __restrict__ o, const T* __restrict__ low,
                                                           const T* __restrict__ dout, HeadRows ds,
                                                    int Tq, int Hq, int D, int stride, float* __restrict__ delta) {
  const int lane = threadIdx.x % 32;
  const int64_t at = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (at >= (int64_t)Tq * Hq) return;
  const int i = (int)(at / Hq), h = (int)(at % Hq);
  const T *a = o + at * D, *b = dout + i * ds.row + h * ds.head;
  float s = 0.f;
  for (int c = lane; c < D; c += 32)
    s = fmaf(low != nullptr ? to_f32(a[c]) + to_f32(low[at * D + c]) : to_f32(a[c]), to_f32(b[c]), s);
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

// ------------------------------------------------------------------------- few queries, many keys
// A tile of 128 queries computes 128 rows of scores for every key that one of them sees. Where a sequence has few
// queries (a pooling query over all tokens of a volume, the next token behind a long context) almost all of that is
// masked, and there are fewer tiles than SMs. Here a CTA takes up to R rows (queries and heads that share a key head)
// of one sequence and a piece of its keys, and the pieces' sums are joined by a second kernel. It is bound by reading
// K and V: LP lanes hold a row's channels, eight each, and a warp has eight 16-byte loads of K and of V a lane under way.
// 16 sequences of 1029 .. 4101 keys, one query, 16 heads of 64 fp16: 805 us by tiles, 46 us here (40 us at 5.4 TB/s and 6 us for joining).
constexpr int kFewThreads = 128;

template <typename T>
__device__ __forceinline__ void store_low(T* o, T* low, int64_t at, float x) {
  const T y = from_f32<T>(x);
  o[at] = y;
  if (low != nullptr) low[at] = from_f32<T>(x - to_f32(y));
}

template <typename T, int LP, int R>
__global__ void __launch_bounds__(kFewThreads) packed_few_kernel(PackedProblem P, PackedFew few, T* __restrict__ o,
                                                                 float* __restrict__ lse) {
  constexpr int KP = 32 / LP, U = 8, W = U * KP;  // keys of a load, loads, keys of a warp at a time
  __shared__ float red[4][R][LP * 8 + 2];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, c = lane % LP, g = lane / LP;
  const int4 item = few.items[blockIdx.x];  // first query, queries, keys [z, w)
  const int hk = blockIdx.y, r0 = blockIdx.z * R, rows = item.y * P.group;
  if (r0 >= rows) return;
  const bool in = c * 8 < P.D;
  float q[R][8], acc[R][8], m[R], l[R];
  int lo[R], hi[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = min(r0 + r, rows - 1), i = item.x + row / P.group, h = hk * P.group + row % P.group;
    Raw8<T> raw = {};
    if (in) raw = load_raw8<T>((const T*)P.q + i * P.qs.row + h * P.qs.head + c * 8);
    unpack8<T>(raw, q[r]);
    const int2 b = P.q_bounds[i];
    lo[r] = b.x;
    hi[r] = b.y;
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[r][e] *= P.scale * kLog2e;
      acc[r][e] = 0.f;
    }
  }
  const T *kp = (const T*)P.k + hk * P.ks.head + c * 8, *vp = (const T*)P.v + hk * P.vs.head + c * 8;
  for (int kb = item.z + warp * W; kb < item.w; kb += 4 * W) {
    Raw8<T> kr[U], vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = kb + u * KP + g;
      kr[u] = vr[u] = {};
      if (in && key < item.w) {
        kr[u] = load_raw8<T>(kp + key * P.ks.row);
        vr[u] = load_raw8<T>(vp + key * P.vs.row);
      }
    }
    float s[R][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8];
      unpack8<T>(kr[u], x);
      const int key = kb + u * KP + g;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf(q[r][e], x[e], d);
#pragma unroll
        for (int w = 1; w < LP; w *= 2) d += __shfl_xor_sync(0xffffffffu, d, w);
        s[r][u] = key >= lo[r] && key < min(hi[r], item.w) ? d : -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float top = s[r][0];
#pragma unroll
      for (int u = 1; u < U; ++u) top = fmaxf(top, s[r][u]);
#pragma unroll
      for (int w = LP; w < 32; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float m_new = fmaxf(m[r], top), ref = m_new == -INFINITY ? 0.f : m_new, fade = exp2f(m[r] - ref);
      m[r] = m_new;
      l[r] *= fade;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r][e] *= fade;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[r][u] = exp2f(s[r][u] - ref);
        l[r] += s[r][u];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[8];
      unpack8<T>(vr[u], x);
      const int key = kb + u * KP + g;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (key >= lo[r] && key < hi[r])  // what a row does not see is not multiplied either
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[r][e] = fmaf(s[r][u], x[e], acc[r][e]);
    }
  }
  // a warp's keys lie in KP groups of lanes, the CTA's in four warps
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int w = LP; w < 32; w *= 2) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[r][e] += __shfl_xor_sync(0xffffffffu, acc[r][e], w);
    }
    if (g == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) red[warp][r][c * 8 + e] = acc[r][e];
      if (c == 0) {
        red[warp][r][LP * 8] = m[r];
        red[warp][r][LP * 8 + 1] = l[r];
      }
    }
  }
  __syncthreads();
  for (int at = threadIdx.x; at < R * LP * 8; at += kFewThreads) {
    const int r = at / (LP * 8), ch = at % (LP * 8), row = r0 + r;
    if (row >= rows || ch >= P.D) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, red[w][r][LP * 8]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, value = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f(red[w][r][LP * 8] - ref);
      sum += f * red[w][r][LP * 8 + 1];
      value += f * red[w][r][ch];
    }
    if (few.partial == nullptr) {
      const int i = item.x + row / P.group, h = hk * P.group + row % P.group;
      const int2 b = P.q_bounds[i];
      store_low<T>(o, (T*)P.o_low, ((int64_t)i * P.Hq + h) * P.D + ch, row_value(b.y > b.x, value, sum));
      if (ch == 0) lse[(int64_t)h * P.lse_stride + i] = row_lse(b.y > b.x, top, sum);
    } else {
      float* part = few.partial + (((int64_t)blockIdx.x * P.Hk + hk) * few.rows + row) * (P.D + 2);
      part[ch] = value;
      if (ch == 0) {
        part[P.D] = top;
        part[P.D + 1] = sum;
      }
    }
  }
}

// Joins the pieces of a sequence's keys in their order, a CTA per row and key head.
template <typename T>
__global__ void __launch_bounds__(128) packed_few_join_kernel(PackedProblem P, PackedFew few, T* __restrict__ o,
                                                              float* __restrict__ lse) {
  const int2 seq = few.pieces[blockIdx.x];  // first item, items
  if (seq.y == 0) return;
  const int4 item = few.items[seq.x];
  const int hk = blockIdx.y, row = blockIdx.z, ch = threadIdx.x;
  if (row >= item.y * P.group) return;
  const int64_t step = (int64_t)P.Hk * few.rows * (P.D + 2);
  const float* part = few.partial + ((int64_t)seq.x * P.Hk + hk) * few.rows * (P.D + 2) + (int64_t)row * (P.D + 2);
  float top = -INFINITY;
  for (int n = 0; n < seq.y; ++n) top = fmaxf(top, part[n * step + P.D]);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, value = 0.f;
  for (int n = 0; n < seq.y; ++n) {
    const float f = exp2f(part[n * step + P.D] - ref);
    sum += f * part[n * step + P.D + 1];
    if (ch < P.D) value += f * part[n * step + ch];
  }
  const int i = item.x + row / P.group, h = hk * P.group + row % P.group;
  const int2 b = P.q_bounds[i];
  if (ch < P.D) store_low<T>(o, (T*)P.o_low, ((int64_t)i * P.Hq + h) * P.D + ch, row_value(b.y > b.x, value, sum));
  if (ch == 0) lse[(int64_t)h * P.lse_stride + i] = row_lse(b.y > b.x, top, sum);
}

int64_t blocks_of(int64_t items, int per) { return (items + per - 1) / per; }
unsigned grid_of(int64_t items, int per) { return (unsigned)blocks_of(items, per); }

}  // namespace

cudaError_t packed_fwd_rows(const PackedProblem& P, void* o, float* lse, cudaStream_t stream) {
  if (blocks_of((int64_t)P.Tq * P.Hq, kWarps) > 0x7fffffff) return cudaErrorInvalidConfiguration;
  by_type(P.type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    packed_fwd_rows_kernel<T><<<grid_of((int64_t)P.Tq * P.Hq, kWarps), kWarps * 32, 0, stream>>>(P, (T*)o, lse);
  });
  return cudaGetLastError();
}

cudaError_t packed_fwd_few(const PackedProblem& P, const PackedFew& few, void* o, float* lse, cudaStream_t stream) {
  const bool wide = P.D > 64, several = few.rows > 1;
  by_type(P.type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto go = [&](auto kernel, int r) {
      kernel<<<dim3(few.count, P.Hk, (few.rows + r - 1) / r), kFewThreads, 0, stream>>>(P, few, (T*)o, lse);
    };
    if (wide) several ? go(packed_few_kernel<T, 16, 4>, 4) : go(packed_few_kernel<T, 16, 1>, 1);
    else several ? go(packed_few_kernel<T, 8, 4>, 4) : go(packed_few_kernel<T, 8, 1>, 1);
    if (few.partial != nullptr)
      packed_few_join_kernel<T><<<dim3(few.sequences, P.Hk, few.rows), 128, 0, stream>>>(P, few, (T*)o, lse);
  });
  return cudaGetLastError();
}

cudaError_t packed_bwd_rows(const PackedProblem& P, const void* o, const void* dout, HeadRows ds, const float* lse,
                            float* delta, void* dq, void* dk, void* dv, cudaStream_t stream) {
  if (blocks_of((int64_t)std::max(P.Tq, P.Tk) * P.Hq, kWarps) > 0x7fffffff) return cudaErrorInvalidConfiguration;
  by_type(P.type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const T* go = (const T*)dout;
    packed_delta_kernel<T><<<grid_of((int64_t)P.Tq * P.Hq, 8), 256, 0, stream>>>(
        (const T*)o, (const T*)P.o_low, go, ds, P.Tq, P.Hq, P.D, P.lse_stride, delta);
    packed_dq_rows_kernel<T><<<grid_of((int64_t)P.Tq * P.Hq, kWarps), kWarps * 32, 0, stream>>>(P, go, ds, lse, delta, (T*)dq);
    packed_dkv_rows_kernel<T><<<grid_of((int64_t)P.Tk * P.Hk, kWarps), kWarps * 32, 0, stream>>>(P, go, ds, lse, delta, (T*)dk,
                                                                                               (T*)dv);
  });
  return cudaGetLastError();
}

}  // namespace mia
