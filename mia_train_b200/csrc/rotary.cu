// Rotation of query and key heads by angles that are computed from the tokens' positions.
//
//   angle[t, p] = sum_a position[t, a] F[a, p]
//   y1 = amplitude (x1 cos - x2 sin),  y2 = amplitude (x2 cos + x1 sin)   for every pair (x1, x2) of the head
//
// (or the angles themselves are given), with the pairs (p, p + P) ("half") or (2 p, 2 p + 1) ("interleaved") of the
// first 2 P channels; the others are copied. The gradient of x is the rotation of dy by the negative angles, that of the table
// dF[a, p] = sum_t position[t, a] sum_heads (dy2 y1 - dy1 y2).
//
// Angles, in turns (1 is 2 pi), where whole turns fall away for nothing: an integer position times the frequency as a
// 64-bit fraction of a turn, modulo 2^64, is exact but for the fraction's own rounding (2^-53 of it); a floating-point
// position and the frequency are pairs of fp32 numbers (48 bits), products with their rounding error by fma, and
// p - rint(p) is exact. Either keeps a position of 2^20 as good as a small one, without the fp64 pipe, whose
// few lanes would take longer than the memory. A block makes the table of frequencies once (this is in fp64); sine and
// cosine are sincospif's. A thread has one place in the head (8 channels, or one pair) and goes through a token's heads
// with the angles in registers.
//
// The pass reads and writes every channel once and is bound by memory. The learned table's gradient stays in the
// thread's registers over all of its tokens; a block's sum goes to one row of partial sums, which a second kernel adds up
// in order (no atomics, the same bits every time).
#include <algorithm>
#include <type_traits>

#include "sequence_kernels.h"
#include "vec8.cuh"

namespace mia {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;

// The position as fp32 for the sums of the frequencies' gradient.
__device__ __forceinline__ float position_of(const RotaryParams& p, int64_t i) {
  if (p.pos_type == 0) return (float)((const int64_t*)p.pos)[i];
  if (p.pos_type == 1) return (float)((const int*)p.pos)[i];
  if (p.pos_type == 2) return ((const float*)p.pos)[i];
  return (float)((const double*)p.pos)[i];
}

__device__ __forceinline__ int64_t position_row(const RotaryParams& p, int64_t token) {
  return p.pos_b == 0 ? token % p.T : token;
}

// Frequency i in turns: a fraction of 2^64, or (high, low) fp32, as the positions are integers or not. A fraction of all
// ones says that the frequency is not finite; none that is comes to that (64-bit floats below 1 end at 1 - 2^-53, and f - floor(f)
// rounds to 1 itself for f just below 0, which is 0 of the next turn).
constexpr uint64_t kNotFinite = ~uint64_t(0);
__device__ __forceinline__ uint2 frequency(const RotaryParams& p, int i) {
  double f = p.freq64 ? ((const double*)p.freq)[i] : (double)((const float*)p.freq)[i];
  f *= 0.15915494309189533577;  // 1 / (2 pi)
  if (p.pos_type <= 1) {
    const double part = f - floor(f);
    const uint64_t u = !isfinite(f) ? kNotFinite : part < 1.0 ? (uint64_t)(part * 18446744073709551616.0) : 0;  // 2^64
    return make_uint2((uint32_t)u, (uint32_t)(u >> 32));
  }
  const float hi = (float)f, lo = (float)(f - (double)hi);
  return make_uint2(__float_as_uint(hi), __float_as_uint(lo));
}

// (cos, sin) of the token's angle of pair i, times the amplitude; `at` is the token's row of positions
__device__ __forceinline__ float2 turn(const RotaryParams& p, const uint2* table, int64_t at, int i) {
  float half;  // in half turns
  if (p.freq == nullptr) {
    const float x = ((const float*)p.pos)[at + i];
    const float hi = 0.15915493667125702f, lo = 6.4206382432985265e-09f;  // 1 / (2 pi) as two fp32
    const float w = x * hi, whole = w - rintf(w) + fmaf(x, lo, fmaf(x, hi, -w));
    half = 2.f * (whole - rintf(whole));
  } else if (p.pos_type <= 1) {
    uint64_t u = 0;
    bool finite = true;
    for (int a = 0; a < p.axes; ++a) {
      const uint2 f = table[a * p.P + i];
      finite = finite && (f.x & f.y) != (uint32_t)kNotFinite;
      const int64_t x = p.pos_type == 0 ? ((const int64_t*)p.pos)[at + a] : (int64_t)((const int*)p.pos)[at + a];
      u += (uint64_t)x * ((uint64_t)f.y << 32 | f.x);
    }
    half = finite ? (float)(int)((u + 0x80000000u) >> 32) * 4.6566128730773926e-10f : NAN;  // 2^-31
  } else {
    float whole = 0.f, rest = 0.f;
    for (int a = 0; a < p.axes; ++a) {
      const uint2 f = table[a * p.P + i];
      const float f_hi = __uint_as_float(f.x), f_lo = __uint_as_float(f.y);
      float hi, lo = 0.f;
      if (p.pos_type == 2) {
        hi = ((const float*)p.pos)[at + a];
      } else {
        const double x = ((const double*)p.pos)[at + a];
        hi = (float)x;
        lo = (float)(x - (double)hi);
        const float w = lo * f_hi;
        whole += w - rintf(w);
        rest += fmaf(lo, f_hi, -w);
      }
      const float w = hi * f_hi;
      whole += w - rintf(w);
      rest += fmaf(hi, f_lo, fmaf(hi, f_hi, -w));
    }
    whole += rest;
    half = 2.f * (whole - rintf(whole));
  }
  float s, c;
  sincospif(half, &s, &c);
  return make_float2(c * p.amplitude, (p.inverse ? -s : s) * p.amplitude);
}

// kVec: 8 channels (of each half) at a time, which needs P (half) or 2 P (interleaved), D and the strides in
// multiples of 8 and 16-byte aligned rows; else one pair or channel at a time.
template <typename T, bool kInter, bool kVec, bool kLearn>
__global__ void __launch_bounds__(kThreads, kLearn ? 2 : 3) rotary_kernel(const RotaryParams p) {
  extern __shared__ uint2 table[];  // (axes, P) frequencies; at the end (slots, axes, P) sums of their gradient
  constexpr int W = kVec ? 8 : 1;
  constexpr int kPairs = kVec ? (kInter ? 4 : 8) : 1;  // pairs of one item
  constexpr int kVecs = kVec && !kInter ? 2 : 1;
  __shared__ float2 angles[kPairs * kThreads];  // a thread's own
  constexpr int kAtOnce = sizeof(T) == 4 || (kLearn && !kInter) ? 2 : 4;  // heads whose loads are under way together
  const int turned = p.P / kPairs;
  const int items = turned + (p.D - 2 * p.P) / W;  // of one head
  const int slots = kThreads / items;
  const int v = threadIdx.x % items, slot = threadIdx.x / items;
  const int H = p.Hq + p.Hk;
  const bool rotates = v < turned;
  // first channels of the item: one vector of the head (interleaved, copied) or two (half)
  const int c1 = rotates ? (kInter ? v * (kVec ? 8 : 2) : v * W) : 2 * p.P + (v - turned) * W;
  const int c2 = kInter ? c1 + 1 : c1 + p.P;
  const int h_begin = blockIdx.y * p.heads, h_end = min(h_begin + p.heads, H);
  float sum[kLearn ? kMaxAxes : 1][kPairs];
  if constexpr (kLearn)
#pragma unroll
    for (int a = 0; a < kMaxAxes; ++a)
#pragma unroll
      for (int e = 0; e < kPairs; ++e) sum[a][e] = 0.f;

  if (p.freq != nullptr) {
    for (int i = threadIdx.x; i < p.axes * p.P; i += kThreads) table[i] = frequency(p, i);
    __syncthreads();
  }
  for (int64_t token = (int64_t)blockIdx.x * slots + slot; slot < slots && token < p.tokens;
       token += (int64_t)gridDim.x * slots) {
    const int64_t b = token / p.T, t = token - b * p.T;
    const int64_t at = position_row(p, token) * (p.freq == nullptr ? p.P : p.axes);
    float2 cs[kPairs];
    float g[kPairs];
#pragma unroll
    for (int e = 0; e < kPairs; ++e) g[e] = 0.f;
    const T *q = (const T*)p.q + b * p.qs.b + t * p.qs.t, *k = (const T*)p.k + b * p.ks.b + t * p.ks.t;
    T *yq = (T*)p.yq + b * p.yqs.b + t * p.yqs.t, *yk = (T*)p.yk + b * p.yks.b + t * p.yks.t;
    const T* xq = kLearn ? (const T*)p.xq + b * p.xqs.b + t * p.xqs.t : nullptr;
    const T* xk = kLearn ? (const T*)p.xk + b * p.xks.b + t * p.xks.t : nullptr;
    for (int h0 = h_begin; h0 < h_end; h0 += kAtOnce) {
      Raw8<T> raw[kAtOnce][kVecs], kept[kLearn ? kAtOnce : 1][kVecs];
      T one[kAtOnce][2], own[kLearn ? kAtOnce : 1][2];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int h = h0 + u;
        if (h >= h_end) break;
        const T* src = h < p.Hq ? q + h * p.qs.h : k + (h - p.Hq) * p.ks.h;
        if constexpr (kVec) {
          raw[u][0] = load_raw8<T>(src + c1);
          if (!kInter && rotates) raw[u][kVecs - 1] = load_raw8<T>(src + c2);
        } else {
          one[u][0] = src[c1];
          if (rotates) one[u][1] = src[c2];
        }
        if constexpr (kLearn) {
          if (!rotates) continue;
          const T* x = h < p.Hq ? xq + h * p.xqs.h : xk + (h - p.Hq) * p.xks.h;
          if constexpr (kVec) {
            kept[u][0] = load_raw8<T>(x + c1);
            if (!kInter) kept[u][kVecs - 1] = load_raw8<T>(x + c2);
          } else {
            own[u][0] = x[c1];
            own[u][1] = x[c2];
          }
        }
      }
      if (h0 == h_begin && rotates) {
        // While the first loads are under way. By way of shared memory, so that the code of one angle is there once:
        // fetching eight copies took longer than a small call's work (3 us more for nine tokens, which take 5).
        float2* mine = angles + threadIdx.x;
#pragma unroll 1
        for (int e = 0; e < kPairs; ++e) mine[e * kThreads] = turn(p, table, at, v * kPairs + e);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) cs[e] = mine[e * kThreads];
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int h = h0 + u;
        if (h >= h_end) break;
        T* dst = h < p.Hq ? yq + h * p.yqs.h : yk + (h - p.Hq) * p.yks.h;
        if (!rotates) {
          if constexpr (kVec) {
#pragma unroll
            for (int w = 0; w < (int)(sizeof(Raw8<T>) / 16); ++w) reinterpret_cast<uint4*>(dst + c1)[w] = raw[u][0].u[w];
          } else {
            dst[c1] = one[u][0];
          }
          continue;
        }
        float x1[kPairs], x2[kPairs];
        auto pairs_of = [&](const Raw8<T>(&r)[kVecs], const T(&single)[2]) {
          if constexpr (!kVec) {
            x1[0] = to_f32(single[0]);
            x2[0] = to_f32(single[1]);
          } else if constexpr (kInter) {
            float x[8];
            unpack8<T>(r[0], x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x1[e] = x[2 * e];
              x2[e] = x[2 * e + 1];
            }
          } else {
            unpack8<T>(r[0], x1);
            unpack8<T>(r[kVecs - 1], x2);
          }
        };
        pairs_of(raw[u], one[u]);
        float y1[kPairs], y2[kPairs];
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          y1[e] = x1[e] * cs[e].x - x2[e] * cs[e].y;
          y2[e] = x2[e] * cs[e].x + x1[e] * cs[e].y;
        }
        if constexpr (!kVec) {
          dst[c1] = from_f32<T>(y1[0]);
          dst[c2] = from_f32<T>(y2[0]);
        } else if constexpr (kInter) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[2 * e] = y1[e];
            y[2 * e + 1] = y2[e];
          }
          store8<T>(dst + c1, y);
        } else {
          store8<T>(dst + c1, y1);
          store8<T>(dst + c2, y2);
        }
        if constexpr (kLearn) {
          // Here x is dy and y its gradient dx = R(-angle) dy: dy2 y1 - dy1 y2 of the forward pass's outputs is the
          // same turned back by the angle, dx2 x1 - dx1 x2 with its inputs.
          pairs_of(kept[u], own[u]);
#pragma unroll
          for (int e = 0; e < kPairs; ++e) g[e] += y2[e] * x1[e] - y1[e] * x2[e];
        }
      }
    }
    if constexpr (kLearn) {
#pragma unroll
      for (int a = 0; a < kMaxAxes; ++a) {
        if (a >= p.axes) break;
        const float at_a = position_of(p, at + a);
#pragma unroll
        for (int e = 0; e < kPairs; ++e) sum[a][e] = fmaf(at_a, g[e], sum[a][e]);
      }
    }
  }
  if constexpr (kLearn) {
    float* block_sums = reinterpret_cast<float*>(table);
    __syncthreads();
    if (slot < slots && rotates)
#pragma unroll
      for (int a = 0; a < kMaxAxes; ++a) {
        if (a >= p.axes) break;
#pragma unroll
        for (int e = 0; e < kPairs; ++e) block_sums[(slot * p.axes + a) * p.P + v * kPairs + e] = sum[a][e];
      }
    __syncthreads();
    const int per = p.axes * p.P;
    for (int i = threadIdx.x; i < per; i += kThreads) {
      float s = 0.f;
      for (int u = 0; u < slots; ++u) s += block_sums[u * per + i];
      p.partial[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * per + i] = s;
    }
  }
}

// dF[i] = sum over the blocks' partial sums, in 64 bits, a warp per element
__global__ void __launch_bounds__(128) rotary_sum_kernel(const float* __restrict__ partial, int blocks, int per,
                                                         float* __restrict__ out) {
  const int i = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (i >= per) return;
  double s = 0.0;
  for (int b = lane; b < blocks; b += 32) s += (double)partial[(int64_t)b * per + i];
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
  if (lane == 0) out[i] = (float)s;
}

template <typename T, bool kInter>
cudaError_t launch(const RotaryParams& p, const RotaryPlan& plan, bool learn, cudaStream_t stream) {
  auto go = [&](auto kernel) {
    kernel<<<dim3(plan.grid, plan.chunks), kThreads, plan.smem, stream>>>(p);
    return cudaGetLastError();
  };
  if (learn) return plan.vec ? go(rotary_kernel<T, kInter, true, true>) : go(rotary_kernel<T, kInter, false, true>);
  return plan.vec ? go(rotary_kernel<T, kInter, true, false>) : go(rotary_kernel<T, kInter, false, false>);
}

}  // namespace

// `aligned`: 16-byte aligned rows and strides in multiples of 8 elements everywhere.
RotaryPlan rotary_plan(const RotaryParams& p, bool aligned, bool interleaved, bool learn) {
  RotaryPlan plan;
  plan.vec = aligned && p.D % 8 == 0 && (interleaved ? 2 * p.P : p.P) % 8 == 0;
  const int pairs = plan.vec ? (interleaved ? 4 : 8) : 1, w = plan.vec ? 8 : 1;
  const int items = p.P / pairs + (p.D - 2 * p.P) / w;
  const int slots = kThreads / items;
  const int H = p.Hq + p.Hk;
  // A block has `slots` tokens at a time; with too few tokens for six blocks on every SM their heads are shared out, four
  // at least to a block as long as that leaves one for every SM (each block computes the angles again).
  const int64_t blocks = (p.tokens + slots - 1) / slots;
  plan.grid = (unsigned)std::min<int64_t>(blocks, learn ? 148 * 4 : 148 * 12);
  int64_t chunks = std::max<int64_t>(1, 6 * 148 / std::max<int64_t>(blocks, 1));
  chunks = std::min<int64_t>(chunks, std::max<int64_t>((H + 3) / 4, 148 / std::max<int64_t>(blocks, 1)));
  chunks = std::min<int64_t>(chunks, H);
  plan.heads = (int)((H + chunks - 1) / chunks);
  plan.chunks = (unsigned)((H + plan.heads - 1) / plan.heads);
  plan.smem = (size_t)p.axes * p.P * std::max<size_t>(sizeof(uint2), learn ? slots * sizeof(float) : 0);
  return plan;
}

cudaError_t rotary_launch(RotaryParams p, const RotaryPlan& plan, SequenceType type, bool interleaved, float* dfreq,
                          cudaStream_t stream) {
  p.heads = plan.heads;
  auto run = [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    return interleaved ? launch<T, true>(p, plan, dfreq != nullptr, stream)
                       : launch<T, false>(p, plan, dfreq != nullptr, stream);
  };
  const cudaError_t status = type == kSeqBf16 ? run((__nv_bfloat16*)nullptr)
                             : type == kSeqF16 ? run((__half*)nullptr)
                                               : run((float*)nullptr);
  if (status != cudaSuccess || dfreq == nullptr) return status;
  const int per = p.axes * p.P;
  if (per == 0) return cudaSuccess;  // no pairs: the table has no element
  rotary_sum_kernel<<<(per + 3) / 4, 128, 0, stream>>>(p.partial, (int)(plan.grid * plan.chunks), per, dfreq);
  return cudaGetLastError();
}

}  // namespace mia
