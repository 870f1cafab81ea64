// Rotation of query and key heads by angles that are computed from the tokens' positions.
//
//   angle[t, p] = sum_a position[t, a] F[a, p]
//   y1 = amplitude (x1 cos - x2 sin),  y2 = amplitude (x2 cos + x1 sin)   for every pair (x1, x2) of the head
//
// with the pairs (p, p + P) ("half") or (2 p, 2 p + 1) ("interleaved") of the first 2 P channels; the others are
// copied. The gradient of x is the rotation of dy by the negative angles, that of the table
// dF[a, p] = sum_t position[t, a] sum_heads (dy2 y1 - dy1 y2).
//
// Angles: the products are formed in 64 bits and reduced to a fraction of a turn there, so that a position of 2^20
// keeps the accuracy of a small one; sine and cosine of the reduced angle are sincospif's. They are computed once per
// token and pair and shared by all heads of the token (a block owns some tokens, its tables are in shared memory).
//
// The pass reads and writes every channel once and is bound by memory. A thread keeps its place within the head, so
// that the learned table's gradient stays in its registers until the end: a block's sum goes to one row of partial
// sums, which a second kernel adds up in order (no atomics, the same bits every time).
#include <algorithm>
#include <type_traits>

#include "sequence_kernels.h"
#include "vec8.cuh"

namespace mia {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;

__device__ __forceinline__ double position_of(const RotaryParams& p, int64_t i) {
  if (p.pos_type == 0) return (double)((const int64_t*)p.pos)[i];
  if (p.pos_type == 1) return (double)((const int*)p.pos)[i];
  if (p.pos_type == 2) return (double)((const float*)p.pos)[i];
  return ((const double*)p.pos)[i];
}

__device__ __forceinline__ int64_t position_row(const RotaryParams& p, int64_t token) {
  return p.pos_b == 0 ? token % p.T : token;
}

// (cos, sin) of the token's angle of pair i, times the amplitude
__device__ __forceinline__ float2 turn(const RotaryParams& p, int64_t token, int i) {
  const int64_t row = position_row(p, token) * p.axes;
  double x = 0.0;
  for (int a = 0; a < p.axes; ++a) {
    const double f = p.freq64 ? ((const double*)p.freq)[a * p.P + i] : (double)((const float*)p.freq)[a * p.P + i];
    x = fma(position_of(p, row + a), f, x);
  }
  double half = x * 0.31830988618379067154;  // in half turns
  half -= 2.0 * rint(0.5 * half);
  float s, c;
  sincospif((float)half, &s, &c);
  return make_float2(c * p.amplitude, (p.inverse ? -s : s) * p.amplitude);
}

// kVec: 8 channels (of each half) at a time, which needs P (half) or 2 P (interleaved), D and the strides in
// multiples of 8 and 16-byte aligned rows; else one pair or channel at a time.
template <typename T, bool kInter, bool kVec, bool kLearn>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryParams p) {
  extern __shared__ float2 table[];  // (group, P); at the end (slots, axes, pairs of a thread) of the frequency sums
  constexpr int W = kVec ? 8 : 1;
  constexpr int kPairs = kVec ? (kInter ? 4 : 8) : 1;  // pairs of one item
  const int turned = p.P / kPairs;
  const int items = turned + (p.D - 2 * p.P) / W;  // of one head
  const int slots = kThreads / items;
  const int v = threadIdx.x % items, slot = threadIdx.x / items;
  const int H = p.Hq + p.Hk;
  const bool rotates = v < turned;
  // first channels of the item: one vector of the head (interleaved, copied) or two (half)
  const int c1 = rotates ? (kInter ? v * (kVec ? 8 : 2) : v * W) : 2 * p.P + (v - turned) * W;
  const int c2 = kInter ? c1 + 1 : c1 + p.P;
  float sum[kLearn ? kMaxAxes : 1][kPairs];
  if constexpr (kLearn)
#pragma unroll
    for (int a = 0; a < kMaxAxes; ++a)
#pragma unroll
      for (int e = 0; e < kPairs; ++e) sum[a][e] = 0.f;

  constexpr int kAtOnce = sizeof(T) == 4 || (kLearn && !kInter) ? 2 : 4;
  const int step_t = slots / H, step_h = slots % H;
  const int64_t groups = (p.tokens + p.group - 1) / p.group;
  for (int64_t gi = blockIdx.x; gi < groups; gi += gridDim.x) {
    const int64_t first = gi * p.group;
    const int n = (int)min((int64_t)p.group, p.tokens - first);
    __syncthreads();
    for (int i = threadIdx.x; i < n * p.P; i += kThreads) table[i] = turn(p, first + i / p.P, i % p.P);
    __syncthreads();
    if (slot >= slots) continue;
    int tk = slot / H, h = slot % H;
    for (int at = slot; at < n * H; at += kAtOnce * slots) {
      // the loads of kAtOnce heads are under way before the first is worked on
      constexpr int kVecs = !kVec ? 1 : kInter ? 1 : 2;
      Raw8<T> raw[kAtOnce][kVecs];
      Raw8<T> kept[kLearn ? kAtOnce : 1][kVecs];
      T one[kAtOnce][2], own[kLearn ? kAtOnce : 1][2];
      int token_of[kAtOnce];
      T* dst[kAtOnce];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        dst[u] = nullptr;
        if (at + u * slots < n * H) {
          const int64_t token = first + tk, b = token / p.T, t = token - b * p.T;
          const bool is_q = h < p.Hq;
          const int hh = is_q ? h : h - p.Hq;
          const TokenRows rs = is_q ? p.qs : p.ks, ws = is_q ? p.yqs : p.yks;
          const T* src = (const T*)(is_q ? p.q : p.k) + b * rs.b + t * rs.t + hh * rs.h;
          dst[u] = (T*)(is_q ? p.yq : p.yk) + b * ws.b + t * ws.t + hh * ws.h;
          token_of[u] = tk;
          if constexpr (kVec) {
            raw[u][0] = load_raw8<T>(src + c1);
            if (!kInter && rotates) raw[u][kVecs - 1] = load_raw8<T>(src + c2);
          } else {
            one[u][0] = src[c1];
            if (rotates) one[u][1] = src[c2];
          }
          if constexpr (kLearn) {
            const TokenRows xs = is_q ? p.xqs : p.xks;
            const T* x = (const T*)(is_q ? p.xq : p.xk) + b * xs.b + t * xs.t + hh * xs.h;
            if (rotates) {
              if constexpr (kVec) {
                kept[u][0] = load_raw8<T>(x + c1);
                if (!kInter) kept[u][kVecs - 1] = load_raw8<T>(x + c2);
              } else {
                own[u][0] = x[c1];
                own[u][1] = x[c2];
              }
            }
          }
        }
        tk += step_t;
        h += step_h;
        if (h >= H) {
          h -= H;
          ++tk;
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (dst[u] == nullptr) break;
        if (!rotates) {
          if constexpr (kVec) {
#pragma unroll
            for (int w = 0; w < (int)(sizeof(Raw8<T>) / 16); ++w) reinterpret_cast<uint4*>(dst[u] + c1)[w] = raw[u][0].u[w];
          } else {
            dst[u][c1] = one[u][0];
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
        const float2* cs = table + token_of[u] * p.P + v * kPairs;
        float y1[kPairs], y2[kPairs];
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
          const float2 r = cs[e];
          y1[e] = x1[e] * r.x - x2[e] * r.y;
          y2[e] = x2[e] * r.x + x1[e] * r.y;
        }
        if constexpr (!kVec) {
          dst[u][c1] = from_f32<T>(y1[0]);
          dst[u][c2] = from_f32<T>(y2[0]);
        } else if constexpr (kInter) {
          float y[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[2 * e] = y1[e];
            y[2 * e + 1] = y2[e];
          }
          store8<T>(dst[u] + c1, y);
        } else {
          store8<T>(dst[u] + c1, y1);
          store8<T>(dst[u] + c2, y2);
        }
        if constexpr (kLearn) {
          // Here x is dy and y its gradient dx = R(-angle) dy: dy2 y1 - dy1 y2 of the forward pass's outputs is the
          // same turned back by the angle, dx2 x1 - dx1 x2 with its inputs.
          pairs_of(kept[u], own[u]);
          const int64_t row = position_row(p, first + token_of[u]) * p.axes;
#pragma unroll
          for (int e = 0; e < kPairs; ++e) x1[e] = y2[e] * x1[e] - y1[e] * x2[e];
#pragma unroll
          for (int a = 0; a < kMaxAxes; ++a) {
            if (a >= p.axes) break;
            const float at_a = (float)position_of(p, row + a);
#pragma unroll
            for (int e = 0; e < kPairs; ++e) sum[a][e] = fmaf(at_a, x1[e], sum[a][e]);
          }
        }
      }
    }
  }
  if constexpr (kLearn) {
    float* out = reinterpret_cast<float*>(table);  // (slots, axes, P)
    __syncthreads();
    if (slot < slots && rotates)
      for (int a = 0; a < p.axes; ++a)
#pragma unroll
        for (int e = 0; e < kPairs; ++e) out[(slot * p.axes + a) * p.P + v * kPairs + e] = sum[a][e];
    __syncthreads();
    const int per = p.axes * p.P;
    for (int i = threadIdx.x; i < per; i += kThreads) {
      float s = 0.f;
      for (int u = 0; u < slots; ++u) s += out[u * per + i];
      p.partial[(int64_t)blockIdx.x * per + i] = s;
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
    kernel<<<plan.grid, kThreads, plan.smem, stream>>>(p);
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
  // Tokens of a block at a time: enough for some sixteen items a thread, few enough that every SM has two blocks, and at
  // most 32 KB of tables.
  const int64_t per_token = (int64_t)items * (p.Hq + p.Hk);
  int64_t group = std::max<int64_t>(1, 16 * kThreads / per_token);
  group = std::min<int64_t>(group, std::max<int64_t>(1, p.tokens / (2 * 148)));
  group = std::min<int64_t>(group, std::max(1, 4096 / std::max(p.P, 1)));
  plan.group = (int)group;
  plan.grid = (unsigned)std::min<int64_t>((p.tokens + group - 1) / group, learn ? 148 * 4 : 148 * 16);
  plan.smem = (size_t)group * p.P * sizeof(float2);
  if (learn) plan.smem = std::max(plan.smem, (size_t)slots * p.axes * p.P * sizeof(float));
  return plan;
}

cudaError_t rotary_launch(RotaryParams p, const RotaryPlan& plan, SequenceType type, bool interleaved, float* dfreq,
                          cudaStream_t stream) {
  p.group = plan.group;
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
  rotary_sum_kernel<<<(per + 3) / 4, 128, 0, stream>>>(p.partial, (int)plan.grid, per, dfreq);
  return cudaGetLastError();
}

}  // namespace mia
