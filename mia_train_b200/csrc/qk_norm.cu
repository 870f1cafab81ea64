// RMS norm of every query and key head with its learned weight, and the position rotation, in one
// pass; forward and backward.
//
//   r = 1 / sqrt(mean_c x[c]^2 + eps),  n[c] = x[c] r w[c]
//   y[i] = n[i] cos a_p - n[j] sin a_p,  y[j] = n[j] cos a_p + n[i] sin a_p     for pair p = (i, j)
//   y[c] = n[c]                                                                for unpaired channels
//
// With C[c] = cos a_p and S[c] = -sin a_p (c first of its pair) or +sin a_p (second), and c' the
// partner of c (C = 1, S = 0 when there is none): y[c] = n[c] C[c] + n[c'] S[c]. Backward:
//   dn[c] = dy[c] C[c] - dy[c'] S[c]
//   dw[c] += dn[c] x[c] r                       (over all heads of all tokens)
//   dx[c] = r (g[c] - x[c] r mean_c(g x r)),    g = dn w
//   da_p  = n[i] dn[j] - n[j] dn[i], summed over the token's query and key heads; dn[c'] needs only
//           dy[c'] C[c] + dy[c] S[c], which the lane of c has, so each lane adds +-n[c] dn[c'] alone
//
// A warp walks whole tokens (forward: query and key heads in turn; backward: one warp of a pair the query
// heads, the other the key heads, their parts of da_p joined in shared memory). The sine and cosine of the
// token's angles are computed once and kept by every lane for its eight channels; the heads then pass
// 256 / D' at a time (D' = D rounded up to a power of two, D' / 8 lanes a head), 16 bytes a lane. The grid
// is as large as fits on the SMs at once; a warp loads several such steps together, the next ones (of the
// next token as well) while it works on the last, and the next token's angles with them.
// Partners: where every lane's eight channels are paired with the same eight of one other lane (rotation by halves, where half
// of a head is a multiple of eight), by shuffles; otherwise (axial chunks) through shared memory
// at index c + c / 8, which spreads the stride of eight between lanes over all banks. Each element is read
// once and written once.
// Weight gradients: registers over a warp's tokens, one partial a CTA, summed in a fixed order by a
// second kernel, so the result does not depend on the order in which CTAs run.
// Measured, 4 x 4101 tokens of 16 query and 16 key heads of 64, bf16, ten launches from a graph: forward 34 us (4.0 TB/s),
// backward 62 us (3.2 TB/s). ncu: 0.6 instructions issued a cycle and scheduler with 16 warps an SM, DRAM at a third: what
// binds is the latency of the chain from a head's load over its sums to its store, with 19 instructions a value forward and
// 37 backward, a third of them the token's table and addresses.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "block_ops.h"
#include "common.cuh"
#include "vec8.cuh"

namespace mia {

constexpr int kQkWarps = 4;
constexpr int kQkMaxD = 256;

struct HeadView {  // (B, T, H, D) with unit channel stride; strides in elements
  void* p;
  int64_t sb, st;
  int sh;
  int heads;
};

struct QkNormParams {
  HeadView x[2];   // q, k (input)
  HeadView dy[2];  // gradients of the outputs (backward)
  HeadView y[2];   // outputs (forward: rotated; backward: dx)
  const float* w[2];
  const float* angles;  // (1 or B, T, P) or nullptr
  int64_t angle_bstride;
  const int* pairs;  // (P, 2)
  int P;
  float* dangles;   // (B, T, P) or nullptr
  float* dw_parts;  // (CTAs, 2, D) or nullptr
  unsigned B, T;
  int D;
  float eps;
};

__device__ __forceinline__ int qk_pad(int c) { return c + (c >> 3); }

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Head h of token `token` of the flattened (B, T); tokens are counted in 32 bits (64-bit division is slow).
template <typename T>
__device__ __forceinline__ T* head_ptr(const HeadView& v, unsigned token, unsigned length, int h) {
  const unsigned b = token / length, t = token - b * length;
  return reinterpret_cast<T*>(v.p) + (int64_t)b * v.sb + (int64_t)t * v.st + h * v.sh;
}

// Shared memory of one CTA: per warp the token's (C, S) table and the exchange rows; the partner of each channel.
template <int LPR>
struct QkSmem {
  static constexpr int kRows = 32 / LPR;             // heads a warp holds at a time
  static constexpr int kCh = LPR * 8;                // channels of a head, rounded up
  static constexpr int kRowFloats = kCh + LPR;       // padded exchange row
  float2 cs[kQkWarps][kCh];
  float ex[kQkWarps][kRows][kRowFloats];
  int partner[kCh];
  int2 pairs[kCh / 2];  // x < 0: left out
  float da[kQkWarps][kRowFloats];  // backward: each warp's part of the token's angle gradient
  int scattered;  // not 0: some lane's channels are paired with channels of several lanes
};

constexpr int kQkAhead = 4;  // steps whose loads are in flight together (backward: half of them, for x and dy)

// Fills partner and pairs; a pair that names a channel outside the head is left out.
template <int LPR>
__device__ __forceinline__ void qk_partners(QkSmem<LPR>& sm, const QkNormParams& p) {
  if (threadIdx.x == 0) sm.scattered = 0;
  for (int c = threadIdx.x; c < QkSmem<LPR>::kCh; c += blockDim.x) {
    sm.partner[c] = c;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < kQkWarps * QkSmem<LPR>::kCh; c += blockDim.x) (&sm.cs[0][0])[c] = make_float2(1.f, 0.f);
  if (p.angles != nullptr)
    for (int i = threadIdx.x; i < p.P; i += blockDim.x) {
      const int a = p.pairs[2 * i], b = p.pairs[2 * i + 1];
      sm.pairs[i] = make_int2(-1, -1);
      if ((unsigned)a < (unsigned)p.D && (unsigned)b < (unsigned)p.D && a != b) {
        sm.partner[a] = b;
        sm.partner[b] = a;
        sm.pairs[i] = make_int2(a, b);
      }
    }
  __syncthreads();
  for (int c = threadIdx.x; c < QkSmem<LPR>::kCh; c += blockDim.x)
    if (sm.partner[c] != (sm.partner[c & ~7] & ~7) + (c & 7)) sm.scattered = 1;
  __syncthreads();
}

// The values of this lane's partner channels: `raw` as loaded, `v` its eight values.
template <int LPR, typename T>
__device__ __forceinline__ void qk_exchange(const Raw8<T>& raw, const float (&v)[8], float (&o)[8], float* ex, int cg,
                                            const int (&part)[8], bool scattered, int source) {
  if (scattered) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) ex[cg * 9 + j] = v[j];
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = ex[part[j]];
  } else {
    Raw8<T> other;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      other.u[i].x = __shfl_sync(0xffffffffu, raw.u[i].x, source);
      other.u[i].y = __shfl_sync(0xffffffffu, raw.u[i].y, source);
      other.u[i].z = __shfl_sync(0xffffffffu, raw.u[i].z, source);
      other.u[i].w = __shfl_sync(0xffffffffu, raw.u[i].w, source);
    }
    unpack8(other, o);
  }
}

// A token's angles, lane i holding i, i + 32, ...
constexpr int kQkAngles = kQkMaxD / 2 / 32;
__device__ __forceinline__ void qk_fetch_angles(const QkNormParams& p, unsigned token, int lane, float (&ang)[kQkAngles]) {
  if (p.angles == nullptr) return;
  const unsigned b = token / p.T, t = token - b * p.T;
  const float* a = p.angles + (int64_t)b * p.angle_bstride + (int64_t)t * p.P;
#pragma unroll
  for (int k = 0; k < kQkAngles; ++k)
    if (lane + 32 * k < p.P) ang[k] = a[lane + 32 * k];
}

// The (C, S) table of a token, by one warp; entries of unpaired channels stay (1, 0) from the start.
template <int LPR>
__device__ __forceinline__ void qk_table(float2* cs, const QkNormParams& p, const int2* pairs, int lane,
                                         const float (&ang)[kQkAngles]) {
  __syncwarp();
  if (p.angles != nullptr) {
#pragma unroll
    for (int k = 0; k < kQkAngles; ++k) {
      const int i = lane + 32 * k;
      if (i < p.P && pairs[i].x >= 0) {
        float s, co;
        sincosf(ang[k], &s, &co);
        cs[pairs[i].x] = make_float2(co, -s);
        cs[pairs[i].y] = make_float2(co, s);
      }
    }
  }
  __syncwarp();
}

// Loads of AHEAD steps of a warp's walk over one token's heads: src is this lane's place in head `row`, the steps
// are heads h0, h0 + 32 / LPR, ... on from there; `left` = heads - row, or none for a lane past the channels.
template <typename T, int LPR, int AHEAD>
__device__ __forceinline__ void qk_load(const T* src, int sh, int h0, int left, Raw8<T> (&raw)[AHEAD]) {
#pragma unroll
  for (int u = 0; u < AHEAD; ++u) {
    const int h = h0 + u * (32 / LPR);
    raw[u] = h < left ? load_raw8(src + h * sh) : Raw8<T>{};
  }
}

template <typename T, int LPR>
__global__ void __launch_bounds__(32 * kQkWarps, 4) qk_norm_fwd_kernel(const QkNormParams p) {
  using S = QkSmem<LPR>;
  constexpr int kAhead = sizeof(T) == 2 ? kQkAhead : kQkAhead / 2;
  __shared__ S sm;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int row = lane / LPR, cg = lane % LPR;
  const bool on = cg * 8 < p.D;
  const unsigned tokens = p.B * p.T, stride = gridDim.x * kQkWarps;
  unsigned token = blockIdx.x * kQkWarps + warp;
  float ang[kQkAngles] = {};
  Raw8<T> next[kAhead];
  if (token < tokens) {
    qk_fetch_angles(p, token, lane, ang);
    qk_load<T, LPR>(head_ptr<const T>(p.x[0], token, p.T, row) + cg * 8, p.x[0].sh, 0, on ? p.x[0].heads - row : 0, next);
  }
  qk_partners<LPR>(sm, p);
  if (token >= tokens) return;
  // y[c] = r (x[c] (w[c] C[c]) + x[c'] (w[c'] S[c])): both factors are made once a token, x itself is exchanged
  float w[2][8], w_other[2][8], C[8], Sn[8];
  int part[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    part[j] = qk_pad(sm.partner[cg * 8 + j]);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      w[s][j] = (on && p.w[s] != nullptr) ? p.w[s][cg * 8 + j] : 1.f;
      w_other[s][j] = (on && p.w[s] != nullptr) ? p.w[s][sm.partner[cg * 8 + j]] : 1.f;
    }
  }
  const bool scattered = sm.scattered != 0;
  const int source = row * LPR + sm.partner[cg * 8] / 8;
  const float inv_d = 1.f / (float)p.D;
  float* ex = sm.ex[warp][row];
  for (; token < tokens; token += stride) {
    qk_table<LPR>(sm.cs[warp], p, sm.pairs, lane, ang);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 v = sm.cs[warp][cg * 8 + j];
      C[j] = v.x;
      Sn[j] = v.y;
    }
    const unsigned after = token + stride;
    if (after < tokens) qk_fetch_angles(p, after, lane, ang);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int heads = p.x[s].heads, sh = p.x[s].sh, left = on ? heads - row : 0;
      const T* const src = head_ptr<const T>(p.x[s], token, p.T, row) + cg * 8;
      T* const dst = head_ptr<T>(p.y[s], token, p.T, row) + cg * 8;
      float a[8], b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        a[j] = w[s][j] * C[j];
        b[j] = w_other[s][j] * Sn[j];
      }
      for (int h0 = 0; h0 < heads; h0 += kAhead * S::kRows) {
        Raw8<T> raw[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) raw[u] = next[u];
        if (h0 + kAhead * S::kRows < heads) {
          qk_load<T, LPR>(src, sh, h0 + kAhead * S::kRows, left, next);
        } else if (s == 0) {
          qk_load<T, LPR>(head_ptr<const T>(p.x[1], token, p.T, row) + cg * 8, p.x[1].sh, 0, on ? p.x[1].heads - row : 0, next);
        } else if (after < tokens) {
          qk_load<T, LPR>(head_ptr<const T>(p.x[0], after, p.T, row) + cg * 8, p.x[0].sh, 0, on ? p.x[0].heads - row : 0, next);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int h = h0 + u * S::kRows;
          if (h >= heads) break;
          float v[8], o[8];
          unpack8(raw[u], v);
          qk_exchange<LPR>(raw[u], v, o, ex, cg, part, scattered, source);
          float ss = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            ss = fmaf(v[j], v[j], ss);
            o[j] = fmaf(o[j], b[j], v[j] * a[j]);
          }
          const float r = rsqrtf(group_sum<LPR>(ss) * inv_d + p.eps);
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] *= r;
          if (h < left) store8(dst + h * p.y[s].sh, o);
        }
      }
    }
  }
}

// Warps 2 i and 2 i + 1 walk the same tokens, the first their query heads, the second their key heads.
template <typename T, int LPR>
__global__ void __launch_bounds__(32 * kQkWarps, 4) qk_norm_bwd_kernel(const QkNormParams p) {
  using S = QkSmem<LPR>;
  constexpr int kAhead = sizeof(T) == 2 ? kQkAhead / 2 : 1;
  constexpr int kPairs = kQkWarps / 2;
  __shared__ S sm;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int pair = warp / 2, s = warp % 2;
  const int row = lane / LPR, cg = lane % LPR;
  const bool on = cg * 8 < p.D;
  const unsigned tokens = p.B * p.T, stride = gridDim.x * kPairs;
  unsigned token = blockIdx.x * kPairs + pair;
  const HeadView xv = p.x[s], gv = p.dy[s], yv = p.y[s];
  const int left = on ? xv.heads - row : 0;
  float ang[kQkAngles] = {};
  Raw8<T> next_x[kAhead], next_g[kAhead];
  if (token < tokens) {
    qk_fetch_angles(p, token, lane, ang);
    qk_load<T, LPR>(head_ptr<const T>(xv, token, p.T, row) + cg * 8, xv.sh, 0, left, next_x);
    qk_load<T, LPR>(head_ptr<const T>(gv, token, p.T, row) + cg * 8, gv.sh, 0, left, next_g);
  }
  qk_partners<LPR>(sm, p);
  int part[8];
  float w[8], dw[8] = {};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    part[j] = qk_pad(sm.partner[cg * 8 + j]);
    w[j] = (on && p.w[s] != nullptr) ? p.w[s][cg * 8 + j] : 1.f;
  }
  const bool scattered = sm.scattered != 0;
  const int source = row * LPR + sm.partner[cg * 8] / 8;
  const float inv_d = 1.f / (float)p.D;
  float* ex = sm.ex[warp][row];
  for (; token < tokens; token += stride) {
    qk_table<LPR>(sm.cs[warp], p, sm.pairs, lane, ang);
    float C[8], Sn[8], da[8] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 v = sm.cs[warp][cg * 8 + j];
      C[j] = v.x;
      Sn[j] = v.y;
    }
    const unsigned after = token + stride;
    if (after < tokens) qk_fetch_angles(p, after, lane, ang);
    // dx may overwrite dy: a lane has loaded all it needs of a head before it stores there
    T* const dst = head_ptr<T>(yv, token, p.T, row) + cg * 8;
    const T* const xs = head_ptr<const T>(xv, token, p.T, row) + cg * 8;
    const T* const gs = head_ptr<const T>(gv, token, p.T, row) + cg * 8;
    for (int h0 = 0; h0 < xv.heads; h0 += kAhead * S::kRows) {
      Raw8<T> xr[kAhead], gr[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        xr[u] = next_x[u];
        gr[u] = next_g[u];
      }
      if (h0 + kAhead * S::kRows < xv.heads) {
        qk_load<T, LPR>(xs, xv.sh, h0 + kAhead * S::kRows, left, next_x);
        qk_load<T, LPR>(gs, gv.sh, h0 + kAhead * S::kRows, left, next_g);
      } else if (after < tokens) {
        qk_load<T, LPR>(head_ptr<const T>(xv, after, p.T, row) + cg * 8, xv.sh, 0, left, next_x);
        qk_load<T, LPR>(head_ptr<const T>(gv, after, p.T, row) + cg * 8, gv.sh, 0, left, next_g);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int h = h0 + u * S::kRows;
        if (h >= xv.heads) break;
        float v[8], g[8], other[8];
        unpack8(xr[u], v);
        unpack8(gr[u], g);
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        // past the last head all is zero: an eps of one keeps the root finite there, whatever the caller's (0 inf is no zero)
        const float eps = h < left ? p.eps : 1.f;
        const float r = rsqrtf(group_sum<LPR>(ss) * inv_d + eps);
        qk_exchange<LPR>(gr[u], g, other, ex, cg, part, scattered, source);
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float dn = fmaf(-other[j], Sn[j], g[j] * C[j]);
          const float dn_other = fmaf(g[j], Sn[j], other[j] * C[j]);
          v[j] *= r;  // normalised
          da[j] = fmaf(v[j], dn_other, da[j]);  // times w[j], after the last head
          dw[j] = fmaf(dn, v[j], dw[j]);
          g[j] = dn * w[j];
          dot = fmaf(g[j], v[j], dot);
        }
        const float m = group_sum<LPR>(dot) * inv_d;
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = r * fmaf(-v[j], m, g[j]);
        if (h < left) store8(dst + h * yv.sh, g);
      }
    }
    if (p.dangles != nullptr) {
      // the rows of a warp, then the pair's two warps, hold parts of the same channels; then the two channels of
      // a rotated pair, with opposite signs
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        da[j] *= w[j];
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) da[j] += __shfl_xor_sync(0xffffffffu, da[j], o);
        if (row == 0) sm.da[warp][cg * 9 + j] = da[j];
      }
      asm volatile("bar.sync %0, 64;" ::"r"(pair + 1) : "memory");
      float* out = p.dangles + (int64_t)token * p.P;
      const float *dq = sm.da[warp - s], *dk = sm.da[warp - s + 1];
      for (int i = lane + 32 * s; i < p.P; i += 64) {
        const int2 ch = sm.pairs[i];
        const int a = qk_pad(max(ch.x, 0)), c = qk_pad(max(ch.y, 0));
        out[i] = ch.x < 0 ? 0.f : (dq[a] + dk[a]) - (dq[c] + dk[c]);
      }
      asm volatile("bar.sync %0, 64;" ::"r"(pair + 1) : "memory");
    }
  }
  if (p.dw_parts != nullptr) {
    // rows of a warp by shuffles, the CTA's warps of one kind through shared memory in warp order
    float* red = reinterpret_cast<float*>(&sm.cs[0][0]);  // kQkWarps x kCh floats of the table's float2s
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int o = LPR; o < 32; o <<= 1) dw[j] += __shfl_xor_sync(0xffffffffu, dw[j], o);
      if (row == 0) red[warp * S::kCh + cg * 8 + j] = dw[j];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * p.D; c += blockDim.x) {
      const int kind = c / p.D, ch = c % p.D;
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) a += red[(2 * k + kind) * S::kCh + ch];
      p.dw_parts[((int64_t)blockIdx.x * 2 + kind) * p.D + ch] = a;
    }
  }
}

// out[s][c] (+)= sum over CTAs of parts[cta][s][c], in a fixed order: a CTA of 32 slices of the list for 32
// channels of one of the two weights, eight loads of a thread in flight.
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* __restrict__ parts, int ctas, int D, float* dq,
                                                          float* dk, int accumulate) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int c = blockIdx.x * 32 + lane, s = blockIdx.y;
  float a = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int k = slice; k < ctas; k += 32) a += parts[((int64_t)k * 2 + s) * D + c];
  }
  red[slice][lane] = a;
  __syncthreads();
  a = red[lane][slice];  // warp `slice` adds the 32 slices of channel `slice`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  const int mine = blockIdx.x * 32 + slice;
  float* out = s == 0 ? dq : dk;
  if (lane == 0 && mine < D && out != nullptr) out[mine] = (accumulate >> s & 1) ? out[mine] + a : a;
}

// ------------------------------------------------------------------------------------------ host

static HeadView head_view(const torch::Tensor& t, const torch::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.dim() == 4 && t.scalar_type() == like.scalar_type() &&
                  t.size(0) == like.size(0) && t.size(1) == like.size(1) && t.size(3) == like.size(3),
              "qk_norm: ", what, " must be a (B, T, H, D) tensor of the query's batch, length, head size and type");
  const int64_t e = 16 / (int64_t)t.element_size();
  auto vec = [&](int64_t stride, int64_t size) { return size <= 1 || stride % e == 0; };
  TORCH_CHECK(t.stride(3) == 1 && vec(t.stride(0), t.size(0)) && vec(t.stride(1), t.size(1)) &&
                  vec(t.stride(2), t.size(2)) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0,
              "qk_norm: ", what, " must have 16-byte aligned heads of contiguous channels");
  TORCH_CHECK(std::abs(t.stride(2)) * t.size(2) < (1ll << 31), "qk_norm: ", what, " has too large a head stride");
  return HeadView{t.data_ptr(), t.stride(0), t.stride(1), (int)t.stride(2), (int)t.size(2)};
}

static QkNormParams qk_params(const torch::Tensor& q, const torch::Tensor& k, const c10::optional<torch::Tensor>& qw,
                              const c10::optional<torch::Tensor>& kw, const c10::optional<torch::Tensor>& angles,
                              const torch::Tensor& pairs, double eps) {
  QkNormParams p{};
  TORCH_CHECK(q.dim() == 4 && q.size(3) % 8 == 0 && q.size(3) >= 8 && q.size(3) <= kQkMaxD,
              "qk_norm: head size must be a multiple of 8 up to ", kQkMaxD);
  TORCH_CHECK(q.size(0) * q.size(1) < (1ll << 30), "qk_norm: too many tokens");
  TORCH_CHECK(q.size(2) >= 1 && k.size(2) >= 1, "qk_norm: at least one query and one key head");
  p.x[0] = head_view(q, q, "q");
  p.x[1] = head_view(k, q, "k");
  p.B = (unsigned)q.size(0);
  p.T = (unsigned)q.size(1);
  p.D = (int)q.size(3);
  p.eps = (float)eps;
  const c10::optional<torch::Tensor>* ws[2] = {&qw, &kw};
  for (int s = 0; s < 2; ++s) {
    if (!ws[s]->has_value()) continue;
    const torch::Tensor& w = **ws[s];
    TORCH_CHECK(w.device() == q.device() && w.scalar_type() == at::kFloat && w.is_contiguous() && w.numel() == p.D,
                "qk_norm: weights must be contiguous fp32 vectors of the head size");
    p.w[s] = w.data_ptr<float>();
  }
  TORCH_CHECK(pairs.device() == q.device() && pairs.scalar_type() == at::kInt && pairs.is_contiguous() &&
                  pairs.dim() == 2 && pairs.size(1) == 2,
              "qk_norm: pairs must be a contiguous int32 (P, 2) tensor");
  p.P = (int)pairs.size(0);
  TORCH_CHECK(p.P <= p.D / 2, "qk_norm: at most D / 2 pairs");
  p.pairs = pairs.data_ptr<int>();
  if (angles.has_value() && p.P > 0) {
    TORCH_CHECK(angles->device() == q.device() && angles->scalar_type() == at::kFloat && angles->is_contiguous() &&
                    angles->dim() == 3 && (angles->size(0) == 1 || angles->size(0) == p.B) &&
                    angles->size(1) == p.T && angles->size(2) == p.P,
                "qk_norm: angles must be contiguous fp32 (1 or B, T, P)");
    p.angles = angles->data_ptr<float>();
    p.angle_bstride = angles->size(0) == 1 ? 0 : (int64_t)p.T * p.P;
  }
  return p;
}

template <typename F>
static void qk_dispatch(const torch::Tensor& q, int D, F&& f) {
  auto by_lanes = [&](auto type) {
    if (D <= 32) f(type, std::integral_constant<int, 4>{});
    else if (D <= 64) f(type, std::integral_constant<int, 8>{});
    else if (D <= 128) f(type, std::integral_constant<int, 16>{});
    else f(type, std::integral_constant<int, 32>{});
  };
  if (q.scalar_type() == at::kBFloat16) by_lanes(__nv_bfloat16{});
  else if (q.scalar_type() == at::kHalf) by_lanes(__half{});
  else if (q.scalar_type() == at::kFloat) by_lanes(float{});
  else TORCH_CHECK(false, "qk_norm: bf16, fp16 or fp32 expected");
}

void qk_norm_fwd(torch::Tensor q, torch::Tensor k, c10::optional<torch::Tensor> qw, c10::optional<torch::Tensor> kw,
                 c10::optional<torch::Tensor> angles, torch::Tensor pairs, torch::Tensor yq, torch::Tensor yk,
                 double eps) {
  QkNormParams p = qk_params(q, k, qw, kw, angles, pairs, eps);
  p.y[0] = head_view(yq, q, "the output of q");
  p.y[1] = head_view(yk, q, "the output of k");
  TORCH_CHECK(p.y[0].heads == p.x[0].heads && p.y[1].heads == p.x[1].heads, "qk_norm: output head counts");
  c10::cuda::CUDAGuard guard(q.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int64_t tokens = (int64_t)p.B * p.T;
  if (tokens == 0) return;
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int blocks = (int)std::min<int64_t>((tokens + kQkWarps - 1) / kQkWarps, 4 * sms);
  qk_dispatch(q, p.D, [&](auto type, auto lanes) {
    qk_norm_fwd_kernel<decltype(type), decltype(lanes)::value><<<blocks, 32 * kQkWarps, 0, stream>>>(p);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// dq / dk may be the very tensors dyq / dyk (each lane reads its channels before it writes them).
// dqw / dkw (fp32, D) are overwritten, or added to where `accumulate` has bit 0 / bit 1.
void qk_norm_bwd(torch::Tensor dyq, torch::Tensor dyk, torch::Tensor q, torch::Tensor k,
                 c10::optional<torch::Tensor> qw, c10::optional<torch::Tensor> kw, c10::optional<torch::Tensor> angles,
                 torch::Tensor pairs, torch::Tensor dq, torch::Tensor dk, c10::optional<torch::Tensor> dqw,
                 c10::optional<torch::Tensor> dkw, int64_t accumulate, c10::optional<torch::Tensor> dangles,
                 double eps) {
  QkNormParams p = qk_params(q, k, qw, kw, angles, pairs, eps);
  p.dy[0] = head_view(dyq, q, "the gradient of q's output");
  p.dy[1] = head_view(dyk, q, "the gradient of k's output");
  p.y[0] = head_view(dq, q, "dq");
  p.y[1] = head_view(dk, q, "dk");
  for (int s = 0; s < 2; ++s)
    TORCH_CHECK(p.dy[s].heads == p.x[s].heads && p.y[s].heads == p.x[s].heads, "qk_norm: gradient head counts");
  float* dws[2] = {nullptr, nullptr};
  const c10::optional<torch::Tensor>* dwt[2] = {&dqw, &dkw};
  for (int s = 0; s < 2; ++s) {
    if (!dwt[s]->has_value()) continue;
    const torch::Tensor& w = **dwt[s];
    TORCH_CHECK(w.device() == q.device() && w.scalar_type() == at::kFloat && w.is_contiguous() && w.numel() == p.D,
                "qk_norm: weight gradients must be contiguous fp32 vectors of the head size");
    dws[s] = w.data_ptr<float>();
  }
  if (dangles.has_value() && p.angles != nullptr) {
    TORCH_CHECK(dangles->device() == q.device() && dangles->scalar_type() == at::kFloat && dangles->is_contiguous() &&
                    dangles->numel() == (int64_t)p.B * p.T * p.P,
                "qk_norm: dangles must be contiguous fp32 (B, T, P)");
    p.dangles = dangles->data_ptr<float>();
  }
  c10::cuda::CUDAGuard guard(q.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int64_t tokens = (int64_t)p.B * p.T;
  const bool want_dw = dws[0] != nullptr || dws[1] != nullptr;
  if (tokens == 0) {
    for (int s = 0; s < 2; ++s)
      if (dws[s] != nullptr && !(accumulate >> s & 1)) C10_CUDA_CHECK(cudaMemsetAsync(dws[s], 0, 4 * p.D, stream));
    return;
  }
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int blocks = (int)std::min<int64_t>((tokens + kQkWarps / 2 - 1) / (kQkWarps / 2), 4 * sms);
  torch::Tensor parts;
  if (want_dw) {
    parts = torch::empty({blocks, 2, p.D}, q.options().dtype(at::kFloat));
    p.dw_parts = parts.data_ptr<float>();
  }
  qk_dispatch(q, p.D, [&](auto type, auto lanes) {
    qk_norm_bwd_kernel<decltype(type), decltype(lanes)::value><<<blocks, 32 * kQkWarps, 0, stream>>>(p);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (want_dw) {
    qk_norm_dw_kernel<<<dim3((p.D + 31) / 32, 2), 1024, 0, stream>>>(p.dw_parts, blocks, p.D, dws[0], dws[1],
                                                                    (int)accumulate);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
}

}  // namespace mia
