// The largest logits of a teacher's rows, and the divergence of a student from a teacher of which only those are kept.
//
// Top logits of a row: the k largest, largest first, equal ones by the lower index, and logsumexp(x / tau). A NaN
// counts as larger than every number. One block owns a row. Pass 1 reads it once: running maximum and sum of the
// log-sum-exp, and the largest value of each of 512 (or 1024) interleaved groups. The k-th largest of those group maxima is a
// value that at least k elements reach, and few more do (65536 normal values and k = 64: about 66). Pass 2 reads the
// row again, from L2 where the rows under way fit there (888 bf16 rows of 65536 are 116 MB, fp32 rows twice that), and
// collects what reaches it; every candidate then counts how many come before it. A row in which too many elements are
// equal takes the exact k-th value by bisection over the bits instead, 32 more passes, and its ties in order of their index
// (1229 x 65536 bf16 logits within a few steps of each other: 1.3 ms; 69 us where they differ).
//
// Distillation: with the teacher's values t_j at classes i_j,
//   p_j = exp(t_j / tau_t - lse_t), lse_t = logsumexp over the given classes, or over all of the teacher's (given):
//         then the classes that are not given are one more, of mass p_T = max(0, 1 - sum p_j)
//   q   = softmax(s / tau), q_T its mass outside the given classes
//   L   = sum_j p_j (log p_j - log q_{i_j}) [+ p_T (log p_T - log q_T)]
//   dL/ds_i = (q_i S - p_i) / tau for the given classes, S = sum p_j (+ p_T);
//             (q_i / q_T) (q_T S - p_T) / tau for the others  (q_i S / tau where there is no p_T).
// The loss is sum_r w_r L_r / norm. A class named twice has the sum of its shares in the gradient and both entries in the sum
// of the loss, an index outside the row is left out, and a row of weight 0 is not read and gives zeros.
//
// What is normalised directly in the pass over the logits are the classes outside the teacher's (a bitmap in shared
// memory tells them apart): a student that has nearly all its mass on the teacher's classes leaves a q_T that could
// not be had as 1 minus the rest. The few per-row figures that differences are taken of are in 64 bits.
#include <algorithm>
#include <type_traits>

#include "pair_math.cuh"
#include "sequence_types.cuh"
#include "vec8.cuh"

namespace mia {
namespace {

// Threads of a row's block: 256, six blocks an SM, so that one row's barriers lie behind another's loads; for long rows
// that are fewer than two for every SM 512, for the row's own time (16 rows of 65536 fp32: 18 -> 14 us; 1024 threads
// wait longer for each other: 15 us, and 11 instead of 5 us for 4 rows of 1000).
constexpr int kMany = 256, kFew = 512;
int threads_for(int rows, int classes) { return rows < 2 * 148 && classes >= 16384 ? kFew : kMany; }

constexpr int kCandidates = 2048;

// Calls f(index, values) for the row's elements, eight aligned ones at a time, and f(index, value) for those at both ends.
template <int NT, typename T, typename F>
__device__ __forceinline__ void for_row(const T* row, int V, F&& f) {
  constexpr int kAlign = 16 / sizeof(T);
  const int ahead = min(V, (int)((kAlign - (reinterpret_cast<uintptr_t>(row) / sizeof(T)) % kAlign) % kAlign));
  const int vecs = (V - ahead) / 8;
  if ((int)threadIdx.x < ahead) {
    float one = to_f32(row[threadIdx.x]);
    f((int)threadIdx.x, one);
  }
  constexpr int kAtOnce = 4;  // loads of a thread under way before the first is worked on
  int i = threadIdx.x;
  for (; i + (kAtOnce - 1) * NT < vecs; i += kAtOnce * NT) {
    Raw8<T> raw[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) raw[u] = load_raw8<T>(row + ahead + (i + u * NT) * 8);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      float v[8];
      unpack8<T>(raw[u], v);
      f(ahead + (i + u * NT) * 8, v);
    }
  }
  for (; i < vecs; i += NT) {
    float v[8];
    unpack8<T>(load_raw8<T>(row + ahead + i * 8), v);
    f(ahead + i * 8, v);
  }
  const int at = ahead + vecs * 8 + threadIdx.x;
  if (at < V) {
    float one = to_f32(row[at]);
    f(at, one);
  }
}

// The largest of eight; NaN if any is.
__device__ __forceinline__ float max8_nan(const float (&v)[8]) {
  float r, q;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]));
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(q) : "f"(v[3]), "f"(v[4]), "f"(v[5]));
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(r), "f"(v[6]), "f"(v[7]));
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(q));
  return r;
}

// log2(e) / tau as two fp32: with one, every exponent would be off by the same 2^-25 of it, which a small divergence (a
// difference of far larger terms) shows.
struct Rate {
  float hi, lo;
  __device__ __forceinline__ explicit Rate(double inv_tau) {
    const double c = inv_tau * 1.4426950408889634074;
    hi = __double2float_rd(c);
    if ((double)hi == c && c > 0.0) hi = __uint_as_float(__float_as_uint(hi) - 1);
    lo = (float)(c - (double)hi);  // positive, so that -inf stays -inf
  }
  __device__ __forceinline__ float operator()(float d) const { return fmaf(d, lo, d * hi); }
  __device__ __forceinline__ f32x2 operator()(f32x2 d) const {
    return fma2(d, pair_of(lo, lo), mul2(d, pair_of(hi, hi)));
  }
};

// Running maximum m (of raw logits) and sum l of exp((s - m) / tau).
struct Soft {
  float m = -INFINITY, l = 0.f;
  __device__ __forceinline__ void add(float s, Rate c) {
    if (s > m) {
      l *= m == -INFINITY ? 0.f : exp2_approx(c(m - s));
      m = s;
    }
    l += s == -INFINITY ? 0.f : exp2_approx(c(s - m));
  }
  // `top` is the largest of the eight, or NaN
  __device__ __forceinline__ void add8(const float (&v)[8], float top, Rate c) {
    if (top > m) {
      l *= m == -INFINITY ? 0.f : exp2_approx(c(m - top));
      m = top;
    }
    // with m = -inf (all of them, or NaN next to them) the differences would be NaN: 0 stands in for m, the terms of
    // -inf are 0 and those of NaN stay NaN
    const float ref = m == -INFINITY ? 0.f : m;
    const f32x2 ref2 = pair_of(-ref, -ref);
    f32x2 sum = 0;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float a, b;
      split(c(add2(pair_of(v[e], v[e + 1]), ref2)), a, b);
      sum = add2(sum, pair_of(exp2_approx(a), exp2_approx(b)));
    }
    float a, b;
    split(sum, a, b);
    l += a + b;
  }
  __device__ __forceinline__ void join(float m2, float l2, Rate c) {
    const float top = fmaxf(m, m2);
    const float ref = top == -INFINITY ? 0.f : top;
    l = l * exp2_approx(c(m - ref)) + l2 * exp2_approx(c(m2 - ref));
    m = top;
  }
};

template <int NT>
__device__ void block_join(Soft& a, Rate c, float* scratch /* 2 * NT / 32 */) {
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, a.m, w), l2 = __shfl_xor_sync(0xffffffffu, a.l, w);
    a.join(m2, l2, c);
  }
  __syncthreads();
  if (threadIdx.x % 32 == 0) {
    scratch[threadIdx.x / 32] = a.m;
    scratch[(NT / 32) + threadIdx.x / 32] = a.l;
  }
  __syncthreads();
  a = Soft();
  for (int w = 0; w < (NT / 32); ++w) a.join(scratch[w], scratch[(NT / 32) + w], c);
}

template <int NT, int N>
__device__ void block_sum(double (&v)[N], double* scratch /* N * NT / 32 */) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], w);
  __syncthreads();
  if (threadIdx.x % 32 == 0)
#pragma unroll
    for (int n = 0; n < N; ++n) scratch[n * (NT / 32) + threadIdx.x / 32] = v[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    v[n] = 0.0;
    for (int w = 0; w < (NT / 32); ++w) v[n] += scratch[n * (NT / 32) + w];
  }
}

// --------------------------------------------------------------------------------------- top logits

// Order of values as unsigned numbers: -0 is 0, NaN is the largest.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The number with a key (for a key that none has, one near it that is not above it); -inf for keys below all.
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key <= 0x007fffffu) return -INFINITY;
  if (key >= 0xff800000u) return INFINITY;
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

template <int NT>
__device__ int block_count(int mine, int* scratch /* NT / 32 */) {
  const int w = __reduce_add_sync(0xffffffffu, mine);
  __syncthreads();
  if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = w;
  __syncthreads();
  int n = 0;
  for (int i = 0; i < (NT / 32); ++i) n += scratch[i];
  return n;
}

// The largest key that at least k of the keys given by `count(threshold)` reach, bit by bit.
template <typename F>
__device__ uint32_t kth_key(int k, F&& count) {
  uint32_t t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t tryit = t | (1u << bit);
    if (count(tryit) >= k) t = tryit;
  }
  return t;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT, NT == kMany ? 6 : 1) top_logits_kernel(const T* __restrict__ x, int64_t stride, int V, int k,
                                                              double inv_tau, T* __restrict__ values,
                                                              int64_t* __restrict__ indices, float* __restrict__ lse) {
  __shared__ uint64_t list[kCandidates];
  __shared__ float red[2 * (NT / 32)];
  __shared__ int counts[(NT / 32)];
  __shared__ int n_list;
  const T* row = x + (int64_t)blockIdx.x * stride;
  const Rate c(inv_tau);
  if (threadIdx.x == 0) n_list = 0;

  Soft soft;
  uint32_t best[2] = {0, 0};  // the two groups of this thread; 0 is below the key of every number
  int turn = 0;
  for_row<NT, T>(row, V, [&](int, auto& v) {
    if constexpr (std::is_same_v<std::decay_t<decltype(v)>, float>) {
      soft.add(v, c);
      if (v != v) soft.l = v;
      best[0] = max(best[0], key_of(v));
    } else {
      const float top = max8_nan(v);
      soft.add8(v, top, c);
      const uint32_t key = key_of(top);
      if (turn) best[1] = max(best[1], key);
      else best[0] = max(best[0], key);
      turn ^= 1;
    }
  });
  block_join<NT>(soft, c, red);
  const bool nan = block_count<NT>(best[0] == 0xffffffffu || best[1] == 0xffffffffu, counts) > 0;
  if (threadIdx.x == 0)
    lse[blockIdx.x] = nan ? NAN : soft.m == INFINITY ? INFINITY : soft.l == 0.f ? -INFINITY : (float)(soft.m * inv_tau + log((double)soft.l));

  // A row shorter than the groups leaves some of them empty, and then the bound may be 0: every element is taken.
  // Any bound that at least k groups reach will do; the search ends where not many more do.
  uint32_t bound = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = bound | (1u << bit);
    const int n = __syncthreads_count(best[0] >= t) + __syncthreads_count(best[1] >= t);
    if (n < k) continue;
    bound = t;
    if (n <= k + k / 4 + 4) break;
  }
  const float floor_of = value_of(bound);
  auto collect = [&](int at, float v, uint32_t least) {
    const uint32_t key = key_of(v);
    if (key >= least) {
      const int n = atomicAdd(&n_list, 1);
      if (n < kCandidates) list[n] = (uint64_t)key << 32 | (0xffffffffu - (uint32_t)at);
    }
  };
  auto scan = [&](uint32_t least, float least_value) {
    for_row<NT, T>(row, V, [&](int at, auto& v) {
      if constexpr (std::is_same_v<std::decay_t<decltype(v)>, float>) {
        collect(at, v, least);
      } else if (!(max8_nan(v) < least_value)) {  // one of them may reach the bound, or is NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) collect(at + e, v[e], least);
      }
    });
  };
  scan(bound, floor_of);
  __syncthreads();
  int n = n_list;
  if (n > kCandidates) {
    // too many: the exact k-th key, everything above it, and of its equals the first in order
    const uint32_t exact = kth_key(k, [&](uint32_t t) {
      int mine = 0;
      for_row<NT, T>(row, V, [&](int, auto& v) {
        if constexpr (std::is_same_v<std::decay_t<decltype(v)>, float>) mine += key_of(v) >= t;
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) mine += key_of(v[e]) >= t;
      });
      return block_count<NT>(mine, counts);
    });
    __syncthreads();
    if (threadIdx.x == 0) n_list = 0;
    __syncthreads();
    if (exact != 0xffffffffu) scan(exact + 1, value_of(exact));
    __syncthreads();
    n = n_list;  // less than k
    int found = 0;
    for (int base = 0; base < V && n + found < k; base += NT) {
      const int at = base + (int)threadIdx.x;
      const bool equal = at < V && key_of(to_f32(row[at])) == exact;
      const uint32_t votes = __ballot_sync(0xffffffffu, equal);
      __syncthreads();
      if (threadIdx.x % 32 == 0) counts[threadIdx.x / 32] = __popc(votes);
      __syncthreads();
      int before = found + __popc(votes & ((1u << (threadIdx.x % 32)) - 1)), all = 0;
      for (int w = 0; w < (NT / 32); ++w) {
        if (w < (int)threadIdx.x / 32) before += counts[w];
        all += counts[w];
      }
      if (equal && n + before < k) list[n + before] = (uint64_t)exact << 32 | (0xffffffffu - (uint32_t)at);
      found += all;
    }
    n = k;
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t me = list[i];
    int before = 0;
    for (int j = 0; j < n; ++j) before += list[j] > me;
    if (before < k) {
      const int at = (int)(0xffffffffu - (uint32_t)me);
      values[(int64_t)blockIdx.x * k + before] = row[at];
      indices[(int64_t)blockIdx.x * k + before] = at;
    }
  }
}

// -------------------------------------------------------------------------------------- distillation

enum { kGenM, kGenL, kGenCoef, kAllM, kAllL, kMass, kLseT, kStats = 8 };

__device__ __forceinline__ double value_at(const DistillParams& p, int64_t i) {
  if (p.value_type == kSeqF32) return (double)((const float*)p.values)[i];
  if (p.value_type == kSeqBf16) return (double)to_f32(((const __nv_bfloat16*)p.values)[i]);
  if (p.value_type == kSeqF16) return (double)to_f32(((const __half*)p.values)[i]);
  return ((const double*)p.values)[i];
}

__device__ __forceinline__ double number_at(const void* x, bool wide, int i) {
  return wide ? ((const double*)x)[i] : (double)((const float*)x)[i];
}

// The class of entry i, -1 where it names none.
__device__ __forceinline__ int index_at(const DistillParams& p, int64_t i) {
  const int64_t at = p.index64 ? ((const int64_t*)p.indices)[i] : (int64_t)((const int*)p.indices)[i];
  return at >= 0 && at < p.V ? (int)at : -1;
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT, NT == kMany ? 6 : 1) distill_fwd_kernel(DistillParams p, double* __restrict__ row_loss) {
  extern __shared__ uint32_t given[];  // a bit per class, where there is a rest
  __shared__ double sums[4 * (NT / 32)];
  __shared__ float red[2 * (NT / 32)];
  const int r = blockIdx.x;
  const double w = p.weights != nullptr ? number_at(p.weights, p.weights64, r) : 1.0;
  if (w == 0.0) {
    if (threadIdx.x == 0) row_loss[r] = 0.0;
    return;
  }
  const T* row = (const T*)p.s + r * p.s_row;
  const int64_t first = (int64_t)r * p.K;
  const double inv_tau = 1.0 / p.tau, inv_tau_t = 1.0 / p.teacher_tau;
  const Rate c(inv_tau);
  const bool tail = p.lse != nullptr;
  Soft gen, top;
  double distinct = 0.0;
  if (tail) {
    for (int i = threadIdx.x; i < (p.V + 31) / 32; i += NT) given[i] = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < p.K; j += NT) {
      const int at = index_at(p, first + j);
      if (at < 0) continue;
      if (atomicOr(&given[at / 32], 1u << (at % 32)) >> (at % 32) & 1) continue;
      distinct += 1.0;
      const float s = to_f32(row[at]);
      top.add(s, c);
      if (s != s) top.l = s;
    }
    __syncthreads();
  }
  for_row<NT, T>(row, p.V, [&](int at, auto& v) {
    if constexpr (std::is_same_v<std::decay_t<decltype(v)>, float>) {
      if (tail && given[at / 32] >> (at % 32) & 1) return;
      gen.add(v, c);
      if (v != v) gen.l = v;
    } else {
      if (tail) {
        uint32_t bits = given[at / 32] >> (at % 32);
        if (at % 32 > 24) bits |= (at / 32 + 1) * 32 < p.V ? given[at / 32 + 1] << (32 - at % 32) : 0;
        if (bits & 0xff)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (bits >> e & 1) v[e] = -INFINITY;
      }
      gen.add8(v, max8_nan(v), c);
    }
  });
  block_join<NT>(gen, c, red);
  Soft all = gen;
  if (tail) {
    block_join<NT>(top, c, red);
    all.join(top.m, top.l, c);
  }
  // the teacher's side: log-sum-exp of the given values, unless that of all of them came along
  double lse_t = tail ? number_at(p.lse, p.lse64, r) : 0.0;
  if (!tail) {
    float m = -INFINITY;
    for (int j = threadIdx.x; j < p.K; j += NT)
      if (index_at(p, first + j) >= 0) m = fmaxf(m, (float)value_at(p, first + j));
    Soft mm;
    mm.m = m;
    block_join<NT>(mm, Rate(0.0), red);
    const double ref = mm.m == -INFINITY ? 0.0 : (double)mm.m * inv_tau_t;
    double sum[1] = {0.0};
    for (int j = threadIdx.x; j < p.K; j += NT)
      if (index_at(p, first + j) >= 0) sum[0] += exp(value_at(p, first + j) * inv_tau_t - ref);
    block_sum<NT, 1>(sum, sums);
    lse_t = sum[0] == 0.0 ? INFINITY : ref + log(sum[0]);  // nothing given: every share is 0
  }
  const double log_all = log((double)all.l);
  double acc[3] = {0.0, 0.0, distinct};  // loss, mass, classes
  for (int j = threadIdx.x; j < p.K; j += NT) {
    const int at = index_at(p, first + j);
    if (at < 0) continue;
    const double log_p = value_at(p, first + j) * inv_tau_t - lse_t, share = exp(log_p);
    const double log_q = ((double)to_f32(row[at]) - all.m) * inv_tau - log_all;
    if (share != 0.0) acc[0] += share * (log_p - log_q);
    acc[1] += share;
  }
  block_sum<NT, 3>(acc, sums);
  if (threadIdx.x != 0) return;
  double loss = acc[0], mass = acc[1], coef = mass;
  if (tail) {
    const double rest = acc[2] < p.V ? fmax(0.0, 1.0 - mass) : 0.0;
    const double log_rest = ((double)gen.m - all.m) * inv_tau + log((double)gen.l) - log_all;  // of the student
    if (rest != 0.0) loss += rest * (log(rest) - log_rest);
    mass += rest;
    coef = acc[2] < p.V ? exp(log_rest) * mass - rest : 0.0;
  }
  row_loss[r] = w * loss;
  double* st = p.stats + (int64_t)r * kStats;
  st[kGenM] = gen.m;
  st[kGenL] = gen.l;
  st[kGenCoef] = coef;
  st[kAllM] = all.m;
  st[kAllL] = all.l;
  st[kMass] = mass;
  st[kLseT] = lse_t;
}

// sum of the rows' losses in order, over norm
template <int NT>
__global__ void __launch_bounds__(NT) distill_sum_kernel(const double* __restrict__ rows, int R, double norm,
                                                               float* __restrict__ out) {
  __shared__ double sums[(NT / 32)];
  double s[1] = {0.0};
  for (int i = threadIdx.x; i < R; i += NT) s[0] += rows[i];
  block_sum<NT, 1>(s, sums);
  if (threadIdx.x == 0) *out = (float)(s[0] / norm);
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_bwd_kernel(DistillParams p, const float* __restrict__ grad,
                                                               T* __restrict__ ds) {
  __shared__ int at_of[kMaxGiven];
  __shared__ float share_of[kMaxGiven];  // off by 2^-25 of it: the student's probability beside it has the 2^-22 of exp2 in its sum
  const int r = p.R - 1 - blockIdx.x;  // the rows that the forward pass read last may still be in L2
  T* out = ds + (int64_t)r * p.V;
  const double w = p.weights != nullptr ? number_at(p.weights, p.weights64, r) : 1.0;
  const int vec_ahead = min(p.V, (int)((8 - (reinterpret_cast<uintptr_t>(out) / sizeof(T)) % 8) % 8));
  if (w == 0.0) {
    for (int i = threadIdx.x; i < p.V; i += NT) out[i] = from_f32<T>(0.f);
    return;
  }
  const T* row = (const T*)p.s + r * p.s_row;
  const int64_t first = (int64_t)r * p.K;
  const double* st = p.stats + (int64_t)r * kStats;
  const double inv_tau = 1.0 / p.tau, inv_tau_t = 1.0 / p.teacher_tau;
  const Rate c(inv_tau);
  const double scale = (double)*grad * w / p.norm * inv_tau;
  const float m = (float)st[kGenM];
  const float ref = m == -INFINITY ? 0.f : m;
  // a rest of no mass at all has no gradient
  const float coef = st[kGenL] == 0.0 ? 0.f : (float)(scale * st[kGenCoef] / st[kGenL]);
  for (int j = threadIdx.x; j < p.K; j += NT) {
    at_of[j] = index_at(p, first + j);
    share_of[j] = at_of[j] < 0 ? 0.f : (float)exp(value_at(p, first + j) * inv_tau_t - st[kLseT]);
  }
  const bool same = (reinterpret_cast<uintptr_t>(row) / sizeof(T)) % 8 == (reinterpret_cast<uintptr_t>(out) / sizeof(T)) % 8;
  if (same) {
    const int vecs = (p.V - vec_ahead) / 8;
    for (int i = threadIdx.x; i < vecs; i += NT) {
      float v[8];
      unpack8<T>(load_raw8<T>(row + vec_ahead + i * 8), v);
      const f32x2 ref2 = pair_of(-ref, -ref), coef2 = pair_of(coef, coef);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        float a, b;
        split(c(add2(pair_of(v[e], v[e + 1]), ref2)), a, b);
        split(mul2(pair_of(exp2_approx(a), exp2_approx(b)), coef2), v[e], v[e + 1]);
      }
      store8<T>(out + vec_ahead + i * 8, v);
    }
    const int end = vec_ahead + vecs * 8;
    for (int i = threadIdx.x; i < vec_ahead + (p.V - end); i += NT) {
      const int at = i < vec_ahead ? i : end + i - vec_ahead;
      out[at] = from_f32<T>(exp2_approx(c(to_f32(row[at]) - ref)) * coef);
    }
  } else {
    for (int i = threadIdx.x; i < p.V; i += NT) out[i] = from_f32<T>(exp2_approx(c(to_f32(row[i]) - ref)) * coef);
  }
  __syncthreads();  // the given classes replace what the pass wrote in their places
  const double inv_l = 1.0 / st[kAllL], all_m = st[kAllM], mass = st[kMass];
  for (int j = threadIdx.x; j < p.K; j += NT) {
    const int at = at_of[j];
    if (at < 0) continue;
    bool again = false;
    double share = 0.0;
    for (int i = 0; i < p.K; ++i)
      if (at_of[i] == at) {
        again = again || i < j;
        share += share_of[i];
      }
    if (again) continue;
    const double q = exp(((double)to_f32(row[at]) - all_m) * inv_tau) * inv_l;
    out[at] = from_f32<T>((float)(scale * (q * mass - share)));
  }
}

}  // namespace

cudaError_t top_logits_rows(const void* x, int64_t stride, int R, int V, int k, double tau, void* values,
                            int64_t* indices, float* lse, SequenceType type, cudaStream_t stream) {
  by_type(type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto go = [&](auto kernel, int threads) {
      kernel<<<R, threads, 0, stream>>>((const T*)x, stride, V, k, 1.0 / tau, (T*)values, indices, lse);
    };
    if (threads_for(R, V) == kMany) go(top_logits_kernel<T, kMany>, kMany);
    else go(top_logits_kernel<T, kFew>, kFew);
  });
  return cudaGetLastError();
}

cudaError_t distill_fwd(const DistillParams& p, double* row_loss, float* loss, cudaStream_t stream) {
  cudaError_t status = cudaSuccess;
  if (p.R > 0) {
    const size_t smem = p.lse != nullptr ? (size_t)(p.V + 31) / 32 * 4 : 0;
    by_type(p.type, [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      auto go = [&](auto kernel, int threads) {
        if (smem > 32 * 1024)
          status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (status == cudaSuccess) kernel<<<p.R, threads, smem, stream>>>(p, row_loss);
      };
      if (threads_for(p.R, p.V) == kMany) go(distill_fwd_kernel<T, kMany>, kMany);
      else go(distill_fwd_kernel<T, kFew>, kFew);
    });
  }
  if (status != cudaSuccess) return status;
  distill_sum_kernel<kMany><<<1, kMany, 0, stream>>>(row_loss, p.R, p.norm, loss);
  return cudaGetLastError();
}

cudaError_t distill_bwd(const DistillParams& p, const float* grad, void* ds, cudaStream_t stream) {
  by_type(p.type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    if (threads_for(p.R, p.V) == kMany) distill_bwd_kernel<T, kMany><<<p.R, kMany, 0, stream>>>(p, grad, (T*)ds);
    else distill_bwd_kernel<T, kFew><<<p.R, kFew, 0, stream>>>(p, grad, (T*)ds);
  });
  return cudaGetLastError();
}

}  // namespace mia
