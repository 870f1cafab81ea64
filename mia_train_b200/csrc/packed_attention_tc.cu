// Packed-sequence attention on the 5th-generation tensor cores (formulas: packed_attention.cu), bf16 and fp16.
//
// Tiles are 128 consecutive rows of the packed array, wherever sequences begin and end: short sequences share a
// tile and a tile's keys are one contiguous range, because the bounds of the rows never fall. A block of keys that
// every row of the tile sees in full skips the mask. Heads of 8 .. 64 channels take 64-column tiles, up to 128 two of
// them side by side; channels past the head are filled with zeros by the TMA unit and the products stop at the
// next multiple of 16.
//
// All second products (P V, dS K, P^T dO, dS^T Q) take their first operand from tensor memory: the threads that
// computed its row write it over the scores they read, half as many columns of 16-bit pairs, so that neither P nor
// dS passes through shared memory.
//
// Masked entries are replaced before any maximum or product of this row, but the second products still multiply their
// zeros with rows of other sequences. Where those hold an infinity or a NaN, the sum becomes NaN: an output row
// that is not finite although its statistics are is computed again by the warp-per-row formulas, which read only what
// the row sees.
//
// The backward pass is two kernels, one per owner of the sums (dQ by query tiles; dK and dV by key tiles): each
// repeats S and dP, seven products instead of five, but no sum leaves its CTA, so there are no atomics, no fp32
// buffers and the result has the same bits every time.
//
// Every wait is bounded (common.cuh); on expiry the kernel records kErrPackedWait, lets its copies and products land,
// frees its tensor memory and returns.
#include <cudaTypedefs.h>

#include <type_traits>

#include "common.cuh"
#include "packed_attention.h"
#include "pair_math.cuh"

namespace mia {
namespace {

constexpr int kRows = 128;  // rows of a tile, keys (or queries) of a block

template <int DP>
struct Tile {
  static constexpr int kBytes = kRows * DP * 2;  // DP / 64 column groups of 128 rows x 128 bytes, swizzled
};

// mbar_wait that looks at the clock and at the abort flag on every 64th failed try only: reading %globaltimer takes
// longer than most of these waits.
__device__ __forceinline__ bool bounded_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  uint64_t start = 0;
#pragma unroll 1
  for (uint32_t n = 1; !mbar_try_wait(bar, parity); ++n) {
    if (n % 64 != 0) continue;
    if (*abort_flag) return false;
    const uint64_t now = globaltimer_ns();
    if (start == 0) start = now;
    if (now - start > MIA_WAIT_LIMIT_NS) {
      record_error(err, kErrPackedWait);
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err) {
  const bool ok = bounded_wait(bar, parity, abort_flag, err);
  return __all_sync(0xffffffffu, ok);
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// 128 rows from `row` of head `h`; DP / 64 boxes
template <int DP>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int row, int h) {
#pragma unroll
  for (int g = 0; g < DP / 64; ++g) tma_load_3d(dst + g * (kRows * 128), map, bar, g * 64, row, h);
}

// Of `issued` loads that go through `stages` stages in turns, the first that may still be in flight; the ones before it have
// been consumed, or their stages would not have been loaded again. A loader that gives up waits for [this, issued) before
// shared memory is given back; the barrier of an earlier load has moved on to a later phase, for which a wait would run out.
constexpr __host__ __device__ int first_in_flight(int issued, int stages) { return issued > stages ? issued - stages : 0; }

constexpr bool waits_for_last_phases(int stages) {
  for (int issued = 0; issued <= 5 * stages; ++issued)
    for (int i = 0; i < issued; ++i) {
      bool last = true;  // phase of its stage
      for (int later = i + 1; later < issued; ++later) last = last && later % stages != i % stages;
      if (last != (i >= first_in_flight(issued, stages))) return false;
    }
  return true;
}
static_assert(waits_for_last_phases(1) && waits_for_last_phases(2) && waits_for_last_phases(3) && waits_for_last_phases(4));

// `bytes` (a multiple of 16, as both addresses) of global memory
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// max of three; NaN if any is
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^x of both on the FMA pipe, for finite x: x = n + f with n the nearest integer (adding 1.5 * 2^23 leaves it in the
// low bits of the sum), 2^f by a polynomial of degree 4 fitted here to the least relative error on [-1/2, 1/2] (2.6e-6,
// iteratively reweighted least squares on 40001 points), n added to the exponent. x below -126 counts as -126.
__device__ __forceinline__ void exp2_fma(f32x2 x, float& p0, float& p1) {
  float a, b;
  split(x, a, b);
  x = pair_of(fmaxf(a, -126.f), fmaxf(b, -126.f));
  const f32x2 magic = pair_of(12582912.f, 12582912.f);
  const f32x2 t = add2(x, magic);
  const f32x2 f = add2(x, mul2(add2(t, pair_of(-12582912.f, -12582912.f)), pair_of(-1.f, -1.f)));
  f32x2 y = fma2(f, pair_of(0.00957005936652422f, 0.00957005936652422f), pair_of(0.055917758494615555f, 0.055917758494615555f));
  y = fma2(y, f, pair_of(0.240247443318367f, 0.240247443318367f));
  y = fma2(y, f, pair_of(0.6931218504905701f, 0.6931218504905701f));
  y = fma2(y, f, pair_of(0.9999992847442627f, 0.9999992847442627f));
  float t0, t1;
  split(t, t0, t1);
  split(y, p0, p1);
  p0 = __int_as_float(__float_as_int(p0) + (__float_as_int(t0) << 23));
  p1 = __int_as_float(__float_as_int(p1) + (__float_as_int(t1) << 23));
}

// D(tmem) (+)= A(tmem, 16-bit pairs along K) * B(smem)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}

template <typename T>
__device__ __forceinline__ uint32_t idesc_of(int n, bool b_mn_major) {
  const uint32_t bf16 = make_idesc_bf16(kRows, n, false, b_mn_major);
  return std::is_same_v<T, __half> ? bf16 & ~((1u << 7) | (1u << 10)) : bf16;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(lo, hi);
  }
}

// A launch of 12 warps with 168 registers a thread shares them out anew: the eight warps that hold rows of scores take
// 216, the four of the loading and issuing group keep 72 (8 * 216 + 4 * 72 = 12 * 168).
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 216;"); }
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); }

// The issuing warp runs its loop as a whole, with one elected lane behind every product: what the products take then
// stays in uniform registers. Issued from a branch of one thread they took 62 cycles each whatever their width
// (128 x 64 x 16: 32 at the full rate), measured on 512 in a row.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

template <typename V>
__device__ __forceinline__ V uniform(V x) { return __shfl_sync(0xffffffffu, x, 0); }

// Descriptor of a tile read along its rows' channels, and of one read along its rows; `tile_step` moves either by a tile.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return make_sdesc_sw<128>(addr, 16, 1024); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) { return make_sdesc_sw<128>(addr, kRows * 128, 1024); }
// 128 rows of 16 bytes one after the other, without swizzle; the second 8 of 16 channels `second` bytes behind.
__device__ __forceinline__ uint64_t desc_columns(uint32_t addr, uint32_t second) {
  return (uint64_t)((addr >> 4) & 0x3FFFu) | (uint64_t)((second >> 4) & 0x3FFFu) << 16 | (uint64_t)(128 >> 4) << 32 |
         (uint64_t)1 << 46;
}
template <int DP>
__device__ __forceinline__ uint32_t tile_step(int n) { return (uint32_t)(n * (Tile<DP>::kBytes / 16)); }

// Scores: d = A B^T over the head's channels.
template <int DP>
__device__ __forceinline__ void mma_scores(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, int D) {
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const uint32_t off = (kk >> 2) * (kRows * 128 / 16) + (kk & 3) * 2;
    if (kk == 0 || kk * 16 < D) tc_mma_f16(d, a + off, b + off, idesc, kk > 0);
  }
}

// Sums: d (+)= A B with A (128 x 128) in 64 columns of tensor memory, B the rows of a tile.
__device__ __forceinline__ void mma_sums(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) mma_ts(d, a + kk * 8, b + kk * 128, idesc, accumulate || kk > 0);
}

// 16 fp32 columns of this lane's row times `f`, as 16-bit values; returns NaN if any is not finite, else 0.
template <typename T>
__device__ __forceinline__ float store16(T* dst, const uint32_t (&v)[16], float f, bool first8, bool last8) {
  float x[16], bad = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    x[e] = __uint_as_float(v[e]) * f;
    bad = fmaf(x[e], 0.f, bad);
  }
#pragma unroll
  for (int g = 0; g < 2; ++g)
    if (g == 0 ? first8 : last8)
      *reinterpret_cast<uint4*>(dst + 8 * g) =
          make_uint4(pack2<T>(x[8 * g], x[8 * g + 1]), pack2<T>(x[8 * g + 2], x[8 * g + 3]),
                     pack2<T>(x[8 * g + 4], x[8 * g + 5]), pack2<T>(x[8 * g + 6], x[8 * g + 7]));
  return bad;
}

// The same of x, which is finite where it is wanted, less what 16 bits keep of it.
template <typename T>
__device__ __forceinline__ void store16_low(T* dst, const uint32_t (&v)[16], float f, bool first8, bool last8) {
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float x = __uint_as_float(v[e]) * f;
    w[e] = __float_as_uint(x - to_f32(from_f32<T>(x)));
  }
  store16<T>(dst, w, 1.f, first8, last8);
}

// ------------------------------------------------------------------------------------------- forward
// A CTA owns NT tiles of 128 queries of one head (two for wide heads). Warps 4 t .. 4 t + 3 hold tile t's rows, one thread per row: S from
// tensor memory, running maximum and sum, P back over S. The accumulator O is rescaled in place, and only when a
// block's maximum exceeds the reference maximum by more than 2^8 (P <= 2^8 until then). The last two warps load
// (TMA) and issue the products. With two tiles, or two CTAs on an SM, one's softmax runs beside the other's products; heads
// of up to 64 channels leave room for P next to S, so that the next S is computed as soon as this one has been read.
//
// Tensor memory: S (128 columns), O (DP) and, for DP = 64, P (64) per tile.
template <int DP, int NT>
struct FwdLayout {
  static_assert(DP == 128 || NT == 1, "two tiles of 64 channels leave no room for P");
  static constexpr int kStages = 2;
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + NT * Tile<DP>::kBytes;
  static constexpr int kV = kK + kStages * Tile<DP>::kBytes;
  static constexpr int kBar = kV + kStages * Tile<DP>::kBytes;
  static constexpr int kBytes = kBar + 256 + 1024;
  static_assert(4 * kRowScratch * 4 <= Tile<DP>::kBytes, "a tile's four warps have their scratch in its queries' place");
  static constexpr int kThreads = NT == 2 ? 384 : 192;
  static constexpr uint32_t kCols = NT == 2 ? 512 : 256;
  static constexpr bool kApart = DP == 64;  // P next to S instead of over it
  static constexpr uint32_t kO = NT * kRows, kP = NT * (kRows + DP);
};

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(NT == 2 ? 384 : 192, NT == 1 ? 2 : 1)
    packed_fwd_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, const PackedProblem P, T* __restrict__ o,
                         float* __restrict__ lse, int* err) {
  using L = FwdLayout<DP, NT>;
  constexpr int S = L::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t *q_full = bar, *k_full = bar + 1, *k_empty = k_full + S, *v_full = k_empty + S, *v_empty = v_full + S;
  uint64_t *s_full = v_empty + S, *s_read = s_full + NT, *p_full = s_read + NT, *o_full = p_full + NT, *drain = o_full + NT;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform((int)threadIdx.x / 32), lane = threadIdx.x % 32;
  const int tiles = (P.Tq + NT * kRows - 1) / (NT * kRows);
  const int h = blockIdx.x % P.Hq;
  const int r0 = (tiles - 1 - (int)(blockIdx.x / P.Hq)) * NT * kRows;  // causal rows see the more keys the later they are
  const int hk = h / P.group;

  // key range of every tile, and of all
  int begin[NT], end[NT];  // blocks
  int from = 0, to = 0;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    begin[t] = end[t] = 0;
    const int a = r0 + t * kRows;
    if (a >= P.Tq) continue;
    const int lo = P.q_bounds[a].x, hi = P.q_bounds[min(a + kRows, P.Tq) - 1].y;
    if (t == 0) from = to = lo;
    if (hi <= lo) continue;
    begin[t] = (lo - from) / kRows;
    end[t] = (hi - from + kRows - 1) / kRows;
    to = max(to, hi);
  }
  const int blocks = (to - from + kRows - 1) / kRows;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < S; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int t = 0; t < NT; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&s_read[t], kRows);
      mbar_init(&p_full[t], kRows);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmQ);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  if (warp == NT * 4 + 1) {
    tmem_alloc(tmem_slot, L::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= NT * 4) {
    if constexpr (NT == 2) fewer_registers();
    if (warp == NT * 4 && lane == 0 && blocks > 0) {
      // ---------------------------------------------------------------------------------- loads
      int nk = 0, nv = 0;
      bool ok = true;
      mbar_arrive_expect_tx(q_full, NT * Tile<DP>::kBytes);
#pragma unroll
      for (int t = 0; t < NT; ++t) load_tile<DP>(smem + L::kQ + t * Tile<DP>::kBytes, &tmQ, q_full, r0 + t * kRows, h);
      for (int j = 0; j < blocks; ++j) {
        const int s = j % S;
        const uint32_t free_parity = ((j / S) & 1) ^ 1;
        if (!bounded_wait(&k_empty[s], free_parity, abort_flag, err)) { ok = false; break; }
        mbar_arrive_expect_tx(&k_full[s], Tile<DP>::kBytes);
        load_tile<DP>(smem + L::kK + s * Tile<DP>::kBytes, &tmK, &k_full[s], from + j * kRows, hk);
        ++nk;
        if (!bounded_wait(&v_empty[s], free_parity, abort_flag, err)) { ok = false; break; }
        mbar_arrive_expect_tx(&v_full[s], Tile<DP>::kBytes);
        load_tile<DP>(smem + L::kV + s * Tile<DP>::kBytes, &tmV, &v_full[s], from + j * kRows, hk);
        ++nv;
      }
      if (!ok) {  // copies in flight land before shared memory is given back
        mbar_wait(q_full, 0, nullptr, nullptr, 0);
        for (int j = first_in_flight(nk, S); j < nk; ++j) mbar_wait(&k_full[j % S], (j / S) & 1, nullptr, nullptr, 0);
        for (int j = first_in_flight(nv, S); j < nv; ++j) mbar_wait(&v_full[j % S], (j / S) & 1, nullptr, nullptr, 0);
      }
    } else if (warp == NT * 4 + 1) {
      // ------------------------------------------------------------------------------- products
      const bool one = elect_one();
      const uint32_t idesc_s = idesc_of<T>(kRows, false), idesc_o = idesc_of<T>((P.D + 15) / 16 * 16, true);
      const uint64_t q_desc = desc_k(uniform(smem_u32(smem + L::kQ))), k_desc = desc_k(uniform(smem_u32(smem + L::kK)));
      const uint64_t v_desc = desc_mn(uniform(smem_u32(smem + L::kV)));
      const uint32_t base = uniform(tmem);
      const int n = uniform(blocks);
      int b0[NT], b1[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        b0[t] = uniform(begin[t]);
        b1[t] = uniform(end[t]);
      }
      auto scores = [&](int t, int j) -> bool {
        if (j < b0[t] || j >= b1[t]) return true;
        const int it = j - b0[t];
        if (L::kApart && it > 0 && !warp_wait(&s_read[t], (it - 1) & 1, abort_flag, err)) return false;
        tc_fence_after();
        if (one) {
          mma_scores<DP>(base + t * kRows, q_desc + tile_step<DP>(t), k_desc + tile_step<DP>(j % S), idesc_s, P.D);
          tc_commit(&s_full[t]);
        }
        return true;
      };
      auto sums = [&](int t, int j) -> bool {
        if (j < b0[t] || j >= b1[t]) return true;
        const int it = j - b0[t];
        if (!warp_wait(&p_full[t], it & 1, abort_flag, err)) return false;
        tc_fence_after();
        if (one) {
          mma_sums(base + L::kO + t * DP, L::kApart ? base + L::kP + t * 64 : base + t * kRows,
                   v_desc + tile_step<DP>(j % S), idesc_o, it > 0);
          tc_commit(&o_full[t]);
        }
        return true;
      };
      bool ok = n == 0 || warp_wait(q_full, 0, abort_flag, err);
      for (int j = 0; j <= n && n > 0 && ok; ++j) {
        if (j < n) ok = warp_wait(&k_full[j % S], (j / S) & 1, abort_flag, err);
        if (ok && j > 0) ok = warp_wait(&v_full[(j - 1) % S], ((j - 1) / S) & 1, abort_flag, err);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if (L::kApart) ok = ok && (j == n || scores(t, j)) && (j == 0 || sums(t, j - 1));
          else ok = ok && (j == 0 || sums(t, j - 1)) && (j == n || scores(t, j));
        }
        if (ok && j < n && one) tc_commit(&k_empty[j % S]);
        if (ok && j > 0 && one) tc_commit(&v_empty[(j - 1) % S]);
      }
      if (!ok && one) {
        tc_commit(drain);
        mbar_wait(drain, 0, nullptr, nullptr, 0);
      }
    }
  } else {
    if constexpr (NT == 2) more_registers();
    // ------------------------------------------------------------------------------------ softmax
    constexpr float kRescale = 8.f;
    const int t = warp / 4, first = r0 + t * kRows;
    const int r = (warp % 4) * 32 + lane, row = first + r;
    const uint32_t lane_off = (uint32_t)((warp % 4) * 32) << 16;
    const uint32_t t_s = tmem + t * kRows + lane_off, t_o = tmem + L::kO + t * DP + lane_off;
    const uint32_t t_p = L::kApart ? tmem + L::kP + t * 64 + lane_off : t_s;
    const float scale_log2 = P.scale * kLog2e;
    const int j0 = t == 0 ? begin[0] : begin[NT - 1], j1 = t == 0 ? end[0] : end[NT - 1];
    const bool real = row < P.Tq;
    const int2 mine = real ? P.q_bounds[row] : make_int2(0, 0);
    int all_lo = 0, all_hi = 0;  // keys that every row of the tile sees
    if (j1 > j0) {
      all_lo = P.q_bounds[min(first + kRows, P.Tq) - 1].x;
      all_hi = P.q_bounds[first].y;
    }
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = j0; j < j1; ++j) {
      if (!warp_wait(&s_full[t], (j - j0) & 1, abort_flag, err)) { ok = false; break; }
      tc_fence_after();
      const int kb = from + j * kRows;
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(t_s + c * 32, v[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_wait_regs(v[c]);
      if constexpr (L::kApart) {
        tc_fence_before();
        mbar_arrive(&s_read[t]);
      }
      const bool masked = kb < all_lo || kb + kRows > all_hi;
      if (masked) {
        const int a = mine.x - kb;
        const uint32_t n = (uint32_t)max(mine.y - mine.x, 0);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if ((uint32_t)(c * 32 + e - a) >= n) v[c][e] = 0xff800000u;
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = max3_nan(__uint_as_float(v[c][0]), __uint_as_float(v[c][1]), __uint_as_float(v[c][2]));
#pragma unroll
        for (int e = 3; e < 31; e += 2) mx[c] = max3_nan(mx[c], __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
      }
      mx[0] = max3_nan(mx[0], mx[1], __uint_as_float(v[0][31]));
      mx[2] = max3_nan(mx[2], mx[3], __uint_as_float(v[1][31]));
      mx[0] = max3_nan(mx[0], __uint_as_float(v[2][31]), __uint_as_float(v[3][31]));
      const float blk = fmaxf(mx[0], mx[2]) * scale_log2;
      // a score of infinity or NaN that this row sees makes it NaN (fmaxf may drop one of two NaN, so both are asked)
      if (!(mx[0] < INFINITY) || !(mx[2] < INFINITY)) m = NAN;
      const bool move = blk > m + kRescale;  // of a first block with a key always
      if (__any_sync(0xffffffffu, move && m != -INFINITY)) {
        if (!warp_wait(&o_full[t], (j - j0 - 1) & 1, abort_flag, err)) { ok = false; break; }
        tc_fence_after();
        const float alpha = move && m != -INFINITY ? exp2_approx(m - blk) : 1.f;
#pragma unroll 1
        for (int c = 0; c * 16 < P.D; ++c) {
          uint32_t w[16];
          tmem_ld_32x32b_x16(t_o + c * 16, w);
          tmem_ld_wait_regs16(w);
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * alpha);
          tmem_st_32x32b_x16(t_o + c * 16, w);
        }
        l *= alpha;
      }
      if (move) m = blk;
      const float ref = m == -INFINITY ? 0.f : m;
      // Where nothing is masked a quarter of the exponentials go to the FMA pipe: the multi-function unit takes 8 cycles
      // for a warp's 32 and is the bound of this loop.
      const f32x2 scale2 = pair_of(scale_log2, scale_log2), ref2 = pair_of(-ref, -ref);
      f32x2 sum[2] = {0, 0};
      auto exponentials = [&](auto mixed) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const f32x2 x = fma2(pair_of(__uint_as_float(v[c][2 * e]), __uint_as_float(v[c][2 * e + 1])), scale2, ref2);
            float p0, p1;
            if (decltype(mixed)::value && e % 4 == 3) {
              exp2_fma(x, p0, p1);
            } else {
              split(x, p0, p1);
              p0 = exp2_approx(p0);
              p1 = exp2_approx(p1);
            }
            sum[e & 1] = add2(sum[e & 1], pair_of(p0, p1));
            v[c / 2][(c & 1) * 16 + e] = pack2<T>(p0, p1);
          }
      };
      if (masked) exponentials(std::false_type{});
      else exponentials(std::true_type{});
      float sum0, sum1;
      split(add2(sum[0], sum[1]), sum0, sum1);
      if (L::kApart && j > j0) {  // the place of P is free once the last P V is done
        if (!warp_wait(&o_full[t], (j - j0 - 1) & 1, abort_flag, err)) { ok = false; break; }
        tc_fence_after();
      }
      tmem_st_32x32b_x32(t_p, v[0]);
      tmem_st_32x32b_x32(t_p + 32, v[1]);
      l += sum0 + sum1;
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[t]);
    }
    if (ok && j1 > j0) ok = warp_wait(&o_full[t], (j1 - j0 - 1) & 1, abort_flag, err);
    const bool sees = mine.y > mine.x;
    // Every score that the row sees is -inf: the exponentials of the FMA pipe, which end at 2^-126, are not 0 then.
    if (m == -INFINITY) l = 0.f;
    if (ok) {
      tc_fence_after();
      const float inv = row_value(sees, 1.f, l);
      T* dst = o + ((int64_t)(real ? row : 0) * P.Hq + h) * P.D;
      float bad = 0.f;
#pragma unroll 1
      for (int c = 0; c * 16 < P.D; ++c) {
        uint32_t w[16];
        if (j1 > j0) {
          tmem_ld_32x32b_x16(t_o + c * 16, w);
          tmem_ld_wait_regs16(w);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = 0;
        }
        const bool both = real && c * 16 + 16 <= P.D;
        bad += store16<T>(dst + c * 16, w, inv, real, both);
        if (P.o_low != nullptr) store16_low<T>((T*)P.o_low + (dst - o) + c * 16, w, inv, real, both);
      }
      if (real) lse[(int64_t)h * P.lse_stride + row] = row_lse(sees, m, l);
      // rows that a masked neighbour's infinity or NaN may have reached
      const bool partly = mine.x > from + j0 * kRows || mine.y < from + j1 * kRows;
      uint32_t again = __ballot_sync(0xffffffffu, real && partly && bad != bad && inv == inv);
      if (again != 0) {
        __syncwarp();
        // in the place of this tile's queries: its last scores are done, and no load and no other tile comes there (K and V
        // may still be loaded and read for the block's other tile)
        float* scratch = reinterpret_cast<float*>(smem + L::kQ + t * Tile<DP>::kBytes) + (warp % 4) * kRowScratch;
        while (again != 0) {
          const int who = __ffs(again) - 1;
          again &= again - 1;
          const int i = first + (warp % 4) * 32 + who;
          const int2 b = P.q_bounds[i];
          float acc[4], stat;
          forward_row<T>((const T*)P.q + i * P.qs.row + h * P.qs.head, (const T*)P.k + hk * P.ks.head,
                         (const T*)P.v + hk * P.vs.head, P.ks.row, P.vs.row, b.x, b.y, P.D, scale_log2, scratch, lane, acc,
                         stat);
          const int64_t out = ((int64_t)i * P.Hq + h) * P.D;
          store_row_low<T>(o + out, P.o_low != nullptr ? (T*)P.o_low + out : nullptr, acc, P.D, lane);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == NT * 4 + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, L::kCols);
  }
}

// --------------------------------------------------------------------------------- backward: delta
// delta_i = do_i . o_i, with o as it was before rounding: where a row has few keys, dP - delta is a small difference. A CTA
// owns 128 rows of a head, 16 lanes a row. For fp16 also the norm of every do row and the block's largest: dS = p (dP - delta)
// is near |do| times a probability and would fall among fp16's subnormals, so the backward kernels scale it by a power of two
// of that size: that of the query's own row for dQ, for dK that of the largest among the queries that see the key, so that no
// other sequence's gradients set the step that this one's are rounded to.
//
// The kernel for dK and dV has its queries along the columns; a statistic per column read from shared memory by every
// thread would take 4 cycles of its port for each 4 columns and warp, as long as the exponentials, and in the way of the
// products' operands. It is subtracted by the tensor core instead: as 8 more channels, -lse / (scale log2 e) and -delta
// as sums of 16-bit values (each what the ones before leave: 24 bits after three bf16, 33 after three fp16) times ones;
// for fp16 times 64, with which they reach 3.3e7. What is beyond becomes NaN, and the rows that it reaches are computed
// again without tensor cores.
template <typename T>
__host__ __device__ constexpr float channel_unit() {
  return std::is_same_v<T, __half> ? 64.f : 1.f;
}

template <typename T>
__device__ __forceinline__ uint4 as_channels(float x) {
  constexpr float kMost = std::is_same_v<T, __half> ? 65504.f : 3.3895314e38f;
  x *= 1.f / channel_unit<T>();
  if (std::is_same_v<T, __half> && fabsf(x) > 8.f * kMost && fabsf(x) < INFINITY) x = NAN;
  float v[8];
  const bool finite = fabsf(x) < INFINITY;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = finite ? to_f32(from_f32<T>(fminf(fmaxf(x, -kMost), kMost))) : e == 0 ? x : 0.f;
    x -= finite ? v[e] : 0.f;
  }
  return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

template <typename T>
__global__ void __launch_bounds__(256) packed_delta_tc_kernel(const T* __restrict__ o, const T* __restrict__ low,
                                                              const T* __restrict__ dout,
                                                              HeadRows ds, int Tq, int Hq, int D, int stride,
                                                              const float* __restrict__ lse, float inv_scale_log2,
                                                              float* __restrict__ delta, uint4* __restrict__ channels,
                                                              float* __restrict__ norms) {
  __shared__ float top[16];
  const int h = blockIdx.x % Hq, block = blockIdx.x / Hq;
  const int lane = threadIdx.x % 16, slot = threadIdx.x / 16;
  const int64_t rows = (int64_t)Hq * stride;
  float most = 0.f;
#pragma unroll 4
  for (int u = 0; u < 8; ++u) {
    const int i = block * kRows + u * 16 + slot;
    float s = 0.f, n = 0.f;
    if (i < Tq && lane * 8 < D) {
      float a[8], b[8];
      unpack8<T>(load_raw8<T>(o + ((int64_t)i * Hq + h) * D + lane * 8), a);
      unpack8<T>(load_raw8<T>(dout + i * ds.row + h * ds.head + lane * 8), b);
      if (low != nullptr) {
        float c[8];
        unpack8<T>(load_raw8<T>(low + ((int64_t)i * Hq + h) * D + lane * 8), c);
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] += c[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s = fmaf(a[e], b[e], s);
        n = fmaf(b[e], b[e], n);
      }
    }
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, w);
      n += __shfl_xor_sync(0xffffffffu, n, w);
    }
    if (i < Tq && lane < 2) {
      const int64_t at = (int64_t)h * stride + i;
      if (lane == 0) delta[at] = s;
      channels[lane * rows + at] = as_channels<T>(lane == 0 ? -lse[at] * inv_scale_log2 : -s);
      if (std::is_same_v<T, __half> && lane == 0) norms[at] = n <= 3e38f ? sqrtf(n) : 0.f;
    }
    if (n <= 3e38f) most = fmaxf(most, n);
  }
  if constexpr (std::is_same_v<T, __half>) {
    if (lane == 0) top[slot] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < 16; ++i) most = fmaxf(most, top[i]);
      norms[rows + (int64_t)h * (stride / kRows) + block] = sqrtf(most);
    }
  }
}

// 2^-e for a (largest) norm of do near 2^e (fp16); dS is then at most 2^8 times the rows of v.
__device__ __forceinline__ float ds_factor(float norm) {
  if (!(norm > 0.f)) return 1.f;
  return exp2f(-fminf(fmaxf(ceilf(log2f(norm)), -100.f), 100.f));
}
constexpr float kHalfShift = 8.f;  // fp16: P is kept times 2^8

// The largest norm of the do rows in [mine.x, mine.y) of `heads` heads from `first`; 0 for none. A whole warp calls it, its
// lanes with the bounds of consecutive keys: lanes whose queries end together (a sequence's keys) share all but the first of
// them, and whole blocks of 128 queries have theirs in `blocks`.
__device__ __forceinline__ float largest_norm(const float* norms, const float* blocks, int stride, int first, int heads,
                                              int2 mine, int lane) {
  float top = 0.f;
  uint32_t left = __ballot_sync(0xffffffffu, mine.y > mine.x);
  while (left != 0) {
    const int leader = __ffs(left) - 1, end = __shfl_sync(0xffffffffu, mine.y, leader);
    const bool member = mine.y > mine.x && mine.y == end;
    const uint32_t members = __ballot_sync(0xffffffffu, member);
    left &= ~members;
    const int begin = __shfl_sync(0xffffffffu, mine.x, leader);
    const int common = __shfl_sync(0xffffffffu, mine.x, 31 - __clz(members));  // the bounds never fall
    const int b0 = (common + kRows - 1) / kRows, b1 = end / kRows;             // whole blocks
    const int head_end = b0 < b1 ? b0 * kRows : end, tail = b0 < b1 ? b1 * kRows : end;
    for (int h = first; h < first + heads; ++h) {
      const float *row = norms + (int64_t)h * stride, *block = blocks + (int64_t)h * (stride / kRows);
      float m = 0.f;
      for (int i = common + lane; i < head_end; i += 32) m = fmaxf(m, row[i]);
      for (int b = b0 + lane; b < b1; b += 32) m = fmaxf(m, block[b]);
      for (int i = tail + lane; i < end; i += 32) m = fmaxf(m, row[i]);
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
      if (member) top = fmaxf(top, m);
      for (int i = begin; i < common; ++i)
        if (member && i >= mine.x) top = fmaxf(top, row[i]);
    }
  }
  return top;
}

// ------------------------------------------------------------------------------------ backward: dQ
// A CTA owns 128 queries of one head and goes through their keys. Two groups of four warps (thread = query) take the
// blocks in turns. A block has 128 of three times 128 columns of tensor memory: S -> P in registers, dP over S, dS over
// dP (64 columns of 16-bit pairs, each written after what it covers has been read) -> dQ += dS K. While one group
// computes exponentials the other one multiplies, and the third place takes the scores of the block after.
template <int DP>
struct DqLayout {
  static constexpr int kKStages = 4, kVStages = DP == 64 ? 3 : 1;
  static constexpr int kQ = 0;
  static constexpr int kDO = kQ + Tile<DP>::kBytes;
  static constexpr int kK = kDO + Tile<DP>::kBytes;
  static constexpr int kV = kK + kKStages * Tile<DP>::kBytes;
  static constexpr int kBar = kV + kVStages * Tile<DP>::kBytes;
  static constexpr int kBytes = kBar + 256 + 1024;
};
constexpr int kBwdThreads = 384;

template <typename T, int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
    packed_dq_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                        const PackedProblem P, const T* __restrict__ dout, HeadRows dos, const float* __restrict__ lse,
                        const float* __restrict__ delta, const float* __restrict__ norms, T* __restrict__ dq, int* err) {
  using L = DqLayout<DP>;
  constexpr int KS = L::kKStages, VS = L::kVStages;
  constexpr bool kHalf = std::is_same_v<T, __half>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t *q_full = bar, *k_full = bar + 1, *k_empty = k_full + KS, *v_full = k_empty + KS, *v_empty = v_full + VS;
  uint64_t *s_full = v_empty + VS, *s_read = s_full + 2, *dp_full = s_read + 2, *ds_full = dp_full + 2;
  uint64_t *dq_full = ds_full + 2, *drain = dq_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform((int)threadIdx.x / 32), lane = threadIdx.x % 32;
  const int tiles = (P.Tq + kRows - 1) / kRows;
  const int h = blockIdx.x % P.Hq;
  const int r0 = (tiles - 1 - (int)(blockIdx.x / P.Hq)) * kRows;
  const int hk = h / P.group;
  const int from = P.q_bounds[r0].x, to = P.q_bounds[min(r0 + kRows, P.Tq) - 1].y;
  const int blocks = to > from ? (to - from + kRows - 1) / kRows : 0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&s_read[s], 128);
      mbar_init(&dp_full[s], 1);
      mbar_init(&ds_full[s], 128);
    }
    mbar_init(dq_full, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmQ);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
    prefetch_tensormap(&tmDO);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t c_dq = tmem + 3 * kRows;

  if (warp >= 8) {
    fewer_registers();
    if (warp == 8 && lane == 0 && blocks > 0) {
      int nk = 0, nv = 0;
      bool ok = true;
      mbar_arrive_expect_tx(q_full, 2 * Tile<DP>::kBytes);
      load_tile<DP>(smem + L::kQ, &tmQ, q_full, r0, h);
      load_tile<DP>(smem + L::kDO, &tmDO, q_full, r0, h);
      for (int j = 0; j < blocks; ++j) {
        if (!bounded_wait(&k_empty[j % KS], ((j / KS) & 1) ^ 1, abort_flag, err)) { ok = false; break; }
        mbar_arrive_expect_tx(&k_full[j % KS], Tile<DP>::kBytes);
        load_tile<DP>(smem + L::kK + (j % KS) * Tile<DP>::kBytes, &tmK, &k_full[j % KS], from + j * kRows, hk);
        ++nk;
        if (!bounded_wait(&v_empty[j % VS], ((j / VS) & 1) ^ 1, abort_flag, err)) { ok = false; break; }
        mbar_arrive_expect_tx(&v_full[j % VS], Tile<DP>::kBytes);
        load_tile<DP>(smem + L::kV + (j % VS) * Tile<DP>::kBytes, &tmV, &v_full[j % VS], from + j * kRows, hk);
        ++nv;
      }
      if (!ok) {
        mbar_wait(q_full, 0, nullptr, nullptr, 0);
        for (int j = first_in_flight(nk, KS); j < nk; ++j) mbar_wait(&k_full[j % KS], (j / KS) & 1, nullptr, nullptr, 0);
        for (int j = first_in_flight(nv, VS); j < nv; ++j) mbar_wait(&v_full[j % VS], (j / VS) & 1, nullptr, nullptr, 0);
      }
    } else if (warp == 9) {
      const bool one = elect_one();
      const uint32_t idesc_s = idesc_of<T>(kRows, false), idesc_g = idesc_of<T>((P.D + 15) / 16 * 16, true);
      const uint64_t q_desc = desc_k(uniform(smem_u32(smem + L::kQ))), do_desc = desc_k(uniform(smem_u32(smem + L::kDO)));
      const uint64_t k_desc = desc_k(uniform(smem_u32(smem + L::kK))), v_desc = desc_k(uniform(smem_u32(smem + L::kV)));
      const uint64_t k_rows = desc_mn(uniform(smem_u32(smem + L::kK)));
      const uint32_t base = uniform(tmem);
      const int n = uniform(blocks);
      auto scores = [&](int j) -> bool {
        if (!warp_wait(&k_full[j % KS], (j / KS) & 1, abort_flag, err)) return false;
        tc_fence_after();
        if (one) {
          mma_scores<DP>(base + (j % 3) * kRows, q_desc, k_desc + tile_step<DP>(j % KS), idesc_s, P.D);
          tc_commit(&s_full[j & 1]);
        }
        return true;
      };
      auto d_probs = [&](int j) -> bool {
        if (!warp_wait(&v_full[j % VS], (j / VS) & 1, abort_flag, err)) return false;
        if (!warp_wait(&s_read[j & 1], (j >> 1) & 1, abort_flag, err)) return false;
        tc_fence_after();
        if (one) {
          mma_scores<DP>(base + (j % 3) * kRows, do_desc, v_desc + tile_step<DP>(j % VS), idesc_s, P.D);
          tc_commit(&v_empty[j % VS]);
          tc_commit(&dp_full[j & 1]);
        }
        return true;
      };
      auto sums = [&](int j) -> bool {
        if (!warp_wait(&ds_full[j & 1], (j >> 1) & 1, abort_flag, err)) return false;
        tc_fence_after();
        if (one) {
          mma_sums(base + 3 * kRows, base + (j % 3) * kRows, k_rows + tile_step<DP>(j % KS), idesc_g, j > 0);
          tc_commit(&k_empty[j % KS]);
        }
        return true;
      };
      bool ok = n == 0 || (warp_wait(q_full, 0, abort_flag, err) && scores(0) && (n < 2 || scores(1)));
      for (int j = 0; j < n && ok; ++j) {
        ok = d_probs(j) && (j == 0 || sums(j - 1)) && (j + 2 >= n || scores(j + 2));
      }
      ok = ok && (n == 0 || sums(n - 1));
      if (one) {
        if (ok) {
          tc_commit(dq_full);
        } else {
          tc_commit(drain);
          mbar_wait(drain, 0, nullptr, nullptr, 0);
        }
      }
    }
  } else {
    more_registers();
    const int group = warp / 4, r = (warp % 4) * 32 + lane, row = r0 + r;
    const uint32_t lane_off = (uint32_t)((warp % 4) * 32) << 16;
    const bool real = row < P.Tq;
    const int2 mine = real ? P.q_bounds[row] : make_int2(0, 0);
    const int all_lo = P.q_bounds[min(r0 + kRows, P.Tq) - 1].x, all_hi = P.q_bounds[r0].y;
    const int64_t stat = (int64_t)h * P.lse_stride + (real ? row : r0);
    const float lse_row = lse[stat], delta_row = delta[stat];
    const float shift = kHalf ? lse_row - kHalfShift : lse_row;
    const float factor = kHalf ? ds_factor(norms[stat]) : 1.f;
    const float scale_log2 = P.scale * kLog2e;
    const f32x2 scale2 = pair_of(scale_log2, scale_log2), shift2 = pair_of(-shift, -shift);
    const f32x2 delta2 = pair_of(-delta_row, -delta_row), factor2 = pair_of(factor, factor);
    bool ok = true;
    for (int j = group; j < blocks; j += 2) {
      const uint32_t parity = (j >> 1) & 1, c_s = tmem + (j % 3) * kRows + lane_off;
      if (!warp_wait(&s_full[group], parity, abort_flag, err)) { ok = false; break; }
      tc_fence_after();
      uint32_t p[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(c_s + c * 32, p[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_wait_regs(p[c]);
      tc_fence_before();
      mbar_arrive(&s_read[group]);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          split(fma2(pair_of(__uint_as_float(p[c][2 * e]), __uint_as_float(p[c][2 * e + 1])), scale2, shift2), x0, x1);
          p[c][2 * e] = __float_as_uint(exp2_approx(x0));
          p[c][2 * e + 1] = __float_as_uint(exp2_approx(x1));
        }
      const int kb = from + j * kRows;
      const bool masked = kb < all_lo || kb + kRows > all_hi;
      const int a = mine.x - kb;
      const uint32_t n = (uint32_t)max(mine.y - mine.x, 0);
      if (!warp_wait(&dp_full[group], parity, abort_flag, err)) { ok = false; break; }
      tc_fence_after();
      uint32_t v[2][32];  // the next 32 columns are on their way while these are worked on
      tmem_ld_32x32b_x32(c_s, v[0]);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t(&x)[32] = v[c & 1];
        tmem_ld_wait_regs(x);
        if (c < 3) tmem_ld_32x32b_x32(c_s + (c + 1) * 32, v[(c + 1) & 1]);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          f32x2 d = mul2(pair_of(__uint_as_float(p[c][2 * e]), __uint_as_float(p[c][2 * e + 1])),
                         add2(pair_of(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])), delta2));
          if constexpr (kHalf) d = mul2(d, factor2);
          float d0, d1;
          split(d, d0, d1);
          p[c][2 * e] = __float_as_uint(d0);
          p[c][2 * e + 1] = __float_as_uint(d1);
        }
        if (masked)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if ((uint32_t)(c * 32 + e - a) >= n) p[c][e] = 0;
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) pk[e] = pack2<T>(__uint_as_float(p[c][2 * e]), __uint_as_float(p[c][2 * e + 1]));
        tmem_st_32x32b_x16(c_s + c * 16, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&ds_full[group]);
    }
    if (ok && blocks > 0) ok = warp_wait(dq_full, 0, abort_flag, err);
    if (ok) {
      tc_fence_after();
      // fp16: the sums hold 2^8 factor dS
      const float f = kHalf ? P.scale / (factor * 256.f) : P.scale;
      T* dst = dq + ((int64_t)(real ? row : 0) * P.Hq + h) * P.D;
      float bad = 0.f;
#pragma unroll 1
      for (int c = group; c * 16 < P.D; c += 2) {
        uint32_t w[16];
        if (blocks > 0) {
          tmem_ld_32x32b_x16(c_dq + lane_off + c * 16, w);
          tmem_ld_wait_regs16(w);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = 0;
        }
        bad += store16<T>(dst + c * 16, w, f, real, real && c * 16 + 16 <= P.D);
      }
      const bool partly = kHalf || mine.x > from || mine.y < from + blocks * kRows;
      const float own = lse_row == INFINITY ? 0.f : fmaf(lse_row, 0.f, delta_row * 0.f);
      uint32_t again = __ballot_sync(0xffffffffu, real && partly && bad != bad && own == own);
      if (again != 0) {
        __syncwarp();
        float* scratch = reinterpret_cast<float*>(smem + L::kK) + warp * kRowScratch;
        while (again != 0) {
          const int who = __ffs(again) - 1;
          again &= again - 1;
          const int i = r0 + (warp % 4) * 32 + who;
          const int2 b = P.q_bounds[i];
          const int64_t at = (int64_t)h * P.lse_stride + i;
          float acc[4];
          dq_row<T>((const T*)P.q + i * P.qs.row + h * P.qs.head, dout + i * dos.row + h * dos.head,
                    (const T*)P.k + hk * P.ks.head, (const T*)P.v + hk * P.vs.head, P.ks.row, P.vs.row, b.x, b.y, P.D,
                    P.scale, lse[at], delta[at], scratch, lane, acc);
          // this warp's columns only: the other group's warp looks after its own
          T* out = dq + ((int64_t)i * P.Hq + h) * P.D;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int c = lane + 32 * u;
            if (c < P.D && ((c >> 4) & 1) == group) out[c] = from_f32<T>(acc[u]);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ----------------------------------------------------------------------------- backward: dK and dV
// A CTA owns 128 keys of one key head and goes through the queries that see them, for every query head of the
// group: S^T = K Q^T -> P^T -> dV += P^T dO, dP^T = V dO^T over S^T as soon as that has been read -> dS^T -> dK += dS^T Q;
// thread = key; lse and delta of the queries are 8 more channels of both products (packed_delta_tc_kernel). Query blocks
// begin at multiples of 128.
//
// DP = 64: two groups of four warps take the blocks in turns, one's exponentials beside the other's dS. Tensor memory
// per group: S^T, then dP^T, then dS^T (128 columns) and P^T (64); dV and dK (64 each).
// DP = 128: dV and dK leave room for one S^T / dP^T (128), P^T and dS^T (64 each): all eight warps share a block, half
// of its queries each, and the products are the bound (2048 cycles a block against 1024 of exponentials).
template <int DP>
struct DkvLayout {
  static constexpr bool kTurns = DP == 64;
  static constexpr int kStages = kTurns ? 4 : 2;
  static constexpr uint32_t kXStep = kTurns ? 192 : 0, kP = 128, kDS = kTurns ? 0 : 192;  // columns
  static constexpr uint32_t kDV = kTurns ? 384 : 256, kDK = kDV + DP;
  static constexpr int kK = 0;
  static constexpr int kV = kK + Tile<DP>::kBytes;
  static constexpr int kQ = kV + Tile<DP>::kBytes;
  static constexpr int kDO = kQ + kStages * Tile<DP>::kBytes;
  static constexpr int kStat = kDO + kStages * Tile<DP>::kBytes;  // channels of lse and delta (2 KB each), per stage
  static constexpr int kOnes = kStat + kStages * 4096;            // 128 rows of 8 times the channels' unit
  static constexpr int kZeros = kOnes + 2048;                     // and of 8 zeros, the other half of a step of 16
  static constexpr int kBar = kZeros + 2048;
  static constexpr int kBytes = kBar + 256 + 1024;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
    packed_dkv_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmDO,
                         const PackedProblem P, const T* __restrict__ dout, HeadRows dos, const float* __restrict__ lse,
                         const float* __restrict__ delta, const uint4* __restrict__ channels,
                         const float* __restrict__ norms, T* __restrict__ dk, T* __restrict__ dv, int* err) {
  using L = DkvLayout<DP>;
  constexpr int S = L::kStages;
  constexpr bool kTurns = L::kTurns;
  constexpr bool kHalf = std::is_same_v<T, __half>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + L::kBar);
  // two of each, in turns; without turns only the first is used
  uint64_t *kv_full = bar, *q_full = bar + 1, *q_empty = q_full + S, *s_full = q_empty + S, *s_read = s_full + 2;
  uint64_t *dp_full = s_read + 2, *dp_read = dp_full + 2, *p_full = dp_read + 2, *ds_full = p_full + 2;
  uint64_t *g_full = ds_full + 2, *drain = g_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform((int)threadIdx.x / 32), lane = threadIdx.x % 32;
  const int g = blockIdx.x % P.Hk;
  const int k0 = (int)(blockIdx.x / P.Hk) * kRows;  // causal keys are seen by the more queries the earlier they are
  const int q_lo = P.k_bounds[k0].x, q_hi = P.k_bounds[min(k0 + kRows, P.Tk) - 1].y;
  const int qb0 = q_lo / kRows, per_head = q_hi > q_lo ? (q_hi + kRows - 1) / kRows - qb0 : 0;
  const int steps = per_head * P.group;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    for (int s = 0; s < S; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      constexpr int kArrive = kTurns ? 128 : 256;
      mbar_init(&s_full[s], 1);
      mbar_init(&s_read[s], kArrive);
      mbar_init(&dp_full[s], 1);
      mbar_init(&dp_read[s], kArrive);
      mbar_init(&p_full[s], kArrive);
      mbar_init(&ds_full[s], kArrive);
    }
    mbar_init(g_full, 1);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmQ);
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
    prefetch_tensormap(&tmDO);
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  {
    const uint32_t one2 = pack2<T>(channel_unit<T>(), channel_unit<T>());
    if (threadIdx.x < 128) reinterpret_cast<uint4*>(smem + L::kOnes)[threadIdx.x] = make_uint4(one2, one2, one2, one2);
    else if (threadIdx.x < 256) reinterpret_cast<uint4*>(smem + L::kZeros)[threadIdx.x - 128] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 8) {
    fewer_registers();
    if (warp == 8 && lane == 0 && steps > 0) {
      int done = 0;
      bool ok = true;
      mbar_arrive_expect_tx(kv_full, 2 * Tile<DP>::kBytes);
      load_tile<DP>(smem + L::kK, &tmK, kv_full, k0, g);
      load_tile<DP>(smem + L::kV, &tmV, kv_full, k0, g);
      for (int i = 0; i < steps; ++i) {
        const int s = i % S, h = g * P.group + i / per_head, q0 = (qb0 + i % per_head) * kRows;
        if (!bounded_wait(&q_empty[s], ((i / S) & 1) ^ 1, abort_flag, err)) { ok = false; break; }
        mbar_arrive_expect_tx(&q_full[s], 2 * Tile<DP>::kBytes + 4096);
        load_tile<DP>(smem + L::kQ + s * Tile<DP>::kBytes, &tmQ, &q_full[s], q0, h);
        load_tile<DP>(smem + L::kDO + s * Tile<DP>::kBytes, &tmDO, &q_full[s], q0, h);
        const int64_t at = (int64_t)h * P.lse_stride + q0;
        bulk_load(smem + L::kStat + s * 4096, channels + at, 2048, &q_full[s]);
        bulk_load(smem + L::kStat + s * 4096 + 2048, channels + (int64_t)P.Hq * P.lse_stride + at, 2048, &q_full[s]);
        ++done;
      }
      if (!ok) {
        mbar_wait(kv_full, 0, nullptr, nullptr, 0);
        for (int i = first_in_flight(done, S); i < done; ++i) mbar_wait(&q_full[i % S], (i / S) & 1, nullptr, nullptr, 0);
      }
    } else if (warp == 9) {
      const bool one = elect_one();
      const uint32_t idesc_s = idesc_of<T>(kRows, false), idesc_g = idesc_of<T>((P.D + 15) / 16 * 16, true);
      const uint64_t k_desc = desc_k(uniform(smem_u32(smem + L::kK))), v_desc = desc_k(uniform(smem_u32(smem + L::kV)));
      const uint64_t q_desc = desc_k(uniform(smem_u32(smem + L::kQ))), do_desc = desc_k(uniform(smem_u32(smem + L::kDO)));
      const uint64_t q_rows = desc_mn(uniform(smem_u32(smem + L::kQ))), do_rows = desc_mn(uniform(smem_u32(smem + L::kDO)));
      const uint32_t base = uniform(tmem);
      const int n = uniform(steps);
      const uint32_t stat_addr = uniform(smem_u32(smem + L::kStat)), ones_addr = uniform(smem_u32(smem + L::kOnes));
      const uint32_t zeros_addr = ones_addr + (L::kZeros - L::kOnes);
      const uint64_t ones_desc = desc_columns(ones_addr, zeros_addr - ones_addr);
      // one more step of 16: the statistics' 8 channels and 8 zeros, times ones (and zeros)
      auto subtract = [&](uint32_t d, int i, int which) {
        const uint32_t from = stat_addr + (i % S) * 4096 + which * 2048;
        tc_mma_f16(d, ones_desc, desc_columns(from, zeros_addr - from), idesc_s, 1);
      };
      auto turn = [&](int i) { return kTurns ? i & 1 : 0; };
      auto phase = [&](int i) -> uint32_t { return kTurns ? (i >> 1) & 1 : i & 1; };
      auto scores = [&](int i) -> bool {
        if (!warp_wait(&q_full[i % S], (i / S) & 1, abort_flag, err)) return false;
        tc_fence_after();
        if (one) {
          mma_scores<DP>(base + turn(i) * L::kXStep, k_desc, q_desc + tile_step<DP>(i % S), idesc_s, P.D);
          subtract(base + turn(i) * L::kXStep, i, 0);
          tc_commit(&s_full[turn(i)]);
        }
        return true;
      };
      auto d_probs = [&](int i) -> bool {
        if (!warp_wait(&s_read[turn(i)], phase(i), abort_flag, err)) return false;
        tc_fence_after();
        if (one) {
          mma_scores<DP>(base + turn(i) * L::kXStep, v_desc, do_desc + tile_step<DP>(i % S), idesc_s, P.D);
          subtract(base + turn(i) * L::kXStep, i, 1);
          tc_commit(&dp_full[turn(i)]);
        }
        return true;
      };
      auto sums_v = [&](int i) -> bool {
        if (!warp_wait(&p_full[turn(i)], phase(i), abort_flag, err)) return false;
        tc_fence_after();
        if (one)
          mma_sums(base + L::kDV, base + turn(i) * L::kXStep + L::kP, do_rows + tile_step<DP>(i % S), idesc_g, i > 0);
        return true;
      };
      auto sums_k = [&](int i) -> bool {
        if (!warp_wait(&ds_full[turn(i)], phase(i), abort_flag, err)) return false;
        tc_fence_after();
        if (one) {
          mma_sums(base + L::kDK, base + turn(i) * L::kXStep + L::kDS, q_rows + tile_step<DP>(i % S), idesc_g, i > 0);
          tc_commit(&q_empty[i % S]);
        }
        return true;
      };
      bool ok = n == 0 || (warp_wait(kv_full, 0, abort_flag, err) && scores(0));
      if constexpr (kTurns) {
        ok = ok && (n < 2 || scores(1));
        for (int i = 0; i < n && ok; ++i)
          ok = d_probs(i) && (i == 0 || (sums_k(i - 1) && (i + 1 >= n || scores(i + 1)))) && sums_v(i);
        ok = ok && (n == 0 || sums_k(n - 1));
      } else {
        for (int i = 0; i < n && ok; ++i) {
          ok = d_probs(i) && sums_v(i);
          if (ok && i + 1 < n) ok = warp_wait(dp_read, i & 1, abort_flag, err) && scores(i + 1);
          ok = ok && sums_k(i);
        }
      }
      if (one) {
        if (ok) {
          tc_commit(g_full);
        } else {
          tc_commit(drain);
          mbar_wait(drain, 0, nullptr, nullptr, 0);
        }
      }
    }
  } else {
    more_registers();
    const int group = warp / 4, r = (warp % 4) * 32 + lane, key = k0 + r;
    const uint32_t lane_off = (uint32_t)((warp % 4) * 32) << 16;
    // a group's own block, or a half of the common block's queries
    constexpr int C = kTurns ? 4 : 2;
    const int bi = kTurns ? group : 0, off = kTurns ? 0 : group * 64;
    const uint32_t t_x = tmem + bi * L::kXStep + off + lane_off;
    const uint32_t t_p = tmem + bi * L::kXStep + L::kP + off / 2 + lane_off;
    const uint32_t t_ds = tmem + bi * L::kXStep + L::kDS + off / 2 + lane_off;
    const bool real = key < P.Tk;
    const int2 mine = real ? P.k_bounds[key] : make_int2(0, 0);
    const int all_lo = P.k_bounds[min(k0 + kRows, P.Tk) - 1].x, all_hi = P.k_bounds[k0].y;
    const float scale_log2 = P.scale * kLog2e;
    float factor = 1.f;
    if constexpr (kHalf)
      factor = ds_factor(largest_norm(norms, norms + (int64_t)P.Hq * P.lse_stride, P.lse_stride, g * P.group, P.group, mine, lane));
    const float shift = kHalf ? kHalfShift : 0.f;
    const f32x2 scale2 = pair_of(scale_log2, scale_log2), shift2 = pair_of(shift, shift), factor2 = pair_of(factor, factor);
    bool ok = true;
    for (int i = kTurns ? group : 0; i < steps; i += kTurns ? 2 : 1) {
      const uint32_t parity = kTurns ? (i >> 1) & 1 : i & 1;
      const int q0 = (qb0 + i % per_head) * kRows + off;
      if (!warp_wait(&s_full[bi], parity, abort_flag, err)) { ok = false; break; }
      tc_fence_after();
      const bool masked = q0 < all_lo || q0 + C * 32 > all_hi;
      const int a = mine.x - q0;
      const uint32_t n = (uint32_t)max(mine.y - mine.x, 0);
      uint32_t p[C][32];
#pragma unroll
      for (int c = 0; c < C; ++c) tmem_ld_32x32b_x32(t_x + c * 32, p[c]);
#pragma unroll
      for (int c = 0; c < C; ++c) tmem_ld_wait_regs(p[c]);
      tc_fence_before();
      mbar_arrive(&s_read[bi]);
      // all exponentials before the first store: the stores keep loads and arithmetic from moving across them
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float x0, x1;
          split(fma2(pair_of(__uint_as_float(p[c][2 * e]), __uint_as_float(p[c][2 * e + 1])), scale2, shift2), x0, x1);
          p[c][2 * e] = __float_as_uint(exp2_approx(x0));
          p[c][2 * e + 1] = __float_as_uint(exp2_approx(x1));
        }
      if (masked)
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if ((uint32_t)(c * 32 + e - a) >= n) p[c][e] = 0;
      // the last P^T there has been multiplied: this S^T came after it
#pragma unroll
      for (int c = 0; c < C; c += 2) {
        uint32_t pk[32];
#pragma unroll
        for (int e = 0; e < 32; ++e)
          pk[e] = pack2<T>(__uint_as_float(p[c + e / 16][2 * e % 32]), __uint_as_float(p[c + e / 16][2 * e % 32 + 1]));
        tmem_st_32x32b_x32(t_p + c * 16, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&p_full[bi]);
      if (!warp_wait(&dp_full[bi], parity, abort_flag, err)) { ok = false; break; }
      tc_fence_after();
      uint32_t v[2][32];
      tmem_ld_32x32b_x32(t_x, v[0]);
      if constexpr (!kTurns) {
        tmem_ld_32x32b_x32(t_x + 32, v[1]);
        tmem_ld_wait_regs(v[0]);
        tmem_ld_wait_regs(v[1]);
        tc_fence_before();
        mbar_arrive(&dp_read[bi]);
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        uint32_t(&x)[32] = v[c & 1];
        if constexpr (kTurns) {  // the next 32 columns are on their way while these are worked on
          tmem_ld_wait_regs(x);
          if (c + 1 < C) tmem_ld_32x32b_x32(t_x + (c + 1) * 32, v[(c + 1) & 1]);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          f32x2 d = mul2(pair_of(__uint_as_float(p[c][2 * e]), __uint_as_float(p[c][2 * e + 1])),
                         pair_of(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1])));
          if constexpr (kHalf) d = mul2(d, factor2);
          float d0, d1;
          split(d, d0, d1);
          p[c][2 * e] = __float_as_uint(d0);
          p[c][2 * e + 1] = __float_as_uint(d1);
        }
        if (masked)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if ((uint32_t)(c * 32 + e - a) >= n) p[c][e] = 0;
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) pk[e] = pack2<T>(__uint_as_float(p[c][2 * e]), __uint_as_float(p[c][2 * e + 1]));
        tmem_st_32x32b_x16(t_ds + c * 16, pk);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&ds_full[bi]);
    }
    if (ok && steps > 0) ok = warp_wait(g_full, 0, abort_flag, err);
    if (ok) {
      tc_fence_after();
      const float fk = kHalf ? P.scale / (factor * 256.f) : P.scale, fv = kHalf ? 1.f / 256.f : 1.f;
      const int64_t at = ((int64_t)(real ? key : 0) * P.Hk + g) * P.D;
      float bad = 0.f;
#pragma unroll 1
      for (int c = group; c * 16 < P.D; c += 2) {
        uint32_t w[16], u[16];
        if (steps > 0) {
          tmem_ld_32x32b_x16(tmem + L::kDK + lane_off + c * 16, w);
          tmem_ld_32x32b_x16(tmem + L::kDV + lane_off + c * 16, u);
          tmem_ld_wait_regs16(w);
          tmem_ld_wait_regs16(u);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = u[e] = 0;
        }
        const bool both = real && c * 16 + 16 <= P.D;
        bad += store16<T>(dk + at + c * 16, w, fk, real, both);
        bad += store16<T>(dv + at + c * 16, u, fv, real, both);
      }
      const bool partly = kHalf || mine.x > qb0 * kRows || mine.y < (qb0 + per_head) * kRows;
      uint32_t again = __ballot_sync(0xffffffffu, real && partly && bad != bad);
      if (again != 0) {
        __syncwarp();
        float* scratch = reinterpret_cast<float*>(smem + L::kQ) + warp * kRowScratch;
        while (again != 0) {
          const int who = __ffs(again) - 1;
          again &= again - 1;
          const int j = k0 + (warp % 4) * 32 + who;
          const int2 b = P.k_bounds[j];
          // a NaN among the statistics of its own queries makes the row NaN: nothing to mend
          float own = 0.f;
          for (int h = g * P.group; h < (g + 1) * P.group; ++h)
            for (int i = b.x + lane; i < b.y; i += 32) {
              const float s = lse[(int64_t)h * P.lse_stride + i];
              if (s != s) own = s;
            }
          if (__any_sync(0xffffffffu, own != own)) continue;
          float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
          for (int h = g * P.group; h < (g + 1) * P.group; ++h)
            dkv_row<T>((const T*)P.k + j * P.ks.row + g * P.ks.head, (const T*)P.v + j * P.vs.row + g * P.vs.head,
                       (const T*)P.q + h * P.qs.head, dout + h * dos.head, P.qs.row, dos.row, b.x, b.y, P.D, P.scale,
                       lse + (int64_t)h * P.lse_stride, delta + (int64_t)h * P.lse_stride, scratch, lane, x, y);
          const int64_t out = ((int64_t)j * P.Hk + g) * P.D;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int c = lane + 32 * u;
            if (c < P.D && ((c >> 4) & 1) == group) {
              dk[out + c] = from_f32<T>(x[u]);
              dv[out + c] = from_f32<T>(y[u]);
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// --------------------------------------------------------------------------------------------- host

PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t status = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found);
    return status == cudaSuccess && found == cudaDriverEntryPointSuccess
               ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr)
               : nullptr;
  }();
  return fn;
}

// Encoding a map needs a current context, which a thread (autograd's, say) has from its first call of the runtime on.
cudaError_t context_current() {
  int device = 0;
  const cudaError_t status = cudaGetDevice(&device);
  return status == cudaSuccess ? cudaSetDevice(device) : status;
}

// (D, rows, H) with boxes of 64 channels of 128 rows; rows past the last sequence and channels past the head read 0.
bool map_rows(CUtensorMap* map, const void* base, HeadRows s, int rows, int H, int D, SequenceType type) {
  if (encode_tiled() == nullptr) return false;
  // a single row or head may come with any stride
  const int64_t row = rows > 1 ? s.row : 8, head = H > 1 ? s.head : 8;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)H};
  cuuint64_t strides[2] = {(cuuint64_t)(row * 2), (cuuint64_t)(head * 2)};
  cuuint32_t box[3] = {64, kRows, 1}, step[3] = {1, 1, 1};
  return encode_tiled()(map, type == kSeqBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K, typename... A>
cudaError_t launch(K kernel, int64_t grid, int threads, int smem, cudaStream_t stream, const A&... args) {
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const cudaError_t status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (status != cudaSuccess) return status;
  kernel<<<(unsigned)grid, threads, smem, stream>>>(args...);
  return cudaGetLastError();
}

template <typename T, int DP>
cudaError_t fwd(const PackedProblem& P, void* o, float* lse, int* err, cudaStream_t stream) {
  CUtensorMap q, k, v;
  const cudaError_t ready = context_current();
  if (ready != cudaSuccess) return ready;
  if (!map_rows(&q, P.q, P.qs, P.Tq, P.Hq, P.D, P.type) || !map_rows(&k, P.k, P.ks, P.Tk, P.Hk, P.D, P.type) ||
      !map_rows(&v, P.v, P.vs, P.Tk, P.Hk, P.D, P.type))
    return cudaErrorInvalidValue;
  const int64_t pairs = (int64_t)((P.Tq + 2 * kRows - 1) / (2 * kRows)) * P.Hq;
  // Heads of up to 64 channels: a tile a CTA and two CTAs an SM, whose softmax fall into turns by themselves (4 x 4101
  // tokens, 16 heads of 64: 446 us; 492 with two tiles in one CTA, which ran in step, when one a CTA took 437). Wider heads have room for
  // one CTA, with two tiles that share the loads of K and V unless that would leave SMs without work (heads of 128, one tile a
  // CTA against two: 38 and 41 us at 64 pairs, 72 and 44 at 128, 104 and 80 at 160, 248 and 147 at 256).
  if constexpr (DP == 128) if (pairs >= 148)
    return launch(packed_fwd_tc_kernel<T, DP, 2>, pairs, FwdLayout<DP, 2>::kThreads, FwdLayout<DP, 2>::kBytes, stream, q,
                  k, v, P, (T*)o, lse, err);
  return launch(packed_fwd_tc_kernel<T, DP, 1>, (int64_t)((P.Tq + kRows - 1) / kRows) * P.Hq, FwdLayout<DP, 1>::kThreads,
                FwdLayout<DP, 1>::kBytes, stream, q, k, v, P, (T*)o, lse, err);
}

template <typename T, int DP>
cudaError_t bwd(const PackedProblem& P, const void* o, const void* dout, HeadRows ds, const float* lse, float* delta,
                void* channels, float* norms, void* dq, void* dk, void* dv, int* err, cudaStream_t stream) {
  CUtensorMap q, k, v, g;
  const cudaError_t ready = context_current();
  if (ready != cudaSuccess) return ready;
  if (!map_rows(&q, P.q, P.qs, P.Tq, P.Hq, P.D, P.type) || !map_rows(&k, P.k, P.ks, P.Tk, P.Hk, P.D, P.type) ||
      !map_rows(&v, P.v, P.vs, P.Tk, P.Hk, P.D, P.type) || !map_rows(&g, dout, ds, P.Tq, P.Hq, P.D, P.type))
    return cudaErrorInvalidValue;
  const int64_t q_tiles = ((int64_t)P.Tq + kRows - 1) / kRows, k_tiles = ((int64_t)P.Tk + kRows - 1) / kRows;
  if (q_tiles * P.Hq > 0x7fffffff) return cudaErrorInvalidConfiguration;
  packed_delta_tc_kernel<T><<<(unsigned)(q_tiles * P.Hq), 256, 0, stream>>>(
      (const T*)o, (const T*)P.o_low, (const T*)dout, ds, P.Tq, P.Hq, P.D, P.lse_stride, lse, 1.f / (P.scale * kLog2e), delta,
      (uint4*)channels, norms);
  cudaError_t status = cudaGetLastError();
  if (status != cudaSuccess) return status;
  status = launch(packed_dq_tc_kernel<T, DP>, q_tiles * P.Hq, kBwdThreads, DqLayout<DP>::kBytes, stream, q, k, v, g, P,
                  (const T*)dout, ds, lse, (const float*)delta, (const float*)norms, (T*)dq, err);
  if (status != cudaSuccess) return status;
  return launch(packed_dkv_tc_kernel<T, DP>, k_tiles * P.Hk, kBwdThreads, DkvLayout<DP>::kBytes, stream, q, k, v, g, P,
                (const T*)dout, ds, lse, (const float*)delta, (const uint4*)channels, (const float*)norms, (T*)dk, (T*)dv, err);
}

}  // namespace

// A positive scale (the running maximum is taken before it) that the statistics can be divided by, 16-bit values and up
// to 128 channels.
bool packed_tc_ok(const PackedProblem& P) {
  return (P.type == kSeqBf16 || P.type == kSeqF16) && P.scale > 1e-12f && P.D <= 128;
}

cudaError_t packed_fwd_tc(const PackedProblem& P, void* o, float* lse, int* err, cudaStream_t stream) {
  if (P.type == kSeqBf16)
    return P.D <= 64 ? fwd<__nv_bfloat16, 64>(P, o, lse, err, stream) : fwd<__nv_bfloat16, 128>(P, o, lse, err, stream);
  return P.D <= 64 ? fwd<__half, 64>(P, o, lse, err, stream) : fwd<__half, 128>(P, o, lse, err, stream);
}

cudaError_t packed_bwd_tc(const PackedProblem& P, const void* o, const void* dout, HeadRows ds, const float* lse,
                          float* delta, void* channels, float* norms, void* dq, void* dk, void* dv, int* err,
                          cudaStream_t stream) {
  if (P.type == kSeqBf16)
    return P.D <= 64 ? bwd<__nv_bfloat16, 64>(P, o, dout, ds, lse, delta, channels, norms, dq, dk, dv, err, stream)
                     : bwd<__nv_bfloat16, 128>(P, o, dout, ds, lse, delta, channels, norms, dq, dk, dv, err, stream);
  return P.D <= 64 ? bwd<__half, 64>(P, o, dout, ds, lse, delta, channels, norms, dq, dk, dv, err, stream)
                   : bwd<__half, 128>(P, o, dout, ds, lse, delta, channels, norms, dq, dk, dv, err, stream);
}

}  // namespace mia
