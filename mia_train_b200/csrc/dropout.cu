// Dropout from a counter-based generator, added to an optional residual; no mask is stored.
//
//   y[i] = residual[i] + (h(i) >= dropped ? x[i] * scale : 0)
//   dropped = round(65536 p),  scale = 65536 / (65536 - dropped)
//
// h(i) is a 16-bit half of a word of Philox4x32-10 (J. Salmon, M. Moraes, R. Dror, D. Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011): elements 8 g .. 8 g + 7 take the eight
// halves, low half first, of the four words for the counter (g, offset with its top bit set) under
// the key `seed`. The mask depends on (seed, offset, i) alone, so backward applies the same kernel
// to dy. 16 bits per decision give p in steps of 1 / 65536 (the scale uses the stepped p, so the
// mean is kept exactly) and halve the generator's cost: ten rounds for eight elements.
// Bound by HBM: x, the residual and y once each. One group of eight a thread, 16-byte loads; the ten rounds
// (two wide products and two three-input logic operations each) hide behind them. Measured: 16384 x 5120 bf16
// with a residual, forward and backward, 164 us for 839 MB (5.1 TB/s); 2048 x 4096 without one 22 us, most of
// it launches and the ramp of two short kernels.
// The offset's top bit keeps these counters apart from those of PyTorch's own kernels, whose upper
// words hold a thread index.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGeneratorImpl.h>
#include <ATen/cuda/PhiloxUtils.cuh>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <mutex>

#include "block_ops.h"
#include "common.cuh"
#include "vec8.cuh"

namespace mia {

struct DropRng {
  const int64_t* given;       // (seed, offset), or nullptr: take `state`
  int64_t* record;            // where the pair is written for the backward pass, or nullptr
  at::PhiloxCudaState state;  // PyTorch's generator; resolved on the device so that a captured graph draws anew
  uint64_t rank_key;          // mixed into a drawn seed
};

__device__ __forceinline__ uint4 philox4x32_10(uint64_t group, uint64_t seed, uint64_t offset) {
  uint4 c = make_uint4((uint32_t)group, (uint32_t)(group >> 32), (uint32_t)offset,
                       (uint32_t)(offset >> 32) | 0x80000000u);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c.x * 0xD2511F53u;
    const uint64_t b = (uint64_t)c.z * 0xCD9E8D57u;
    c = make_uint4((uint32_t)(b >> 32) ^ c.y ^ k0, (uint32_t)b, (uint32_t)(a >> 32) ^ c.w ^ k1, (uint32_t)a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}

template <typename T, bool RES, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                                                      T* __restrict__ y, int64_t n, uint32_t dropped, float scale,
                                                      DropRng rng) {
  uint64_t seed, offset;
  if (rng.given != nullptr) {
    seed = (uint64_t)rng.given[0];
    offset = (uint64_t)rng.given[1];
  } else {
    const auto so = at::cuda::philox::unpack(rng.state);
    seed = std::get<0>(so) ^ rng.rank_key;
    offset = std::get<1>(so);
  }
  if (rng.record != nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
    rng.record[0] = (int64_t)seed;
    rng.record[1] = (int64_t)offset;
  }
  const int64_t g = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t i = 8 * g;
  if (i >= n) return;
  const bool full = VEC && i + 8 <= n;
  float v[8], r[8];
  if (full) {
    const Raw8<T> xr = load_raw8(x + i);
    if (RES) unpack8(load_raw8(residual + i), r);
    unpack8(xr, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = i + j < n ? to_f32(x[i + j]) : 0.f;
      if (RES) r[j] = i + j < n ? to_f32(residual[i + j]) : 0.f;
    }
  }
  const uint4 w = philox4x32_10((uint64_t)g, seed, offset);
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t h = (j & 1) ? words[j / 2] >> 16 : words[j / 2] & 0xFFFFu;
    // a select, not a product: a dropped infinity or NaN leaves nothing behind
    const float kept = h >= dropped ? v[j] * scale : 0.f;
    v[j] = RES ? r[j] + kept : kept;
  }
  if (full) {
    store8(y + i, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) y[i + j] = from_f32<T>(v[j]);
  }
}

template <typename T>
static void launch_dropout(const torch::Tensor& x, const c10::optional<torch::Tensor>& residual, torch::Tensor& y,
                           uint32_t dropped, float scale, const DropRng& rng, cudaStream_t stream) {
  const int64_t n = x.numel();
  const T* xp = reinterpret_cast<const T*>(x.data_ptr());
  const T* rp = residual.has_value() ? reinterpret_cast<const T*>(residual->data_ptr()) : nullptr;
  T* yp = reinterpret_cast<T*>(y.data_ptr());
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const bool vec = aligned(xp) && aligned(yp) && (rp == nullptr || aligned(rp));
  const int64_t blocks = (n + 8 * 256 - 1) / (8 * 256);
  TORCH_CHECK(blocks <= INT32_MAX, "dropout: too many elements");
  auto run = [&](auto res, auto v) {
    dropout_kernel<T, decltype(res)::value, decltype(v)::value>
        <<<(unsigned)blocks, 256, 0, stream>>>(xp, rp, yp, n, dropped, scale, rng);
  };
  if (rp != nullptr) vec ? run(std::true_type{}, std::true_type{}) : run(std::true_type{}, std::false_type{});
  else vec ? run(std::false_type{}, std::true_type{}) : run(std::false_type{}, std::false_type{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// y = residual + dropout(x). `rng` holds (seed, offset); without it the pair is drawn from PyTorch's
// CUDA generator of that device, the seed taken apart by `rank_key` (ranks seed their generators alike). `record` receives
// the pair that was used: the caller may advance its own tensor before the backward pass.
void dropout_launch(torch::Tensor x, c10::optional<torch::Tensor> residual, torch::Tensor y, int64_t dropped,
                    c10::optional<torch::Tensor> rng, c10::optional<torch::Tensor> record, int64_t rank_key) {
  TORCH_CHECK(x.is_cuda() && x.is_contiguous() && y.is_contiguous(), "dropout: contiguous CUDA tensors expected");
  TORCH_CHECK(y.device() == x.device() && y.scalar_type() == x.scalar_type() && y.numel() == x.numel(),
              "dropout: output must match the input");
  if (residual.has_value())
    TORCH_CHECK(residual->device() == x.device() && residual->scalar_type() == x.scalar_type() &&
                    residual->is_contiguous() && residual->numel() == x.numel(),
                "dropout: residual must match the input");
  auto check_pair = [&](const torch::Tensor& t) {
    TORCH_CHECK(t.device() == x.device() && t.scalar_type() == at::kLong && t.is_contiguous() && t.numel() == 2,
                "dropout: (seed, offset) must be a contiguous int64 pair on the input's device");
  };
  TORCH_CHECK(dropped >= 0 && dropped <= 65536, "dropout: dropped must be within 0..65536");
  c10::cuda::CUDAGuard guard(x.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  DropRng r{};
  if (rng.has_value()) {
    check_pair(*rng);
    r.given = rng->data_ptr<int64_t>();
  } else {
    auto gen = at::get_generator_or_default<at::CUDAGeneratorImpl>(
        c10::nullopt, at::cuda::detail::getDefaultCUDAGenerator(x.get_device()));
    std::lock_guard<std::mutex> lock(gen->mutex_);
    r.state = gen->philox_cuda_state(4);
    r.rank_key = (uint64_t)rank_key;
  }
  if (record.has_value()) {
    check_pair(*record);
    r.record = record->data_ptr<int64_t>();
  }
  if (x.numel() == 0) {
    if (record.has_value()) record->zero_();
    return;
  }
  const float scale = dropped == 65536 ? 0.f : (float)(65536.0 / (double)(65536 - dropped));
  if (x.scalar_type() == at::kBFloat16) launch_dropout<__nv_bfloat16>(x, residual, y, (uint32_t)dropped, scale, r, stream);
  else if (x.scalar_type() == at::kHalf) launch_dropout<__half>(x, residual, y, (uint32_t)dropped, scale, r, stream);
  else if (x.scalar_type() == at::kFloat) launch_dropout<float>(x, residual, y, (uint32_t)dropped, scale, r, stream);
  else TORCH_CHECK(false, "dropout: bf16, fp16 or fp32 expected");
}

void dropout_apply(torch::Tensor x, c10::optional<torch::Tensor> residual, torch::Tensor y, int64_t dropped,
                   c10::optional<torch::Tensor> rng, c10::optional<torch::Tensor> record) {
  dropout_launch(x, residual, y, dropped, rng, record, 0);
}

}  // namespace mia
