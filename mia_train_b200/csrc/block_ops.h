// Launchers of the dropout, query/key norm and 8-bit kernels, shared by their autograd nodes (block_ops.cpp).
#pragma once

#include <torch/extension.h>

namespace mia {

using OptTensor = c10::optional<at::Tensor>;

void dropout_launch(at::Tensor x, OptTensor residual, at::Tensor y, int64_t dropped, OptTensor rng, OptTensor record,
                    int64_t rank_key);
void dropout_apply(at::Tensor x, OptTensor residual, at::Tensor y, int64_t dropped, OptTensor rng, OptTensor record);
void qk_norm_fwd(at::Tensor q, at::Tensor k, OptTensor qw, OptTensor kw, OptTensor angles, at::Tensor pairs,
                 at::Tensor yq, at::Tensor yk, double eps);
void qk_norm_bwd(at::Tensor dyq, at::Tensor dyk, at::Tensor q, at::Tensor k, OptTensor qw, OptTensor kw,
                 OptTensor angles, at::Tensor pairs, at::Tensor dq, at::Tensor dk, OptTensor dqw, OptTensor dkw,
                 int64_t accumulate, OptTensor dangles, double eps);
void fp8_quantize(at::Tensor x, OptTensor aux, OptTensor gamma, bool block, bool e5m2, OptTensor q, OptTensor q_scale,
                  OptTensor qt, OptTensor qt_scale, OptTensor sums, bool accumulate);
void fp8_gemm(at::Tensor a, at::Tensor a_scale, bool a_block, at::Tensor b, at::Tensor b_scale, bool b_block, int64_t k,
              at::Tensor d, OptTensor bias, OptTensor residual, OptTensor gamma, OptTensor aux_out, int64_t act,
              bool accumulate);

}  // namespace mia
