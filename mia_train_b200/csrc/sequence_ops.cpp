// Autograd nodes of packed attention, rotation by positions and distillation from top logits, in C++ for the reason
// that block_ops.cpp gives: small calls are bound by the host.
//
// Every backward pass is differentiable once: with create_graph it refuses to run where its result depends on
// anything that wants a gradient, the incoming gradient or an operand.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>

#include "block_ops.h"
#include "errors.h"
#include "sequence_kernels.h"

namespace mia {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

using BelowAutograd = at::AutoDispatchBelowADInplaceOrView;

void once_differentiable(const at::Tensor& grad, bool open, const char* what) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && (open || (grad.defined() && grad.requires_grad()))), what,
              ": the backward pass is differentiable once only");
}

// `x` itself when its rows of channels can be read 16 bytes at a time, else a contiguous copy.
at::Tensor heads(const at::Tensor& x) {
  const int64_t e = 16 / x.element_size(), last = x.dim() - 1;
  bool ok = x.stride(last) == 1 && (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0;
  for (int i = 0; i < last && ok; ++i) ok = (x.stride(i) > 0 && x.stride(i) % e == 0) || x.size(i) <= 1;
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

at::Tensor value(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

SequenceType type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return kSeqBf16;
    case at::kHalf: return kSeqF16;
    case at::kFloat: return kSeqF32;
    default: return kSeqF64;
  }
}

// ------------------------------------------------------------------------------- packed attention

HeadRows rows_of(const at::Tensor& x) { return {x.stride(0), x.stride(1)}; }

PackedProblem problem(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_bounds,
                      const at::Tensor& k_bounds, double scale) {
  PackedProblem P;
  P.q = q.data_ptr();
  P.k = k.data_ptr();
  P.v = v.data_ptr();
  P.qs = rows_of(q);
  P.ks = rows_of(k);
  P.vs = rows_of(v);
  P.q_bounds = reinterpret_cast<const int2*>(q_bounds.data_ptr<int>());
  P.k_bounds = reinterpret_cast<const int2*>(k_bounds.data_ptr<int>());
  P.Tq = (int)q_bounds.size(0);
  P.Tk = (int)k_bounds.size(0);
  P.Hq = (int)q.size(1);
  P.Hk = (int)k.size(1);
  P.group = P.Hq / P.Hk;
  P.D = (int)q.size(2);
  P.lse_stride = (P.Tq + 127) / 128 * 128;
  P.scale = (float)scale;
  P.type = type_of(q);
  P.o_low = nullptr;
  return P;
}

// The bounds belong to the caller's plan, which may have been made on another stream and may go before its launches end.
void keep_for(const at::Tensor& t, const c10::cuda::CUDAStream& stream) {
  if (t.numel()) c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), stream);
}

// Whether few queries over many keys go piece by piece. Tiles compute `tile_pairs` scores a head at some 2.2e6 a
// microsecond on all 148 SMs (4 x 4101 tokens, 16 heads of 64: 1.08e9 in 453 us, a little less behind masks); the pieces read K and V once for up to
// four rows at some 4.2e6 bytes a microsecond, behind 12 us of two launches and their tails.
bool few_is_faster(const PackedProblem& P, int64_t max_queries, int64_t tile_pairs, int64_t pairs) {
  const int64_t rows = max_queries * P.group;
  if (rows > 65535 || P.Hk > 65535) return false;
  const double share = (double)std::min<int64_t>(rows, 4);  // rows that one reading of K and V serves
  const int width = P.type == kSeqF32 ? 8 : 4;               // bytes of K and V per channel
  const double few = 12.0 + (double)pairs * P.Hq / share * width * P.D / 4.2e6;
  const double ctas = (double)((P.Tq + 127) / 128) * P.Hq;
  const double tiles = 6.0 + (double)tile_pairs * P.Hq / 2.2e6 * std::max(1.0, 148.0 / ctas);
  return few < tiles;
}

// An output whose rows behind the sequences are zeros.
at::Tensor rows_out(const at::Tensor& like, int64_t used) {
  at::Tensor out = at::empty(like.sizes(), like.options());
  if (used < out.size(0)) out.narrow(0, used, out.size(0) - used).zero_();
  return out;
}

struct PackedAttentionNode : Function<PackedAttentionNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& q_bounds, const at::Tensor& k_bounds, double scale,
                            const OptTensor& items, const OptTensor& pieces, int64_t max_queries, int64_t tile_pairs,
                            int64_t pairs, bool grad) {
    BelowAutograd below;
    const at::Tensor qc = heads(q), kc = heads(k), vc = heads(v);
    const int64_t used = q_bounds.size(0);
    at::Tensor o = rows_out(q, used);
    at::Tensor lse = at::empty({q.size(1), (used + 127) / 128 * 128}, q.options().dtype(at::kFloat));
    const c10::cuda::CUDAGuard guard(q.device());
    const auto stream = at::cuda::getCurrentCUDAStream();
    keep_for(q_bounds, stream);
    PackedProblem P = problem(qc, kc, vc, q_bounds, k_bounds, scale);
    at::Tensor low;
    if (grad && P.type != kSeqF32) low = at::empty(o.sizes(), o.options());
    P.o_low = low.defined() ? low.data_ptr() : nullptr;
    if (P.Tk == 0) {  // nobody sees anything
      o.zero_();
      lse.fill_(INFINITY);
      if (low.defined()) low.zero_();
    } else if (used > 0 && items.has_value() && few_is_faster(P, max_queries, tile_pairs, pairs)) {
      PackedFew few;
      few.items = reinterpret_cast<const int4*>(items->data_ptr<int>());
      few.pieces = reinterpret_cast<const int2*>(pieces->data_ptr<int>());
      few.count = (int)items->size(0);
      few.sequences = (int)pieces->size(0);
      few.rows = (int)max_queries * P.group;
      keep_for(*items, stream);
      keep_for(*pieces, stream);
      at::Tensor partial;
      if (few.count > few.sequences)
        partial = at::empty({few.count, P.Hk, few.rows, P.D + 2}, lse.options());
      few.partial = partial.defined() ? partial.data_ptr<float>() : nullptr;
      C10_CUDA_CHECK(packed_fwd_few(P, few, o.data_ptr(), lse.data_ptr<float>(), stream));
    } else if (used > 0) {
      C10_CUDA_CHECK(packed_tc_ok(P) ? packed_fwd_tc(P, o.data_ptr(), lse.data_ptr<float>(),
                                                     error_word(q.get_device()), stream)
                                     : packed_fwd_rows(P, o.data_ptr(), lse.data_ptr<float>(), stream));
    }
    ctx->save_for_backward({qc, kc, vc, q_bounds, k_bounds, o, lse, low});
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_differentiable(grads[0], true, "packed_attention");
    const variable_list s = ctx->get_saved_variables();
    BelowAutograd below;
    const at::Tensor dout = heads(grads[0]);
    at::Tensor dq = rows_out(s[0], s[3].size(0)), dk = rows_out(s[1], s[4].size(0)), dv = rows_out(s[2], s[4].size(0));
    at::Tensor delta = at::empty_like(s[6]);
    const c10::cuda::CUDAGuard guard(dout.device());
    const auto stream = at::cuda::getCurrentCUDAStream();
    keep_for(s[3], stream);
    keep_for(s[4], stream);
    PackedProblem P = problem(s[0], s[1], s[2], s[3], s[4], ctx->saved_data["scale"].toDouble());
    P.o_low = s[7].defined() ? s[7].data_ptr() : nullptr;
    const float* lse = s[6].data_ptr<float>();
    if (P.Tq == 0 || P.Tk == 0) {
      for (at::Tensor* x : {&dq, &dk, &dv}) x->zero_();
    } else if (packed_tc_ok(P)) {
      at::Tensor norms = at::empty({P.type == kSeqF16 ? s[6].numel() / 128 * 129 : 0}, s[6].options());
      at::Tensor channels = at::empty({2 * s[6].numel() * 8}, s[0].options());
      C10_CUDA_CHECK(packed_bwd_tc(P, s[5].data_ptr(), dout.data_ptr(), rows_of(dout), lse, delta.data_ptr<float>(),
                                   channels.data_ptr(), norms.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                   error_word(dout.get_device()), stream));
    } else {
      C10_CUDA_CHECK(packed_bwd_rows(P, s[5].data_ptr(), dout.data_ptr(), rows_of(dout), lse, delta.data_ptr<float>(),
                                     dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), stream));
    }
    return {dq, dk, dv, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor(), at::Tensor()};
  }
};

// --------------------------------------------------------------------------------------- rotation

TokenRows token_rows(const at::Tensor& x) { return {x.stride(0), x.stride(1), x.stride(2)}; }

bool in_vectors(const at::Tensor& x) {
  bool ok = (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (x.stride(i) % 8 == 0 || x.size(i) <= 1);
  return ok || x.size(2) == 0;
}

// q, k (B, T, H, D) -> yq, yk; `inverse` turns back. With xq and xk (the forward pass's inputs, where q and k are
// gradients) also dfreq (axes, P) fp32. k may have no heads.
void rotate(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions, const OptTensor& freq,
            bool interleaved, double amplitude, bool inverse, const at::Tensor& yq, const at::Tensor& yk,
            const OptTensor& xq, const OptTensor& xk, const OptTensor& dfreq) {
  const bool learn = dfreq.has_value();
  RotaryParams p;
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.yq = yq.data_ptr();
  p.yk = yk.data_ptr();
  p.xq = learn ? xq->data_ptr() : nullptr;
  p.xk = learn ? xk->data_ptr() : nullptr;
  p.qs = token_rows(q);
  p.ks = token_rows(k);
  p.yqs = token_rows(yq);
  p.yks = token_rows(yk);
  p.xqs = learn ? token_rows(*xq) : p.qs;
  p.xks = learn ? token_rows(*xk) : p.ks;
  p.pos = positions.data_ptr();
  const at::ScalarType pt = positions.scalar_type();
  p.pos_type = pt == at::kLong ? 0 : pt == at::kInt ? 1 : pt == at::kFloat ? 2 : 3;
  p.pos_b = positions.size(0) == 1 ? 0 : 1;
  p.freq = freq.has_value() ? freq->data_ptr() : nullptr;
  p.freq64 = freq.has_value() && freq->scalar_type() == at::kDouble;
  p.axes = freq.has_value() ? (int)freq->size(0) : 1;
  p.P = (int)positions.size(2);
  if (freq.has_value()) p.P = (int)freq->size(1);
  p.D = (int)q.size(3);
  p.T = (int)q.size(1);
  p.Hq = (int)q.size(2);
  p.Hk = (int)k.size(2);
  p.tokens = q.size(0) * q.size(1);
  p.amplitude = (float)amplitude;
  p.inverse = inverse;
  p.partial = nullptr;
  if (p.tokens == 0 || p.Hq + p.Hk == 0 || p.D == 0) {
    if (learn) dfreq->zero_();
    return;
  }
  const c10::cuda::CUDAGuard guard(q.device());
  const auto stream = at::cuda::getCurrentCUDAStream();
  const bool aligned = in_vectors(q) && in_vectors(k) && in_vectors(yq) && in_vectors(yk) &&
                       (!learn || (in_vectors(*xq) && in_vectors(*xk)));
  const RotaryPlan plan = rotary_plan(p, aligned, interleaved, learn);
  at::Tensor partial;
  if (learn) {
    partial = at::empty({(int64_t)plan.grid * plan.chunks, p.axes, p.P}, q.options().dtype(at::kFloat));
    p.partial = partial.data_ptr<float>();
  }
  C10_CUDA_CHECK(rotary_launch(p, plan, type_of(q), interleaved, learn ? dfreq->data_ptr<float>() : nullptr, stream));
}

struct RotaryNode : Function<RotaryNode> {
  // q, k (B, T, H, D); positions (1 or B, T, axes) and freq (axes, P), or angles (1 or B, T, P) alone
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                               const OptTensor& freq, bool interleaved, double amplitude) {
    BelowAutograd below;
    const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), Hk = k.size(2), D = q.size(3);
    const at::Tensor qc = heads(q), kc = heads(k), pos = positions.contiguous();
    const OptTensor f = freq.has_value() ? OptTensor(freq->contiguous()) : OptTensor();
    at::Tensor out = at::empty({B, T, Hq + Hk, D}, q.options());
    at::Tensor yq = out.narrow(2, 0, Hq), yk = out.narrow(2, Hq, Hk);
    rotate(qc, kc, pos, f, interleaved, amplitude, false, yq, yk, {}, {}, {});
    const bool learn = freq.has_value() && freq->requires_grad();
    ctx->save_for_backward({pos, value(f), learn ? qc : at::Tensor(), learn ? kc : at::Tensor()});
    auto& d = ctx->saved_data;
    d["interleaved"] = interleaved;
    d["amplitude"] = amplitude;
    d["learn"] = learn;
    d["q_heads"] = Hq;
    d["k_heads"] = Hk;
    // the rotation is linear in q and k: their gradients depend on the frequencies alone, those of the frequencies on
    // q, k and the frequencies
    d["open"] = learn;
    return {yq, yk};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    auto& d = ctx->saved_data;
    for (const at::Tensor& g : grads) once_differentiable(g, d["open"].toBool(), "rotary");
    const variable_list s = ctx->get_saved_variables();
    BelowAutograd below;
    const at::Tensor& one = grads[0].defined() ? grads[0] : grads[1];
    const int64_t B = one.size(0), T = one.size(1), D = one.size(3), Hk = d["k_heads"].toInt();
    const int64_t Hq = d["q_heads"].toInt();
    const at::Tensor gq = grads[0].defined() ? heads(grads[0]) : at::zeros({B, T, Hq, D}, one.options());
    const at::Tensor gk = grads[1].defined() ? heads(grads[1]) : at::zeros({B, T, Hk, D}, one.options());
    at::Tensor out = at::empty({B, T, Hq + Hk, D}, one.options());
    at::Tensor dq = out.narrow(2, 0, Hq), dk = out.narrow(2, Hq, Hk);
    OptTensor xq, xk, df;
    if (d["learn"].toBool()) {
      xq = s[2];
      xk = s[3];
      df = at::empty(s[1].sizes(), one.options().dtype(at::kFloat));
    }
    rotate(gq, gk, s[0], opt(s[1]), d["interleaved"].toBool(), d["amplitude"].toDouble(), true, dq, dk, xq, xk, df);
    at::Tensor dfreq;
    if (df.has_value()) dfreq = df->to(s[1].scalar_type());
    return {dq, dk, at::Tensor(), dfreq, at::Tensor(), at::Tensor()};
  }
};

// ----------------------------------------------------------------------------------- distillation

DistillParams distill_params(const at::Tensor& s, const at::Tensor& values, const at::Tensor& indices,
                             const OptTensor& lse, const OptTensor& weights, double tau, double teacher_tau, double norm,
                             const at::Tensor& stats) {
  DistillParams p;
  p.s = s.data_ptr();
  p.s_row = s.stride(0);
  p.values = values.data_ptr();
  p.indices = indices.data_ptr();
  p.lse = lse.has_value() ? lse->data_ptr() : nullptr;
  p.weights = weights.has_value() ? weights->data_ptr() : nullptr;
  p.lse64 = lse.has_value() && lse->scalar_type() == at::kDouble;
  p.weights64 = weights.has_value() && weights->scalar_type() == at::kDouble;
  p.type = type_of(s);
  p.value_type = type_of(values);
  p.index64 = indices.scalar_type() == at::kLong;
  p.R = (int)s.size(0);
  p.V = (int)s.size(1);
  p.K = (int)values.size(1);
  p.tau = tau;
  p.teacher_tau = teacher_tau;
  p.norm = norm;
  p.stats = stats.data_ptr<double>();
  return p;
}

// A number per row in fp32, or in fp64 if it came so: the rest of 1 is a difference of what the lse gives.
OptTensor row_numbers(const OptTensor& x) {
  if (!x.has_value()) return x;
  return x->scalar_type() == at::kDouble ? x->contiguous() : x->to(at::kFloat).contiguous();
}

struct DistillNode : Function<DistillNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& student, const at::Tensor& values,
                            const at::Tensor& indices, const OptTensor& teacher_lse, const OptTensor& weights, double tau,
                            double teacher_tau, double norm) {
    BelowAutograd below;
    const at::Tensor s = student.stride(1) == 1 || student.size(1) <= 1 ? student : student.contiguous();
    const at::Tensor t = values.contiguous(), at_ = indices.contiguous();
    const OptTensor lse = row_numbers(teacher_lse), w = row_numbers(weights);
    at::Tensor stats = at::empty({s.size(0), 8}, s.options().dtype(at::kDouble));
    at::Tensor loss = at::empty({}, s.options().dtype(at::kFloat));
    at::Tensor rows = at::empty({s.size(0)}, stats.options());
    const c10::cuda::CUDAGuard guard(s.device());
    C10_CUDA_CHECK(distill_fwd(distill_params(s, t, at_, lse, w, tau, teacher_tau, norm, stats), rows.data_ptr<double>(),
                               loss.data_ptr<float>(), at::cuda::getCurrentCUDAStream()));
    ctx->save_for_backward({s, t, at_, value(w), stats});
    auto& d = ctx->saved_data;
    d["tau"] = tau;
    d["teacher_tau"] = teacher_tau;
    d["norm"] = norm;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_differentiable(grads[0], true, "top_logit_distillation");
    const variable_list s = ctx->get_saved_variables();
    BelowAutograd below;
    auto& d = ctx->saved_data;
    at::Tensor ds = at::empty(s[0].sizes(), s[0].options());
    const at::Tensor g = grads[0].to(at::kFloat).contiguous();
    const c10::cuda::CUDAGuard guard(ds.device());
    if (ds.numel() > 0)
      C10_CUDA_CHECK(distill_bwd(distill_params(s[0], s[1], s[2], {}, opt(s[3]), d["tau"].toDouble(),
                                                d["teacher_tau"].toDouble(), d["norm"].toDouble(), s[4]),
                                 g.data_ptr<float>(), ds.data_ptr(), at::cuda::getCurrentCUDAStream()));
    return {ds, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace

at::Tensor packed_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_bounds,
                            const at::Tensor& k_bounds, double scale, const OptTensor& items, const OptTensor& pieces,
                            int64_t max_queries, int64_t tile_pairs, int64_t pairs) {
  return PackedAttentionNode::apply(q, k, v, q_bounds, k_bounds, scale, items, pieces, max_queries, tile_pairs, pairs,
                                    at::GradMode::is_enabled() &&
                                        (q.requires_grad() || k.requires_grad() || v.requires_grad()));
}

std::tuple<at::Tensor, at::Tensor> rotary(const at::Tensor& q, const at::Tensor& k, const at::Tensor& positions,
                                          const OptTensor& freq, bool interleaved, double amplitude) {
  variable_list out = RotaryNode::apply(q, k, positions, freq, interleaved, amplitude);
  return {out[0], out[1]};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> top_logits(const at::Tensor& x, int64_t k, double tau) {
  at::NoGradGuard no_grad;
  BelowAutograd below;
  const at::Tensor c = x.stride(1) == 1 || x.size(1) <= 1 ? x : x.contiguous();
  at::Tensor values = at::empty({x.size(0), k}, x.options()), indices = at::empty({x.size(0), k}, x.options().dtype(at::kLong));
  at::Tensor lse = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
  const c10::cuda::CUDAGuard guard(x.device());
  if (x.size(0) > 0)
    C10_CUDA_CHECK(top_logits_rows(c.data_ptr(), c.stride(0), (int)x.size(0), (int)x.size(1), (int)k, tau,
                                   values.data_ptr(), indices.data_ptr<int64_t>(), lse.data_ptr<float>(), type_of(x),
                                   at::cuda::getCurrentCUDAStream()));
  return {values, indices, lse};
}

at::Tensor top_logit_distillation(const at::Tensor& s, const at::Tensor& values, const at::Tensor& indices,
                                  const OptTensor& teacher_lse, const OptTensor& weights, double tau,
                                  double teacher_tau, double norm) {
  return DistillNode::apply(s, values, indices, teacher_lse, weights, tau, teacher_tau, norm);
}

}  // namespace mia
