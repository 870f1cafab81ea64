// Autograd nodes of dropout, the query/key norm with rotation and the 8-bit linear layer. They are C++ because
// small calls are bound by the host: a Python autograd.Function costs 40 to 100 us for forward and backward, more
// than these kernels run for below some ten million elements.
//
// Every backward pass is differentiable once: with create_graph it refuses to run where its result depends on
// anything that wants a gradient, the incoming gradient or an operand.
#include <ATen/ATen.h>
#include <torch/extension.h>

#include "block_ops.h"

namespace mia {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

namespace {

// Inside a node nothing is recorded: views, copies and allocations go past the autograd dispatch keys. In a backward
// pass only once the saved variables are there: fetching them may run a checkpointed forward pass again.
using BelowAutograd = at::AutoDispatchBelowADInplaceOrView;

at::Tensor value(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor opt(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
bool wants(const OptTensor& t) { return t.has_value() && t->defined() && t->requires_grad(); }

// `open`: whether the gradients depend on an operand that itself wants a gradient. Without create_graph nothing is
// missed; with it, even a constant incoming gradient would leave the result without the graph it should have.
void once_differentiable(const at::Tensor& grad, bool open, const char* what) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && (open || (grad.defined() && grad.requires_grad()))), what,
              ": the backward pass is differentiable once only");
}

// A parameter's `main_grad`. Not a saved variable: it is written between forward and backward (cleared, or added to
// by other layers), which saved variables may not be.
void keep_sink(AutogradContext* ctx, const char* name, const OptTensor& sink) {
  if (sink.has_value()) ctx->saved_data[name] = *sink;
}
at::Tensor kept_sink(AutogradContext* ctx, const char* name) {
  const auto it = ctx->saved_data.find(name);
  return it == ctx->saved_data.end() ? at::Tensor() : it->second.toTensor();
}

bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

at::Tensor aligned(const at::Tensor& t) {
  at::Tensor c = t.contiguous();
  return aligned16(c) ? c : c.clone(at::MemoryFormat::Contiguous);
}

// ---------------------------------------------------------------------------------------- dropout

struct DropoutNode : Function<DropoutNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& residual, int64_t dropped,
                            const OptTensor& rng, int64_t rank_key) {
    BelowAutograd below;
    const at::Tensor xc = x.contiguous();
    const OptTensor res = residual.has_value() ? OptTensor(residual->contiguous()) : OptTensor();
    at::Tensor used = at::empty({2}, x.options().dtype(at::kLong));
    at::Tensor y = at::empty_like(xc);
    dropout_launch(xc, res, y, dropped, rng.has_value() ? OptTensor(rng->contiguous()) : OptTensor(), used, rank_key);
    ctx->save_for_backward({used});
    ctx->saved_data["dropped"] = dropped;
    ctx->saved_data["need_x"] = x.requires_grad();
    ctx->saved_data["need_r"] = wants(residual);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor dy = grads[0];
    once_differentiable(dy, false, "dropout");  // linear in dy, and of x it knows only the place
    const at::Tensor used = ctx->get_saved_variables()[0];
    BelowAutograd below;
    at::Tensor dx;
    if (ctx->saved_data["need_x"].toBool()) {
      const at::Tensor dyc = dy.contiguous();
      dx = at::empty_like(dyc);
      dropout_apply(dyc, {}, dx, ctx->saved_data["dropped"].toInt(), used, {});
    }
    return {dx, ctx->saved_data["need_r"].toBool() ? dy : at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// ------------------------------------------------------------------- query / key norm with rotation

// `x` itself when its heads can be read 16 bytes at a time, else a contiguous copy.
at::Tensor heads(const at::Tensor& x) {
  const int64_t e = 16 / x.element_size();
  bool ok = x.stride(3) == 1 && aligned16(x);
  for (int i = 0; i < 3 && ok; ++i) ok = x.stride(i) % e == 0 || x.size(i) <= 1;
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

// fp32 values of an operand that is kept for the backward pass: the operand itself where nothing needs converting,
// never a detached alias. Below the autograd keys an alias has a version counter of its own, and a change of the
// operand between forward and backward would go unseen.
OptTensor fp32_values(const OptTensor& w) {
  return w.has_value() ? OptTensor(w->to(at::kFloat).contiguous()) : OptTensor();
}

struct QkNormNode : Function<QkNormNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const OptTensor& qw,
                               const OptTensor& kw, const OptTensor& angles, const OptTensor& pairs, double eps,
                               const OptTensor& q_sink, const OptTensor& k_sink) {
    BelowAutograd below;
    const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), D = q.size(3), Hk = k.size(2);
    const at::Tensor qc = heads(q), kc = heads(k);
    const OptTensor qf = fp32_values(qw), kf = fp32_values(kw);
    const bool rotate = angles.has_value() && pairs.has_value() && pairs->numel() > 0;
    const OptTensor ang = rotate ? fp32_values(angles) : OptTensor();
    const at::Tensor pr = rotate ? pairs->to(q.device(), at::kInt).contiguous()
                                 : at::empty({0, 2}, q.options().dtype(at::kInt));
    at::Tensor out = at::empty({B, T, Hq + Hk, D}, q.options());
    at::Tensor yq = out.narrow(2, 0, Hq), yk = out.narrow(2, Hq, Hk);
    qk_norm_fwd(qc, kc, qf, kf, ang, pr, yq, yk, eps);
    ctx->save_for_backward({qc, kc, value(qf), value(kf), value(ang), pr});
    keep_sink(ctx, "q_sink", q_sink);
    keep_sink(ctx, "k_sink", k_sink);
    ctx->saved_data["eps"] = eps;
    // each gradient depends on q, k and the angles; the weights' own are constant in the weights
    ctx->saved_data["open"] = q.requires_grad() || k.requires_grad() || (rotate && wants(angles));
    ctx->saved_data["need_qw"] = wants(qw);
    ctx->saved_data["need_kw"] = wants(kw);
    ctx->saved_data["need_angles"] = rotate && wants(angles);
    if (rotate) {
      ctx->saved_data["one_angle"] = angles->size(0) == 1;
      ctx->saved_data["angle_type"] = (int64_t)angles->scalar_type();
    }
    ctx->saved_data["qw_type"] = (int64_t)(qw.has_value() ? qw->scalar_type() : at::kFloat);
    ctx->saved_data["kw_type"] = (int64_t)(kw.has_value() ? kw->scalar_type() : at::kFloat);
    return {yq, yk};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool open = ctx->saved_data["open"].toBool();
    once_differentiable(grads[0], open, "qk_norm_rope");
    once_differentiable(grads[1], open, "qk_norm_rope");
    const variable_list saved = ctx->get_saved_variables();
    BelowAutograd below;
    const at::Tensor q = saved[0], k = saved[1], pairs = saved[5];
    const int64_t B = q.size(0), T = q.size(1), Hq = q.size(2), D = q.size(3), Hk = k.size(2);
    const at::Tensor dyq = grads[0].defined() ? heads(grads[0]) : at::zeros_like(q, at::MemoryFormat::Contiguous);
    const at::Tensor dyk = grads[1].defined() ? heads(grads[1]) : at::zeros_like(k, at::MemoryFormat::Contiguous);
    at::Tensor buf = at::empty({B, T, Hq + Hk, D}, q.options());
    at::Tensor dq = buf.narrow(2, 0, Hq), dk = buf.narrow(2, Hq, Hk);
    const char* need[2] = {"need_qw", "need_kw"};
    const char* type[2] = {"qw_type", "kw_type"};
    const at::Tensor sinks[2] = {kept_sink(ctx, "q_sink"), kept_sink(ctx, "k_sink")};
    OptTensor dw[2];
    int64_t accumulate = 0;
    for (int s = 0; s < 2; ++s) {
      if (!ctx->saved_data[need[s]].toBool()) continue;
      const at::Tensor sink = sinks[s];
      if (sink.defined()) accumulate |= 1 << s;
      dw[s] = sink.defined() ? sink.view({D}) : at::empty({D}, q.options().dtype(at::kFloat));
    }
    at::Tensor dangles;
    if (ctx->saved_data["need_angles"].toBool())
      dangles = at::empty({B, T, pairs.size(0)}, q.options().dtype(at::kFloat));
    qk_norm_bwd(dyq, dyk, q, k, opt(saved[2]), opt(saved[3]), opt(saved[4]), pairs, dq, dk, dw[0], dw[1], accumulate,
                opt(dangles), ctx->saved_data["eps"].toDouble());
    at::Tensor grad_w[2];
    for (int s = 0; s < 2; ++s)
      if (dw[s].has_value() && !(accumulate >> s & 1))
        grad_w[s] = dw[s]->to((at::ScalarType)ctx->saved_data[type[s]].toInt());
    if (dangles.defined()) {
      if (ctx->saved_data["one_angle"].toBool() && B != 1) dangles = dangles.sum(0, true);
      dangles = dangles.to((at::ScalarType)ctx->saved_data["angle_type"].toInt());
    }
    return {dq, dk, grad_w[0], grad_w[1], dangles, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// ------------------------------------------------------------------------------ 8-bit linear layer

constexpr int64_t kBlk = 128;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Q8 {
  at::Tensor data, scale;
  int64_t cols = 0;
};

Q8 empty_q8(int64_t rows, int64_t cols, bool block, const at::Tensor& like) {
  Q8 q;
  q.cols = cols;
  q.data = at::empty({rows, ceil_div(cols, 16) * 16}, like.options().dtype(at::kFloat8_e4m3fn));
  q.scale = at::empty({ceil_div(cols, kBlk), block ? ceil_div(rows, kBlk) : rows}, like.options().dtype(at::kFloat));
  return q;
}

void quantize_both(const at::Tensor& x, bool block, bool rows, bool cols, Q8& q, Q8& qt, const OptTensor& aux = {},
                   const OptTensor& gamma = {}, const OptTensor& sums = {}, bool accumulate = false) {
  if (rows) q = empty_q8(x.size(0), x.size(1), block, x);
  if (cols) qt = empty_q8(x.size(1), x.size(0), block, x);
  fp8_quantize(x, aux, gamma, block, false, opt(q.data), opt(q.scale), opt(qt.data), opt(qt.scale), sums, accumulate);
}

// A row-major (rows, cols) view of x, or a copy.
at::Tensor matrix(const at::Tensor& x, int64_t cols) {
  at::Tensor m = x.reshape({-1, cols});
  return m.stride(1) == 1 || cols == 1 ? m : m.contiguous();
}

OptTensor aligned_vector(const OptTensor& v) {  // not detached: see fp32_values
  return v.has_value() ? OptTensor(aligned(v->to(at::kFloat))) : OptTensor();
}

struct Fp8LinearNode : Function<Fp8LinearNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias,
                            const OptTensor& residual, const OptTensor& gamma, int64_t act, bool bf16,
                            const OptTensor& shadow, const OptTensor& w_sink, const OptTensor& b_sink, bool grad) {
    BelowAutograd below;
    const int64_t N = weight.size(0), K = weight.numel() / N;
    const at::ScalarType type = bf16 ? at::kBFloat16 : at::kFloat;
    const at::Tensor x2 = matrix(x, K);
    const at::Tensor w = matrix((shadow.has_value() ? *shadow : weight).detach(), K);
    // under no_grad nothing is kept for a backward pass
    const bool need_x = grad && x.requires_grad(), need_w = grad && weight.requires_grad();
    const bool need_b = grad && wants(bias), need_g = grad && wants(gamma);
    Q8 xq, xt, wq, wt;
    quantize_both(x2, false, true, need_w, xq, xt);
    quantize_both(w, true, true, need_x, wq, wt);
    const OptTensor g = aligned_vector(gamma), b = aligned_vector(bias);
    const int64_t M = x2.size(0);
    OptTensor res, pre;
    if (residual.has_value()) res = aligned(residual->detach().reshape({M, N}).to(type));
    // the pre-activation is read by the gradients of the product alone; without it the epilogue also stages one output less
    if (act != 0 && (need_x || need_w || need_b)) pre = at::empty({M, N}, x.options().dtype(type));
    at::Tensor y = at::empty({M, N}, x.options().dtype(type));
    fp8_gemm(xq.data, xq.scale, false, wq.data, wq.scale, true, K, y, b, res, g, pre, act, false);
    if (!need_g) xq = wq = Q8();
    // gamma scales the gradient of the product; the bias is in the activation that gamma's own gradient recomputes
    const at::Tensor kept_g = need_x || need_w || need_b ? value(g) : at::Tensor();
    const at::Tensor kept_b = need_g ? value(b) : at::Tensor();
    ctx->save_for_backward({value(pre), kept_g, kept_b, xt.data, xt.scale, wt.data, wt.scale, xq.data, xq.scale,
                            wq.data, wq.scale});
    keep_sink(ctx, "w_sink", w_sink);
    keep_sink(ctx, "b_sink", b_sink);
    auto& d = ctx->saved_data;
    d["act"] = act;
    // y is linear in x, weight, bias and gamma alone, but not in two that are multiplied, nor behind an activation
    d["open"] = (need_x && need_w) || ((act != 0 || need_g) && (need_x || need_w || need_b));
    d["need_x"] = need_x;
    d["need_w"] = need_w;
    d["need_b"] = need_b;
    d["need_r"] = wants(residual);
    d["need_g"] = need_g;
    d["x_shape"] = x.sizes().vec();
    d["w_shape"] = weight.sizes().vec();
    d["w_type"] = (int64_t)weight.scalar_type();
    d["b_type"] = (int64_t)(bias.has_value() ? bias->scalar_type() : at::kFloat);
    d["g_type"] = (int64_t)(gamma.has_value() ? gamma->scalar_type() : at::kFloat);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = N;
    return y.view(shape);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor dy = grads[0];
    once_differentiable(dy, ctx->saved_data["open"].toBool(), "fp8_linear");
    const variable_list s = ctx->get_saved_variables();
    BelowAutograd below;
    auto& d = ctx->saved_data;
    const std::vector<int64_t> x_shape = d["x_shape"].toIntVector(), w_shape = d["w_shape"].toIntVector();
    const int64_t N = w_shape[0], K = x_shape.back();
    const int64_t act = d["act"].toInt();
    const bool need_x = d["need_x"].toBool(), need_w = d["need_w"].toBool(), need_b = d["need_b"].toBool();
    at::Tensor dz = matrix(dy, N);
    if (dz.size(0) > 1 && dz.stride(0) < N) dz = dz.contiguous();  // an expanded gradient
    const int64_t M = dz.size(0);
    at::Tensor dgamma;
    if (d["need_g"].toBool()) {
      // d(gamma * h) / d gamma needs h = act(x W^T + b): recomputed once, from the saved operands
      at::Tensor h = at::empty({M, N}, dz.options().dtype(at::kFloat));
      fp8_gemm(s[7], s[8], false, s[9], s[10], true, K, h, opt(s[2]), {}, {}, {}, act, false);
      dgamma = dz.to(at::kFloat).mul_(h).sum(0).to((at::ScalarType)d["g_type"].toInt());
    }
    const at::Tensor w_sink = kept_sink(ctx, "w_sink"), b_sink = kept_sink(ctx, "b_sink");
    at::Tensor db;
    OptTensor sums;
    if (need_b) {
      if (!b_sink.defined()) db = at::empty({N}, dz.options().dtype(at::kFloat));
      sums = b_sink.defined() ? b_sink : db;
    }
    Q8 dq, dt;
    quantize_both(dz, false, need_x, need_w, dq, dt, opt(s[0]), opt(s[1]), sums, b_sink.defined());
    at::Tensor dx, dw;
    if (need_x) {
      dx = at::empty({M, K}, dz.options());
      fp8_gemm(dq.data, dq.scale, false, s[5], s[6], true, N, dx, {}, {}, {}, {}, 0, false);
      dx = dx.view(x_shape);
    }
    if (need_w) {
      const bool sink = w_sink.defined();
      at::Tensor out = sink ? w_sink.view({N, K}) : at::empty({N, K}, dz.options().dtype(at::kFloat));
      fp8_gemm(dt.data, dt.scale, false, s[3], s[4], false, M, out, {}, {}, {}, {}, 0, sink);
      if (!sink) dw = out.to((at::ScalarType)d["w_type"].toInt()).view(w_shape);
    }
    if (db.defined()) db = db.to((at::ScalarType)d["b_type"].toInt());
    return {dx, dw, db, d["need_r"].toBool() ? dy : at::Tensor(), dgamma, at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace

at::Tensor dropout(const at::Tensor& x, const OptTensor& residual, int64_t dropped, const OptTensor& rng,
                   int64_t rank_key) {
  return DropoutNode::apply(x, residual, dropped, rng, rank_key);
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw,
                                                const OptTensor& kw, const OptTensor& angles, const OptTensor& pairs,
                                                double eps, const OptTensor& q_sink, const OptTensor& k_sink) {
  variable_list out = QkNormNode::apply(q, k, qw, kw, angles, pairs, eps, q_sink, k_sink);
  return {out[0], out[1]};
}

at::Tensor fp8_linear(const at::Tensor& x, const at::Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                      const OptTensor& gamma, int64_t act, bool bf16, const OptTensor& shadow, const OptTensor& w_sink,
                      const OptTensor& b_sink) {
  return Fp8LinearNode::apply(x, weight, bias, residual, gamma, act, bf16, shadow, w_sink, b_sink,
                              at::GradMode::is_enabled());
}

// y = residual + gamma * act(x W^T + bias) on a weight that was quantised once; no backward.
at::Tensor fp8_linear_quantized(const at::Tensor& x, const at::Tensor& data, const at::Tensor& scale, bool block,
                                int64_t K, const OptTensor& bias, const OptTensor& residual, const OptTensor& gamma,
                                int64_t act, bool bf16) {
  at::NoGradGuard no_grad;
  BelowAutograd below;
  const at::ScalarType type = bf16 ? at::kBFloat16 : at::kFloat;
  const at::Tensor x2 = matrix(x, K);
  const int64_t M = x2.size(0), N = data.size(0);
  Q8 xq, none;
  quantize_both(x2, false, true, false, xq, none);
  OptTensor res;
  if (residual.has_value()) res = aligned(residual->reshape({M, N}).to(type));
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  at::Tensor y = at::empty({M, N}, x.options().dtype(type));
  fp8_gemm(xq.data, xq.scale, false, data, scale, block, K, y, aligned_vector(bias), res, aligned_vector(gamma), {}, act,
           false);
  return y.view(shape);
}

}  // namespace mia
