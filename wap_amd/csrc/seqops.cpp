// Autograd of the sequence operators on the GPU: argument checks, layout, and
// the nodes that call the kernels' entry points (gscan.hip, seqloss.hip,
// ctrdrop.hip).
//
// In C++ because the smallest calls are bound by the host: a training step of
// the decoder's own sizes spends 10 to 20 us in these kernels, and a node
// written in Python costs several times that in its forward and backward pass.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <tuple>
#include <vector>

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

// ---- the kernels' entry points
std::vector<Tensor> gated_scan_fwd(Tensor g, OptTensor h0, OptTensor mask,
                                   bool keep);
std::vector<Tensor> gated_scan_bwd(Tensor g, OptTensor h0, OptTensor mask,
                                   OptTensor marks, OptTensor dh,
                                   OptTensor dlast);
std::vector<Tensor> token_logprob_fwd(Tensor logits, Tensor y, OptTensor w);
Tensor token_logprob_bwd(Tensor logits, Tensor y, OptTensor w, Tensor stats,
                         Tensor dlogp);
std::vector<Tensor> policy_loss_fwd(Tensor logits, Tensor y, Tensor w,
                                    Tensor old_logp, Tensor adv, OptTensor ref,
                                    double lo, double hi, double beta,
                                    bool grad);
void policy_loss_bwd(Tensor logits, Tensor y, Tensor w, Tensor rows, bool again,
                     Tensor up, Tensor dlogits);
int64_t capture_of(const Tensor& like);
std::vector<Tensor> preference_loss_fwd(Tensor logits, Tensor y, Tensor w,
                                        Tensor ref, double beta, double eps);
Tensor preference_loss_bwd(Tensor logits, Tensor y, Tensor w, Tensor rows,
                           Tensor up);
std::vector<Tensor> counter_dropout_run(Tensor x, OptTensor residual, double p,
                                        OptTensor rng, int64_t seed,
                                        int64_t step, int64_t stream,
                                        bool keep_used);

namespace {

// Whether a gradient is wanted by t.  A tangent, which no kernel here carries
// on, is refused: without it the output would read as a zero derivative.
bool tracked(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what,
                              " has no forward-mode derivative");
  return at::GradMode::is_enabled() && t.requires_grad();
}

bool tracked(const Tensor& t, const OptTensor& u, const char* what) {
  const bool second = u.has_value() && tracked(*u, what);
  return tracked(t, what) || second;
}

OptTensor given(const Tensor& t) {
  return t.defined() ? OptTensor(t) : OptTensor();
}

// These gradients have no gradient of their own: whoever differentiates
// through them is told.
variable_list once(const char* what, variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + ": its gradient cannot be differentiated again",
      (int64_t)grads.size());
  return (*node)(std::move(grads));
}

// The kernels step over rows by stride; the last axis has to be dense.
Tensor dense(const Tensor& t) {
  return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}

// A constant beside the data, in f32.
Tensor plain(const Tensor& t) {
  // (each call into the dispatcher that is not made is about 1 us)
  if (t.scalar_type() == at::kFloat && t.is_contiguous() && !t.requires_grad())
    return t;
  return t.detach().to(at::kFloat).contiguous();
}

// ------------------------------------------------------ gated recurrence

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, Tensor g, OptTensor h0,
                               OptTensor mask) {
    ctx->set_materialize_grads(false);
    g = dense(g);
    OptTensor h;
    if (h0.has_value()) {
      h = h0->to(at::kFloat).contiguous();
      ctx->saved_data["h0"] = (int64_t)h0->scalar_type();
    }
    auto out = gated_scan_fwd(g, h, mask, true);
    ctx->save_for_backward({g, h.value_or(Tensor()), mask.value_or(Tensor()),
                            out.size() > 2 ? out[2] : Tensor()});
    return {out[0], out[1]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    auto s = ctx->get_saved_variables();
    variable_list grads(3);
    if (up[0].defined() || up[1].defined()) {
      OptTensor dh, dlast;
      if (up[0].defined()) dh = dense(up[0]);
      if (up[1].defined()) dlast = up[1].contiguous();
      auto d = gated_scan_bwd(s[0], given(s[1]), given(s[2]), given(s[3]), dh,
                              dlast);
      grads[0] = d[0];
      if (s[1].defined())
        grads[1] = d[1].to((at::ScalarType)ctx->saved_data["h0"].toInt());
    }
    return once("gated_scan", std::move(grads));
  }
};

void check_gates(const Tensor& g, int64_t dim, const char* what) {
  TORCH_CHECK_VALUE(g.dim() == dim && g.size(-1) % 2 == 0, what, ": g must be [",
                    dim == 3 ? "B, T, " : "B, ", "2*D], got ", g.sizes());
}

void check_state(const Tensor& h, const Tensor& g, const char* what) {
  TORCH_CHECK_VALUE(h.dim() == 2 && h.size(0) == g.size(0) &&
                        h.size(1) == g.size(-1) / 2,
                    what, ": state must be [B, D] = [", g.size(0), ", ",
                    g.size(-1) / 2, "], got ", h.sizes());
  TORCH_CHECK_VALUE(h.device() == g.device() && h.is_floating_point(), what,
                    ": state must be floating point on ", g.device());
}

// ------------------------------------------------------ token probabilities

struct TokenLogprob : torch::autograd::Function<TokenLogprob> {
  static Tensor forward(AutogradContext* ctx, Tensor logits, Tensor y,
                        OptTensor w) {
    auto out = token_logprob_fwd(logits, y, w);
    ctx->save_for_backward({logits, y, w.value_or(Tensor()), out[1]});
    return out[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    auto s = ctx->get_saved_variables();
    variable_list grads(3);
    grads[0] =
        token_logprob_bwd(s[0], s[1], given(s[2]), s[3], up[0].contiguous());
    return once("token_logprob", std::move(grads));
  }
};

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext* ctx, Tensor logits, Tensor y,
                               Tensor w, Tensor old_logp, Tensor adv,
                               OptTensor ref, double lo, double hi,
                               double beta) {
    ctx->set_materialize_grads(false);
    // the gradient of a row needs nothing but the row: it is made while the
    // row is at hand, for an upstream gradient of one
    auto out = policy_loss_fwd(logits, y, w, old_logp, adv, ref, lo, hi, beta,
                               true);
    ctx->save_for_backward({logits, y, w, out[3]});
    // not among the saved tensors: it is handed out, and from then on the
    // caller's to write into
    ctx->saved_data["made"] = out[2];
    ctx->saved_data["capture"] = capture_of(logits);
    ctx->mark_non_differentiable({out[1]});
    return {out[0], out[1]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    auto s = ctx->get_saved_variables();
    variable_list grads(9);
    if (up[0].defined()) {
      // Handed out once, and only where the forward pass runs whenever this
      // pass does: eagerly, or in the same captured graph.  A pass that is
      // replayed without the forward pass would find what the caller has
      // written there, and a forward pass that is replayed without this one
      // would write into what the caller was given.  Any other walk makes the
      // gradient anew.
      auto made = ctx->saved_data.find("made");
      const bool take = made != ctx->saved_data.end() &&
                        ctx->saved_data["capture"].toInt() == capture_of(s[0]);
      if (take) {
        grads[0] = made->second.toTensor();
        ctx->saved_data.erase(made);
      } else {
        grads[0] = torch::empty(s[0].sizes(), s[0].options());
      }
      policy_loss_bwd(s[0], s[1], s[2], s[3], take, plain(up[0]), grads[0]);
    }
    return once("policy_loss", std::move(grads));
  }
};

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, Tensor logits, Tensor y,
                               Tensor w, Tensor ref, double beta, double eps) {
    ctx->set_materialize_grads(false);
    auto out = preference_loss_fwd(logits, y, w, ref, beta, eps);
    ctx->save_for_backward({logits, y, w, out[2]});
    ctx->mark_non_differentiable({out[1]});
    return {out[0], out[1]};
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    auto s = ctx->get_saved_variables();
    variable_list grads(6);
    if (up[0].defined())
      grads[0] = preference_loss_bwd(s[0], s[1], s[2], s[3], plain(up[0]));
    return once("preference_loss", std::move(grads));
  }
};

bool same_rows(const Tensor& t, const Tensor& logits) {
  return t.dim() == 2 && t.size(0) == logits.size(0) &&
         t.size(1) == logits.size(1) && t.device() == logits.device();
}

Tensor per_token(const Tensor& t, const Tensor& logits, const char* what,
                 const char* name) {
  TORCH_CHECK_VALUE(same_rows(t, logits), what, ": ", name, " must be [",
                    logits.size(0), ", ", logits.size(1), "] on ",
                    logits.device(), ", got ", t.sizes(), " on ", t.device());
  return plain(t);
}

// Checked and laid out.
void check_rows(Tensor& logits, Tensor& y, const char* what) {
  TORCH_CHECK_VALUE(logits.dim() == 3 && logits.size(2) >= 1, what,
                    ": logits must be [B, T, K], got ", logits.sizes());
  TORCH_CHECK_TYPE(!y.is_floating_point() && !y.is_complex() &&
                       y.scalar_type() != at::kBool,
                   what, ": y must hold whole numbers, got ", y.scalar_type());
  TORCH_CHECK_VALUE(same_rows(y, logits), what, ": y must be [", logits.size(0),
                    ", ", logits.size(1), "] on ", logits.device(), ", got ",
                    y.sizes(), " on ", y.device());
  logits = dense(logits);
  if (y.scalar_type() != at::kLong || !y.is_contiguous())
    y = y.to(at::kLong).contiguous();
}

// ------------------------------------------------------ dropout

// 0: as it lies; else the channels-last order of 4 or 5 axes.
int64_t order_of(const Tensor& x) {
  if (x.is_contiguous()) return 0;
  if (x.dim() == 4 && x.is_contiguous(at::MemoryFormat::ChannelsLast)) return 4;
  if (x.dim() == 5 && x.is_contiguous(at::MemoryFormat::ChannelsLast3d))
    return 5;
  return 0;
}

Tensor in_order(const Tensor& t, int64_t order) {
  if (order == 0) return t.contiguous();
  if (order == 4)
    return t.contiguous(at::MemoryFormat::ChannelsLast).permute({0, 2, 3, 1});
  return t.contiguous(at::MemoryFormat::ChannelsLast3d)
      .permute({0, 2, 3, 4, 1});
}

Tensor back(const Tensor& t, int64_t order) {
  if (order == 0) return t;
  return order == 4 ? t.permute({0, 3, 1, 2}) : t.permute({0, 4, 1, 2, 3});
}

std::vector<Tensor> drop(const Tensor& x, const OptTensor& residual,
                         int64_t order, double p, const OptTensor& rng,
                         int64_t seed, int64_t step, int64_t stream,
                         bool keep) {
  OptTensor res;
  if (residual.has_value()) res = in_order(*residual, order);
  auto out = counter_dropout_run(in_order(x, order), res, p, rng, seed, step,
                                 stream, keep);
  out[0] = back(out[0], order);
  return out;
}

struct CounterDropout : torch::autograd::Function<CounterDropout> {
  static Tensor forward(AutogradContext* ctx, Tensor x, OptTensor residual,
                        double p, OptTensor rng, int64_t seed, int64_t step,
                        int64_t stream) {
    const int64_t order = order_of(x);
    auto out = drop(x, residual, order, p, rng, seed, step, stream, true);
    auto& d = ctx->saved_data;
    d["p"] = p;
    d["seed"] = seed;
    d["step"] = step;
    d["stream"] = stream;
    d["order"] = order;
    d["residual"] = residual.has_value();
    // what the kernel read, not what the caller's tensor holds by then
    if (rng.has_value()) ctx->save_for_backward({out[1]});
    return out[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    auto& d = ctx->saved_data;
    auto s = ctx->get_saved_variables();
    variable_list grads(7);
    if (ctx->needs_input_grad(0))
      grads[0] = drop(up[0], {}, d["order"].toInt(), d["p"].toDouble(),
                      s.empty() ? OptTensor() : OptTensor(s[0]),
                      d["seed"].toInt(), d["step"].toInt(),
                      d["stream"].toInt(), false)[0];
    grads = once("counter_dropout", std::move(grads));
    if (d["residual"].toBool()) grads[1] = up[0];
    return grads;
  }
};

}  // namespace

std::tuple<Tensor, Tensor> gated_scan(Tensor g, OptTensor h0, OptTensor mask) {
  const char* what = "gated_scan";
  check_gates(g, 3, what);
  if (h0.has_value()) check_state(*h0, g, what);
  if (mask.has_value()) {
    TORCH_CHECK_VALUE(same_rows(*mask, g), what, ": mask must be [", g.size(0),
                      ", ", g.size(1), "] on ", g.device(), ", got ",
                      mask->sizes(), " on ", mask->device());
    mask = plain(mask->scalar_type() == at::kFloat ? *mask : mask->gt(0));
  }
  if (tracked(g, h0, what)) {
    auto out = GatedScan::apply(g, h0, mask);
    return {out[0], out[1]};
  }
  if (h0.has_value()) h0 = plain(*h0);
  auto out = gated_scan_fwd(dense(g), h0, mask, false);
  return {out[0], out[1]};
}

std::tuple<Tensor, Tensor> gated_step_run(Tensor g, Tensor h);

std::tuple<Tensor, Tensor> gated_step(Tensor g, Tensor h) {
  check_gates(g, 2, "gated_step");
  check_state(h, g, "gated_step");
  return gated_step_run(dense(g.detach()), plain(h));
}

Tensor token_logprob(Tensor logits, Tensor y, OptTensor mask) {
  const char* what = "token_logprob";
  check_rows(logits, y, what);
  OptTensor w;
  if (mask.has_value()) w = per_token(*mask, logits, what, "mask");
  if (tracked(logits, what)) return TokenLogprob::apply(logits, y, w);
  return token_logprob_fwd(logits, y, w)[0];
}

std::tuple<Tensor, Tensor> policy_loss(Tensor logits, Tensor y, Tensor mask,
                                       Tensor old_logp, Tensor advantage,
                                       OptTensor ref_logp, double lo, double hi,
                                       double beta) {
  const char* what = "policy_loss";
  check_rows(logits, y, what);
  Tensor w = per_token(mask, logits, what, "mask");
  Tensor old = per_token(old_logp, logits, what, "old_logp");
  OptTensor ref;
  if (ref_logp.has_value())
    ref = per_token(*ref_logp, logits, what, "ref_logp");
  if (beta == 0.0) ref.reset();  // no term, not 0 times an infinite one
  if (advantage.dim() == 1 && advantage.size(0) == logits.size(0))
    advantage = advantage.unsqueeze(1).expand({logits.size(0), logits.size(1)});
  TORCH_CHECK_VALUE(same_rows(advantage, logits), what,
                    ": advantage must be [B, T] or [B] on ", logits.device(),
                    ", got ", advantage.sizes(), " on ", advantage.device());
  if (advantage.scalar_type() != at::kFloat || advantage.requires_grad())
    advantage = advantage.detach().to(at::kFloat);
  if (tracked(logits, what)) {
    auto out =
        PolicyLoss::apply(logits, y, w, old, advantage, ref, lo, hi, beta);
    return {out[0], out[1]};
  }
  auto out = policy_loss_fwd(logits, y, w, old, advantage, ref, lo, hi, beta,
                             false);
  return {out[0], out[1]};
}

std::tuple<Tensor, Tensor> preference_loss(Tensor logits, Tensor y, Tensor mask,
                                           Tensor ref_logp, double beta,
                                           double eps) {
  const char* what = "preference_loss";
  check_rows(logits, y, what);
  Tensor w = per_token(mask, logits, what, "mask");
  Tensor ref = per_token(ref_logp, logits, what, "ref_logp");
  if (tracked(logits, what)) {
    auto out = PreferenceLoss::apply(logits, y, w, ref, beta, eps);
    return {out[0], out[1]};
  }
  auto out = preference_loss_fwd(logits, y, w, ref, beta, eps);
  return {out[0], out[1]};
}

Tensor counter_dropout(Tensor x, OptTensor residual, double p, OptTensor rng,
                       int64_t seed, int64_t step, int64_t stream) {
  if (rng.has_value()) {
    TORCH_CHECK_VALUE(rng->scalar_type() == at::kLong && rng->dim() == 1 &&
                          rng->size(0) == 2 && rng->device() == x.device(),
                      "counter_dropout: rng must be int64 [2] on ", x.device(),
                      ", got ", rng->scalar_type(), " ", rng->sizes(), " on ",
                      rng->device());
    rng = rng->detach().contiguous();
  }
  if (residual.has_value())
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() &&
                          residual->scalar_type() == x.scalar_type() &&
                          residual->device() == x.device(),
                      "counter_dropout: residual must have x's shape, type and "
                      "device, got ",
                      residual->sizes(), " ", residual->scalar_type());
  if (tracked(x, residual, "counter_dropout"))
    return CounterDropout::apply(x, residual, p, rng, seed, step, stream);
  return drop(x, residual, order_of(x), p, rng, seed, step, stream, false)[0];
}
