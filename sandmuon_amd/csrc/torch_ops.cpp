// The differentiable operators of a training step as torch functions: argument
// checks, allocation, the call of the C ABI on the current stream, autograd.
//
// A small call's time is the host's.  In Python, checks, descriptors and above
// all the hand-over of the interpreter lock to autograd's device thread took 120
// to 200 us of a forward and backward whose kernels take 15 to 65; here neither
// forward nor backward runs Python code.
//
// Nothing is computed here: every operation is an entry point of
// libsandmuon_amd.so, and errors are its status and message.
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <optional>
#include <string>
#include <tuple>

#include "../../include/sandmuon_amd.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ---------------------------------------------------------------- calls ---
void *stream_of(const Tensor &t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream();
}

void check(int rc, const char *what) {
  if (rc == SMX_OK) return;
  static const char *const names[] = {"SMX_EINVAL", "SMX_ESHAPE", "SMX_EDTYPE", "SMX_EALIGN", "SMX_EWORKSPACE", "SMX_ELAUNCH"};
  const char *name = rc <= -1 && rc >= -6 ? names[-rc - 1] : "error";
  TORCH_CHECK_VALUE(rc < -5, what, ": ", name, ": ", smx_last_error());
  TORCH_CHECK(false, what, ": ", name, ": ", smx_last_error());
}

int dtype_of(const Tensor &t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return SMX_F32;
    case torch::kBFloat16: return SMX_BF16;
    case torch::kFloat16: return SMX_F16;
    default: return -1;
  }
}

void need_float(const Tensor &t, const std::string &what) {
  TORCH_CHECK(t.is_cuda(), what, ": sandmuon_amd runs on ROCm GPU tensors only (got ", t.device(), ")");
  TORCH_CHECK_VALUE(dtype_of(t) >= 0, what, ": unsupported dtype ", t.scalar_type(),
                    "; expected float32, bfloat16 or float16");
}

void same_device(const char *what, const Tensor &first, std::initializer_list<const OptTensor *> others) {
  for (const OptTensor *t : others)
    TORCH_CHECK_VALUE(!t->has_value() || (*t)->device() == first.device(), what, ": tensors on ", first.device(), " and ",
                      (*t)->device());
}

bool integral(const Tensor &t) { return c10::isIntegralType(t.scalar_type(), false); }

// t, or a contiguous copy where its last dimension has no unit stride.
Tensor unit_last(const Tensor &t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// And where its rows overlap (the gradient of a sum over them is one row
// repeated): the entry points take rows that lie behind each other.
Tensor apart_rows(const Tensor &t) {
  return t.size(-2) > 1 && t.stride(-2) < t.size(-1) ? t.contiguous() : unit_last(t);
}

template <typename T = void>
T *ptr(const OptTensor &t) {
  return t.has_value() && t->defined() ? static_cast<T *>(t->data_ptr()) : nullptr;
}

bool wants_grad(const OptTensor &t) { return t.has_value() && t->defined() && t->requires_grad(); }

OptTensor some(const Tensor &t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// A backward's result has no graph of its own.
void no_double_backward(const char *what) {
  TORCH_CHECK(!torch::GradMode::is_enabled(), what, ": its gradient cannot be differentiated (create_graph)");
}

// Nor has anything here a forward-mode one: a tangent is refused where no autograd
// function sees it, and the result would count as a constant.
void no_tangent(const char *what, std::initializer_list<const OptTensor *> inputs) {
  for (const OptTensor *t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->has_value() || !(*t)->defined() || !(*t)->_fw_grad(0).defined(), what,
                                ": no forward-mode derivative");
}

// ------------------------------------------------------ qk_norm_rotary ---
struct QkRest {
  int64_t position0, style;
  double eps;
};

void fill_side(smx_qk_side *s, const Tensor &x, const OptTensor &w, const Tensor &y, const Tensor *dy, Tensor *dw) {
  s->x = x.data_ptr(), s->weight = ptr(w), s->y = y.data_ptr(), s->heads = x.size(2);
  for (int i = 0; i < 3; ++i) {
    s->x_stride[i] = x.stride(i), s->y_stride[i] = y.stride(i);
    if (dy) s->dy_stride[i] = dy->stride(i);
  }
  if (dy) s->dy = dy->data_ptr();
  if (dw && dw->defined()) s->dw = dw->data_ptr();
  if (s->weight) s->weight_dtype = dtype_of(*w);
}

smx_qk_desc qk_desc(const Tensor &x, const Tensor &cos, const Tensor &sin, const OptTensor &positions, const QkRest &rest) {
  smx_qk_desc d{};
  d.cos = cos.data_ptr<float>(), d.sin = sin.data_ptr<float>();
  if (positions.has_value()) {
    d.positions = positions->data_ptr<int64_t>();
    d.pos_stride[0] = positions->stride(0), d.pos_stride[1] = positions->stride(1);
  }
  d.position0 = rest.position0, d.table_rows = cos.size(0);
  d.batch = x.size(0), d.seq = x.size(1), d.dim = x.size(3), d.rot = 2 * cos.size(1);
  d.eps = rest.eps, d.dtype = dtype_of(x), d.style = static_cast<int32_t>(rest.style);
  return d;
}

void qk_forward(const Tensor &q, const Tensor &k, const OptTensor &qw, const OptTensor &kw, const Tensor &cos,
                const Tensor &sin, const OptTensor &positions, const QkRest &rest, const Tensor &yq, const Tensor &yk) {
  smx_qk_desc d = qk_desc(q, cos, sin, positions, rest);
  fill_side(&d.q, q, qw, yq, nullptr, nullptr);
  fill_side(&d.k, k, kw, yk, nullptr, nullptr);
  const c10::DeviceGuard guard(q.device());
  check(smx_qk_norm_rotary(&d, stream_of(q)), "smx_qk_norm_rotary");
}

struct QkNormRotary : torch::autograd::Function<QkNormRotary> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const OptTensor &qw,
                               const OptTensor &kw, const Tensor &cos, const Tensor &sin, const OptTensor &positions,
                               int64_t position0, double eps, int64_t style) {
    const Tensor yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
    qk_forward(q, k, qw, kw, cos, sin, positions, {position0, style, eps}, yq, yk);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, qw.value_or(Tensor()), kw.value_or(Tensor()), cos, sin, positions.value_or(Tensor())});
    ctx->saved_data["position0"] = position0;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["style"] = style;
    ctx->saved_data["needs"] =
        static_cast<int64_t>(q.requires_grad() | k.requires_grad() << 1 | wants_grad(qw) << 2 | wants_grad(kw) << 3);
    return {yq, yk};
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    no_double_backward("qk_norm_rotary");
    const auto saved = ctx->get_saved_variables();
    const int64_t needs = ctx->saved_data["needs"].toInt();
    const Tensor &q = saved[0], &cos = saved[4];
    variable_list out(10);
    smx_qk_desc d = qk_desc(q, cos, saved[5], some(saved[6]),
                            {ctx->saved_data["position0"].toInt(), ctx->saved_data["style"].toInt(),
                             ctx->saved_data["eps"].toDouble()});
    Tensor dy[2], dx[2], dw[2];
    for (int i = 0; i < 2; ++i) {
      const bool need_x = needs >> i & 1, need_w = needs >> (2 + i) & 1;
      if (!grads[i].defined() || !(need_x || need_w)) continue;  // (a side with no heads is left out)
      const Tensor &x = saved[i];
      dy[i] = unit_last(grads[i].to(x.scalar_type()));
      dx[i] = at::empty(x.sizes(), x.options());
      if (need_w) dw[i] = at::empty(saved[2 + i].sizes(), saved[2 + i].options());
      fill_side(i ? &d.k : &d.q, x, some(saved[2 + i]), dx[i], &dy[i], &dw[i]);
      if (need_x) out[i] = dx[i];
      if (need_w) out[2 + i] = dw[i];
    }
    if (!dx[0].defined() && !dx[1].defined()) return out;
    Tensor work;
    int64_t bytes = 0;
    if (dw[0].defined() || dw[1].defined()) {
      bytes = smx_qk_workspace_bytes(q.size(3));
      work = at::empty({bytes}, q.options().dtype(torch::kUInt8));
    }
    const c10::DeviceGuard guard(q.device());
    check(smx_qk_norm_rotary_backward(&d, bytes ? work.data_ptr() : nullptr, bytes, stream_of(q)),
          "smx_qk_norm_rotary_backward");
    return out;
  }
};

OptTensor checked_weight(const OptTensor &w, const Tensor &x, const char *name) {
  if (!w.has_value()) return w;
  need_float(*w, std::string("qk_norm_rotary: ") + name);
  TORCH_CHECK_VALUE(w->dim() == 1 && w->size(0) == x.size(3), "qk_norm_rotary: ", name, " ", w->sizes(), " of heads of ",
                    x.size(3));
  return w->contiguous();
}

std::tuple<Tensor, Tensor> qk_norm_rotary(Tensor q, Tensor k, OptTensor qw, OptTensor kw, Tensor cos, Tensor sin,
                                          OptTensor positions, int64_t position0, double eps, int64_t style,
                                          std::optional<std::tuple<Tensor, Tensor>> out) {
  const char *what = "qk_norm_rotary";
  need_float(q, what);
  need_float(k, what);
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(1) == k.size(1) &&
                        q.size(3) == k.size(3) && q.scalar_type() == k.scalar_type(),
                    what, ": q ", q.sizes(), " ", q.scalar_type(), " and k ", k.sizes(), " ", k.scalar_type(),
                    "; expected [batch, seq, heads, dim] of one type, alike but for heads");
  TORCH_CHECK_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.scalar_type() == torch::kFloat32 &&
                        sin.scalar_type() == torch::kFloat32 && 2 * cos.size(1) <= q.size(3),
                    what, ": cos ", cos.sizes(), " ", cos.scalar_type(), " and sin ", sin.sizes(), " ", sin.scalar_type(),
                    "; expected float32 [positions, rot / 2] with rot at most dim");
  qw = checked_weight(qw, q, "q_weight");
  kw = checked_weight(kw, k, "k_weight");
  const OptTensor others[] = {k, cos, sin};
  same_device(what, q, {&others[0], &others[1], &others[2], &qw, &kw, &positions});
  const OptTensor first = q;
  no_tangent(what, {&first, &others[0], &others[1], &others[2], &qw, &kw});
  if (positions.has_value()) {
    TORCH_CHECK_VALUE(integral(*positions) && (positions->dim() == 1 || positions->dim() == 2), what, ": positions ",
                      positions->sizes(), " ", positions->scalar_type(), "; expected integers [seq] or [batch, seq]");
    positions = positions->to(torch::kInt64).expand({q.size(0), q.size(1)});
  }
  cos = cos.contiguous(), sin = sin.contiguous();
  q = unit_last(q), k = unit_last(k);
  const bool grad =
      torch::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || wants_grad(qw) || wants_grad(kw));
  if (grad) {
    TORCH_CHECK_VALUE(!out.has_value(), what, ": out= is not supported under autograd");
    const auto y = QkNormRotary::apply(q, k, qw, kw, cos, sin, positions, position0, eps, style);
    return {y[0], y[1]};
  }
  const bool given = out.has_value();
  if (given) {
    for (const auto &[o, x] : {std::tie(std::get<0>(*out), q), std::tie(std::get<1>(*out), k)}) {
      TORCH_CHECK_VALUE(o.sizes() == x.sizes() && o.scalar_type() == x.scalar_type() && o.device() == x.device() &&
                            (o.size(3) <= 1 || o.stride(3) == 1),
                        what, ": out ", o.sizes(), " ", o.scalar_type(), " for ", x.sizes(), " ", x.scalar_type(),
                        "; the last stride must be one");
      for (int d = 0; d < 3; ++d)
        TORCH_CHECK_VALUE(o.size(d) <= 1 || o.stride(d) != 0 || o.numel() == 0, what, ": out of strides ", o.strides(),
                          " names places twice");
      TORCH_CHECK_VALUE(!torch::GradMode::is_enabled() || !o.requires_grad(), what,
                        ": out= that requires a gradient is not supported under autograd");
    }
    // written while the other side, or another place of its own, is still read
    const auto &[oq, ok] = *out;
    at::assert_no_partial_overlap(oq, q);
    at::assert_no_partial_overlap(ok, k);
    at::assert_no_overlap(oq, k);
    at::assert_no_overlap(ok, q);
    at::assert_no_overlap(oq, ok);
  } else {
    out = {at::empty(q.sizes(), q.options()), at::empty(k.sizes(), k.options())};
  }
  const auto &[oq, ok] = *out;
  qk_forward(q, k, qw, kw, cos, sin, positions, {position0, style, eps}, oq, ok);
  // (a graph that saved what was there notices)
  if (given) oq.unsafeGetTensorImpl()->bump_version(), ok.unsafeGetTensorImpl()->bump_version();
  return *out;
}

// --------------------------------------------------------------- losses ---
void check_logits(const char *what, Tensor *logits, Tensor *targets, OptTensor *mask) {
  need_float(*logits, what);
  TORCH_CHECK_VALUE(logits->dim() == 3 && logits->size(2) > 0, what, ": logits ", logits->sizes(),
                    "; expected [batch, seq, vocab]");
  TORCH_CHECK_VALUE(targets->dim() == 2 && targets->size(0) == logits->size(0) && targets->size(1) == logits->size(1) &&
                        integral(*targets),
                    what, ": targets ", targets->sizes(), " ", targets->scalar_type(), " of logits ", logits->sizes(),
                    "; expected integers [batch, seq]");
  if (mask->has_value()) {
    const auto type = (*mask)->scalar_type();
    TORCH_CHECK_VALUE((*mask)->sizes() == targets->sizes() && (type == torch::kBool || type == torch::kUInt8), what,
                      ": mask ", (*mask)->sizes(), " ", type, "; expected bool [batch, seq]");
    *mask = (*mask)->contiguous();
  }
  const OptTensor t = *targets, z = *logits;
  same_device(what, *logits, {&t, mask});
  no_tangent(what, {&z});
  *logits = apart_rows(*logits);
  *targets = targets->to(torch::kInt64).contiguous();
}

// A per-token float tensor as contiguous FP32.
OptTensor token_floats(const char *what, const char *name, const OptTensor &t, const Tensor &targets) {
  if (!t.has_value()) return t;
  TORCH_CHECK_VALUE(t->sizes() == targets.sizes() && t->is_floating_point(), what, ": ", name, " ", t->sizes(), " ",
                    t->scalar_type(), "; expected floats ", targets.sizes());
  same_device(what, targets, {&t});
  return t->detach().to(torch::kFloat32).contiguous();
}

struct Rows {
  const void *z;
  int dtype;
  int64_t batch, seq, vocab, batch_stride, row_stride;
  const int64_t *targets;
  const uint8_t *mask;
};

Rows rows_of(const Tensor &logits, const Tensor &targets, const OptTensor &mask) {
  return {logits.data_ptr(), dtype_of(logits), logits.size(0), logits.size(1), logits.size(2), logits.stride(0),
          logits.stride(1), targets.data_ptr<int64_t>(), ptr<uint8_t>(mask)};
}

#define ROWS(r) r.z, r.dtype, r.batch, r.seq, r.vocab, r.batch_stride, r.row_stride, r.targets, r.mask

Tensor fp32(const Tensor &like, at::IntArrayRef sizes) { return at::empty(sizes, like.options().dtype(torch::kFloat32)); }

std::pair<Tensor, Tensor> logprobs(const Tensor &logits, const Tensor &targets, const OptTensor &mask, bool want_stats) {
  const Tensor lp = fp32(logits, targets.sizes());
  Tensor stats;
  if (want_stats) stats = fp32(logits, {targets.size(0), targets.size(1), 2});
  const Rows r = rows_of(logits, targets, mask);
  const c10::DeviceGuard guard(logits.device());
  check(smx_token_logprobs(ROWS(r), lp.data_ptr<float>(), want_stats ? stats.data_ptr<float>() : nullptr,
                           stream_of(logits)),
        "smx_token_logprobs");
  return {lp, stats};
}

Tensor logprobs_backward(const Tensor &logits, const Tensor &targets, const OptTensor &mask, const Tensor &stats,
                         const Tensor &coef, int64_t batch_stride, int64_t row_stride, const OptTensor &scale) {
  const Tensor out = at::empty(logits.sizes(), logits.options());
  const Rows r = rows_of(logits, targets, mask);
  const c10::DeviceGuard guard(logits.device());
  check(smx_token_logprobs_backward(ROWS(r), stats.data_ptr<float>(), coef.data_ptr<float>(), batch_stride, row_stride,
                                    ptr<float>(scale), out.data_ptr(), stream_of(logits)),
        "smx_token_logprobs_backward");
  return out;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Tensor &targets, const OptTensor &mask) {
    const auto [lp, stats] = logprobs(logits, targets, mask, true);
    ctx->save_for_backward({logits, targets, mask.value_or(Tensor()), stats});
    return lp;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    no_double_backward("token_logprobs");
    const auto s = ctx->get_saved_variables();
    const Tensor coef = grads[0].to(torch::kFloat32);
    return {logprobs_backward(s[0], s[1], some(s[2]), s[3], coef, coef.stride(0), coef.stride(1), std::nullopt), Tensor(),
            Tensor()};
  }
};

Tensor token_logprobs(Tensor logits, Tensor targets, OptTensor mask) {
  check_logits("token_logprobs", &logits, &targets, &mask);
  if (torch::GradMode::is_enabled() && logits.requires_grad()) return TokenLogprobs::apply(logits, targets, mask);
  return logprobs(logits, targets, mask, false).first;
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  // The gradient of FP32 and BF16 logits is made with the loss, in the pass that
  // reads them.  Of FP16 ones, at unit scale, most would round to zero before a
  // loss scaler's factor arrives: theirs is made in the backward, and rounded once
  // with the factor in it.
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &targets, const OptTensor &mask,
                               const OptTensor &old, const OptTensor &ref, const Tensor &adv, double low, double high,
                               double kl, int64_t reduction, double scale, bool want_grad) {
    const Tensor loss = fp32(logits, {}), lp = fp32(logits, targets.sizes());
    const bool later = want_grad && logits.scalar_type() == torch::kFloat16;
    Tensor grad, stats, coef;
    if (later) {
      stats = fp32(logits, {targets.size(0), targets.size(1), 2}), coef = fp32(logits, targets.sizes());
    } else if (want_grad) {
      grad = at::empty(logits.sizes(), logits.options());
    }
    const Rows r = rows_of(logits, targets, mask);
    const int64_t bytes = smx_policy_loss_workspace_bytes(r.batch, r.seq);
    const Tensor work = at::empty({bytes}, logits.options().dtype(torch::kUInt8));
    const c10::DeviceGuard guard(logits.device());
#define POLICY(r)                                                                                             \
  ROWS(r), ptr<float>(old), ptr<float>(ref), adv.data_ptr<float>(), adv.stride(0),                            \
      adv.dim() == 2 ? adv.stride(1) : 0, low, high, kl, static_cast<int>(reduction), scale, loss.data_ptr<float>(), \
      lp.data_ptr<float>()
    if (later) {
      check(smx_policy_loss_coef(POLICY(r), stats.data_ptr<float>(), coef.data_ptr<float>(), work.data_ptr(), bytes,
                                 stream_of(logits)),
            "smx_policy_loss_coef");
    } else {
      check(smx_policy_loss(POLICY(r), want_grad ? grad.data_ptr() : nullptr, work.data_ptr(), bytes, stream_of(logits)),
            "smx_policy_loss");
    }
#undef POLICY
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({lp});
    ctx->saved_data["later"] = later;
    if (later) {
      ctx->save_for_backward({logits, targets, mask.value_or(Tensor()), stats, coef});
    } else if (want_grad) {
      ctx->saved_data["grad"] = grad;
    }
    return {loss, lp};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    no_double_backward("policy_loss");
    variable_list out(12);
    if (!grads[0].defined()) return out;
    const Tensor scale = grads[0].to(torch::kFloat32);
    if (ctx->saved_data["later"].toBool()) {
      const auto s = ctx->get_saved_variables();
      out[0] = logprobs_backward(s[0], s[1], some(s[2]), s[3], s[4], s[4].stride(0), s[4].stride(1), scale);
      return out;
    }
    const auto it = ctx->saved_data.find("grad");
    TORCH_CHECK(it != ctx->saved_data.end(),
                "policy_loss: the gradient is made with the loss and handed out once; call policy_loss again to go "
                "through it a second time");
    out[0] = it->second.toTensor();
    ctx->saved_data.erase(it);
    const c10::DeviceGuard guard(out[0].device());
    check(smx_scale(out[0].data_ptr(), dtype_of(out[0]), out[0].numel(), scale.data_ptr<float>(), stream_of(out[0])),
          "smx_scale");
    return out;
  }
};

std::tuple<Tensor, Tensor> policy_loss(Tensor logits, Tensor targets, Tensor advantages, OptTensor old, OptTensor ref,
                                       OptTensor mask, double low, double high, double kl, int64_t reduction,
                                       double scale) {
  const char *what = "policy_loss";
  check_logits(what, &logits, &targets, &mask);
  TORCH_CHECK_VALUE(kl == 0 || ref.has_value(), what, ": kl_coef without ref_logprobs");
  old = token_floats(what, "old_logprobs", old, targets);
  ref = kl != 0 ? token_floats(what, "ref_logprobs", ref, targets) : std::nullopt;
  TORCH_CHECK_VALUE(advantages.is_floating_point() &&
                        (advantages.sizes() == targets.sizes() ||
                         (advantages.dim() == 1 && advantages.size(0) == targets.size(0))),
                    what, ": advantages ", advantages.sizes(), " ", advantages.scalar_type(),
                    "; expected floats [batch] or [batch, seq]");
  const OptTensor a = advantages;
  same_device(what, logits, {&a});
  const bool grad = torch::GradMode::is_enabled() && logits.requires_grad();
  const auto y = PolicyLoss::apply(logits, targets, mask, old, ref, advantages.detach().to(torch::kFloat32), low, high, kl,
                                   reduction, scale, grad);
  return {y[0], y[1]};
}

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &targets, const OptTensor &mask,
                               const Tensor &ref, double beta, double smoothing, bool want_grad) {
    const int64_t pairs = logits.size(0) / 2;
    const auto [lp, stats] = logprobs(logits, targets, mask, want_grad);
    const Tensor loss = fp32(logits, {}), margins = fp32(logits, {pairs}), coef = fp32(logits, {2 * pairs});
    const c10::DeviceGuard guard(logits.device());
    check(smx_preference_loss(lp.data_ptr<float>(), ref.data_ptr<float>(), ptr<uint8_t>(mask), pairs, logits.size(1), beta,
                              smoothing, loss.data_ptr<float>(), margins.data_ptr<float>(), coef.data_ptr<float>(),
                              stream_of(logits)),
          "smx_preference_loss");
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({margins});
    if (want_grad) ctx->save_for_backward({logits, targets, mask.value_or(Tensor()), stats, coef});
    return {loss, margins};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    no_double_backward("preference_loss");
    variable_list out(7);
    if (!grads[0].defined()) return out;
    const auto s = ctx->get_saved_variables();
    out[0] = logprobs_backward(s[0], s[1], some(s[2]), s[3], s[4], 1, 0, grads[0].to(torch::kFloat32));
    return out;
  }
};

std::tuple<Tensor, Tensor> preference_loss(Tensor logits, Tensor targets, OptTensor ref, OptTensor mask, double beta,
                                           double smoothing) {
  const char *what = "preference_loss";
  check_logits(what, &logits, &targets, &mask);
  TORCH_CHECK_VALUE(logits.size(0) % 2 == 0, what, ": ", logits.size(0), " sequences are no pairs");
  TORCH_CHECK_VALUE(ref.has_value(), what, ": ref_logprobs is needed");
  const bool grad = torch::GradMode::is_enabled() && logits.requires_grad();
  const auto y = PreferenceLoss::apply(logits, targets, mask, *token_floats(what, "ref_logprobs", ref, targets), beta,
                                       smoothing, grad);
  return {y[0], y[1]};
}

// ----------------------------------------------------------------- act8 ---
// A kept activation: codes [rows, pitch], then scale bytes [rows, pitch / 32].
struct Kept {
  Tensor data;
  int64_t rows, cols, pitch;
  // A new one for an activation like `x`.
  static Kept for_rows(const Tensor &x, int64_t rows, int64_t cols) {
    const int64_t pitch = (cols + 31) / 32 * 32;
    return {at::empty({rows * (pitch + pitch / 32)}, x.options().dtype(torch::kUInt8)), rows, cols, pitch};
  }
  // The one in `data`, of an activation of this shape.
  static Kept in(const Tensor &data, at::IntArrayRef shape) {
    TORCH_CHECK_VALUE(!shape.empty(), "a kept activation has at least one dimension");
    const int64_t rows = c10::multiply_integers(shape.slice(0, shape.size() - 1)), cols = shape.back();
    const int64_t pitch = (cols + 31) / 32 * 32;
    TORCH_CHECK_VALUE(data.is_cuda() && data.scalar_type() == torch::kUInt8 && data.is_contiguous() &&
                          data.numel() == rows * (pitch + pitch / 32),
                      "the bytes of a kept ", shape, ": ", data.sizes(), " ", data.scalar_type(), " on ", data.device());
    return {data, rows, cols, pitch};
  }
  uint8_t *codes() const { return data.data_ptr<uint8_t>(); }
  uint8_t *scales() const { return codes() + rows * pitch; }
};

// x as [rows, cols] with unit column stride (a copy where its strides allow no such view).
Tensor rows2d(const Tensor &x, const char *what) {
  need_float(x, what);
  TORCH_CHECK_VALUE(x.dim() >= 1, what, ": expected at least one dimension");
  const Tensor t = x.requires_grad() ? x.detach() : x;
  if (t.dim() == 2) return apart_rows(t);
  const int64_t cols = t.size(-1);
  return apart_rows(t.reshape({cols ? t.numel() / cols : c10::multiply_integers(t.sizes().slice(0, t.dim() - 1)), cols}));
}

int out_dtype(torch::ScalarType type) {
  switch (type) {
    case torch::kFloat32: return SMX_F32;
    case torch::kBFloat16: return SMX_BF16;
    case torch::kFloat16: return SMX_F16;
    default: TORCH_CHECK_VALUE(false, "unsupported dtype ", type, "; expected float32, bfloat16 or float16");
  }
}

Tensor act8_encode(const Tensor &x, int64_t fmt) {
  const Tensor r = rows2d(x, "act8.encode");
  const Kept k = Kept::for_rows(r, r.size(0), r.size(1));
  const c10::DeviceGuard guard(r.device());
  check(smx_act8_encode(r.data_ptr(), dtype_of(r), k.rows, k.cols, r.stride(0), static_cast<int>(fmt), k.codes(),
                        k.scales(), k.pitch, stream_of(r)),
        "smx_act8_encode");
  return k.data;
}

Tensor act8_decode(const Tensor &data, at::IntArrayRef shape, int64_t fmt, torch::ScalarType type) {
  const int code = out_dtype(type);
  const Kept k = Kept::in(data, shape);
  const Tensor out = at::empty(shape, data.options().dtype(type));
  const c10::DeviceGuard guard(data.device());
  check(smx_act8_decode(k.codes(), k.scales(), static_cast<int>(fmt), k.rows, k.cols, k.pitch, out.data_ptr(), code, k.cols,
                        stream_of(data)),
        "smx_act8_decode");
  return out;
}

std::tuple<Tensor, OptTensor, OptTensor> act8_gelu(const Tensor &h, int64_t fmt, bool keep_input, bool keep_output) {
  const Tensor r = rows2d(h, "act8.gelu_forward");
  const Tensor y = at::empty(h.sizes(), r.options());
  const int64_t rows = r.size(0), cols = r.size(1), pitch = (cols + 31) / 32 * 32;
  std::optional<Kept> kh, ky;
  if (keep_input) kh = Kept::for_rows(r, rows, cols);
  if (keep_output) ky = Kept::for_rows(r, rows, cols);
  const c10::DeviceGuard guard(r.device());
  check(smx_act8_gelu(r.data_ptr(), dtype_of(r), rows, cols, r.stride(0), static_cast<int>(fmt), y.data_ptr(), cols,
                      kh ? kh->codes() : nullptr, kh ? kh->scales() : nullptr, ky ? ky->codes() : nullptr,
                      ky ? ky->scales() : nullptr, pitch, stream_of(r)),
        "smx_act8_gelu");
  return {y, kh ? OptTensor(kh->data) : std::nullopt, ky ? OptTensor(ky->data) : std::nullopt};
}

Tensor act8_gelu_backward(const Tensor &dy, const Tensor &data, at::IntArrayRef shape, int64_t fmt) {
  const char *what = "act8.gelu_backward";
  const Tensor r = rows2d(dy, what);
  TORCH_CHECK_VALUE(dy.sizes() == shape, what, ": cotangent ", dy.sizes(), " of a kept ", shape);
  const OptTensor d = data;
  same_device(what, dy, {&d});
  const Kept k = Kept::in(data, shape);
  const Tensor dh = at::empty(dy.sizes(), r.options());
  const c10::DeviceGuard guard(r.device());
  check(smx_act8_gelu_backward(r.data_ptr(), dtype_of(r), k.rows, k.cols, r.stride(0), k.codes(), k.scales(),
                               static_cast<int>(fmt), k.pitch, dh.data_ptr(), k.cols, stream_of(r)),
        "smx_act8_gelu_backward");
  return dh;
}

std::tuple<Tensor, OptTensor> act8_linear_backward(const Tensor &delta, const Tensor &data, at::IntArrayRef shape,
                                                   int64_t fmt, std::optional<torch::ScalarType> type, bool bias) {
  const char *what = "act8.linear_backward";
  const Tensor r = rows2d(delta, what);
  TORCH_CHECK_VALUE(delta.dim() == static_cast<int64_t>(shape.size()) &&
                        delta.sizes().slice(0, delta.dim() - 1) == shape.slice(0, shape.size() - 1),
                    what, ": cotangent ", delta.sizes(), " of a kept input ", shape);
  const OptTensor d = data;
  same_device(what, delta, {&d});
  const auto out = r.options().dtype(type.value_or(r.scalar_type()));
  const int code = out_dtype(type.value_or(r.scalar_type()));
  const Kept k = Kept::in(data, shape);
  const int64_t n = r.size(1);
  const Tensor dw = at::empty({n, k.cols}, out);
  OptTensor db;
  if (bias) db = at::empty({n}, out);
  // (a refusal is the call's below)
  const int64_t bytes = std::max<int64_t>(0, smx_act8_wgrad_workspace_bytes(k.rows, n, k.cols, dtype_of(r)));
  const Tensor work = at::empty({bytes}, r.options().dtype(torch::kUInt8));
  const c10::DeviceGuard guard(r.device());
  check(smx_act8_wgrad(r.data_ptr(), dtype_of(r), k.rows, n, r.stride(0), k.codes(), k.scales(), static_cast<int>(fmt),
                       k.cols, k.pitch, dw.data_ptr(), ptr(db), code, work.data_ptr(), bytes, stream_of(r)),
        "smx_act8_wgrad");
  return {dw, db};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.attr("abi_version") = smx_abi_version();
  m.def("qk_norm_rotary", &qk_norm_rotary);
  m.def("token_logprobs", &token_logprobs);
  m.def("policy_loss", &policy_loss);
  m.def("preference_loss", &preference_loss);
  m.def("act8_encode", &act8_encode);
  m.def("act8_decode", &act8_decode);
  m.def("act8_gelu", &act8_gelu);
  m.def("act8_gelu_backward", &act8_gelu_backward);
  m.def("act8_linear_backward", &act8_linear_backward);
}
