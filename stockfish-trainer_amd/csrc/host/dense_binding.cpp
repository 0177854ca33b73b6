// The dense head's operators for eager torch programs: argument checks, workspaces,
// streams and autograd nodes in C++ over the C ABI (include/sft_ft.h).
//
// Calls for a few positions, and steps of small batches, take less time on the GPU
// than their host work in Python does: a ctypes call, its checks and a Python autograd
// function came to 13 us for one row and to 150 us for a small training step, most of
// it in handing Python's lock to the autograd thread and back.  Programs that are
// being compiled use the operators in src/model/modules/dense/ops.py instead.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <cmath>
#include <string>

#include "sft_ft.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A refused argument, as the package's Python checks report it.
void require(bool ok, const char *what, PyObject *type = PyExc_AssertionError) {
  if (ok) return;
  PyErr_SetString(type, what);
  throw py::error_already_set();
}
void check(int rc, const char *what) {
  TORCH_CHECK(rc == SFT_OK, what, " failed (code ", rc, "): ", sft_last_error());
}

int type_code(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return SFT_TYPE_F32;
    case at::kHalf:
      return SFT_TYPE_F16;
    case at::kBFloat16:
      return SFT_TYPE_BF16;
    default:
      return -1;
  }
}
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *stream(const Tensor &t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
Tensor empty(at::IntArrayRef size, const Tensor &like, at::ScalarType type) {
  return at::empty(size, like.options().dtype(type).requires_grad(false));
}

// A 2-D tensor's row stride; a tensor of one row or column has any.
int64_t rows_of(const Tensor &t) {
  const int64_t cols = t.size(1), ld = t.stride(0);
  return t.size(0) > 1 && ld >= cols ? ld : cols;
}
// t, or a copy where its rows are not dense, overlap or lie in descending order.
Tensor dense_rows(const Tensor &t) {
  if (!t.defined() || t.is_contiguous()) return t;
  const int64_t rows = t.size(0), cols = t.size(1);
  if ((cols == 1 || t.stride(1) == 1) && (rows == 1 || t.stride(0) >= cols)) return t;
  return t.contiguous();
}
// Whether products read the matrix where it lies.
bool in_place(const Tensor &t) {
  const int64_t stride = rows_of(t) * (int64_t)t.element_size();
  return ((uintptr_t)t.data_ptr() | (uintptr_t)stride) % 16 == 0 && stride <= ((int64_t)1 << 23);
}

struct Workspace {
  Tensor buffer;
  size_t bytes = 0;
  void take(const Tensor &like) {
    if (bytes) buffer = empty({(int64_t)bytes}, like, at::kByte);
  }
  void *at() const { return ptr(buffer); }
};

// A backward that is not differentiable itself: asking for its derivative is an error.
variable_list once(variable_list grads, const char *name) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list inputs;
  for (Tensor &g : grads)
    if (g.defined()) inputs.push_back(g.detach().set_requires_grad(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " is differentiable once only", (int64_t)inputs.size());
  inputs = (*error)(std::move(inputs));
  size_t i = 0;
  for (Tensor &g : grads)
    if (g.defined()) g = inputs[i++];
  return grads;
}

// ---- linear ----
void linear_forward(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &r, int64_t act, const Tensor &y,
                    const Tensor &deriv) {
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  const int type = type_code(x);
  Workspace ws;
  check(sft_linear_fwd_workspace_size(type, M, K, N, in_place(x) && in_place(w) ? 0 : SFT_LINEAR_COPY, &ws.bytes),
        "sft_linear_fwd_workspace_size");
  ws.take(x);
  check(sft_linear_fwd(type, x.data_ptr(), rows_of(x), w.data_ptr(), rows_of(w), ptr(b), ptr(r),
                       r.defined() ? rows_of(r) : 0, y.data_ptr(), N, ptr(deriv), M, K, N, (int32_t)act, ws.at(),
                       ws.bytes, stream(x)),
        "sft_linear_fwd");
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x_, const Tensor &w_, const std::optional<Tensor> &bias,
                        const std::optional<Tensor> &residual, int64_t act) {
    const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
    const Tensor x = dense_rows(x_), w = dense_rows(w_);
    const bool need_x = x_.requires_grad(), need_w = w_.requires_grad(), need_b = b.defined() && b.requires_grad();
    const Tensor y = empty({x.size(0), w.size(0)}, x, x.scalar_type());
    Tensor deriv;
    if (act != SFT_ACT_NONE && (need_x || need_w || need_b))
      deriv = empty(y.sizes(), x, x.scalar_type() == at::kFloat ? at::kFloat : at::kShort);
    linear_forward(x, w, b.defined() ? b.contiguous() : b, dense_rows(r), act, y, deriv);
    ctx->save_for_backward({x, w, deriv});
    ctx->saved_data["act"] = act;
    ctx->saved_data["need"] = (int64_t)(need_x | need_w << 1 | need_b << 2 | (r.defined() && r.requires_grad()) << 3);
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &deriv = saved[2];
    const int64_t act = ctx->saved_data["act"].toInt(), need = ctx->saved_data["need"].toInt();
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    Tensor dx, dw, db;
    if (need & 7) {
      const c10::OptionalDeviceGuard guard(x.device());
      const Tensor dy = dense_rows(grads[0]);
      if (need & 1) dx = empty({M, K}, x, x.scalar_type());
      if (need & 2) dw = empty({N, K}, x, x.scalar_type());
      if (need & 4) db = empty({N}, x, x.scalar_type());
      const int type = type_code(x);
      Workspace ws;
      check(sft_linear_bwd_workspace_size(type, M, K, N, (int32_t)act,
                                          in_place(dy) && in_place(x) && in_place(w) ? 0 : SFT_LINEAR_COPY, &ws.bytes),
            "sft_linear_bwd_workspace_size");
      ws.take(x);
      check(sft_linear_bwd(type, dy.data_ptr(), rows_of(dy), ptr(deriv), x.data_ptr(), rows_of(x), w.data_ptr(),
                           rows_of(w), ptr(dx), ptr(dw), ptr(db), M, K, N, (int32_t)act, ws.at(), ws.bytes, stream(x)),
            "sft_linear_bwd");
    }
    return once({dx, dw, db, need & 8 ? grads[0] : Tensor(), Tensor()}, "fused_linear");
  }
};

Tensor linear(const Tensor &x, const Tensor &w, const std::optional<Tensor> &bias,
              const std::optional<Tensor> &residual, int64_t act) {
  const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
  require(x.is_cuda() && type_code(x) >= 0, "x must be a float32, float16 or bfloat16 CUDA tensor");
  require(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1) && w.size(0) > 0 && w.size(1) > 0,
          "x must be [..., K] and weight [N, K], K and N at least 1");
  const int64_t K = w.size(1), N = w.size(0);
  for (const Tensor *t : {&w, &b, &r})
    require(!t->defined() || (t->device() == x.device() && t->scalar_type() == x.scalar_type()),
            "weight, bias and residual must be on x's device and of its type");
  require(!b.defined() || (b.dim() == 1 && b.size(0) == N), "bias must be [N]");
  if (r.defined()) {
    auto shape = x.sizes().vec();
    shape.back() = N;
    require(r.sizes() == at::IntArrayRef(shape), "residual must be [..., N]");
  }
  const c10::OptionalDeviceGuard guard(x.device());
  const bool flat = x.dim() == 2;
  const Tensor x2 = flat ? x : x.reshape({-1, K}), r2 = flat || !r.defined() ? r : r.reshape({-1, N});
  Tensor y;
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (b.defined() && b.requires_grad()) ||
                                     (r.defined() && r.requires_grad()))) {
    y = LinearFunction::apply(x2, w, bias, r2.defined() ? std::optional<Tensor>(r2) : std::nullopt, act);
  } else {
    y = empty({x2.size(0), N}, x, x.scalar_type());
    linear_forward(dense_rows(x2), dense_rows(w), b.defined() ? b.contiguous() : b, dense_rows(r2), act, y, Tensor());
  }
  if (flat) return y;
  auto shape = x.sizes().vec();
  shape.back() = N;
  return y.view(shape);
}

// ---- balance ----
struct BalanceFunction : torch::autograd::Function<BalanceFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits_, const std::optional<Tensor> &mask_,
                               int64_t top_k) {
    const Tensor mask = mask_.value_or(Tensor());
    const Tensor logits = dense_rows(logits_);
    const int type = type_code(logits);
    const int32_t E = (int32_t)logits.size(1);
    Workspace ws;
    check(sft_balance_fwd_workspace_size(type, logits.size(0), E, &ws.bytes), "sft_balance_fwd_workspace_size");
    ws.take(logits);
    const Tensor loss = empty({}, logits, at::kFloat), counts = empty({E}, logits, at::kLong),
                 kept = empty({}, logits, at::kLong);
    check(sft_balance_fwd(type, logits.data_ptr(), rows_of(logits), static_cast<uint8_t *>(ptr(mask)), logits.size(0),
                          E, (int32_t)top_k, loss.data_ptr<float>(), counts.data_ptr<int64_t>(),
                          kept.data_ptr<int64_t>(), ws.at(), ws.bytes, stream(logits)),
          "sft_balance_fwd");
    if (ctx) {
      ctx->save_for_backward({logits, mask, counts, kept});
      ctx->saved_data["top_k"] = top_k;
      ctx->mark_non_differentiable({counts});
    }
    return {loss, counts};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &mask = saved[1];
    const c10::OptionalDeviceGuard guard(logits.device());
    const Tensor grad = grads[0].to(at::kFloat), out = empty(logits.sizes(), logits, logits.scalar_type());
    check(sft_balance_bwd(type_code(logits), logits.data_ptr(), rows_of(logits), static_cast<uint8_t *>(ptr(mask)),
                          logits.size(0), (int32_t)logits.size(1), (int32_t)ctx->saved_data["top_k"].toInt(),
                          saved[2].data_ptr<int64_t>(), saved[3].data_ptr<int64_t>(), grad.data_ptr<float>(),
                          out.data_ptr(), stream(logits)),
          "sft_balance_bwd");
    return once({out, Tensor(), Tensor()}, "expert_balance");
  }
};

py::tuple balance(const Tensor &logits, int64_t top_k, const std::optional<Tensor> &mask_) {
  Tensor mask = mask_.value_or(Tensor());
  require(logits.is_cuda() && type_code(logits) >= 0 && logits.dim() >= 1,
          "logits must be a float32, float16 or bfloat16 CUDA tensor [..., E]");
  const int64_t E = logits.size(-1);
  require(E >= 1 && E <= SFT_BALANCE_MAX_EXPERTS, "the number of experts must be in [1, 1024]");
  require(top_k >= 1 && top_k <= E, "top_k must be in [1, E]");
  if (mask.defined()) {
    require(mask.scalar_type() == at::kBool && mask.device() == logits.device(), "mask must be bool, on logits' device");
    require(mask.sizes() == logits.sizes().slice(0, logits.dim() - 1), "mask must be logits' shape without the last");
    mask = mask.reshape({-1}).contiguous();
  }
  const c10::OptionalDeviceGuard guard(logits.device());
  const Tensor flat = logits.dim() == 2 ? logits : logits.reshape({-1, E});
  const std::optional<Tensor> kept = mask.defined() ? std::optional<Tensor>(mask) : std::nullopt;
  const variable_list out = at::GradMode::is_enabled() && logits.requires_grad()
                                ? BalanceFunction::apply(flat, kept, top_k)
                                : BalanceFunction::forward(nullptr, flat, kept, top_k);
  return py::make_tuple(out[0], out[1]);
}

// ---- distillation ----
void distill_call(const Tensor &s, const Tensor &t, const Tensor &i, double tau, const Tensor &weight,
                  const Tensor &loss, const Tensor &grad) {
  check(sft_distill(type_code(s), s.data_ptr(), rows_of(s), type_code(t), t.data_ptr(), i.data_ptr(),
                    (int32_t)i.element_size(), s.size(0), s.size(1), (int32_t)t.size(1), (float)tau,
                    static_cast<float *>(ptr(weight)), static_cast<float *>(ptr(loss)), ptr(grad), stream(s)),
        "sft_distill");
}

struct DistillFunction : torch::autograd::Function<DistillFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &s_, const Tensor &t, const Tensor &i, double tau) {
    const Tensor s = dense_rows(s_), loss = empty({s.size(0)}, s, at::kFloat);
    distill_call(s, t, i, tau, Tensor(), loss, Tensor());
    if (ctx) {
      ctx->save_for_backward({s, t, i});
      ctx->saved_data["tau"] = tau;
    }
    return loss;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &s = saved[0];
    const c10::OptionalDeviceGuard guard(s.device());
    const Tensor grad = empty(s.sizes(), s, s.scalar_type());
    distill_call(s, saved[1], saved[2], ctx->saved_data["tau"].toDouble(), grads[0].to(at::kFloat).contiguous(),
                 Tensor(), grad);
    return once({grad, Tensor(), Tensor(), Tensor()}, "distill_loss");
  }
};

void distill_checks(const Tensor &s, const Tensor &t, const Tensor &i, double tau) {
  require(s.is_cuda() && s.dim() == 2 && s.size(1) >= 1 && type_code(s) >= 0,
          "student logits must be a float32, float16 or bfloat16 CUDA tensor [R, V]");
  require(type_code(t) >= 0 && (i.scalar_type() == at::kInt || i.scalar_type() == at::kLong),
          "teacher logits must be float32, float16 or bfloat16, their indices int32 or int64");
  require(t.dim() == 2 && t.sizes() == i.sizes() && t.size(0) == s.size(0) && t.size(1) >= 1 &&
              t.size(1) <= SFT_DISTILL_MAX_K,
          "teacher logits and indices must be [R, k], k in [1, 256]");
  require(t.device() == s.device() && i.device() == s.device(), "teacher tensors must be on the student's device");
  require(tau > 0 && std::isfinite(tau), "temperature must be positive and finite", PyExc_ValueError);
}

Tensor distill_loss(const Tensor &s, const Tensor &t, const Tensor &i, double tau) {
  distill_checks(s, t, i, tau);
  const c10::OptionalDeviceGuard guard(s.device());
  const Tensor td = t.detach().contiguous(), id = i.contiguous();
  if (at::GradMode::is_enabled() && s.requires_grad()) return DistillFunction::apply(s, td, id, tau);
  return DistillFunction::forward(nullptr, s, td, id, tau);
}

py::tuple distill_loss_and_grad(const Tensor &s_, const Tensor &t, const Tensor &i,
                                const std::optional<Tensor> &weight_, double tau) {
  distill_checks(s_, t, i, tau);
  Tensor weight = weight_.value_or(Tensor());
  if (weight.defined()) {
    require(weight.dim() == 1 && weight.size(0) == s_.size(0) && weight.scalar_type() == at::kFloat,
            "row_weight must be float32 [R]");
    require(weight.device() == s_.device(), "row_weight must be on the student's device");
    weight = weight.detach().contiguous();
  }
  const c10::OptionalDeviceGuard guard(s_.device());
  const Tensor s = dense_rows(s_.detach());
  const Tensor loss = empty({s.size(0)}, s, at::kFloat), grad = empty(s.sizes(), s, s.scalar_type());
  distill_call(s, t.detach().contiguous(), i.contiguous(), tau, weight, loss, grad);
  return py::make_tuple(loss, grad);
}

}  // namespace

PYBIND11_MODULE(_sft_dense, m) {
  m.def("linear", &linear);
  m.def("balance", &balance);
  m.def("distill_loss", &distill_loss);
  m.def("distill_loss_and_grad", &distill_loss_and_grad);
}
