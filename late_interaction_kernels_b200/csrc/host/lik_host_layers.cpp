// Native host path of the layers in front of the document head (layer_norm, linear, gated_feed_forward): checks of the
// arguments, launches, and the autograd nodes.
#include "lik_host.h"

#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <mutex>
#include <sstream>

namespace lik_host {

namespace {

using OptTensor = std::optional<Tensor>;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using Named = std::initializer_list<std::pair<const char*, const Tensor*>>;

[[noreturn]] void value_error(const std::string& what) { throw pybind11::value_error(what); }
Tensor opt(const OptTensor& t) { return t ? *t : Tensor(); }
template <typename T = void>
T* ptr(const Tensor& t) {
  return t.defined() && t.numel() ? (T*)t.data_ptr() : nullptr;
}
std::string shape(at::IntArrayRef s) {
  std::ostringstream o;
  o << s;
  return o.str();
}
bool float_type(at::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

// all on x's GPU, in a type that has kernels, no tangents
void require_layer_inputs(const char* op, const Tensor& x, Named others) {
  if (!x.is_cuda()) throw std::runtime_error(std::string(op) + " requires CUDA tensors; got a tensor on " + x.device().str() + ". There is no CPU fallback.");
  if (!float_type(x.scalar_type())) value_error(std::string(op) + ": dtype " + c10::toString(x.scalar_type()) + " is not supported (float32, float16, bfloat16)");
  if (x.dim() < 1) value_error("x must have at least one dimension");
  TORCH_CHECK_NOT_IMPLEMENTED(!x._fw_grad(0).defined(), op, " has no forward-mode derivative.");
  for (const auto& [name, t] : others) {
    if (!t->defined()) continue;
    if (t->device() != x.device()) value_error(std::string(name) + " must be on the same device as x; got " + t->device().str() + " vs " + x.device().str() + ".");
    if (!float_type(t->scalar_type())) value_error(std::string(name) + ": dtype " + c10::toString(t->scalar_type()) + " is not supported (float32, float16, bfloat16)");
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), op, " has no forward-mode derivative.");
  }
}
void require_vector(const char* name, const Tensor& t, int64_t n) {
  if (t.defined() && (t.dim() != 1 || t.size(0) != n)) value_error(std::string(name) + " must be [" + std::to_string(n) + "]; got " + shape(t.sizes()));
}
constexpr int64_t FEATURES_END = int64_t(1) << 30;  // (the kernels count features in 32 bits)
void require_features(const Tensor& x) {
  if (x.size(-1) < 1 || x.size(-1) >= FEATURES_END) value_error("x must have at least one feature, and less than 2^30; got " + shape(x.sizes()));
}
void require_matrix(const char* name, const Tensor& t, int64_t rows, const char* cols_name, int64_t cols) {
  if (t.dim() == 2 && t.size(0) >= FEATURES_END) value_error(std::string(name) + " must have less than 2^30 rows; got " + shape(t.sizes()));
  if (t.dim() != 2 || t.size(1) != cols || (rows >= 0 && t.size(0) != rows) || t.size(0) < 1)
    value_error(std::string(name) + " must be [" + (rows >= 0 ? std::to_string(rows) : "features >= 1") + ", " + cols_name + "=" + std::to_string(cols) + "]; got " + shape(t.sizes()));
}
void require_residual(const Tensor& residual, const Tensor& x, int64_t out) {
  if (!residual.defined()) return;
  auto want = x.sizes().vec();
  want.back() = out;
  if (residual.sizes() != at::IntArrayRef(want)) value_error("residual must have the result's shape " + shape(want) + "; got " + shape(residual.sizes()));
}
int activation_code(const std::optional<std::string>& name) {
  static const std::pair<const char*, int> known[] = {{"relu", LIK_ACT_RELU}, {"silu", LIK_ACT_SILU}, {"gelu", LIK_ACT_GELU}, {"gelu_tanh", LIK_ACT_GELU_TANH},
                                                      {"tanh", LIK_ACT_TANH}, {"sigmoid", LIK_ACT_SIGMOID}};
  if (!name) return LIK_ACT_NONE;
  for (const auto& [n, code] : known)
    if (*name == n) return code;
  value_error("activation must be None, 'relu', 'silu', 'gelu', 'gelu_tanh', 'tanh' or 'sigmoid'; got '" + *name + "'");
}

// [.., n] -> [rows, n] with unit stride inside a row and rows that do not overlap; a copy (inside the graph) only where it has to be
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / std::max<int64_t>(t.size(-1), 1), t.size(-1)});
  return (r.size(1) > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < r.size(1)) ? r.contiguous() : r;
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? std::max(t.stride(0), t.size(1)) : t.size(1); }
// as the kernels read it: in the call's type (fp32 weights have to be, as the tensor core's operands; biases and residuals are with them, so that a call
// has one type and one epilogue: half a step of a term that is added to a sum which is rounded to the same type), unit stride inside rows that do not overlap
Tensor as_rows(const Tensor& t, at::ScalarType dt) {
  if (!t.defined()) return t;
  Tensor r = t.scalar_type() == dt ? t : t.to(dt);
  if (r.dim() == 1) return r.contiguous();
  return rows_of(r);
}
// matrices that kernels write and read again, one behind the other: rows that start on 16 bytes
Tensor kept_rows(int64_t n, int64_t rows, int64_t cols, const Tensor& like) {
  const int64_t v = 16 / (int64_t)like.element_size();
  return at::empty({n, rows, (cols + v - 1) / v * v}, like.options());
}
void* matrix_of(const Tensor& kept, int64_t i) { return kept.numel() ? (char*)kept.data_ptr() + i * kept.stride(0) * kept.element_size() : nullptr; }
struct Workspace {
  Tensor t;
  void* p = nullptr;
  size_t bytes = 0;
  Workspace(size_t n, const at::Device& dev) : bytes(n) {
    if (!n) return;
    t = at::empty({(int64_t)n}, at::TensorOptions().device(dev).dtype(at::kByte));
    p = t.data_ptr();
  }
};

// Gradients are taken in the call's type where all parameters have it, in fp32 otherwise, and handed over in each parameter's own.
int param_dtype(at::ScalarType dt, std::initializer_list<const Tensor*> params) {
  for (const Tensor* p : params)
    if (p->defined() && p->scalar_type() != dt) return LIK_F32;
  return dtype_code(dt);
}
at::ScalarType scalar_of(int code) { return code == LIK_F32 ? at::kFloat : (code == LIK_F16 ? at::kHalf : at::kBFloat16); }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// A leaf's gradient accumulator belongs to the stream on which the first live graph of that leaf was built.  A backward pass that is being
// captured waits for that stream and draws it into the capture, which the legacy default stream cannot be: CUDA ends the capture in the
// engine's thread, where the error ends the process.  So the call says so before anything is recorded.
void refuse_foreign_accumulators(const char* op, std::initializer_list<const Tensor*> ts) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  for (const Tensor* t : ts) {
    if (!t->defined() || !t->requires_grad() || t->grad_fn()) continue;
    const auto acc = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto made = acc ? acc->stream() : std::nullopt;
    if (made && c10::cuda::CUDAStream(*made).stream() == nullptr)
      throw std::runtime_error(std::string(op) + ": a graph of the same leaf tensors, built on the default stream, is still alive; drop it (the loss or output that holds it) "
                               "before this call is captured into a CUDA graph.");
  }
}
// gradients of gradients do not exist: whoever differentiates the returned gradients is told so
variable_list once(variable_list&& grads, const char* op) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  variable_list out(grads.size());
  for (size_t i = 0; i < grads.size(); ++i)
    if (grads[i].defined()) {
      auto err = std::make_shared<torch::autograd::DelayedError>(std::string(op) + " has no second derivative.", 1);
      out[i] = err->apply({grads[i].detach().requires_grad_(true)})[0];
    }
  return out;
}

// ---------------------------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------------------------
// weight and bias as the kernels read them: both in the call's type or both in fp32
std::pair<Tensor, Tensor> norm_params(const Tensor& w, const Tensor& b, at::ScalarType dt) {
  const auto pt = scalar_of(param_dtype(dt, {&w, &b}));
  return {as_rows(w, pt), as_rows(b, pt)};
}
lik_norm_args norm_args(const Tensor& x, const Tensor& w, const Tensor& b, double eps) {
  lik_norm_args a{};
  a.x = ptr(x);
  a.x_stride = row_stride(x);
  a.rows = x.size(0);
  a.width = (int32_t)x.size(1);
  a.dtype = dtype_code(x.scalar_type());
  a.weight = ptr(w);
  a.bias = ptr(b);
  a.param_dtype = w.defined() ? dtype_code(w.scalar_type()) : (b.defined() ? dtype_code(b.scalar_type()) : a.dtype);
  a.eps = (float)eps;
  return a;
}

struct LayerNormBackward : public torch::autograd::Node {
  SavedVariable x, w, b, stats;
  at::ScalarType w_type = at::kFloat, b_type = at::kFloat;
  double eps = 0;

  std::string name() const override { return "LayerNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&x, &w, &b, &stats}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(3);
    if (!grads[0].defined()) return out;
    const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
    Tensor X, W, B, S;
    {
      // (before the autograd keys are switched off: unpacking may run the caller's hooks)
      const std::lock_guard<std::mutex> lock(mutex_);
      X = x.unpack();
      W = w.unpack();
      B = b.unpack();
      S = stats.unpack();
    }
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::cuda::CUDAGuard guard(X.device());
      const auto dt = X.scalar_type();
      const Tensor dy = grads[0].contiguous();
      auto [pw, pb] = norm_params(W, B, dt);
      X = as_rows(X, dt);
      lik_norm_args a = norm_args(X, pw, pb, eps);
      const auto popt = X.options().dtype(scalar_of(a.param_dtype));
      a.mean = ptr<float>(S);
      a.rstd = a.mean ? a.mean + X.size(0) : nullptr;
      a.dy = ptr(dy);
      if (need_x) out[0] = at::empty(X.sizes(), X.options());
      if (need_w) out[1] = at::empty({X.size(1)}, popt);
      if (need_b) out[2] = at::empty({X.size(1)}, popt);
      a.dx = ptr(out[0]);
      a.dweight = ptr(out[1]);
      a.dbias = ptr(out[2]);
      const Workspace ws(lik_layer_norm_bwd_workspace(&a), X.device());
      a.workspace = ws.p;
      a.workspace_bytes = ws.bytes;
      check(lik_layer_norm_bwd(&a, c10::cuda::getCurrentCUDAStream(X.device().index()).stream()), "lik_layer_norm_bwd");
      if (need_w) out[1] = out[1].to(w_type);
      if (need_b) out[2] = out[2].to(b_type);
    }
    return once(std::move(out), "layer_norm");
  }
};

Tensor layer_norm(const Tensor& x_, const OptTensor& weight_, const OptTensor& bias_, double eps) {
  const Tensor w = opt(weight_), b = opt(bias_);
  require_layer_inputs("layer_norm", x_, {{"weight", &w}, {"bias", &b}});
  const int64_t width = x_.size(-1);
  require_features(x_);
  require_vector("weight", w, width);
  require_vector("bias", b, width);
  if (!(eps >= 0) || eps > 3e38) value_error("eps must be a number that is not negative; got " + std::to_string(eps));
  const Tensor x = rows_of(x_);
  const c10::cuda::CUDAGuard guard(x.device());
  const bool grad = wants_grad({&x, &w, &b});
  if (grad) refuse_foreign_accumulators("layer_norm", {&x_, &w, &b});
  Tensor y, stats;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    auto [pw, pb] = norm_params(w, b, x.scalar_type());
    lik_norm_args a = norm_args(x, pw, pb, eps);
    y = at::empty(x.sizes(), x.options());
    a.y = ptr(y);
    if (grad) {
      stats = at::empty({2, x.size(0)}, x.options().dtype(at::kFloat));
      a.mean = ptr<float>(stats);
      a.rstd = a.mean ? a.mean + x.size(0) : nullptr;
    }
    check(lik_layer_norm_fwd(&a, c10::cuda::getCurrentCUDAStream(x.device().index()).stream()), "lik_layer_norm_fwd");
  }
  if (grad) {
    auto node = std::shared_ptr<LayerNormBackward>(new LayerNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    node->x = SavedVariable(x, false);
    node->w = SavedVariable(w, false);
    node->b = SavedVariable(b, false);
    node->stats = SavedVariable(stats, false);
    if (w.defined()) node->w_type = w.scalar_type();
    if (b.defined()) node->b_type = b.scalar_type();
    node->eps = eps;
    torch::autograd::set_history(y, node);
  }
  return x_.dim() == 2 ? y : y.view(x_.sizes());
}

// ---------------------------------------------------------------------------------------------
// linear
// ---------------------------------------------------------------------------------------------
lik_linear_args linear_args(const Tensor& x, const Tensor& w, int act) {
  lik_linear_args a{};
  a.x = ptr(x);
  a.x_stride = row_stride(x);
  a.w = ptr(w);
  a.w_stride = row_stride(w);
  a.rows = x.size(0);
  a.in = (int32_t)x.size(1);
  a.out = (int32_t)w.size(0);
  a.dtype = a.param_dtype = dtype_code(x.scalar_type());
  a.activation = act;
  a.status = status_ptr(x.device());
  return a;
}

struct LinearBackward : public torch::autograd::Node {
  SavedVariable x, w, z;
  at::ScalarType w_type = at::kFloat, b_type = at::kFloat;
  int act = LIK_ACT_NONE, grad_type = LIK_F32;

  std::string name() const override { return "LinearBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&x, &w, &z}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
    Tensor X, W, Z;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      X = x.unpack();
      W = w.unpack();
      Z = z.unpack();
    }
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::cuda::CUDAGuard guard(X.device());
      const auto dt = X.scalar_type();
      X = as_rows(X, dt);
      W = as_rows(W, dt);
      const Tensor dy = rows_of(grads[0]);
      lik_linear_args a = linear_args(X, W, act);
      a.param_dtype = grad_type;
      const auto popt = X.options().dtype(scalar_of(grad_type));
      a.z = ptr(Z);
      a.z_stride = Z.defined() ? Z.size(2) : 0;
      a.dy = ptr(dy);
      a.dy_stride = row_stride(dy);
      if (need_x) out[0] = at::empty(X.sizes(), X.options());
      if (need_w) out[1] = at::empty(W.sizes(), popt);
      if (need_b) out[2] = at::empty({W.size(0)}, popt);
      a.dx = ptr(out[0]);
      a.dw = ptr(out[1]);
      a.dbias = ptr(out[2]);
      const Workspace ws(lik_linear_bwd_workspace(&a), X.device());
      a.workspace = ws.p;
      a.workspace_bytes = ws.bytes;
      check(lik_linear_bwd(&a, c10::cuda::getCurrentCUDAStream(X.device().index()).stream()), "lik_linear_bwd");
      if (need_w) out[1] = out[1].to(w_type);
      if (need_b) out[2] = out[2].to(b_type);
      if (task_should_compute_output(3)) out[3] = grads[0];
    }
    return once(std::move(out), "linear");
  }
};

Tensor linear(const Tensor& x_, const Tensor& w, const OptTensor& bias_, const std::optional<std::string>& activation, const OptTensor& residual_) {
  const Tensor b = opt(bias_), r_ = opt(residual_);
  require_layer_inputs("linear", x_, {{"weight", &w}, {"bias", &b}, {"residual", &r_}});
  const int64_t in = x_.size(-1);
  require_features(x_);
  require_matrix("weight", w, -1, "in_features", in);
  const int64_t out = w.size(0);
  require_vector("bias", b, out);
  require_residual(r_, x_, out);
  const int act = activation_code(activation);
  const auto dt = x_.scalar_type();
  const Tensor x = rows_of(x_);
  const Tensor r = r_.defined() ? rows_of(r_.scalar_type() == dt ? r_ : r_.to(dt)) : r_;
  const c10::cuda::CUDAGuard guard(x.device());
  const bool grad = wants_grad({&x, &w, &b, &r});
  if (grad) refuse_foreign_accumulators("linear", {&x_, &w, &b, &r_});
  Tensor y, z, pw;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    pw = as_rows(w, dt);
    const Tensor pb = as_rows(b, dt);
    lik_linear_args a = linear_args(x, pw, act);
    a.bias = ptr(pb);
    a.residual = ptr(r);
    a.residual_stride = r.defined() ? row_stride(r) : 0;
    y = at::empty({x.size(0), out}, x.options());
    a.y = ptr(y);
    if (act != LIK_ACT_NONE && wants_grad({&x, &w, &b})) {  // (a residual's gradient is dy)
      z = kept_rows(1, x.size(0), out, x);
      a.z = ptr(z);
      a.z_stride = z.size(2);
    }
    const Workspace ws(lik_linear_fwd_workspace(&a), x.device());
    a.workspace = ws.p;
    a.workspace_bytes = ws.bytes;
    check(lik_linear_fwd(&a, c10::cuda::getCurrentCUDAStream(x.device().index()).stream()), "lik_linear_fwd");
  }
  if (grad) {
    auto node = std::shared_ptr<LinearBackward>(new LinearBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b, r));
    node->x = SavedVariable(x, false);
    node->w = SavedVariable(w.scalar_type() == dt ? w : pw, false);
    node->z = SavedVariable(z, false);
    node->w_type = w.scalar_type();
    if (b.defined()) node->b_type = b.scalar_type();
    node->act = act;
    node->grad_type = param_dtype(dt, {&w, &b});
    torch::autograd::set_history(y, node);
  }
  if (x_.dim() == 2) return y;
  auto sizes = x_.sizes().vec();
  sizes.back() = out;
  return y.view(sizes);
}

// ---------------------------------------------------------------------------------------------
// gated feed-forward block
// ---------------------------------------------------------------------------------------------
lik_gated_args gated_args(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int act) {
  lik_gated_args a{};
  a.x = ptr(x);
  a.x_stride = row_stride(x);
  a.w_gate = ptr(wg);
  a.w_gate_stride = row_stride(wg);
  a.w_up = ptr(wu);
  a.w_up_stride = row_stride(wu);
  a.w_down = ptr(wd);
  a.w_down_stride = row_stride(wd);
  a.rows = x.size(0);
  a.in = (int32_t)x.size(1);
  a.hidden = (int32_t)wg.size(0);
  a.out = (int32_t)wd.size(0);
  a.dtype = a.param_dtype = dtype_code(x.scalar_type());
  a.activation = act;
  a.status = status_ptr(x.device());
  return a;
}
constexpr int N_GATED_PARAMS = 6;  // w_gate, w_up, w_down, b_gate, b_up, b_down

struct GatedFeedForwardBackward : public torch::autograd::Node {
  SavedVariable x, wg, wu, wd, kept;  // kept: the factors of the gradients of gate and up, and h
  std::array<at::ScalarType, N_GATED_PARAMS> types{};
  int act = LIK_ACT_NONE, grad_type = LIK_F32;

  std::string name() const override { return "GatedFeedForwardBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* v : {&x, &wg, &wu, &wd, &kept}) v->reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    variable_list out(2 + N_GATED_PARAMS);
    if (!grads[0].defined()) return out;
    Tensor X, WG, WU, WD, K;
    {
      const std::lock_guard<std::mutex> lock(mutex_);
      X = x.unpack();
      WG = wg.unpack();
      WU = wu.unpack();
      WD = wd.unpack();
      K = kept.unpack();
    }
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const c10::cuda::CUDAGuard guard(X.device());
      const auto dt = X.scalar_type();
      X = as_rows(X, dt);
      WG = as_rows(WG, dt);
      WU = as_rows(WU, dt);
      WD = as_rows(WD, dt);
      const Tensor dy = rows_of(grads[0]);
      lik_gated_args a = gated_args(X, WG, WU, WD, act);
      a.param_dtype = grad_type;
      const auto popt = X.options().dtype(scalar_of(grad_type));
      if (K.defined()) {
        a.gate_factor = matrix_of(K, 0);
        a.up_factor = matrix_of(K, 1);
        a.h = matrix_of(K, 2);
        a.kept_stride = K.size(2);
      }
      a.dy = ptr(dy);
      a.dy_stride = row_stride(dy);
      if (task_should_compute_output(0)) out[0] = at::empty(X.sizes(), X.options());
      a.dx = ptr(out[0]);
      const int64_t f = WG.size(0), in = WG.size(1), o = WD.size(0);
      void** const to[N_GATED_PARAMS] = {&a.dw_gate, &a.dw_up, &a.dw_down, &a.db_gate, &a.db_up, &a.db_down};
      const std::vector<int64_t> sizes[N_GATED_PARAMS] = {{f, in}, {f, in}, {o, f}, {f}, {f}, {o}};
      for (int i = 0; i < N_GATED_PARAMS; ++i)
        if (task_should_compute_output(1 + i)) {
          out[1 + i] = at::empty(sizes[i], popt);
          *to[i] = ptr(out[1 + i]);
        }
      const Workspace ws(lik_gated_bwd_workspace(&a), X.device());
      a.workspace = ws.p;
      a.workspace_bytes = ws.bytes;
      check(lik_gated_bwd(&a, c10::cuda::getCurrentCUDAStream(X.device().index()).stream()), "lik_gated_bwd");
      for (int i = 0; i < N_GATED_PARAMS; ++i)
        if (out[1 + i].defined()) out[1 + i] = out[1 + i].to(types[i]);
      if (task_should_compute_output(1 + N_GATED_PARAMS)) out[1 + N_GATED_PARAMS] = grads[0];
    }
    return once(std::move(out), "gated_feed_forward");
  }
};

Tensor gated_feed_forward(const Tensor& x_, const Tensor& wg, const Tensor& wu, const Tensor& wd, const OptTensor& bg_, const OptTensor& bu_, const OptTensor& bd_,
                          const std::optional<std::string>& activation, const OptTensor& residual_) {
  const Tensor bg = opt(bg_), bu = opt(bu_), bd = opt(bd_), r_ = opt(residual_);
  require_layer_inputs("gated_feed_forward", x_,
                       {{"w_gate", &wg}, {"w_up", &wu}, {"w_down", &wd}, {"b_gate", &bg}, {"b_up", &bu}, {"b_down", &bd}, {"residual", &r_}});
  const int64_t in = x_.size(-1);
  require_features(x_);
  require_matrix("w_gate", wg, -1, "in_features", in);
  const int64_t f = wg.size(0);
  require_matrix("w_up", wu, f, "in_features", in);
  require_matrix("w_down", wd, -1, "hidden_features", f);
  const int64_t out = wd.size(0);
  require_vector("b_gate", bg, f);
  require_vector("b_up", bu, f);
  require_vector("b_down", bd, out);
  require_residual(r_, x_, out);
  const int act = activation_code(activation);
  const auto dt = x_.scalar_type();
  const Tensor x = rows_of(x_);
  const Tensor r = r_.defined() ? rows_of(r_.scalar_type() == dt ? r_ : r_.to(dt)) : r_;
  const c10::cuda::CUDAGuard guard(x.device());
  const bool grad = wants_grad({&x, &wg, &wu, &wd, &bg, &bu, &bd, &r});
  if (grad) refuse_foreign_accumulators("gated_feed_forward", {&x_, &wg, &wu, &wd, &bg, &bu, &bd, &r_});
  Tensor y, kept, pg, pu, pd;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    pg = as_rows(wg, dt);
    pu = as_rows(wu, dt);
    pd = as_rows(wd, dt);
    const Tensor qg = as_rows(bg, dt), qu = as_rows(bu, dt), qd = as_rows(bd, dt);
    lik_gated_args a = gated_args(x, pg, pu, pd, act);
    a.b_gate = ptr(qg);
    a.b_up = ptr(qu);
    a.b_down = ptr(qd);
    a.residual = ptr(r);
    a.residual_stride = r.defined() ? row_stride(r) : 0;
    y = at::empty({x.size(0), out}, x.options());
    a.y = ptr(y);
    if (wants_grad({&x, &wg, &wu, &wd, &bg, &bu})) {  // (b_down's and a residual's gradients are made of dy alone)
      kept = kept_rows(3, x.size(0), f, x);
      a.gate_factor = matrix_of(kept, 0);
      a.up_factor = matrix_of(kept, 1);
      a.h = matrix_of(kept, 2);
      a.kept_stride = kept.size(2);
    }
    const Workspace ws(lik_gated_fwd_workspace(&a), x.device());
    a.workspace = ws.p;
    a.workspace_bytes = ws.bytes;
    check(lik_gated_fwd(&a, c10::cuda::getCurrentCUDAStream(x.device().index()).stream()), "lik_gated_fwd");
  }
  if (grad) {
    auto node = std::shared_ptr<GatedFeedForwardBackward>(new GatedFeedForwardBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, wg, wu, wd, bg, bu, bd, r));
    node->x = SavedVariable(x, false);
    node->wg = SavedVariable(wg.scalar_type() == dt ? wg : pg, false);
    node->wu = SavedVariable(wu.scalar_type() == dt ? wu : pu, false);
    node->wd = SavedVariable(wd.scalar_type() == dt ? wd : pd, false);
    node->kept = SavedVariable(kept, false);
    const Tensor* const params[N_GATED_PARAMS] = {&wg, &wu, &wd, &bg, &bu, &bd};
    for (int i = 0; i < N_GATED_PARAMS; ++i)
      if (params[i]->defined()) node->types[i] = params[i]->scalar_type();
    node->act = act;
    node->grad_type = param_dtype(dt, {&wg, &wu, &wd, &bg, &bu, &bd});
    torch::autograd::set_history(y, node);
  }
  if (x_.dim() == 2) return y;
  auto sizes = x_.sizes().vec();
  sizes.back() = out;
  return y.view(sizes);
}

}  // namespace

void bind_layers(pybind11::module_& m) {
  m.def("layer_norm", torch::wrap_pybind_function_no_gil(&layer_norm));
  m.def("linear", torch::wrap_pybind_function_no_gil(&linear));
  m.def("gated_feed_forward", torch::wrap_pybind_function_no_gil(&gated_feed_forward));
}

}  // namespace lik_host
