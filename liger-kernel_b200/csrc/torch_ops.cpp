// torch-side binding of the norms and of the router's balance loss: argument checks, allocation, autograd nodes.  The kernels stay behind the C ABI of
// libflce_b200.so, whose entry points are looked up at load time (liger_b200_bind); no torch type crosses it.
//
// Why not ctypes and a Python autograd.Function, as for the losses: those run once per step, a norm runs dozens of times and
// its kernels last as little as 3 us.  RMSNorm of 64 x 1024 rows through Python: forward 34 us, forward + backward 154 us (most of
// it in the backward thread); through this binding 10 and 66 us, where torch's own layer norm takes 66.
//
// Each operator has an autograd kernel, which looks at no data and no sizes: it goes through the dispatcher once more, to the
// kernel for CUDA tensors that checks, allocates and launches, and sets up the gradient.  What the dispatcher puts between the two
// therefore sees the launch as an operator: tracers record it (its results' shapes are given in _torch_ops.py), and torch.func's
// transforms, nested ones too, find an autograd kernel at each of their levels.
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include "flce_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ------------------------------------------------------------------ the library's entry points
struct Library {
  decltype(&flce_b200_norm_forward) norm_forward = nullptr;
  decltype(&flce_b200_norm_workspace_bytes) norm_workspace_bytes = nullptr;
  decltype(&flce_b200_norm_backward) norm_backward = nullptr;
  decltype(&flce_b200_balance_workspace_bytes) balance_workspace_bytes = nullptr;
  decltype(&flce_b200_balance_forward) balance_forward = nullptr;
  decltype(&flce_b200_balance_backward) balance_backward = nullptr;
  decltype(&flce_b200_status_string) status_string = nullptr;
  decltype(&flce_b200_last_error) last_error = nullptr;
  bool host_memory = false;     // the tests' emulation of the library computes on host memory
};
Library g_lib;

void check(int status) {
  TORCH_CHECK(status == FLCE_OK, "libflce_b200: ", g_lib.status_string(status), ": ", g_lib.last_error());
}

void require_device(const Tensor& t) {
  TORCH_CHECK(t.is_cuda() || (g_lib.host_memory && t.is_cpu()),
              "liger_kernel_b200 runs on CUDA (sm_100a) tensors only; there is no CPU path");
}

// the tensor's device is the current one inside; `stream` is the current stream there
struct OnDevice {
  explicit OnDevice(const Tensor& t) {
    if (t.is_cuda()) {
      guard.set_index(t.get_device());
      stream = c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
    }
  }
  c10::cuda::OptionalCUDAGuard guard;
  void* stream = nullptr;
};

int dtype_of(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return FLCE_BF16;
    case at::kHalf: return FLCE_FP16;
    case at::kFloat: return FLCE_FP32;
    default: TORCH_CHECK_TYPE(false, "unsupported ", what, "dtype ", t.scalar_type());
  }
}

// Where a tensor's elements lie.  Wrapper tensors (distributed ones, for instance) have none of their own: nullptr would mean
// "not given" to the library.
const void* elements(const Tensor& t, const char* what) {
  const void* p = t.const_data_ptr();
  TORCH_CHECK(p != nullptr || t.numel() == 0, what, " has no storage: pass the local tensor");
  return p;
}

// Tangents of forward-mode differentiation would be lost below autograd, and with them a part of the derivative.
void refuse_tangent(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                              "liger_kernel_b200 has no forward-mode derivatives: an input or an upstream gradient carries a forward gradient");
}

// A gradient of a gradient would need the graph of the kernels' own arithmetic, which does not exist: what backward returns
// under create_graph is attached to a node that says so.
template <class... Of>
variable_list once_differentiable(variable_list&& grads, const Of&... of) {
  if (!torch::autograd::compute_requires_grad(of...)) return std::move(grads);
  auto error = std::shared_ptr<torch::autograd::Error>(
      new torch::autograd::Error("trying to differentiate twice a function that was marked with @once_differentiable",
                                 torch::autograd::collect_next_edges(of...)),
      torch::autograd::deleteNode);
  for (auto& g : grads) {
    if (g.defined()) torch::autograd::set_history(g, error);
  }
  return std::move(grads);
}

// the operator of that name, for calls that go through the dispatcher
template <class Signature>
c10::TypedOperatorHandle<Signature> operator_of(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

// ------------------------------------------------------------------ layer norm and RMSNorm
struct NormOperands {
  flce_norm_t p{};
  Tensor x, w, b;               // as the kernels read them; they keep p's pointers alive
};

// [rows, hidden] with adjacent elements: a view wherever one exists
Tensor as_rows(const Tensor& t, int64_t hidden) {
  Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / hidden, hidden});
  return r.stride(1) == 1 || hidden == 1 ? r : r.contiguous();
}

const Tensor& check_parameter(const char* name, const Tensor& t, const Tensor& x, int64_t hidden) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == hidden, name, " must be [", hidden, "], got ", t.sizes());
  dtype_of(t, name[0] == 'w' ? "weight " : "bias ");
  TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", the input on ", x.device());
  return t;
}

NormOperands norm_operands(int64_t kind, const Tensor& x, const Tensor& w, const Tensor& b, double eps, double offset,
                           bool round_xhat) {
  require_device(x);
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "expected [..., H] with H >= 1, got ", x.sizes());
  NormOperands o;
  const int64_t hidden = x.size(-1);
  o.p.dtype = dtype_of(x, "");
  o.x = as_rows(x, hidden);
  // the kernels take parameters of the rows' type or fp32, both alike: anything else is widened
  at::ScalarType wtype = x.scalar_type();
  for (const Tensor* t : {&w, &b}) {
    if (t->defined() && check_parameter(t == &w ? "weight" : "bias", *t, x, hidden).scalar_type() != wtype) wtype = at::kFloat;
  }
  if (w.defined()) o.w = w.to(wtype).contiguous();
  if (b.defined()) o.b = b.to(wtype).contiguous();
  o.p.n_rows = o.x.size(0);
  o.p.hidden = hidden;
  o.p.ld_x = o.x.stride(0);
  o.p.kind = static_cast<int32_t>(kind);
  o.p.weight_dtype = wtype == at::kFloat ? FLCE_FP32 : o.p.dtype;
  o.p.round_xhat = round_xhat;
  o.p.eps = static_cast<float>(eps);
  o.p.offset = static_cast<float>(offset);
  o.p.x = elements(o.x, "the input");
  o.p.weight = w.defined() ? elements(o.w, "weight") : nullptr;
  o.p.bias = b.defined() ? elements(o.b, "bias") : nullptr;
  return o;
}

Tensor norm_rows(const Tensor& x, const Tensor& w, const Tensor& b, int64_t kind, double eps, double offset, bool round_xhat,
                 Tensor* stats) {
  const NormOperands o = norm_operands(kind, x, w, b, eps, offset, round_xhat);
  OnDevice on(x);
  Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  float *rstd = nullptr, *mean = nullptr;
  if (stats != nullptr) {
    *stats = at::empty({kind == FLCE_LAYER_NORM ? 2 : 1, o.p.n_rows}, x.options().dtype(at::kFloat));
    rstd = stats->data_ptr<float>();
    mean = kind == FLCE_LAYER_NORM ? rstd + o.p.n_rows : nullptr;
  }
  check(g_lib.norm_forward(&o.p, y.data_ptr(), mean, rstd, on.stream));
  return y;
}

Tensor norm_launch(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, int64_t kind, double eps, double offset,
                   bool round_xhat) {
  return norm_rows(x, weight.value_or(Tensor()), bias.value_or(Tensor()), kind, eps, offset, round_xhat, nullptr);
}

// y and [2 or 1, rows] fp32: rstd, mean
std::tuple<Tensor, Tensor> norm_with_statistics_launch(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                                                       int64_t kind, double eps, double offset, bool round_xhat) {
  Tensor stats;
  Tensor y = norm_rows(x, weight.value_or(Tensor()), bias.value_or(Tensor()), kind, eps, offset, round_xhat, &stats);
  return {y, stats};
}

// the gradients of x, weight and bias, the latter undefined where not wanted
std::tuple<Tensor, Tensor, Tensor> norm_backward_launch(const Tensor& grad, const Tensor& x, const optional<Tensor>& weight,
                                                        const optional<Tensor>& bias, const Tensor& stats, int64_t kind, double eps,
                                                        double offset, bool round_xhat, bool need_w, bool need_b) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  OnDevice on(x);
  const NormOperands o = norm_operands(kind, x, w, b, eps, offset, round_xhat);
  TORCH_CHECK_VALUE(grad.sizes() == x.sizes() && grad.scalar_type() == x.scalar_type() && grad.device() == x.device(),
                    "the gradient must agree with the input in shape, type and device");
  const int64_t planes = kind == FLCE_LAYER_NORM ? 2 : 1;
  TORCH_CHECK_VALUE(stats.dim() == 2 && stats.size(0) == planes && stats.size(1) == o.p.n_rows && stats.scalar_type() == at::kFloat &&
                        stats.device() == x.device(),
                    "the statistics must be [", planes, ", ", o.p.n_rows, "] in fp32 on the input's device");
  TORCH_CHECK_VALUE((w.defined() || !need_w) && (b.defined() || !need_b), "the gradient of a parameter that is not given");
  const Tensor dy = as_rows(grad, o.p.hidden), kept = stats.contiguous();
  Tensor dx = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)), dw, db, workspace;
  size_t bytes = 0;
  if (need_w) dw = at::empty_like(o.w);
  if (need_b) db = at::empty_like(o.b);
  if (need_w || need_b) {
    bytes = g_lib.norm_workspace_bytes(&o.p);
    workspace = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  }
  const float* rstd = kept.const_data_ptr<float>();
  check(g_lib.norm_backward(&o.p, elements(dy, "the gradient"), dy.stride(0), kind == FLCE_LAYER_NORM ? rstd + o.p.n_rows : nullptr, rstd,
                            dx.data_ptr(), need_w ? dw.data_ptr() : nullptr, need_b ? db.data_ptr() : nullptr,
                            workspace.defined() ? workspace.data_ptr() : nullptr, bytes, on.stream));
  return {dx, need_w ? dw.to(w.scalar_type()) : dw, need_b ? db.to(b.scalar_type()) : db};
}

std::tuple<Tensor, Tensor, Tensor> norm_backward(const Tensor& grad, const Tensor& x, const optional<Tensor>& weight,
                                                 const optional<Tensor>& bias, const Tensor& stats, int64_t kind, double eps, double offset,
                                                 bool round_xhat, bool need_w, bool need_b) {
  static const auto next = operator_of<decltype(norm_backward_launch)>("liger_b200::_norm_backward");
  refuse_tangent(grad);
  variable_list out(3);
  {
    at::AutoDispatchBelowAutograd below;
    std::tie(out[0], out[1], out[2]) = next.call(grad, x, weight, bias, stats, kind, eps, offset, round_xhat, need_w, need_b);
  }
  out = once_differentiable(std::move(out), grad, x, weight.value_or(Tensor()));
  return {out[0], out[1], out[2]};
}

struct NormBackward : public torch::autograd::Node {
  SavedVariable x, w, b;
  Tensor stats;
  int64_t kind = 0;
  double eps = 0, offset = 0;
  bool round_xhat = false;

  std::string name() const override { return kind == FLCE_LAYER_NORM ? "LigerLayerNormBackward" : "LigerRMSNormBackward"; }

  void release_variables() override {
    x.reset_data();
    w.reset_data();
    b.reset_data();
    stats.reset();
  }

  variable_list apply(variable_list&& grads) override {
    static const auto backward = operator_of<decltype(norm_backward_launch)>("liger_b200::_norm_backward");
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);
    const Tensor& grad = grads[0];
    if (!grad.defined()) return out;
    const Tensor xs = x.unpack(), ws = w.unpack(), bs = b.unpack();
    TORCH_CHECK(stats.defined(), torch::autograd::ERR_BACKWARD_TWICE);
    const bool need_w = ws.defined() && task_should_compute_output(1), need_b = bs.defined() && task_should_compute_output(2);
    std::tie(out[0], out[1], out[2]) = backward.call(grad, xs, ws, bs, stats, kind, eps, offset, round_xhat, need_w, need_b);
    if (!task_should_compute_output(0)) out[0] = Tensor();
    return out;
  }
};

std::tuple<Tensor, Tensor> norm_with_statistics(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, int64_t kind,
                                                double eps, double offset, bool round_xhat) {
  static const auto next = operator_of<decltype(norm_with_statistics_launch)>("liger_b200::_norm_with_statistics");
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  for (const Tensor* t : {&x, &w, &b}) refuse_tangent(*t);
  Tensor y, stats;
  {
    at::AutoDispatchBelowAutograd below;
    std::tie(y, stats) = next.call(x, weight, bias, kind, eps, offset, round_xhat);
  }
  if (torch::autograd::compute_requires_grad(x, w, b)) {
    auto node = std::shared_ptr<NormBackward>(new NormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    node->x = SavedVariable(x, false);
    node->w = SavedVariable(w, false);
    node->b = SavedVariable(b, false);
    node->stats = stats;
    node->kind = kind;
    node->eps = eps;
    node->offset = offset;
    node->round_xhat = round_xhat;
    torch::autograd::set_history(y, node);
  }
  return {y, stats};
}

// the row statistics are kept only where a gradient may be asked for
Tensor norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, int64_t kind, double eps, double offset,
            bool round_xhat) {
  static const auto next = operator_of<decltype(norm_launch)>("liger_b200::norm");
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  if (torch::autograd::compute_requires_grad(x, w, b))
    return std::get<0>(norm_with_statistics(x, weight, bias, kind, eps, offset, round_xhat));
  for (const Tensor* t : {&x, &w, &b}) refuse_tangent(*t);
  at::AutoDispatchBelowAutograd below;
  return next.call(x, weight, bias, kind, eps, offset, round_xhat);
}

// ------------------------------------------------------------------ the router's load-balancing loss
struct BalanceOperands {
  flce_balance_t p{};
  std::vector<Tensor> logits;   // [tokens, experts] each, one pitch for all
  std::vector<const void*> pointers;
  Tensor mask;
};

BalanceOperands balance_operands(at::TensorList logits, int64_t num_experts, int64_t top_k, const Tensor& mask, double lse_square_scale) {
  TORCH_CHECK_VALUE(!logits.empty(), "expected the router logits of at least one layer");
  TORCH_CHECK_VALUE(num_experts >= 1, "num_experts must be at least 1, got ", num_experts);
  BalanceOperands o;
  const Tensor& head = logits[0];
  require_device(head);
  o.p.dtype = dtype_of(head, "");
  bool same_pitch = true;
  for (const Tensor& t : logits) {
    TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) == num_experts, "router logits must be [..., ", num_experts, "], got ", t.sizes());
    TORCH_CHECK_VALUE(t.scalar_type() == head.scalar_type() && t.device() == head.device() && t.numel() == head.numel(),
                      "the router logits of all layers must agree in type, device and number of tokens");
    o.logits.push_back(as_rows(t, num_experts));
    same_pitch = same_pitch && o.logits.back().stride(0) == o.logits[0].stride(0);
  }
  TORCH_CHECK_VALUE(top_k >= 1 && top_k <= num_experts, "top_k must be in [1, ", num_experts, "], got ", top_k);
  TORCH_CHECK_NOT_IMPLEMENTED(num_experts <= 1024, "at most 1024 experts, got ", num_experts);
  o.p.n_layers = static_cast<int64_t>(o.logits.size());
  o.p.n_tokens = o.logits[0].size(0);
  o.p.n_experts = num_experts;
  o.p.top_k = top_k;
  for (Tensor& t : o.logits) {
    if (!same_pitch) t = t.contiguous();
    o.pointers.push_back(elements(t, "a layer's router logits"));
  }
  o.p.ld = same_pitch ? o.logits[0].stride(0) : num_experts;
  o.p.lse_square_scale = static_cast<float>(lse_square_scale);
  if (mask.defined()) {
    TORCH_CHECK_VALUE(mask.numel() == o.p.n_tokens, "the attention mask has ", mask.numel(), " elements, a layer's router logits ",
                      o.p.n_tokens, " tokens");
    const auto type = mask.scalar_type();
    o.mask = type == at::kBool || type == at::kByte || type == at::kChar || type == at::kInt || type == at::kLong ? mask : mask.ne(0);
    o.mask = o.mask.to(head.device()).contiguous();
    o.p.mask_bytes = static_cast<int32_t>(o.mask.element_size());
    o.p.mask = o.p.n_tokens > 0 ? elements(o.mask, "the attention mask") : nullptr;
  }
  return o;
}

// Dense elements of `whole` from `offset` on, in the given shape, as a tensor that shares its storage: what select and view give,
// without a trip through the dispatcher for each of dozens of layers.
Tensor piece_of(const Tensor& whole, int64_t offset, at::IntArrayRef sizes) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  t.unsafeGetTensorImpl()->set_storage_offset(whole.storage_offset() + offset);
  return t;
}

// One fp32 buffer: what backward needs, [experts + 1], then the loss and its lse^2 term.
int64_t loss_at(int64_t num_experts) { return num_experts + 1; }

// that buffer and the counts, [layers, experts]
std::tuple<Tensor, Tensor> balance_launch(at::TensorList logits, int64_t num_experts, int64_t top_k, const optional<Tensor>& attention_mask,
                                          double lse_square_scale) {
  const BalanceOperands o = balance_operands(logits, num_experts, top_k, attention_mask.value_or(Tensor()), lse_square_scale);
  OnDevice on(logits[0]);
  const auto options = o.logits[0].options();
  const Tensor values = at::empty({loss_at(num_experts) + 2}, options.dtype(at::kFloat));
  const Tensor counts = at::empty({o.p.n_layers, num_experts}, options.dtype(at::kLong));
  const size_t bytes = g_lib.balance_workspace_bytes(&o.p);
  const Tensor workspace = at::empty({static_cast<int64_t>(bytes)}, options.dtype(at::kByte));
  float* f = values.data_ptr<float>();
  check(g_lib.balance_forward(&o.p, o.pointers.data(), f + loss_at(num_experts), counts.data_ptr<int64_t>(), f, workspace.data_ptr(), bytes,
                              on.stream));
  return {values, counts};
}

// the gradients of all layers' logits: [layers, tokens, experts]
Tensor balance_backward_launch(const Tensor& grad, at::TensorList logits, const optional<Tensor>& attention_mask, const Tensor& values,
                               int64_t num_experts, int64_t top_k, double lse_square_scale) {
  OnDevice on(logits[0]);
  const BalanceOperands o = balance_operands(logits, num_experts, top_k, attention_mask.value_or(Tensor()), lse_square_scale);
  TORCH_CHECK_VALUE(grad.numel() == 1 && grad.device() == logits[0].device(), "the gradient must be one number on the logits' device");
  TORCH_CHECK_VALUE(values.dim() == 1 && values.size(0) > num_experts && values.scalar_type() == at::kFloat &&
                        values.device() == logits[0].device(),
                    "the coefficients must be ", num_experts + 1, " fp32 numbers or more on the logits' device");
  const Tensor up = grad.to(at::kFloat).contiguous(), coef = values.contiguous();
  Tensor all = at::empty({o.p.n_layers, o.p.n_tokens, num_experts}, logits[0].options().memory_format(at::MemoryFormat::Contiguous));
  check(g_lib.balance_backward(&o.p, o.pointers.data(), coef.const_data_ptr<float>(), up.const_data_ptr<float>(), all.data_ptr(),
                               on.stream));
  return all;
}

Tensor balance_backward(const Tensor& grad, at::TensorList logits, const optional<Tensor>& attention_mask, const Tensor& values,
                        int64_t num_experts, int64_t top_k, double lse_square_scale) {
  static const auto next = operator_of<decltype(balance_backward_launch)>("liger_b200::_load_balancing_loss_backward");
  refuse_tangent(grad);
  variable_list out(1);
  {
    at::AutoDispatchBelowAutograd below;
    out[0] = next.call(grad, logits, attention_mask, values, num_experts, top_k, lse_square_scale);
  }
  return once_differentiable(std::move(out), grad, logits)[0];
}

// Whether nobody but autograd sees what is done with the tensors: no tracer, no mode, no transform, no wrapper around them.
bool is_plain(at::TensorList tensors) {
  using c10::DispatchKey;
  static const c10::DispatchKeySet usual =
      c10::DispatchKeySet({DispatchKey::CUDA, DispatchKey::CPU, DispatchKey::BackendSelect, DispatchKey::ADInplaceOrView,
                           DispatchKey::AutogradCUDA, DispatchKey::AutogradCPU, DispatchKey::AutocastCUDA, DispatchKey::AutocastCPU});
  c10::DispatchKeySet keys = c10::impl::tls_local_dispatch_key_set().included_;
  for (const Tensor& t : tensors) {
    if (!t.is_cuda() && !t.is_cpu()) return false;
    keys = keys | t.key_set();
  }
  return ((keys - usual).raw_repr() & ~c10::full_backend_mask) == 0;      // the difference keeps the backends' bits
}

struct BalanceBackward : public torch::autograd::Node {
  std::vector<SavedVariable> logits;
  SavedVariable mask;
  Tensor values;
  bool of_values = false;       // the node stands behind the buffer, not behind the loss cut from it
  int64_t num_experts = 0, top_k = 0;
  double lse_square_scale = 0;

  std::string name() const override { return "LigerLoadBalancingLossBackward"; }

  void release_variables() override {
    for (auto& t : logits) t.reset_data();
    mask.reset_data();
    values.reset();
  }

  variable_list apply(variable_list&& grads) override {
    static const auto backward = operator_of<decltype(balance_backward_launch)>("liger_b200::_load_balancing_loss_backward");
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(logits.size());
    const Tensor grad = of_values ? grads[0].select(0, loss_at(num_experts)) : grads[0];
    variable_list x;
    x.reserve(logits.size());
    for (auto& t : logits) x.push_back(t.unpack());
    const Tensor m = mask.unpack();
    TORCH_CHECK(values.defined(), torch::autograd::ERR_BACKWARD_TWICE);
    const Tensor all = backward.call(grad, x, m, values, num_experts, top_k, lse_square_scale);
    // The layers' pieces of it start on any boundary.  A compiler has to see where: through the dispatcher then, and also where
    // the pieces need a history.
    const bool quick = is_plain(all) && !all.requires_grad();
    variable_list out(x.size());
    for (size_t l = 0; l < x.size(); ++l) {
      if (!task_should_compute_output(l)) continue;
      out[l] = quick ? piece_of(all, static_cast<int64_t>(l) * all.stride(0), x[l].sizes())
                     : all.select(0, static_cast<int64_t>(l)).view_symint(x[l].sym_sizes());
    }
    return out;
  }
};

void set_balance_history(const Tensor& result, bool of_values, const Tensor& values, at::TensorList logits, int64_t num_experts,
                         int64_t top_k, const optional<Tensor>& attention_mask, double lse_square_scale) {
  auto node = std::shared_ptr<BalanceBackward>(new BalanceBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(logits));
  node->logits.reserve(logits.size());
  for (const Tensor& t : logits) node->logits.emplace_back(t, false);
  node->mask = SavedVariable(attention_mask.value_or(Tensor()), false);
  node->values = of_values ? values.detach() : values;
  node->of_values = of_values;
  node->num_experts = num_experts;
  node->top_k = top_k;
  node->lse_square_scale = lse_square_scale;
  torch::autograd::set_history(result, node);
}

std::tuple<Tensor, Tensor> balance(at::TensorList logits, int64_t num_experts, int64_t top_k, const optional<Tensor>& attention_mask,
                                   double lse_square_scale) {
  static const auto next = operator_of<decltype(balance_launch)>("liger_b200::_load_balancing_loss");
  for (const Tensor& t : logits) refuse_tangent(t);
  Tensor values, counts;
  {
    at::AutoDispatchBelowAutograd below;
    std::tie(values, counts) = next.call(logits, num_experts, top_k, attention_mask, lse_square_scale);
  }
  if (torch::autograd::compute_requires_grad(logits))
    set_balance_history(values, true, values, logits, num_experts, top_k, attention_mask, lse_square_scale);
  return {values, counts};
}

// loss, its lse^2 term, counts [layers, experts]: a composite.  Where nobody looks on, the two numbers are cut out without the
// dispatcher and the node stands right behind the loss.
std::tuple<Tensor, Tensor, Tensor> load_balancing_loss(at::TensorList logits, int64_t num_experts, int64_t top_k,
                                                       const optional<Tensor>& attention_mask, double lse_square_scale) {
  static const auto forward = operator_of<decltype(balance_launch)>("liger_b200::_load_balancing_loss");
  TORCH_CHECK_VALUE(!logits.empty(), "expected the router logits of at least one layer");      // the dispatch goes by their device
  if (!is_plain(logits)) {
    auto [values, counts] = forward.call(logits, num_experts, top_k, attention_mask, lse_square_scale);
    return {values.select(0, loss_at(num_experts)), values.detach().select(0, loss_at(num_experts) + 1), counts};
  }
  for (const Tensor& t : logits) refuse_tangent(t);
  Tensor values, counts;
  {
    at::AutoDispatchBelowAutograd below;
    std::tie(values, counts) = forward.call(logits, num_experts, top_k, attention_mask, lse_square_scale);
  }
  const Tensor loss = piece_of(values, loss_at(num_experts), {}), z_loss = piece_of(values, loss_at(num_experts) + 1, {});
  if (torch::autograd::compute_requires_grad(logits))
    set_balance_history(loss, false, values, logits, num_experts, top_k, attention_mask, lse_square_scale);
  return {loss, z_loss, counts};
}

TORCH_LIBRARY(liger_b200, m) {
  m.def("load_balancing_loss(Tensor[] logits, int num_experts, int top_k, Tensor? attention_mask, float lse_square_scale) -> "
        "(Tensor, Tensor, Tensor)", load_balancing_loss);
  m.def("norm(Tensor x, Tensor? weight, Tensor? bias, int kind, float eps, float offset, bool round_xhat) -> Tensor");
  m.def("_norm_with_statistics(Tensor x, Tensor? weight, Tensor? bias, int kind, float eps, float offset, bool round_xhat) -> "
        "(Tensor, Tensor)");
  m.def("_norm_backward(Tensor grad, Tensor x, Tensor? weight, Tensor? bias, Tensor statistics, int kind, float eps, float offset, "
        "bool round_xhat, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)");
  m.def("_load_balancing_loss(Tensor[] logits, int num_experts, int top_k, Tensor? attention_mask, float lse_square_scale) -> "
        "(Tensor, Tensor)");
  m.def("_load_balancing_loss_backward(Tensor grad, Tensor[] logits, Tensor? attention_mask, Tensor values, int num_experts, "
        "int top_k, float lse_square_scale) -> Tensor");
}

// Tensors on the CPU get as far as require_device, which knows whether the library computes there.
void register_launches(torch::Library& m) {
  m.impl("norm", norm_launch);
  m.impl("_norm_with_statistics", norm_with_statistics_launch);
  m.impl("_norm_backward", norm_backward_launch);
  m.impl("_load_balancing_loss", balance_launch);
  m.impl("_load_balancing_loss_backward", balance_backward_launch);
}
TORCH_LIBRARY_IMPL(liger_b200, CUDA, m) { register_launches(m); }
TORCH_LIBRARY_IMPL(liger_b200, CPU, m) { register_launches(m); }
TORCH_LIBRARY_IMPL(liger_b200, Autograd, m) {
  m.impl("norm", norm);
  m.impl("_norm_with_statistics", norm_with_statistics);
  m.impl("_norm_backward", norm_backward);
  m.impl("_load_balancing_loss", balance);
  m.impl("_load_balancing_loss_backward", balance_backward);
}

}  // namespace

// torch's C++ interface changes between its versions: the Python side looks for this in the file before it loads it.
extern "C" __attribute__((used)) const char liger_b200_built_against[] = "liger_b200 built against torch " LIGER_TORCH_VERSION ";";

// Looks the entry points up in the library at `path` (one that is loaded already is not loaded again); host_memory: it is the
// tests' emulation.  Returns nullptr, or what is missing.  The string is valid until the thread's next call.
extern "C" const char* liger_b200_bind(const char* path, int host_memory) {
  static thread_local char message[256];
  void* handle = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (handle == nullptr) {
    snprintf(message, sizeof(message), "%s", dlerror());
    return message;
  }
  Library lib;
  lib.host_memory = host_memory != 0;
  const char* missing = nullptr;
  auto find = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(dlsym(handle, name));
    if (fn == nullptr) missing = name;
  };
  find(lib.norm_forward, "flce_b200_norm_forward");
  find(lib.norm_workspace_bytes, "flce_b200_norm_workspace_bytes");
  find(lib.norm_backward, "flce_b200_norm_backward");
  find(lib.balance_workspace_bytes, "flce_b200_balance_workspace_bytes");
  find(lib.balance_forward, "flce_b200_balance_forward");
  find(lib.balance_backward, "flce_b200_balance_backward");
  find(lib.status_string, "flce_b200_status_string");
  find(lib.last_error, "flce_b200_last_error");
  if (missing != nullptr) {
    snprintf(message, sizeof(message), "%s has no %s", path, missing);
    return message;
  }
  g_lib = lib;
  return nullptr;
}
