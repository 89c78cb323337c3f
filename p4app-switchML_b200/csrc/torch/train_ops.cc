// lib/torch_switchml_train.so: the operators of a training step around its gradients, for ops/layer_norm.py and
// ops/adamw.py. Arguments are checked and kernels launched without Python: a step of BERT-large's optimizer has 298
// parameters to ask for their gradients, and layer norm's backward pass runs on the engine's thread.
#include <ATen/autocast_mode.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <memory>
#include <mutex>
#include <string>
#include <vector>

#include "kernels/adamw.h"
#include "kernels/layer_norm.h"

namespace {

using torch::Tensor;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

void* CurrentStream() { return at::cuda::getCurrentCUDAStream().stream(); }

void Check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed: ", rc == -4 ? "kernel launch" : "bad argument"); }

bool Known(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }

int NormType(const Tensor& t) { return t.scalar_type() == at::kFloat ? SML_NORM_F32 : SML_NORM_BF16; }

// (Null says that a tensor is not there: one that is, but has no memory, must not look like that.)
void* Data(const Tensor& t) {
  if (!t.defined()) return nullptr;
  void* const data = const_cast<void*>(t.const_data_ptr());
  TORCH_CHECK(data || !t.numel(), "a tensor of the shape ", t.sizes(), " has no memory");
  return data;
}

// For a kernel that writes: a lazy clone of the tensor gets its own memory first.
void* Writable(const Tensor& t) {
  if (!t.defined()) return nullptr;
  void* const data = t.mutable_data_ptr();
  TORCH_CHECK(data || !t.numel(), "a tensor of the shape ", t.sizes(), " has no memory");
  return data;
}

// Whether the memory of a tensor does not hold its values: a view that says they are to be negated (imag() of a conjugate), or
// zeros that autograd has not written out.
bool Implied(const Tensor& t) {
  return t.key_set().has_any(c10::DispatchKeySet{c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
}

Tensor Written(const Tensor& t) { return at::zeros(t.sizes(), t.options()).copy_(t); }

// As the kernels read it.
Tensor Contiguous(const Tensor& t) { return Implied(t) ? Written(t) : t.contiguous(); }

// What records operations to run them again (torch.jit.trace, make_fx, export) sees the allocation of a result here, but not the
// kernel that writes it: the recording would return memory that nothing has written.
void RefuseTracing(const char* what) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  const bool modes = c10::impl::dispatch_mode_enabled();
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) &&
                  !(modes && (TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY).has_value() ||
                              TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE).has_value())),
              what, " cannot be traced");
}

// Dual tensors are such while a level of forward mode is open: asked once per call, since to ask a view looks at its base.
bool DualsExist() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

void RefuseDual(const Tensor& t, const char* what) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), what, " has no forward-mode gradient");
}

// ---- layer norm ----

constexpr int64_t kMaxFeatures = 1 << 30;

void CheckParameter(const Tensor& p, const char* name, const Tensor& x, const Tensor& other) {
  if (!p.defined()) return;
  TORCH_CHECK_VALUE(p.device() == x.device(), "layer_norm: ", name, " is on ", p.device(), ", x on ", x.device());
  TORCH_CHECK_VALUE(p.dim() == 1 && p.size(0) == x.size(-1), "layer_norm: ", name, " has the shape ", p.sizes(), ", the last dimension of x is ",
              x.size(-1));
  TORCH_CHECK_TYPE(p.scalar_type() == at::kFloat || p.scalar_type() == x.scalar_type(), "layer_norm: ", name, " is ", p.scalar_type(),
              ": float32 or the type of x (", x.scalar_type(), ") is wanted");
  TORCH_CHECK_TYPE(!other.defined() || other.scalar_type() == p.scalar_type(), "layer_norm: weight and bias are of different types");
}

// y, with a residual the sum, and with `stats` mean and 1 / deviation of every row.
struct Normed {
  Tensor y, sum, stats, x, weight, bias;  // the inputs as they were read
};

Normed Normalize(const Tensor& x_in, const OptTensor& residual_in, const OptTensor& weight_in, const OptTensor& bias_in, double eps,
                 bool with_stats) {
  at::AutoDispatchBelowADInplaceOrView below_autograd;
  const c10::cuda::OptionalCUDAGuard device(x_in.device());
  const bool add = residual_in.has_value();
  Normed r;
  r.x = Contiguous(x_in);
  const Tensor residual = add ? Contiguous(*residual_in) : Tensor();
  if (weight_in) r.weight = Contiguous(*weight_in);
  if (bias_in) r.bias = Contiguous(*bias_in);
  const int64_t n = r.x.size(-1), rows = r.x.numel() / n;
  r.y = at::empty_like(r.x);
  if (add) r.sum = at::empty_like(r.x);
  if (with_stats) r.stats = at::empty({2, rows}, r.x.options().dtype(at::kFloat));
  float* mean = with_stats ? r.stats.data_ptr<float>() : nullptr;
  if (rows > 0) {
    const Tensor& p = r.weight.defined() ? r.weight : r.bias;
    Check(switchml_layer_norm_forward(Data(r.x), Data(residual), Data(r.weight), Data(r.bias), r.y.data_ptr(), Data(r.sum), mean,
                                      mean ? mean + rows : nullptr, rows, static_cast<int>(n), static_cast<float>(eps), NormType(r.x),
                                      p.defined() ? NormType(p) : SML_NORM_F32, CurrentStream()),
          "layer_norm");
  }
  return r;
}

// A node of its own: with torch::autograd::Function forward and backward of a small input took 73 us of host time, where the
// engine alone takes 35.
struct LayerNormBackward : public torch::autograd::Node {
  torch::autograd::SavedVariable s, weight, stats;
  bool add = false;  // there was a residual
  bool has_weight = false;
  at::ScalarType type = at::kFloat;  // of s
  std::vector<int64_t> sizes;
  at::Device where = at::kCPU;
  at::ScalarType parameter_type = at::kFloat;

  std::string name() const override { return "LayerNormBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    s.reset_data();
    weight.reset_data();
    stats.reset_data();
  }

  // What the forward pass has saved, as the kernels take it. It may come back as another tensor: from hooks on saved tensors, and
  // because a leaf is saved as itself, of which .data may have been exchanged.
  Tensor Unpacked(const torch::autograd::SavedVariable& saved, const char* name, at::ScalarType its_type, at::IntArrayRef its_sizes,
                  std::shared_ptr<torch::autograd::Node> node = nullptr) const {
    const Tensor t = saved.unpack(std::move(node));
    TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.scalar_type() == its_type && t.sizes() == its_sizes && t.device() == where,
                "layer_norm: the ", name, " that the backward pass finds is not what the forward pass saved: ", its_type, " ", its_sizes, " on ", where);
    return Contiguous(t);
  }

  // Edges: x, residual, weight, bias; those of tensors that are not there lead nowhere.
  variable_list apply(variable_list&& grads) override {
    RefuseTracing("layer_norm");
    TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm has no gradient of its gradient (create_graph)");
    if (DualsExist()) {
      for (const Tensor& t : grads) RefuseDual(t, "layer_norm");
    }
    std::lock_guard<std::mutex> lock(mutex_);
    const c10::cuda::OptionalCUDAGuard device(where);
    const int64_t n = sizes.back(), rows = c10::multiply_integers(sizes) / n;
    const Tensor s_ = Unpacked(s, "input", type, sizes, add ? shared_from_this() : nullptr);
    const Tensor stats_ = Unpacked(stats, "statistics", at::kFloat, {2, rows});
    const Tensor weight_ = has_weight ? Unpacked(weight, "weight", parameter_type, {n}) : Tensor();
    for (const Tensor& t : grads)
      TORCH_CHECK(!t.defined() || (t.layout() == at::kStrided && t.scalar_type() == type && t.sizes() == sizes && t.device() == where),
                  "layer_norm: a gradient is ", t.scalar_type(), " ", t.sizes(), " on ", t.device(), ", the input ", type, " ", sizes, " on ", where);
    const bool want_weight = task_should_compute_output(2), want_bias = task_should_compute_output(3);
    const Tensor dsum = grads.size() > 1 && grads[1].defined() ? Contiguous(grads[1]) : Tensor();
    variable_list out(4);
    Tensor dx;
    if (!grads[0].defined()) {  // only the sum was used
      dx = dsum;
    } else {
      const Tensor dy = Contiguous(grads[0]);
      dx = at::empty_like(s_);
      if (want_weight) out[2] = at::empty({n}, s_.options().dtype(parameter_type));
      if (want_bias) out[3] = at::empty({n}, s_.options().dtype(parameter_type));
      if (rows > 0) {
        Tensor workspace;
        if (want_weight || want_bias)
          workspace = at::empty({switchml_layer_norm_workspace(rows, static_cast<int>(n), NormType(s_))}, s_.options().dtype(at::kFloat));
        const float* mean = stats_.const_data_ptr<float>();
        Check(switchml_layer_norm_backward(Data(dy), Data(dsum), Data(s_), Data(weight_), mean, mean + rows, dx.data_ptr(), Data(out[2]),
                                           Data(out[3]), static_cast<float*>(Data(workspace)), rows, static_cast<int>(n), NormType(s_),
                                           parameter_type == at::kFloat ? SML_NORM_F32 : SML_NORM_BF16, CurrentStream()),
              "layer_norm");
      } else {
        if (want_weight) out[2].zero_();
        if (want_bias) out[3].zero_();
      }
    }
    if (task_should_compute_output(0)) out[0] = dx;
    if (add && task_should_compute_output(1)) out[1] = dx;
    return out;
  }
};

variable_list LayerNormForward(Tensor x, OptTensor residual, const OptTensor& weight, const OptTensor& bias, double eps) {
  RefuseTracing("layer_norm");
  // (A dual tensor need not require a gradient: this is asked whether a backward pass comes or not.)
  if (DualsExist()) {
    for (const Tensor& t : {x, residual.value_or(Tensor()), weight.value_or(Tensor()), bias.value_or(Tensor())}) RefuseDual(t, "layer_norm");
  }
  const bool autocast = x.is_cuda() && at::autocast::is_autocast_enabled(at::kCUDA);
  c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::AutocastCUDA);
  if (autocast) {
    const auto type = at::autocast::get_autocast_dtype(at::kCUDA);
    const auto cast = [&](const Tensor& t) { return t.is_floating_point() && t.scalar_type() != at::kDouble ? t.to(type) : t; };
    x = cast(x);
    if (residual) residual = cast(*residual);
  }
  TORCH_CHECK_TYPE(Known(x), "layer_norm: x is ", x.scalar_type(), ": float32 or bfloat16 is wanted");
  TORCH_CHECK_VALUE(x.is_cuda(), "layer_norm: x is on ", x.device(), ": a CUDA device is wanted");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= kMaxFeatures, "layer_norm: x has the shape ", x.sizes(),
                    ": a last dimension of 1 to 2^30 is wanted");
  TORCH_CHECK_VALUE(eps >= 0, "layer_norm: eps is ", eps);
  if (residual) {
    TORCH_CHECK_VALUE(residual->device() == x.device() && residual->scalar_type() == x.scalar_type() && residual->sizes() == x.sizes(),
                      "layer_norm: the residual is ", residual->scalar_type(), " ", residual->sizes(), " on ", residual->device(), ", x is ",
                      x.scalar_type(), " ", x.sizes(), " on ", x.device());
  }
  CheckParameter(weight.value_or(Tensor()), "weight", x, Tensor());
  CheckParameter(bias.value_or(Tensor()), "bias", x, weight.value_or(Tensor()));
  const auto wants = [](const OptTensor& t) { return t && t->requires_grad(); };
  const bool backward_comes = at::GradMode::is_enabled() && (x.requires_grad() || wants(residual) || wants(weight) || wants(bias));
  if (!backward_comes) {
    const Normed r = Normalize(x, residual, weight, bias, eps, false);
    return residual ? variable_list{r.y, r.sum} : variable_list{r.y};
  }
  const Normed r = Normalize(x, residual, weight, bias, eps, true);
  const std::shared_ptr<LayerNormBackward> node(new LayerNormBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, residual.value_or(Tensor()), weight.value_or(Tensor()), bias.value_or(Tensor())));
  node->add = residual.has_value();
  node->has_weight = r.weight.defined();
  node->type = r.x.scalar_type(), node->sizes = r.x.sizes().vec(), node->where = r.x.device();
  if (r.weight.defined()) node->parameter_type = r.weight.scalar_type();
  else if (r.bias.defined()) node->parameter_type = r.bias.scalar_type();
  variable_list out = residual ? variable_list{r.y, r.sum} : variable_list{r.y};
  torch::autograd::set_history(out, node);
  node->s = torch::autograd::SavedVariable(node->add ? out[1] : r.x, node->add);
  node->weight = torch::autograd::SavedVariable(r.weight, false);
  node->stats = torch::autograd::SavedVariable(r.stats, false);
  return out;
}

// ---- gradient norm ----

int AdamwType(const Tensor& t) { return t.scalar_type() == at::kFloat ? SML_ADAMW_F32 : SML_ADAMW_BF16; }

// Same values in the same places of memory, without gaps: what an elementwise pass over memory may take.
bool Dense(const Tensor& t) { return t.is_non_overlapping_and_dense(); }

Tensor NormWorkspace(size_t tensors, const at::TensorOptions& where) {
  return at::empty({switchml_grad_norm_workspace(static_cast<int>(tensors))}, where.dtype(at::kDouble));
}

void NormOf(const std::vector<SmlNormTensor>& list, const Tensor& workspace, int* ticket, const Tensor& out) {
  Check(switchml_grad_norm(list.data(), static_cast<int>(list.size()), workspace.data_ptr<double>(), ticket, out.data_ptr<float>(), CurrentStream()),
        "grad_norm");
}

// Takes a list as it is: a vector of tensors would count every one of them up and down.
Tensor GradNorm(const py::list& tensors) {
  RefuseTracing("grad_norm");
  const Py_ssize_t count = PyList_GET_SIZE(tensors.ptr());
  TORCH_CHECK_VALUE(count > 0, "grad_norm: no tensors");
  std::vector<SmlNormTensor> list;
  std::vector<Tensor> keep;
  list.reserve(count);
  at::Device where(at::kCPU);
  const bool grad_mode = at::GradMode::is_enabled(), duals = DualsExist();
  at::NoGradGuard no_grad;
  std::optional<c10::cuda::CUDAGuard> device;
  for (Py_ssize_t i = 0; i < count; i++) {
    PyObject* const item = PyList_GET_ITEM(tensors.ptr(), i);
    TORCH_CHECK_TYPE(THPVariable_CheckExact(item) || THPVariable_Check(item), "grad_norm: tensors are wanted");
    const Tensor* t = &THPVariable_Unpack(item);
    TORCH_CHECK_TYPE(t->layout() == at::kStrided && Known(*t), "grad_norm: a tensor is ", t->layout(), " ", t->scalar_type(),
                     ": strided float32 or bfloat16 is wanted");
    if (duals) RefuseDual(*t, "grad_norm");
    TORCH_CHECK(!grad_mode || !t->requires_grad(),
                "grad_norm has no gradient: a tensor that requires one is wanted detached, or the call under no_grad");
    if (i == 0) where = t->device();
    TORCH_CHECK_VALUE(t->is_cuda() && t->device() == where, "grad_norm: tensors on ", where, " and ", t->device(), ": one CUDA device is wanted");
    if (i == 0) device.emplace(where);
    if (!Dense(*t) || Implied(*t)) {
      keep.push_back(Contiguous(*t));
      t = &keep.back();
    }
    list.push_back({Data(*t), t->numel(), AdamwType(*t)});
  }
  const Tensor out = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(where));
  NormOf(list, NormWorkspace(list.size(), out.options()), nullptr, out);
  return out;
}

// ---- AdamW ----

struct Group {
  std::vector<Tensor> params;
  std::vector<int64_t> numel, place;  // place: in units of SML_ADAMW_ALIGN values
  std::vector<at::ScalarType> type;
  std::vector<std::vector<int64_t>> sizes, strides;  // as the state lies; empty for contiguous parameters
  Tensor exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, remainder, steps;
  int64_t first = 0;
};

class Adamw {
 public:
  Adamw(int bits, int64_t seed) : bits_(bits), seed_(static_cast<unsigned>(seed)) {}

  void AddGroup(std::vector<Tensor> params, std::vector<int64_t> place, Tensor exp_avg, Tensor exp_avg_sq, OptTensor exp_avg_scale,
                OptTensor exp_avg_sq_scale, OptTensor remainder, Tensor steps, int64_t first) {
    Group g;
    for (const Tensor& p : params) {
      g.numel.push_back(p.numel()), g.type.push_back(p.scalar_type());
      g.sizes.push_back(p.is_contiguous() ? std::vector<int64_t>() : p.sizes().vec());
      g.strides.push_back(p.is_contiguous() ? std::vector<int64_t>() : p.strides().vec());
    }
    g.params = std::move(params), g.place = std::move(place);
    g.exp_avg = std::move(exp_avg), g.exp_avg_sq = std::move(exp_avg_sq), g.steps = std::move(steps), g.first = first;
    g.exp_avg_scale = exp_avg_scale.value_or(Tensor()), g.exp_avg_sq_scale = exp_avg_sq_scale.value_or(Tensor());
    g.remainder = remainder.value_or(Tensor());
    // Steps may have been captured with the workspace that there was: it stays.
    count_ += g.params.size();
    workspaces_.push_back(NormWorkspace(count_, g.exp_avg.options()));
    if (!norm_.defined()) {  // (the last one that is made)
      ticket_ = at::zeros({1}, g.exp_avg.options().dtype(at::kInt));
      norm_ = at::zeros({}, g.exp_avg.options().dtype(at::kFloat));
    }
    groups_.push_back(std::move(g));
  }

  // settings: (lr, beta1, beta2, eps, weight decay) of every group; lr_tensors: lr in device memory, or None.
  void Step(const std::vector<std::array<double, 5>>& settings, const std::vector<OptTensor>& lr_tensors, std::optional<double> max_norm) {
    RefuseTracing("FusedAdamW");
    TORCH_CHECK(settings.size() == groups_.size() && lr_tensors.size() == groups_.size(), "FusedAdamW: groups have come or gone");
    const c10::cuda::OptionalCUDAGuard device(ticket_.device());
    at::NoGradGuard no_grad;
    tensors_.clear(), norms_.clear(), stepped_.clear();
    std::vector<Tensor> keep;
    struct Run { size_t begin, end; int type; };
    std::vector<std::pair<size_t, Run>> runs;  // of tensors whose gradients are of one type, by group
    for (size_t k = 0; k < groups_.size(); k++) {
      Group& g = groups_[k];
      for (const int type : {SML_ADAMW_F32, SML_ADAMW_BF16}) {
        const size_t begin = tensors_.size();
        for (size_t i = 0; i < g.params.size(); i++) {
          const Tensor& p = g.params[i];
          if (TypeOf(g, i) != type) continue;
          const Tensor* grad = &p.grad();
          if (!grad->defined()) continue;
          CheckParam(g, i);
          CheckGrad(p, *grad);
          if ((!(p.is_contiguous() && grad->is_contiguous()) && p.strides() != grad->strides()) || Implied(*grad)) {
            keep.push_back(at::empty_strided(p.sizes(), p.strides(), grad->options()).copy_(*grad));
            grad = &keep.back();
          }
          void* const grad_data = Data(*grad);
          tensors_.push_back({Writable(p), grad_data, g.numel[i], static_cast<unsigned>(g.place[i]), static_cast<int>(i)});
          stepped_.push_back(p.unsafeGetTensorImpl());
          if (max_norm) norms_.push_back({grad_data, g.numel[i], type});
        }
        if (tensors_.size() > begin) runs.push_back({k, {begin, tensors_.size(), type}});
      }
    }
    if (max_norm) NormOf(norms_, workspaces_.back(), ticket_.data_ptr<int>(), norm_);
    for (const auto& [k, run] : runs) {
      const Group& g = groups_[k];
      const SmlAdamwState state{Writable(g.exp_avg), Writable(g.exp_avg_sq), static_cast<unsigned char*>(Writable(g.exp_avg_scale)),
                                static_cast<unsigned char*>(Writable(g.exp_avg_sq_scale)), static_cast<short*>(Writable(g.remainder)), g.steps.data_ptr<int>(), ticket_.data_ptr<int>(), bits_, seed_, static_cast<unsigned long long>(g.first)};
      const auto& s = settings[k];
      const SmlAdamwStep step{s[0], s[1], s[2], s[3], s[4], lr_tensors[k] ? lr_tensors[k]->const_data_ptr<float>() : nullptr,
                              max_norm ? norm_.data_ptr<float>() : nullptr, static_cast<float>(max_norm.value_or(0.0))};
      Check(switchml_adamw_step(&tensors_[run.begin], static_cast<int>(run.end - run.begin), &state, &step, run.type, CurrentStream()),
            "FusedAdamW");
    }
    for (c10::TensorImpl* p : stepped_) p->bump_version();
  }

  // The fp32 values of a group's parameters, in the layout of its state.
  Tensor Masters(size_t k) {
    RefuseTracing("FusedAdamW");
    const c10::cuda::OptionalCUDAGuard device(ticket_.device());
    const Group& g = groups_.at(k);
    const auto options = g.exp_avg.options().dtype(at::kFloat);
    // (A group of empty tensors has a block of state too, which belongs to none of them.)
    const bool any = std::any_of(g.numel.begin(), g.numel.end(), [](int64_t n) { return n > 0; });
    Tensor out = any ? at::empty({g.exp_avg.numel()}, options) : at::zeros({g.exp_avg.numel()}, options);
    for (const int type : {SML_ADAMW_F32, SML_ADAMW_BF16}) {
      tensors_.clear();
      for (size_t i = 0; i < g.params.size(); i++) {
        CheckParam(g, i);
        if (TypeOf(g, i) == type)
          tensors_.push_back({Data(g.params[i]), nullptr, g.numel[i], static_cast<unsigned>(g.place[i]), static_cast<int>(i)});
      }
      if (tensors_.empty()) continue;
      Check(switchml_adamw_masters(tensors_.data(), static_cast<int>(tensors_.size()), static_cast<short*>(Data(g.remainder)),
                                   out.data_ptr<float>(), type, CurrentStream()),
            "FusedAdamW");
    }
    return out;
  }

  Tensor norm() const { return norm_; }

 private:
  static int TypeOf(const Group& g, size_t i) { return g.type[i] == at::kFloat ? SML_ADAMW_F32 : SML_ADAMW_BF16; }
  // What a parameter's storage has become: p.data may have been exchanged.
  void CheckParam(const Group& g, size_t i) const {
    const Tensor& p = g.params[i];
    TORCH_CHECK(p.numel() == g.numel[i] && Dense(p) && !Implied(p) && p.scalar_type() == g.type[i] && p.device() == ticket_.device(),
                "FusedAdamW: a parameter has another size, type or device than when its state was made, or gaps in memory");
    TORCH_CHECK(SameOrder(g, i), "FusedAdamW: a parameter's values lie in another order than when its state was made (sizes ", p.sizes(),
                ", strides ", p.strides(), "): a memory format is chosen before the optimizer is made");
  }
  // Values and state meet by their places in memory.
  static bool SameOrder(const Group& g, size_t i) {
    const Tensor& p = g.params[i];
    if (g.sizes[i].empty()) return p.is_contiguous();
    if (p.sizes() != g.sizes[i]) return false;
    for (int64_t d = 0; d < p.dim(); d++)
      if (p.size(d) > 1 && p.stride(d) != g.strides[i][d]) return false;
    return true;
  }
  static void CheckGrad(const Tensor& p, const Tensor& grad) {
    TORCH_CHECK(grad.layout() == at::kStrided, "FusedAdamW: a gradient is ", grad.layout(), ": strided is wanted");
    TORCH_CHECK(grad.scalar_type() == p.scalar_type() && grad.device() == p.device() && grad.sizes() == p.sizes(),
                "FusedAdamW: a parameter is ", p.scalar_type(), " ", p.sizes(), " on ", p.device(), ", its gradient ", grad.scalar_type(), " ",
                grad.sizes(), " on ", grad.device());
  }

  const int bits_;
  const unsigned seed_;
  std::vector<Group> groups_;
  Tensor ticket_, norm_;
  std::vector<Tensor> workspaces_;  // the last one is for all groups
  size_t count_ = 0;                // of all parameters
  std::vector<SmlAdamwTensor> tensors_;
  std::vector<SmlNormTensor> norms_;
  std::vector<c10::TensorImpl*> stepped_;  // parameters of this step
};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("layer_norm", &LayerNormForward);
  m.def("grad_norm", &GradNorm);
  m.attr("ALIGN") = static_cast<int>(SML_ADAMW_ALIGN);
  py::class_<Adamw>(m, "Adamw")
      .def(py::init<int, int64_t>())
      .def("add_group", &Adamw::AddGroup)
      .def("step", &Adamw::Step)
      .def("masters", &Adamw::Masters)
      .def_property_readonly("norm", &Adamw::norm);
}
