// titanet_amd — host side of the optimizer step and of the 8-bit product for torch tensors (Python module titanet_amd._host).
//
// The kernels of these operators take microseconds; reading a few hundred tensors' addresses, types and gradients through Python
// took longer than the step of a whole model (560 us against 48 us of kernels for 428 tensors; now 35).  What is checked and collected in
// every call is therefore done here, and the launches go through the C entries of libtitanet_amd.so like every other caller's.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <ATen/core/grad_mode.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <cmath>
#include <optional>
#include <vector>

#include "../../include/titanet_amd.h"

namespace py = pybind11;

namespace {

int type_code(c10::ScalarType t) {
  return t == at::kFloat ? TN_DTYPE_F32 : t == at::kBFloat16 ? TN_DTYPE_BF16 : t == at::kHalf ? TN_DTYPE_F16 : -1;
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed: ", rc == TN_E_BADARG ? "TN_E_BADARG" : rc == TN_E_UNSUPPORTED ? "TN_E_UNSUPPORTED" : "hipError_t ", rc > 0 ? std::to_string(rc) : "");
}

void* current_stream(const c10::Device& d) { return (void*)c10::hip::getCurrentHIPStream(d.index()).stream(); }

// ------------------------------------------------------------------------------------------------------------- optimizer
struct Lists {                         // the tensors of one type that a step touches
  std::vector<void*> p;
  std::vector<const void*> g;
  std::vector<int64_t> numel, first;
  std::vector<int32_t> index, slot;
  void reserve(size_t n) {
    p.reserve(n);
    g.reserve(n);
    numel.reserve(n);
    first.reserve(n);
    index.reserve(n);
    slot.reserve(n);
  }
  tn_adamw_lists c(int code) const { return {(int32_t)p.size(), code, p.data(), g.data(), numel.data(), first.data(), slot.data()}; }
};

struct GroupWork {
  std::array<Lists, 3> by_type;
  std::vector<int32_t> slots;
  tn_adamw_hyper h;
  at::Tensor lr_dev;
};

struct Norm {                          // partial sums of several lists, then their norm
  static int64_t partials(const std::vector<std::pair<int, Lists*>>& lists) {
    int64_t n = 0;
    for (auto& [code, l] : lists) n += tn_grad_sumsq_partials((int32_t)l->numel.size(), l->numel.data());
    return n;
  }
  static int64_t sums(const std::vector<std::pair<int, Lists*>>& lists, double* out, void* stream) {
    int64_t at = 0, written = 0;
    for (auto& [code, l] : lists) {
      check(tn_grad_sumsq((int32_t)l->numel.size(), l->g.data(), l->numel.data(), code, out + at, &written, stream), "tn_grad_sumsq");
      at += written;
    }
    return at;
  }
};

class Stepper {
 public:
  Stepper(int bits) : bits_(bits) {}

  void layout(std::vector<int64_t> numel, std::vector<int64_t> first, std::vector<int32_t> sets, int64_t blocks, at::Tensor exp_avg,
              at::Tensor exp_avg_sq, std::optional<at::Tensor> scale1, std::optional<at::Tensor> scale2, at::Tensor steps, at::Tensor corr, at::Tensor owner, const py::list& params) {
    numel_ = std::move(numel);
    first_ = std::move(first);
    blocks_ = blocks;
    exp_avg_ = exp_avg;
    exp_avg_sq_ = exp_avg_sq;
    scale1_ = scale1.value_or(at::Tensor());
    scale2_ = scale2.value_or(at::Tensor());
    steps_ = steps;
    corr_ = corr;
    owner_ = owner;
    params_.clear();
    for (const auto& p : params) params_.push_back(p.ptr());
    if (!norm_.defined()) norm_ = at::zeros({}, corr.options());
    put_sets(std::move(sets));
  }
  std::vector<int32_t> sets() const { return sets_; }
  void put_sets(std::vector<int32_t> s) {
    TORCH_CHECK(s.size() == numel_.size());
    sets_ = std::move(s);
  }
  bool captured() const { return captured_; }

  // the moments as float32 values; 32 bits: the buffers themselves
  std::pair<at::Tensor, at::Tensor> moments() const {
    if (bits_ == 32) return {exp_avg_, exp_avg_sq_};
    const at::NoGradGuard no_grad;
    const c10::OptionalDeviceGuard guard(exp_avg_.device());
    at::Tensor m = at::empty(exp_avg_.sizes(), scale1_.options()), v = at::empty(exp_avg_.sizes(), scale1_.options());
    check(tn_moments_decode(exp_avg_.const_data_ptr(), exp_avg_sq_.const_data_ptr(), scale1_.const_data_ptr<float>(), scale2_.const_data_ptr<float>(),
                            m.mutable_data_ptr<float>(), v.mutable_data_ptr<float>(), blocks_, current_stream(exp_avg_.device())),
          "tn_moments_decode");
    return {m, v};
  }

  // one step of all groups; the norm before clipping (0-dim float32) where max_norm > 0
  std::optional<at::Tensor> step(const py::list& groups, double max_norm, double grad_mult) {
    const at::NoGradGuard no_grad;
    const c10::Device dev = exp_avg_.device();
    const c10::OptionalDeviceGuard guard(dev);
    const bool capturing = c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
    std::vector<at::Tensor> keep;                // gradients laid out anew
    std::vector<c10::TensorImpl*> stepped;       // parameters (the group's list holds them)
    stepped.reserve(numel_.size());
    std::vector<GroupWork> work;
    std::vector<char> active(numel_.size(), 0);
    work.reserve(groups.size());
    bool moved = false;
    int32_t at = 0;
    for (const auto& item : groups) {
      const py::dict group = py::reinterpret_borrow<py::dict>(item);
      const py::list params = group["params"];
      GroupWork w;
      bool any = false;
      const Py_ssize_t count = PyList_GET_SIZE(params.ptr());
      for (Py_ssize_t k = 0; k < count; ++k) {
        PyObject* obj = PyList_GET_ITEM(params.ptr(), k);
        const int32_t i = at++;
        TORCH_CHECK(THPVariable_Check(obj) && (size_t)i < numel_.size(), "AdamW: the parameter list changed; use add_param_group");
        moved |= obj != params_[i];
        const at::Tensor& p = THPVariable_Unpack(obj);
        const at::Tensor& given = p.grad();
        if (!given.defined()) continue;
        TORCH_CHECK(given.layout() == at::kStrided, "AdamW does not take sparse gradients");
        const int code = type_code(p.scalar_type());
        TORCH_CHECK(code >= 0 && p.device() == dev && given.device() == dev && given.scalar_type() == p.scalar_type() && p.numel() == numel_[i] &&
                        given.numel() == numel_[i] && p.is_contiguous(),
                    "parameter ", i, " is no longer what this optimizer was built for (device, type, size or layout changed)");
        w.slots.push_back(i);
        if (numel_[i] == 0) continue;
        const void* g = given.const_data_ptr();
        if (!given.is_contiguous()) {
          keep.push_back(given.contiguous());
          g = keep.back().const_data_ptr();
        }
        Lists& l = w.by_type[code];
        if (l.p.empty()) l.reserve((size_t)count);
        l.p.push_back(p.mutable_data_ptr());
        l.g.push_back(g);
        l.numel.push_back(numel_[i]);
        l.first.push_back(first_[i]);
        l.index.push_back(i);
        active[i] = 1;
        any = true;
        stepped.push_back(p.unsafeGetTensorImpl());
      }
      if (!any) continue;
      hyper(group, dev, capturing, w);
      work.push_back(std::move(w));
    }
    // Moments belong to positions.  A parameter that was exchanged for another of its size keeps its position's; where some were taken out of
    // the groups, those that are left must be at theirs.
    TORCH_CHECK(!moved || (size_t)at == numel_.size(), "AdamW: the parameter list changed; use add_param_group");
    if (work.empty()) return std::nullopt;
    split(active, capturing);
    // Every tensor has a count of its own, at its own place on the device, which is advanced in every step that it takes part in.  Tensors of
    // one set read that of the set's first, so that neighbours in memory are stepped as one run.  In a graph every block looks up its own
    // tensor's: it is replayed when later eager steps may have parted the set.
    std::vector<int32_t> first_of(numel_.size(), -1);
    for (auto& w : work)
      for (auto& l : w.by_type)
        for (int32_t i : l.index) {
          int32_t& f = first_of[sets_[i]];
          if (f < 0) f = i;
          l.slot.push_back(f);
        }
    captured_ |= capturing;
    void* stream = current_stream(dev);
    const tn_adamw_state state = {bits_, blocks_, exp_avg_.mutable_data_ptr(), exp_avg_sq_.mutable_data_ptr(),
                                  scale1_.defined() ? scale1_.mutable_data_ptr<float>() : nullptr,
                                  scale2_.defined() ? scale2_.mutable_data_ptr<float>() : nullptr, steps_.mutable_data_ptr<int32_t>(),
                                  corr_.mutable_data_ptr<float>(), capturing ? owner_.const_data_ptr<int32_t>() : nullptr};
    std::vector<std::pair<int, Lists*>> lists;
    for (auto& w : work)
      for (int code = 0; code < 3; ++code)
        if (!w.by_type[code].p.empty()) lists.emplace_back(code, &w.by_type[code]);
    at::Tensor norm, partials;
    // A tensor of its own for every eager step, so that norms can be collected; once there is a graph, one that every step and replay writes:
    // the host does not see which of several graphs ran last.
    if (max_norm > 0.0) norm = captured_ ? norm_ : at::empty({}, norm_.options());
    float* norm_ptr = norm.defined() ? norm.mutable_data_ptr<float>() : nullptr;
    int small = TN_E_UNSUPPORTED;
    if (lists.size() == 1) {
      const tn_adamw_lists l = lists[0].second->c(lists[0].first);
      small = tn_adamw_step_small(&l, &state, &work[0].h, (int32_t)work[0].slots.size(), work[0].slots.data(), grad_mult, max_norm, norm_ptr, stream);
      if (small != TN_E_UNSUPPORTED) check(small, "tn_adamw_step_small");
    }
    if (small == TN_E_UNSUPPORTED) {
      double* ctl = nullptr;
      int64_t count = 0;
      if (max_norm > 0.0) {
        partials = at::empty({Norm::partials(lists) + 2}, at::TensorOptions().dtype(at::kDouble).device(dev));
        ctl = partials.mutable_data_ptr<double>();             // two for the factor, then the sums
        count = Norm::sums(lists, ctl + 2, stream);
      }
      bool first = max_norm > 0.0;
      for (auto& w : work) {
        check(tn_adamw_tick((int32_t)w.slots.size(), w.slots.data(), &state, &w.h, first ? ctl + 2 : nullptr, count, grad_mult, max_norm, norm_ptr, ctl, stream),
              "tn_adamw_tick");
        first = false;
        for (int code = 0; code < 3; ++code) {
          if (w.by_type[code].p.empty()) continue;
          const tn_adamw_lists l = w.by_type[code].c(code);
          check(tn_adamw_apply(&l, &state, &w.h, grad_mult, ctl, stream), "tn_adamw_apply");
        }
      }
    }
    for (c10::TensorImpl* p : stepped)
      if (!p->is_inference()) p->bump_version();      // autograd has to see that the values changed
    if (max_norm > 0.0) return norm;
    return std::nullopt;
  }

 private:
  void hyper(const py::dict& group, const c10::Device& dev, bool capturing, GroupWork& w) {
    const py::object lr = group["lr"];
    w.h.lr = 0.0;
    w.h.lr_dev = nullptr;
    if (THPVariable_Check(lr.ptr())) {
      w.lr_dev = THPVariable_Unpack(lr.ptr());
      TORCH_CHECK_VALUE(w.lr_dev.scalar_type() == at::kFloat && w.lr_dev.dim() == 0 && w.lr_dev.device() == dev,
                        "a tensor lr must be a 0-dim float32 tensor on the parameters' device");
      w.h.lr_dev = w.lr_dev.const_data_ptr<float>();
    } else {
      TORCH_CHECK(!capturing, "AdamW: give lr as a 0-dim device tensor to capture a step (a number would be frozen into the graph)");
      w.h.lr = lr.cast<double>();
      TORCH_CHECK_VALUE(w.h.lr >= 0.0, "Invalid learning rate: ", w.h.lr);
    }
    const py::sequence betas = group["betas"];
    w.h.beta1 = betas[0].cast<double>();
    w.h.beta2 = betas[1].cast<double>();
    w.h.eps = group["eps"].cast<double>();
    w.h.weight_decay = group["weight_decay"].cast<double>();
    TORCH_CHECK_VALUE(w.h.beta1 >= 0.0 && w.h.beta1 < 1.0 && w.h.beta2 >= 0.0 && w.h.beta2 < 1.0, "betas must be two numbers in [0, 1)");
    TORCH_CHECK_VALUE(w.h.eps >= 0.0 && w.h.weight_decay >= 0.0, "eps and weight_decay must not be negative");
  }

  // A set holds tensors of one group whose counts are equal.  Where some of its tensors have a gradient and others have not, those that
  // have become a set of their own.  (There are as many numbers as tensors, so one is free whenever two tensors share one.)  Sets are
  // only ever parted once a step has been captured: a replay advances its tensors without this host code, but always all of a set.
  void split(const std::vector<char>& active, bool capturing) {
    const size_t n = sets_.size();
    std::vector<int32_t> some(n, 0), every(n, 0);
    for (size_t i = 0; i < n; ++i) {
      if (numel_[i] == 0) continue;
      every[sets_[i]]++;
      some[sets_[i]] += active[i];
    }
    for (size_t s = 0; s < n; ++s) {
      if (some[s] == 0 || some[s] == every[s]) continue;
      TORCH_CHECK(!capturing, "AdamW: other parameters than before have gradients in a captured step: run such a step once before capturing it");
      std::vector<char> used(n, 0);
      for (int32_t k : sets_) used[k] = 1;
      size_t free = 0;
      while (used[free]) ++free;
      for (size_t i = 0; i < n; ++i)
        if (sets_[i] == (int32_t)s && active[i]) sets_[i] = (int32_t)free;
    }
  }

  int bits_;
  int64_t blocks_ = 0;
  std::vector<int64_t> numel_, first_;
  std::vector<int32_t> sets_;
  std::vector<PyObject*> params_;        // compared only: the Python side holds them
  bool captured_ = false;
  at::Tensor exp_avg_, exp_avg_sq_, scale1_, scale2_, steps_, corr_, owner_, norm_;
};

at::Tensor grad_norm(const std::vector<at::Tensor>& tensors) {
  const at::NoGradGuard no_grad;
  TORCH_CHECK_VALUE(!tensors.empty(), "grad_norm needs at least one tensor");
  const c10::Device dev = tensors[0].device();
  for (const auto& t : tensors) {
    TORCH_CHECK_TYPE(t.layout() == at::kStrided && type_code(t.scalar_type()) >= 0, "grad_norm takes dense float32, bfloat16 or float16 tensors");
    TORCH_CHECK(t.is_cuda(), "titanet_amd.optim needs ROCm device tensors; there is no CPU execution path");
    TORCH_CHECK_VALUE(t.device() == dev, "grad_norm takes tensors of one device, got ", dev, " and ", t.device());
  }
  const c10::OptionalDeviceGuard guard(dev);
  std::vector<at::Tensor> keep;
  std::array<Lists, 3> by_type;
  for (const auto& t : tensors) {
    keep.push_back(t.is_contiguous() ? t : t.contiguous());
    Lists& l = by_type[type_code(t.scalar_type())];
    l.g.push_back(keep.back().const_data_ptr());
    l.numel.push_back(t.numel());
  }
  std::vector<std::pair<int, Lists*>> lists;
  for (int code = 0; code < 3; ++code)
    if (!by_type[code].g.empty()) lists.emplace_back(code, &by_type[code]);
  void* stream = current_stream(dev);
  at::Tensor partials = at::empty({Norm::partials(lists) + 1}, at::TensorOptions().dtype(at::kDouble).device(dev));
  at::Tensor norm = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev));
  const int64_t count = Norm::sums(lists, partials.mutable_data_ptr<double>(), stream);
  check(tn_grad_norm_finish(partials.const_data_ptr<double>(), count, 1.0, INFINITY, norm.mutable_data_ptr<float>(), nullptr, stream), "tn_grad_norm_finish");
  return norm;
}

// --------------------------------------------------------------------------------------------------------- 8-bit product
// what flows through these operators is not differentiated: an operand that asks for it is refused, not cut off
void need_no_gradient(const at::Tensor& t, const char* what) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what, " has no backward pass: detach its operands or call it under torch.no_grad()");
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), what, " has no backward pass and no forward-mode derivative: unpack its operands' primals");
}

// torch.jit.trace records torch's own operators only: a module traced through here would return memory that nothing has written
void need_no_trace(const char* what) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced (torch.jit.trace, torch.onnx.export): its kernels are no operators of torch");
}

std::pair<at::Tensor, at::Tensor> quantize_rows(const at::Tensor& given) {
  need_no_trace("quantize_rows");
  TORCH_CHECK_TYPE(type_code(given.scalar_type()) >= 0 && given.layout() == at::kStrided, "quantize_rows takes a float32, bfloat16 or float16 matrix, got ", given.scalar_type());
  TORCH_CHECK_VALUE(given.dim() == 2 && given.size(1) >= 1, "quantize_rows takes a matrix with at least one column, got ", given.sizes());
  TORCH_CHECK_VALUE(given.size(1) <= TN_INT8_MAX_K, "rows of more than ", TN_INT8_MAX_K, " values could overflow the 32-bit sums");
  TORCH_CHECK(given.is_cuda(), "titanet_amd.int8: x must be a ROCm device tensor; there is no CPU execution path");
  need_no_gradient(given, "quantize_rows");
  const at::NoGradGuard no_grad;
  const c10::OptionalDeviceGuard guard(given.device());
  const at::Tensor x = given.stride(1) == 1 || given.size(1) == 1 ? given : given.contiguous();
  const int64_t rows = x.size(0), cols = x.size(1), ld = (cols + 63) / 64 * 64;
  at::Tensor codes = at::empty({rows, ld}, x.options().dtype(at::kChar)), scales = at::empty({rows}, x.options().dtype(at::kFloat));
  check(tn_int8_quantize_rows(x.const_data_ptr(), type_code(x.scalar_type()), rows, cols, x.stride(0), codes.mutable_data_ptr(), ld,
                              scales.mutable_data_ptr<float>(), current_stream(x.device())),
        "tn_int8_quantize_rows");
  return {codes, scales};
}

// Rows of codes as the kernels read them.  A module's buffers can be moved or replaced after they were checked: a kernel that gets a host
// address takes the device down.
void need_rows(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, const char* what) {
  TORCH_CHECK(codes.is_cuda() && scales.is_cuda(), "titanet_amd.int8: ", what, " must be on a ROCm device, got ", codes.device(), " and ", scales.device(),
              "; there is no CPU execution path");
  TORCH_CHECK_VALUE(codes.device() == scales.device(), "codes and scales are on different devices: ", codes.device(), " and ", scales.device());
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kChar && scales.scalar_type() == at::kFloat, what, " must be int8 codes and float32 scales, got ", codes.scalar_type(),
                   " and ", scales.scalar_type());
  TORCH_CHECK_VALUE(codes.dim() == 2 && codes.is_contiguous() && codes.size(1) >= cols && scales.dim() == 1 && scales.is_contiguous() &&
                        scales.size(0) == codes.size(0),
                    what, ": codes ", codes.sizes(), " and scales ", scales.sizes(), " do not belong together");
}

struct Out {
  at::Tensor bias, y;
  const float* bias_ptr = nullptr;
};

Out prepare_out(const c10::Device& dev, int64_t cols_a, int64_t cols, int64_t m, const at::Tensor& b, const std::optional<at::Tensor>& bias,
                c10::ScalarType out) {
  TORCH_CHECK_TYPE(type_code(out) >= 0, "out_dtype must be float32, bfloat16 or float16, got ", out);
  TORCH_CHECK_VALUE(cols_a == cols, "operands of ", cols_a, " and ", cols, " columns");
  TORCH_CHECK_VALUE(dev == b.device(), "operands on different devices: ", dev, " and ", b.device());
  Out o;
  const int64_t n = b.size(0);
  if (bias) {
    TORCH_CHECK_VALUE(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == n && bias->device() == b.device(), "bias must be float32 [", n, "] on ",
                      b.device(), ", got ", bias->scalar_type(), " ", bias->sizes(), " on ", bias->device());
    o.bias = bias->is_contiguous() ? *bias : bias->contiguous();
    o.bias_ptr = o.bias.const_data_ptr<float>();
  }
  o.y = at::empty({m, n}, b.options().dtype(out));
  return o;
}

void product(const at::Tensor& a, const at::Tensor& a_scales, const at::Tensor& b, const at::Tensor& b_scales, int64_t cols, Out& o) {
  check(tn_int8_matmul(a.const_data_ptr(), a_scales.const_data_ptr<float>(), a.size(1), b.const_data_ptr(), b_scales.const_data_ptr<float>(), b.size(1),
                       o.bias_ptr, o.y.mutable_data_ptr(), type_code(o.y.scalar_type()), b.size(0), a.size(0), b.size(0), cols, current_stream(b.device())),
        "tn_int8_matmul");
}

at::Tensor matmul_rows(const at::Tensor& a, const at::Tensor& a_scales, int64_t cols_a, const at::Tensor& b, const at::Tensor& b_scales, int64_t cols,
                       const std::optional<at::Tensor>& bias, std::optional<c10::ScalarType> out) {
  need_no_trace("int8_matmul");
  need_rows(a, a_scales, cols_a, "the first operand");
  need_rows(b, b_scales, cols, "the second operand");
  const c10::OptionalDeviceGuard guard(b.device());
  if (bias) need_no_gradient(*bias, "int8_matmul");
  const at::NoGradGuard no_grad;
  Out o = prepare_out(a.device(), cols_a, cols, a.size(0), b, bias, out.value_or(at::kFloat));
  product(a, a_scales, b, b_scales, cols, o);
  return o.y;
}

at::Tensor matmul_float(const at::Tensor& x, const at::Tensor& b, const at::Tensor& b_scales, int64_t cols, const std::optional<at::Tensor>& bias,
                        std::optional<c10::ScalarType> out) {
  need_no_trace("int8_matmul");
  TORCH_CHECK_TYPE(type_code(x.scalar_type()) >= 0 && x.layout() == at::kStrided,
                   "the first operand must be Int8Rows or a float32, bfloat16 or float16 tensor, got ", x.scalar_type());
  TORCH_CHECK_VALUE(x.dim() >= 1, "the first operand needs at least one dimension");
  need_rows(b, b_scales, cols, "the second operand");
  need_no_gradient(x, "int8_matmul");
  if (bias) need_no_gradient(*bias, "int8_matmul");
  const at::NoGradGuard no_grad;
  const c10::OptionalDeviceGuard guard(b.device());
  const int64_t cols_a = x.size(-1);
  TORCH_CHECK_VALUE(cols_a == cols, "operands of ", cols_a, " and ", cols, " columns");
  const at::Tensor flat = x.dim() == 2 ? x : x.reshape({-1, cols});
  Out o = prepare_out(x.device(), cols_a, cols, flat.size(0), b, bias, out.value_or(x.scalar_type()));
  const at::Tensor rows = flat.stride(1) == 1 || cols == 1 ? flat : flat.contiguous();
  const int64_t bytes = tn_int8_linear_workspace(rows.size(0), cols);
  at::Tensor workspace;
  if (bytes > 0) workspace = at::empty({bytes}, b.options());
  check(tn_int8_linear(rows.const_data_ptr(), type_code(x.scalar_type()), rows.stride(0), b.const_data_ptr(), b_scales.const_data_ptr<float>(), b.size(1),
                       o.bias_ptr, o.y.mutable_data_ptr(), type_code(o.y.scalar_type()), b.size(0), rows.size(0), b.size(0), cols,
                       bytes > 0 ? workspace.mutable_data_ptr() : nullptr, bytes, current_stream(b.device())),
        "tn_int8_linear");
  if (x.dim() == 2) return o.y;
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = b.size(0);
  return o.y.view(shape);
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  py::class_<Stepper>(m, "Stepper")
      .def(py::init<int>())
      .def("layout", &Stepper::layout)
      .def("step", &Stepper::step)
      .def("moments", &Stepper::moments)
      .def_property("sets", &Stepper::sets, &Stepper::put_sets)
      .def_property_readonly("captured", &Stepper::captured);
  m.def("grad_norm", &grad_norm);
  m.def("quantize_rows", &quantize_rows);
  m.def("matmul_rows", &matmul_rows);
  m.def("matmul_float", &matmul_float);
}
