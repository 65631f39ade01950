// Torch front end of the list entry points (gradient norm, clipping, AdamW step): the loops over parameter tensors and
// their checks run here rather than in Python, and a step of a few hundred tensors costs the host microseconds.
// Host code only; the C ABI is bound at run time with that of the residual losses (pde_amd_torch_bind).
#include <dlfcn.h>

#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <tuple>
#include <vector>

#include <ATen/ATen.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/custom_class.h>
#include <torch/library.h>

#include "../../include/pde_amd.h"

namespace {

struct Abi {
  decltype(&pde_amd_multi_workspace_bytes) workspace_bytes = nullptr;
  decltype(&pde_amd_multi_norm) norm = nullptr;
  decltype(&pde_amd_multi_clip) clip = nullptr;
  decltype(&pde_amd_multi_norm_clip) norm_clip = nullptr;
  decltype(&pde_amd_multi_adamw) adamw = nullptr;
  decltype(&pde_amd_status_string) status_string = nullptr;
  decltype(&pde_amd_diag_poison_lds) poison_lds = nullptr;
} abi;

void check(int st, const char* what) {
  TORCH_CHECK(st == 0, "pde_amd: ", what, " failed: ", abi.status_string ? abi.status_string(st) : "?", " (", st, ")");
}

void check_bound() { TORCH_CHECK(abi.norm != nullptr, "pde_amd: the kernel library is not bound (pde_amd_torch_bind)"); }

int32_t type_of(const at::Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return PDE_AMD_F32;
    case at::kBFloat16: return PDE_AMD_BF16;
    case at::kHalf: return PDE_AMD_F16;
    default: TORCH_CHECK_TYPE(false, "pde_amd: ", what, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

// PDE_AMD_POISON_LDS=1: NaNs into every workspace and every CU's LDS ahead of a call
bool poison() {
  static const bool on = [] { const char* e = std::getenv("PDE_AMD_POISON_LDS"); return e && !std::strcmp(e, "1"); }();
  return on;
}

at::Tensor workspace(const at::Device& dev, int32_t n, void* stream) {
  at::Tensor ws = at::empty({(int64_t)abi.workspace_bytes(n)}, at::TensorOptions().dtype(at::kByte).device(dev));
  if (poison()) {
    ws.fill_(255);
    check(abi.poison_lds(stream), "diag_poison_lds");
  }
  return ws;
}

// A list of tensors as the C ABI takes it
struct List {
  std::vector<const void*> ptr;
  std::vector<int64_t> numel;
  std::vector<int32_t> dtype;
  std::vector<at::Tensor> keep;      // copies of tensors that are not dense
  at::Device dev = at::kCPU;

  void reserve(size_t n) { ptr.reserve(n); numel.reserve(n); dtype.reserve(n); }

  void add(const at::Tensor& t, const char* what, bool in_place) {
    TORCH_CHECK_TYPE(t.layout() == at::kStrided, "pde_amd: ", what, " must be dense tensors, got layout ", t.layout());
    const int32_t dt = type_of(t, what);
    if (ptr.empty()) dev = t.device();
    TORCH_CHECK_VALUE(t.device() == dev, "pde_amd: ", what, " must all be on one device, got ", dev, " and ", t.device());
    if (t.is_non_overlapping_and_dense()) {
      ptr.push_back(t.const_data_ptr());
    } else {
      TORCH_CHECK_VALUE(!in_place, "pde_amd: ", what, " that are written must be dense in memory (no gaps, no repeated elements), got sizes ",
                        t.sizes(), " with strides ", t.strides());
      keep.push_back(t.contiguous());
      ptr.push_back(keep.back().const_data_ptr());
    }
    numel.push_back(t.numel());
    dtype.push_back(dt);
  }

  int32_t size() const { return (int32_t)ptr.size(); }

  void check_device(const char* what) const {
    TORCH_CHECK(dev.is_cuda(), "pde_amd: ", what, " must be on a HIP device (there is no CPU fallback), got ", dev);
  }
};

struct Range {
  uintptr_t lo, hi;
};

// Memory that is written in one launch must belong to one tensor only.  Tensors mostly come in the order of their
// addresses; only others are sorted first.
void check_apart(std::vector<Range>& r, const char* what) {
  const auto before = [](const Range& a, const Range& b) { return a.lo < b.lo; };
  if (!std::is_sorted(r.begin(), r.end(), before)) std::sort(r.begin(), r.end(), before);
  for (size_t i = 1; i < r.size(); ++i)
    TORCH_CHECK_VALUE(r[i].lo >= r[i - 1].hi, "pde_amd: ", what, " share memory (the same tensor twice, or overlapping views)");
}

void add_range(std::vector<Range>& r, const void* p, int64_t bytes) {
  if (bytes > 0) r.push_back({(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes});
}

void check_apart(const List& l, const char* what) {
  std::vector<Range> r;
  r.reserve(l.ptr.size());
  for (size_t i = 0; i < l.ptr.size(); ++i) add_range(r, l.ptr[i], l.numel[i] * (l.dtype[i] == PDE_AMD_F32 ? 4 : 2));
  check_apart(r, what);
}

void written(const at::Tensor& t) {      // autograd has to know that saved values are gone
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

// [total], or [total, norms of the tensors]
std::vector<at::Tensor> total_norm(at::TensorList tensors, int64_t norm_type, bool each) {
  check_bound();
  List l;
  l.reserve(tensors.size());
  for (const auto& t : tensors) l.add(t, "tensors", false);
  if (!l.size()) {
    at::Tensor zero = at::zeros({}, at::kFloat);
    return each ? std::vector<at::Tensor>{zero, at::zeros({0}, at::kFloat)} : std::vector<at::Tensor>{zero};
  }
  l.check_device("tensors");
  c10::hip::HIPGuard guard(l.dev.index());
  void* stream = c10::hip::getCurrentHIPStream(l.dev.index()).stream();
  const auto opt = at::TensorOptions().dtype(at::kFloat).device(l.dev);
  std::vector<at::Tensor> out{at::empty({}, opt)};
  if (each) out.push_back(at::empty({l.size()}, opt));
  at::Tensor ws = workspace(l.dev, l.size(), stream);
  check(abi.norm(l.ptr.data(), l.numel.data(), l.dtype.data(), l.size(), (int32_t)norm_type, out[0].data_ptr<float>(),
                 each ? out[1].data_ptr<float>() : nullptr, ws.data_ptr(), (size_t)ws.numel(), stream),
        "multi_norm");
  return out;
}

std::vector<at::Tensor> grads_of(at::TensorList parameters) {
  std::vector<at::Tensor> g;
  g.reserve(parameters.size());
  for (const auto& p : parameters) {
    const at::Tensor& x = p.grad();
    if (x.defined()) g.push_back(x);
  }
  return g;
}

List written_list(const std::vector<at::Tensor>& grads) {
  List l;
  l.reserve(grads.size());
  for (const auto& g : grads) l.add(g, "gradients", true);
  check_apart(l, "gradients");
  if (l.size()) l.check_device("gradients");
  return l;
}

at::Tensor clip_grad_norm(at::TensorList parameters, double max_norm, int64_t norm_type) {
  check_bound();
  const std::vector<at::Tensor> grads = grads_of(parameters);
  const List l = written_list(grads);
  if (!l.size()) return at::zeros({}, at::kFloat);
  c10::hip::HIPGuard guard(l.dev.index());
  void* stream = c10::hip::getCurrentHIPStream(l.dev.index()).stream();
  at::Tensor total = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(l.dev));
  at::Tensor ws = workspace(l.dev, l.size(), stream);
  check(abi.norm_clip((void* const*)l.ptr.data(), l.numel.data(), l.dtype.data(), l.size(), (int32_t)norm_type, (float)max_norm,
                      total.data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream),
        "multi_norm_clip");
  for (const auto& g : grads) written(g);
  return total;
}

// the norm as a fp32 scalar on the gradients' device
at::Tensor norm_scalar(const at::Tensor& total, const at::Device& dev) {
  TORCH_CHECK_VALUE(total.numel() == 1, "pde_amd: total_norm must hold one value, got sizes ", total.sizes());
  TORCH_CHECK_TYPE(at::isFloatingType(total.scalar_type()), "pde_amd: total_norm must be a floating point tensor, got ", total.scalar_type());
  return total.to(at::TensorOptions().dtype(at::kFloat).device(dev)).contiguous();
}

void clip_grads_with_norm(at::TensorList parameters, double max_norm, const at::Tensor& total_norm) {
  check_bound();
  const std::vector<at::Tensor> grads = grads_of(parameters);
  const List l = written_list(grads);
  if (!l.size()) return;
  c10::hip::HIPGuard guard(l.dev.index());
  void* stream = c10::hip::getCurrentHIPStream(l.dev.index()).stream();
  const at::Tensor total = norm_scalar(total_norm, l.dev);
  check(abi.clip((void* const*)l.ptr.data(), l.numel.data(), l.dtype.data(), l.size(), (float)max_norm, total.data_ptr<float>(), stream),
        "multi_clip");
  for (const auto& g : grads) written(g);
}

// The parameters of an optimizer with their state, described once in device memory.  The description is made again when
// a tensor has moved; older ones are kept, since a captured step reads the one it was captured with.
struct AdamWPlan : torch::CustomClassHolder {
  std::vector<at::Tensor> params, exp_avg, exp_avg_sq, master, step;      // a parameter without state has undefined entries' stand-ins
  std::vector<bool> has_state;
  std::vector<pde_amd_adamw_tensor> table;
  std::vector<pde_amd_adamw_group> groups;
  std::vector<at::Tensor> tables;      // [table, groups] on the device, the current ones last
  at::Device dev = at::kCPU;

  // state: indices of the parameters that have state; exp_avg ... belong to those, in that order.  master: the parameter
  // itself where it is fp32.
  AdamWPlan(std::vector<at::Tensor> params_, std::vector<int64_t> groups, std::vector<int64_t> state, std::vector<at::Tensor> exp_avg_,
            std::vector<at::Tensor> exp_avg_sq_, std::vector<at::Tensor> master_, std::vector<at::Tensor> step_)
      : params(std::move(params_)) {
    check_bound();
    const size_t n = params.size();
    TORCH_CHECK_VALUE(groups.size() == n && exp_avg_.size() == state.size() && exp_avg_sq_.size() == state.size() &&
                          master_.size() == state.size() && step_.size() == state.size(),
                      "pde_amd: an optimizer's lists must have one entry per parameter");
    exp_avg.resize(n);
    exp_avg_sq.resize(n);
    master.resize(n);
    step.resize(n);
    has_state.resize(n);
    table.resize(n);
    std::vector<Range> ranges;
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor& p = params[i];
      TORCH_CHECK_TYPE(p.layout() == at::kStrided && (p.scalar_type() == at::kFloat || p.scalar_type() == at::kBFloat16),
                       "pde_amd: parameters must be dense float32 or bfloat16 tensors, got ", p.scalar_type(), " ", p.layout());
      TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(), "pde_amd: parameters must be dense in memory, got sizes ", p.sizes(), " with strides ",
                        p.strides());
      if (i == 0) dev = p.device();
      TORCH_CHECK_VALUE(p.device() == dev, "pde_amd: parameters must all be on one device, got ", dev, " and ", p.device());
      table[i] = pde_amd_adamw_tensor{};
      table[i].numel = p.numel();
      table[i].dtype = p.scalar_type() == at::kFloat ? PDE_AMD_F32 : PDE_AMD_BF16;
      table[i].group = (int32_t)groups[i];
      add_range(ranges, p.const_data_ptr(), p.numel() * (int64_t)p.element_size());
    }
    for (size_t k = 0; k < state.size(); ++k) {
      TORCH_CHECK_VALUE(state[k] >= 0 && (size_t)state[k] < n && !has_state[state[k]], "pde_amd: bad state index");
      const size_t i = (size_t)state[k];
      has_state[i] = true;
      exp_avg[i] = exp_avg_[k];
      exp_avg_sq[i] = exp_avg_sq_[k];
      step[i] = step_[k];
      if (table[i].dtype == PDE_AMD_BF16) master[i] = master_[k];
      for (const at::Tensor* t : {&exp_avg[i], &exp_avg_sq[i], &master[i]}) {
        if (!t->defined()) continue;
        TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->device() == dev && t->sizes() == params[i].sizes() &&
                              (t->strides() == params[i].strides() || t->numel() == 0),
                          "pde_amd: an optimizer's state must be float32 tensors laid out as the parameter (sizes ", params[i].sizes(), ", strides ",
                          params[i].strides(), ") on its device, got ", t->scalar_type(), " ", t->sizes(), " with strides ", t->strides(), " on ",
                          t->device());
        add_range(ranges, t->const_data_ptr(), t->numel() * 4);
      }
      TORCH_CHECK_VALUE(step[i].scalar_type() == at::kFloat && step[i].device() == dev && step[i].numel() == 1,
                        "pde_amd: an optimizer's step counts must be float32 scalars on the parameter's device");
      add_range(ranges, step[i].const_data_ptr(), 4);
    }
    check_apart(ranges, "parameters and optimizer state");
    TORCH_CHECK(n == 0 || dev.is_cuda(), "pde_amd: parameters must be on a HIP device (there is no CPU fallback), got ", dev);
  }

  void describe(const std::vector<pde_amd_adamw_group>& now) {
    const size_t table_bytes = table.size() * sizeof(pde_amd_adamw_tensor), group_bytes = now.size() * sizeof(pde_amd_adamw_group);
    bool same = !tables.empty() && groups.size() == now.size() && !std::memcmp(groups.data(), now.data(), group_bytes);
    for (size_t i = 0; i < params.size(); ++i) {
      pde_amd_adamw_tensor& t = table[i];
      void* p = params[i].mutable_data_ptr();
      float *m = nullptr, *v = nullptr, *w = nullptr, *s = nullptr;
      if (has_state[i]) {
        m = exp_avg[i].mutable_data_ptr<float>();
        v = exp_avg_sq[i].mutable_data_ptr<float>();
        s = step[i].mutable_data_ptr<float>();
        if (master[i].defined()) w = master[i].mutable_data_ptr<float>();
      }
      same = same && t.param == p && t.exp_avg == m && t.exp_avg_sq == v && t.master == w && t.step == s;
      t.param = p;
      t.exp_avg = m;
      t.exp_avg_sq = v;
      t.master = w;
      t.step = s;
    }
    if (same) return;
    TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None,
                "pde_amd: an optimizer's first step, or the first one after its tensors changed, cannot be captured into a graph: run one step before");
    groups = now;
    at::Tensor host = at::empty({(int64_t)(table_bytes + group_bytes)}, at::kByte);
    std::memcpy(host.mutable_data_ptr(), table.data(), table_bytes);
    std::memcpy((char*)host.mutable_data_ptr() + table_bytes, now.data(), group_bytes);
    tables.push_back(host.to(dev));      // waits for the copy
  }

  // hyper: lr, beta1, beta2, eps, weight_decay of every group; lr_tensors[lr_index[g]] replaces lr where lr_index[g] >= 0.
  // max_norm < 0: no clipping.  given: [] or [norm].  Returns ([norm] where one was computed, indices of parameters that
  // have a gradient but no state: nothing was done then).
  typedef std::tuple<std::vector<at::Tensor>, std::vector<int64_t>> Result;

  Result run(std::vector<double> hyper, std::vector<int64_t> lr_index, std::vector<at::Tensor> lr_tensors, double max_norm,
             bool skip_nonfinite, std::vector<at::Tensor> given) {
    const size_t n = params.size(), n_groups = lr_index.size();
    TORCH_CHECK_VALUE(hyper.size() == 5 * n_groups, "pde_amd: five values per parameter group");
    std::vector<const void*> grads(n);
    std::vector<at::Tensor> keep;
    std::vector<int64_t> missing;
    bool any = false;
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor& p = params[i];
      const at::Tensor& g = p.grad();
      if (!g.defined()) continue;
      if (!has_state[i]) {
        missing.push_back((int64_t)i);
        continue;
      }
      TORCH_CHECK_TYPE(g.layout() == at::kStrided, "pde_amd: gradients must be dense tensors, got layout ", g.layout());
      TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type(), "pde_amd: a gradient must have its parameter's type, got ", g.scalar_type(), " for ",
                       p.scalar_type());
      TORCH_CHECK_VALUE(g.device() == dev && g.sizes() == p.sizes(), "pde_amd: a gradient must have its parameter's sizes and device");
      if (g.strides() == p.strides() || (g.is_contiguous() && p.is_contiguous())) {
        grads[i] = g.const_data_ptr();
      } else {
        at::Tensor c = at::empty_strided(p.sizes(), p.strides(), p.options());
        c.copy_(g.detach());
        keep.push_back(c);
        grads[i] = c.const_data_ptr();
      }
      any = any || p.numel() > 0;
      if (p.numel() == 0) grads[i] = nullptr;
    }
    if (!missing.empty() || !any) return Result(std::vector<at::Tensor>(), missing);
    c10::hip::HIPGuard guard(dev.index());
    void* stream = c10::hip::getCurrentHIPStream(dev.index()).stream();
    std::vector<pde_amd_adamw_group> now(n_groups);
    std::vector<float> lr(n_groups);
    for (size_t k = 0; k < n_groups; ++k) {
      lr[k] = (float)hyper[5 * k];
      now[k].beta1 = hyper[5 * k + 1];
      now[k].beta2 = hyper[5 * k + 2];
      now[k].eps = (float)hyper[5 * k + 3];
      now[k].weight_decay = (float)hyper[5 * k + 4];
      now[k].lr_device = nullptr;
      if (lr_index[k] >= 0) {
        const at::Tensor& t = lr_tensors.at((size_t)lr_index[k]);
        TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.numel() == 1 && t.device() == dev,
                          "pde_amd: a learning rate on the device must be one float32 value on the parameters' device");
        now[k].lr_device = t.const_data_ptr<float>();
      }
    }
    describe(now);
    std::vector<at::Tensor> out;
    const bool need = max_norm >= 0 || skip_nonfinite;
    at::Tensor norm;
    if (need && !given.empty()) norm = norm_scalar(given[0], dev);
    if (need && given.empty()) out.push_back(at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev)));
    at::Tensor ws = workspace(dev, (int32_t)n, stream);
    check(abi.adamw(table.data(), (const pde_amd_adamw_tensor*)tables.back().const_data_ptr(), grads.data(), (int32_t)n,
                    (const pde_amd_adamw_group*)((const char*)tables.back().const_data_ptr() + n * sizeof(pde_amd_adamw_tensor)),
                    (int32_t)n_groups, lr.data(), (float)max_norm, skip_nonfinite ? 1 : 0, norm.defined() ? norm.const_data_ptr<float>() : nullptr,
                    out.empty() ? nullptr : out[0].data_ptr<float>(), ws.data_ptr(), (size_t)ws.numel(), stream),
          "multi_adamw");
    for (size_t i = 0; i < n; ++i) {
      if (!grads[i]) continue;
      written(params[i]);
      written(exp_avg[i]);
      written(exp_avg_sq[i]);
      written(step[i]);
      if (master[i].defined()) written(master[i]);
    }
    return Result(out, std::vector<int64_t>());
  }
};

}  // namespace

TORCH_LIBRARY_FRAGMENT(pde_amd, m) {
  m.def("total_norm(Tensor[] tensors, int norm_type, bool each) -> Tensor[]", &total_norm);
  m.def("clip_grad_norm_(Tensor[] parameters, float max_norm, int norm_type) -> Tensor", &clip_grad_norm);
  m.def("clip_grads_with_norm_(Tensor[] parameters, float max_norm, Tensor total_norm) -> ()", &clip_grads_with_norm);
  m.class_<AdamWPlan>("AdamWPlan")
      .def(torch::init<std::vector<at::Tensor>, std::vector<int64_t>, std::vector<int64_t>, std::vector<at::Tensor>, std::vector<at::Tensor>,
                       std::vector<at::Tensor>, std::vector<at::Tensor>>())
      .def("run", &AdamWPlan::run);
}

// The part of pde_amd_torch_bind that belongs to this file.
int pde_amd_torch_bind_optim(void* h) {
#define PDE_AMD_BIND(field, sym)                                        \
  abi.field = reinterpret_cast<decltype(abi.field)>(dlsym(h, #sym));    \
  if (!abi.field) return -1;
  PDE_AMD_BIND(workspace_bytes, pde_amd_multi_workspace_bytes)
  PDE_AMD_BIND(clip, pde_amd_multi_clip)
  PDE_AMD_BIND(norm_clip, pde_amd_multi_norm_clip)
  PDE_AMD_BIND(adamw, pde_amd_multi_adamw)
  PDE_AMD_BIND(status_string, pde_amd_status_string)
  PDE_AMD_BIND(poison_lds, pde_amd_diag_poison_lds)
  PDE_AMD_BIND(norm, pde_amd_multi_norm)
#undef PDE_AMD_BIND
  return 0;
}
