// Torch front end of the list entry points (gradient norm, clipping, AdamW step): the loops over parameter tensors and
// their checks run here rather than in Python.  The functions are a Python extension module (_pde_amd_optim, a library of its
// own: the operators' loads without Python) and not dispatcher operators: boxing the lists of a call costs more than the
// call's GPU time where the tensors are small (norm of 48 tensors: 15.9 us boxed, GPU 5.5 us).
// Host code only; the C ABI is bound at run time (pde_amd_optim_bind).
#include <torch/csrc/python_headers.h>

#include <dlfcn.h>

#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <vector>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include "../../include/pde_amd.h"

namespace {

struct Abi {
  decltype(&pde_amd_multi_workspace_bytes) workspace_bytes = nullptr;
  decltype(&pde_amd_multi_norm) norm = nullptr;
  decltype(&pde_amd_multi_clip) clip = nullptr;
  decltype(&pde_amd_multi_norm_clip) norm_clip = nullptr;
  decltype(&pde_amd_multi_adamw_groups) adamw_groups = nullptr;
  decltype(&pde_amd_multi_adamw) adamw = nullptr;
  decltype(&pde_amd_status_string) status_string = nullptr;
  decltype(&pde_amd_diag_poison_lds) poison_lds = nullptr;
} capi;

void check(int st, const char* what) {
  TORCH_CHECK(st == 0, "pde_amd: ", what, " failed: ", capi.status_string ? capi.status_string(st) : "?", " (", st, ")");
}

void check_bound() { TORCH_CHECK(capi.norm != nullptr, "pde_amd: the kernel library is not bound (pde_amd_optim_bind)"); }

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

// Scratch of one call: memory of torch's allocator on the current stream, handed back (in the stream's order) at the
// call's end, so that no two calls, streams or graphs share any
struct Workspace {
  size_t bytes;
  c10::DataPtr data;
  Workspace(const at::Device& dev, int32_t n, void* stream) : bytes(capi.workspace_bytes(n)), data(c10::GetAllocator(at::kCUDA)->allocate(bytes)) {
    if (!poison()) return;
    at::from_blob(data.get(), {(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev)).fill_(255);
    check(capi.poison_lds(stream), "diag_poison_lds");
  }
};

// Tensors whose memory does not hold their values: those of a negative view are the negated ones, and a tensor that is
// known to be zero has none.  Copying makes ordinary ones of them.
bool is_lazy(const at::Tensor& t) { return t.is_neg() || t._is_zerotensor(); }

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
    // (a norm is that of the negated values, and scaling these scales the negative)
    if (t._is_zerotensor()) {
      TORCH_CHECK_VALUE(!in_place, "pde_amd: ", what, " that are written must have memory of their own");
      keep.push_back(at::zeros(t.sizes(), t.options()));
      ptr.push_back(keep.back().const_data_ptr());
    } else if (t.is_non_overlapping_and_dense()) {
      ptr.push_back(in_place ? t.mutable_data_ptr() : t.const_data_ptr());      // written, a lazy clone gets memory of its own
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

// ----------------------------------------------------------------------------------------------------------------------
// Python arguments
// ----------------------------------------------------------------------------------------------------------------------
struct Ref {      // an owned Python object
  PyObject* o;
  explicit Ref(PyObject* p) : o(p) {}
  ~Ref() { Py_XDECREF(o); }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
};

const at::Tensor& tensor_of(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "pde_amd: %s must be a tensor, got %.100s", what, Py_TYPE(o)->tp_name);
    throw python_error();
  }
  return THPVariable_Unpack(o);
}

// The tensors of one tensor or of any iterable, alive as long as the object is
struct TensorSeq {
  PyObject* single = nullptr;
  Ref seq;
  const char* what;
  TensorSeq(PyObject* o, const char* what_) : seq(THPVariable_Check(o) ? nullptr : PySequence_Fast(o, "pde_amd: a tensor or an iterable of tensors is needed")), what(what_) {
    if (THPVariable_Check(o)) single = o;
    else if (!seq.o) throw python_error();
  }
  size_t size() const { return single ? 1 : (size_t)PySequence_Fast_GET_SIZE(seq.o); }
  PyObject* object(size_t i) const { return single ? single : PySequence_Fast_GET_ITEM(seq.o, (Py_ssize_t)i); }
  const at::Tensor& operator[](size_t i) const { return tensor_of(object(i), what); }
  std::vector<at::Tensor> all() const {
    std::vector<at::Tensor> v;
    v.reserve(size());
    for (size_t i = 0; i < size(); ++i) v.push_back((*this)[i]);
    return v;
  }
};

double number_of(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw python_error();
  return x;
}

// names of the entries of a parameter group, and of a parameter's state
struct Names {
  PyObject *params = PyUnicode_InternFromString("params"), *lr = PyUnicode_InternFromString("lr"), *betas = PyUnicode_InternFromString("betas"),
           *eps = PyUnicode_InternFromString("eps"), *weight_decay = PyUnicode_InternFromString("weight_decay"),
           *amsgrad = PyUnicode_InternFromString("amsgrad"), *maximize = PyUnicode_InternFromString("maximize"),
           *decoupled = PyUnicode_InternFromString("decoupled_weight_decay"), *step = PyUnicode_InternFromString("step"),
           *exp_avg = PyUnicode_InternFromString("exp_avg"), *exp_avg_sq = PyUnicode_InternFromString("exp_avg_sq"),
           *master = PyUnicode_InternFromString("master");
};

const Names& names() {
  static const Names n;
  return n;
}

PyObject* entry_of(PyObject* dict, PyObject* name) {      // borrowed; NULL where there is none
  PyObject* v = PyDict_Check(dict) ? PyDict_GetItemWithError(dict, name) : nullptr;
  if (!v && PyErr_Occurred()) throw python_error();
  return v;
}

PyObject* item_of(PyObject* dict, PyObject* name) {
  PyObject* v = entry_of(dict, name);
  TORCH_CHECK_VALUE(v, "pde_amd: a parameter group has no entry '", PyUnicode_AsUTF8(name), "'");
  return v;
}

bool true_of(PyObject* o) {
  const int t = PyObject_IsTrue(o);
  if (t < 0) throw python_error();
  return t != 0;
}

void need_args(Py_ssize_t got, Py_ssize_t want) { TORCH_CHECK_TYPE(got == want, "pde_amd: ", want, " arguments are needed, got ", got); }

// total_norm(tensors, norm code, each) -> total, or (total, norms of the tensors)
PyObject* py_total_norm(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  need_args(n_args, 3);
  check_bound();
  at::NoGradGuard no_grad;
  const TensorSeq tensors(args[0], "tensors");
  const int64_t norm_type = PyLong_AsLongLong(args[1]);
  const bool each = args[2] == Py_True;
  List l;
  l.reserve(tensors.size());
  for (size_t i = 0; i < tensors.size(); ++i) l.add(tensors[i], "tensors", false);
  if (!l.size()) {
    at::Tensor zero = at::zeros({}, at::kFloat);
    if (!each) return THPVariable_Wrap(zero);
    const Ref a(THPVariable_Wrap(zero)), b(THPVariable_Wrap(at::zeros({0}, at::kFloat)));
    return PyTuple_Pack(2, a.o, b.o);
  }
  l.check_device("tensors");
  c10::hip::HIPGuard guard(l.dev.index());
  void* stream = c10::hip::getCurrentHIPStream(l.dev.index()).stream();
  const auto opt = at::TensorOptions().dtype(at::kFloat).device(l.dev);
  at::Tensor total = at::empty({}, opt), norms;
  if (each) norms = at::empty({l.size()}, opt);
  const Workspace ws(l.dev, l.size(), stream);
  check(capi.norm(l.ptr.data(), l.numel.data(), l.dtype.data(), l.size(), (int32_t)norm_type, total.data_ptr<float>(),
                 each ? norms.data_ptr<float>() : nullptr, ws.data.get(), ws.bytes, stream),
        "multi_norm");
  if (!each) return THPVariable_Wrap(total);
  const Ref a(THPVariable_Wrap(total)), b(THPVariable_Wrap(norms));
  return PyTuple_Pack(2, a.o, b.o);
  END_HANDLE_TH_ERRORS
}

// the gradients of the parameters that have one, to be written in place
List written_list(const TensorSeq& parameters) {
  List l;
  l.reserve(parameters.size());
  for (size_t i = 0; i < parameters.size(); ++i) {
    const at::Tensor& g = parameters[i].grad();
    if (g.defined()) l.add(g, "gradients", true);
  }
  check_apart(l, "gradients");
  if (l.size()) l.check_device("gradients");
  return l;
}

void written_grads(const TensorSeq& parameters) {
  for (size_t i = 0; i < parameters.size(); ++i) {
    const at::Tensor& g = parameters[i].grad();
    if (g.defined()) written(g);
  }
}

// clip_grad_norm_(parameters, max_norm, norm code) -> the norm
PyObject* py_clip_grad_norm(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  need_args(n_args, 3);
  check_bound();
  at::NoGradGuard no_grad;
  const TensorSeq parameters(args[0], "parameters");
  const double max_norm = number_of(args[1]);
  const int64_t norm_type = PyLong_AsLongLong(args[2]);
  const List l = written_list(parameters);
  if (!l.size()) return THPVariable_Wrap(at::zeros({}, at::kFloat));
  c10::hip::HIPGuard guard(l.dev.index());
  void* stream = c10::hip::getCurrentHIPStream(l.dev.index()).stream();
  at::Tensor total = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(l.dev));
  const Workspace ws(l.dev, l.size(), stream);
  check(capi.norm_clip((void* const*)l.ptr.data(), l.numel.data(), l.dtype.data(), l.size(), (int32_t)norm_type, (float)max_norm,
                      total.data_ptr<float>(), ws.data.get(), ws.bytes, stream),
        "multi_norm_clip");
  written_grads(parameters);
  return THPVariable_Wrap(total);
  END_HANDLE_TH_ERRORS
}

// the norm as a fp32 scalar on the gradients' device
at::Tensor norm_scalar(const at::Tensor& total, const at::Device& dev) {
  TORCH_CHECK_VALUE(total.numel() == 1, "pde_amd: total_norm must hold one value, got sizes ", total.sizes());
  TORCH_CHECK_TYPE(at::isFloatingType(total.scalar_type()), "pde_amd: total_norm must be a floating point tensor, got ", total.scalar_type());
  const auto opt = at::TensorOptions().dtype(at::kFloat).device(dev);
  if (is_lazy(total)) return at::empty({}, opt).copy_(total.reshape({}));
  return total.to(opt).contiguous();
}

// clip_grads_with_norm_(parameters, max_norm, norm)
PyObject* py_clip_grads_with_norm(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  need_args(n_args, 3);
  check_bound();
  at::NoGradGuard no_grad;
  const TensorSeq parameters(args[0], "parameters");
  const double max_norm = number_of(args[1]);
  const at::Tensor& given = tensor_of(args[2], "total_norm");
  const List l = written_list(parameters);
  if (!l.size()) Py_RETURN_NONE;
  c10::hip::HIPGuard guard(l.dev.index());
  void* stream = c10::hip::getCurrentHIPStream(l.dev.index()).stream();
  at::Tensor total = norm_scalar(given, l.dev);
  const uintptr_t at = (uintptr_t)total.const_data_ptr();
  for (size_t i = 0; i < l.ptr.size(); ++i)      // a norm inside a gradient that is about to be scaled by it
    if (at >= (uintptr_t)l.ptr[i] && at < (uintptr_t)l.ptr[i] + (uintptr_t)(l.numel[i] * (l.dtype[i] == PDE_AMD_F32 ? 4 : 2))) {
      total = total.clone();
      break;
    }
  check(capi.clip((void* const*)l.ptr.data(), l.numel.data(), l.dtype.data(), l.size(), (float)max_norm, total.data_ptr<float>(), stream),
        "multi_clip");
  written_grads(parameters);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// A number that is another one after every change of the dictionary
uint64_t version_of(PyObject* dict) {
#if PY_VERSION_HEX < 0x030C0000
  return reinterpret_cast<PyDictObject*>(dict)->ma_version_tag;
#else
  static uint64_t next = 0;      // not to be had any more: taken to have changed
  return ++next;
#endif
}

// A dictionary as it was when it was looked at
struct Seen {
  Ref dict;
  uint64_t version;
  explicit Seen(PyObject* d) : dict((Py_INCREF(d), d)), version(version_of(d)) {}
  bool unchanged() const { return version == version_of(dict.o); }
};

// Device memory that steps read.  Given back, it goes to the stream that it was made on, so the allocator has to know of
// the others; where a graph reads it, it must stay as long as the plan.
struct Block {
  at::Tensor memory;
  std::vector<c10::hip::HIPStream> streams;      // where it was made, and where steps have read it
  bool in_graph = false;

  void read_on(const c10::hip::HIPStream& stream, bool capturing) {
    in_graph = in_graph || capturing;
    if (capturing || std::find(streams.begin(), streams.end(), stream) != streams.end()) return;
    c10::hip::HIPCachingAllocator::recordStream(memory.storage().data_ptr(), stream);
    streams.push_back(stream);
  }
  void replace(const at::Tensor& by, const c10::hip::HIPStream& stream, std::vector<at::Tensor>& kept) {
    if (in_graph) kept.push_back(memory);
    memory = by;
    streams.assign(1, stream);
    in_graph = false;
  }
};

// The parameters of an optimizer with their state, described once in device memory.  The description is made again when
// a tensor has moved, the groups' settings are written again when one of them has changed; older ones are kept where a
// captured step reads them, and given back otherwise.
struct AdamWPlan {
  std::vector<at::Tensor> params, exp_avg, exp_avg_sq, master, step;      // state undefined where there is none
  std::vector<bool> has_state;
  std::vector<pde_amd_adamw_tensor> table;
  std::vector<pde_amd_adamw_group> groups;
  Block described, settings;           // table and groups on the device
  bool captured = false;               // a graph reads something of this plan
  std::vector<at::Tensor> kept;        // what graphs read beside the present blocks
  std::unique_ptr<Seen> seen;          // the optimizer's dictionary of states, and the states in it, found to be these
  std::vector<std::unique_ptr<Seen>> seen_states;
  std::vector<const void*> apart;      // gradients found apart from what table says is written
  at::Device dev = at::kCPU;

  // state: indices of the parameters that have state; exp_avg ... belong to those, in that order.  master: not looked at
  // where the parameter is fp32.
  AdamWPlan(std::vector<at::Tensor> params_, const std::vector<int64_t>& group_of, const std::vector<int64_t>& state, std::vector<at::Tensor> exp_avg_,
            std::vector<at::Tensor> exp_avg_sq_, std::vector<at::Tensor> master_, std::vector<at::Tensor> step_)
      : params(std::move(params_)) {
    const size_t n = params.size();
    TORCH_CHECK_VALUE(group_of.size() == n && exp_avg_.size() == state.size() && exp_avg_sq_.size() == state.size() &&
                          master_.size() == state.size() && step_.size() == state.size(),
                      "pde_amd: an optimizer's lists must have one entry per parameter");
    exp_avg.resize(n);
    exp_avg_sq.resize(n);
    master.resize(n);
    step.resize(n);
    has_state.resize(n);
    table.resize(n);
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor& p = params[i];
      TORCH_CHECK_TYPE(p.layout() == at::kStrided && (p.scalar_type() == at::kFloat || p.scalar_type() == at::kBFloat16),
                       "pde_amd: parameters must be dense float32 or bfloat16 tensors, got ", p.scalar_type(), " ", p.layout());
      TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(), "pde_amd: parameters must be dense in memory, got sizes ", p.sizes(), " with strides ",
                        p.strides());
      TORCH_CHECK_VALUE(!is_lazy(p), "pde_amd: parameters must hold their values (no negative views)");
      if (i == 0) dev = p.device();
      TORCH_CHECK_VALUE(p.device() == dev, "pde_amd: parameters must all be on one device, got ", dev, " and ", p.device());
      std::memset(&table[i], 0, sizeof(table[i]));
      table[i].numel = p.numel();
      table[i].dtype = p.scalar_type() == at::kFloat ? PDE_AMD_F32 : PDE_AMD_BF16;
      table[i].group = (int32_t)group_of[i];
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
        TORCH_CHECK_VALUE(!is_lazy(*t), "pde_amd: an optimizer's state must hold its values (no negative views)");
        TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->device() == dev && t->sizes() == params[i].sizes() &&
                              (t->strides() == params[i].strides() || t->numel() == 0),
                          "pde_amd: an optimizer's state must be float32 tensors laid out as the parameter (sizes ", params[i].sizes(), ", strides ",
                          params[i].strides(), ") on its device, got ", t->scalar_type(), " ", t->sizes(), " with strides ", t->strides(), " on ",
                          t->device());
      }
      TORCH_CHECK_VALUE(step[i].scalar_type() == at::kFloat && step[i].device() == dev && step[i].numel() == 1 && !is_lazy(step[i]),
                        "pde_amd: an optimizer's step counts must be float32 scalars on the parameter's device");
    }
    check_memory();
    TORCH_CHECK(n == 0 || dev.is_cuda(), "pde_amd: parameters must be on a HIP device (there is no CPU fallback), got ", dev);
  }

  // Nothing is written twice, and no gradient lies in what is written
  void check_memory(const std::vector<const void*>* grads = nullptr) const {
    std::vector<Range> ranges;
    ranges.reserve(6 * params.size());
    for (size_t i = 0; i < params.size(); ++i) {
      add_range(ranges, params[i].mutable_data_ptr(), params[i].numel() * (int64_t)params[i].element_size());
      if (!has_state[i]) continue;
      for (const at::Tensor* t : {&exp_avg[i], &exp_avg_sq[i], &master[i], &step[i]})
        if (t->defined()) add_range(ranges, t->mutable_data_ptr(), t->numel() * 4);
    }
    check_apart(ranges, "parameters and optimizer state");
    if (!grads) return;
    for (size_t i = 0; i < params.size(); ++i) {      // ranges is sorted now; gradients may well share memory among themselves
      if (!(*grads)[i]) continue;
      const uintptr_t lo = (uintptr_t)(*grads)[i], hi = lo + (uintptr_t)(table[i].numel * (table[i].dtype == PDE_AMD_F32 ? 4 : 2));
      const auto next = std::upper_bound(ranges.begin(), ranges.end(), lo, [](uintptr_t a, const Range& r) { return a < r.hi; });
      TORCH_CHECK_VALUE(next == ranges.end() || next->lo >= hi, "pde_amd: a gradient shares memory with parameters or optimizer state");
    }
  }

  // The device's description is that of the tensors as they are now
  void describe(const c10::hip::HIPStream& stream, bool capturing) {
    bool same = described.memory.defined();
    for (size_t i = 0; same && i < params.size(); ++i) same = at_same_addresses(i);
    if (same) return;
    check_memory();
    TORCH_CHECK(!capturing, "pde_amd: an optimizer's first step, or the first one after its tensors changed, cannot be captured into a graph: run one "
                "step before");
    std::vector<pde_amd_adamw_tensor> fresh = table;
    for (size_t i = 0; i < params.size(); ++i) {
      pde_amd_adamw_tensor& t = fresh[i];
      t.param = params[i].mutable_data_ptr();
      if (!has_state[i]) continue;
      t.exp_avg = exp_avg[i].mutable_data_ptr<float>();
      t.exp_avg_sq = exp_avg_sq[i].mutable_data_ptr<float>();
      t.step = step[i].mutable_data_ptr<float>();
      if (master[i].defined()) t.master = master[i].mutable_data_ptr<float>();
    }
    const size_t bytes = fresh.size() * sizeof(pde_amd_adamw_tensor);
    at::Tensor host = at::empty({(int64_t)bytes}, at::kByte);
    std::memcpy(host.mutable_data_ptr(), fresh.data(), bytes);
    described.replace(host.to(dev), stream, kept);      // waits for the copy
    table = std::move(fresh);
    apart.clear();
  }

  // The groups on the device, as they are now; the memory that holds them.  Never waits.
  const void* settle(const std::vector<pde_amd_adamw_group>& now, const c10::hip::HIPStream& stream, bool capturing) {
    const size_t bytes = now.size() * sizeof(pde_amd_adamw_group);
    if (!settings.memory.defined() || groups.size() != now.size() || std::memcmp(groups.data(), now.data(), bytes)) {
      at::Tensor fresh = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
      auto* to = static_cast<pde_amd_adamw_group*>(fresh.mutable_data_ptr());
      check(capi.adamw_groups(now.data(), (int32_t)now.size(), to, stream.stream()), "multi_adamw_groups");
      if (capturing) {      // written by the graph's replays, and of no use to other steps
        kept.push_back(fresh);
        return to;
      }
      settings.replace(fresh, stream, kept);
      groups = now;
    }
    settings.read_on(stream, capturing);
    return settings.memory.const_data_ptr();
  }

  // (addresses for writing: a tensor that has been cloned lazily since gets memory of its own)
  bool at_same_addresses(size_t i) const {
    const pde_amd_adamw_tensor& t = table[i];
    return t.param == params[i].mutable_data_ptr() &&
           (!has_state[i] || (t.exp_avg == exp_avg[i].mutable_data_ptr() && t.exp_avg_sq == exp_avg_sq[i].mutable_data_ptr() &&
                              t.step == step[i].mutable_data_ptr() && (!master[i].defined() || t.master == master[i].mutable_data_ptr())));
  }

  bool fits(const at::Tensor& state, int64_t numel) const {
    return state.numel() == numel && state.scalar_type() == at::kFloat && state.device() == dev;
  }

  // A parameter and its state have the type, size, layout and device that they had when the plan was made
  bool unchanged(size_t i) const {
    const at::Tensor& p = params[i];
    const int64_t n = table[i].numel;
    if (p.numel() != n || p.scalar_type() != (table[i].dtype == PDE_AMD_F32 ? at::kFloat : at::kBFloat16) || p.device() != dev ||
        !p.is_non_overlapping_and_dense())
      return false;
    if (!has_state[i]) return true;
    for (const at::Tensor* t : {&exp_avg[i], &exp_avg_sq[i], &master[i]})
      if (t->defined() && (!fits(*t, n) || (n != 0 && t->strides() != p.strides()))) return false;
    return fits(step[i], 1);
  }

  bool is_state(size_t i, PyObject* state) const {
    const auto same = [state](PyObject* name, const at::Tensor& t) {
      PyObject* o = entry_of(state, name);
      return o && THPVariable_Check(o) && THPVariable_Unpack(o).is_same(t);
    };
    return same(names().step, step[i]) && same(names().exp_avg, exp_avg[i]) && same(names().exp_avg_sq, exp_avg_sq[i]) &&
           (!master[i].defined() || same(names().master, master[i]));
  }

  // The tensors in the optimizer's state are those of the plan: looked up where a dictionary has changed since
  bool matches_state(PyObject* state, PyObject* param_groups) {
    if (seen && seen->dict.o == state && seen->unchanged() &&
        std::all_of(seen_states.begin(), seen_states.end(), [](const std::unique_ptr<Seen>& s) { return !s || s->unchanged(); }))
      return true;
    TORCH_CHECK_TYPE(PyDict_Check(state), "pde_amd: an optimizer's state must be a dictionary");
    seen.reset();
    auto now = std::make_unique<Seen>(state);
    seen_states.clear();
    seen_states.resize(params.size());
    size_t i = 0;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(param_groups); ++k) {
      const TensorSeq ps(item_of(PyList_GET_ITEM(param_groups, k), names().params), "parameters");
      for (size_t j = 0; j < ps.size(); ++j, ++i) {
        PyObject* one = entry_of(state, ps.object(j));
        if (one && PyDict_Check(one)) {
          seen_states[i] = std::make_unique<Seen>(one);
          if (has_state[i] ? !is_state(i, one) : PyDict_GET_SIZE(one) != 0) return false;
        } else if (one || has_state[i]) {
          return false;
        }
      }
    }
    seen = std::move(now);
    return true;
  }

  // The parameters of param_groups are those of the plan, in the plan's order
  bool matches(PyObject* param_groups) const {
    size_t i = 0;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(param_groups); ++k) {
      const TensorSeq ps(item_of(PyList_GET_ITEM(param_groups, k), names().params), "parameters");
      for (size_t j = 0; j < ps.size(); ++j, ++i)
        if (i >= params.size() || !params[i].is_same(ps[j]) || table[i].group != (int32_t)k || !unchanged(i)) return false;
    }
    return i == params.size();
  }

  // The hyperparameters of a group, checked; the learning rate is left in the group where it lives on the device
  static float read_group(PyObject* group, const at::Device& dev, pde_amd_adamw_group& out, std::vector<at::Tensor>& device_rates) {
    PyObject *lr = item_of(group, names().lr), *betas = item_of(group, names().betas);
    std::memset(&out, 0, sizeof(out));
    double rate = 0.0;
    if (THPVariable_Check(lr)) {
      const at::Tensor& t = THPVariable_Unpack(lr);
      TORCH_CHECK_VALUE(t.numel() == 1, "pde_amd: a learning rate must hold one value, got sizes ", t.sizes());
      if (t.is_cuda()) {
        TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && t.device() == dev && !is_lazy(t),
                          "pde_amd: a learning rate on the device must be one float32 value on the parameters' device");
        out.lr_device = t.const_data_ptr<float>();
        device_rates.push_back(t);
      } else {
        rate = t.item<double>();
      }
    } else {
      rate = number_of(lr);
    }
    const Ref pair(PySequence_Fast(betas, "pde_amd: betas must be a pair of numbers"));
    if (!pair.o) throw python_error();
    TORCH_CHECK_VALUE(PySequence_Fast_GET_SIZE(pair.o) == 2, "pde_amd: betas must be a pair of numbers");
    out.beta1 = number_of(PySequence_Fast_GET_ITEM(pair.o, 0));
    out.beta2 = number_of(PySequence_Fast_GET_ITEM(pair.o, 1));
    const double eps = number_of(item_of(group, names().eps)), decay = number_of(item_of(group, names().weight_decay));
    TORCH_CHECK_VALUE(rate >= 0 && out.beta1 >= 0 && out.beta1 < 1 && out.beta2 >= 0 && out.beta2 < 1 && eps >= 0 && decay >= 0,
                      "pde_amd: need lr >= 0, 0 <= betas < 1, eps >= 0 and weight_decay >= 0, got lr=", rate, ", betas=(", out.beta1, ", ", out.beta2,
                      "), eps=", eps, ", weight_decay=", decay);
    for (PyObject* name : {names().amsgrad, names().maximize}) {
      PyObject* o = entry_of(group, name);
      TORCH_CHECK_VALUE(!o || !true_of(o), "pde_amd: ClippedAdamW has no ", PyUnicode_AsUTF8(name));
    }
    PyObject* decoupled = entry_of(group, names().decoupled);
    TORCH_CHECK_VALUE(decay == 0 || !decoupled || true_of(decoupled),
                      "pde_amd: ClippedAdamW has no weight decay that is added to the gradients (decoupled_weight_decay=False)");
    out.eps = (float)eps;
    out.weight_decay = (float)decay;
    return (float)rate;
  }

  // max_norm < 0: no clipping.  given: the norm, or undefined.  norm: where it was computed here.  missing: parameters
  // that have a gradient but no state; nothing was done then.
  void run(PyObject* param_groups, double max_norm, bool skip_nonfinite, const at::Tensor& given, at::Tensor& out, std::vector<int64_t>& missing) {
    const size_t n = params.size(), n_groups = (size_t)PyList_GET_SIZE(param_groups);
    std::vector<pde_amd_adamw_group> now(n_groups);
    std::vector<float> lr(n_groups);
    std::vector<at::Tensor> device_rates;
    for (size_t k = 0; k < n_groups; ++k) lr[k] = read_group(PyList_GET_ITEM(param_groups, (Py_ssize_t)k), dev, now[k], device_rates);
    std::vector<const void*> grads(n);
    std::vector<at::Tensor> keep;
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
      if ((g.strides() == p.strides() || (g.is_contiguous() && p.is_contiguous())) && !is_lazy(g)) {
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
    if (!missing.empty()) return;
    const bool need = max_norm >= 0 || skip_nonfinite;
    if (!any) {      // nothing to update
      if (need && !given.defined()) out = at::zeros({}, at::TensorOptions().dtype(at::kFloat).device(dev));
      return;
    }
    c10::hip::HIPGuard guard(dev.index());
    const c10::hip::HIPStream stream = c10::hip::getCurrentHIPStream(dev.index());
    const bool capturing = c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
    describe(stream, capturing);
    if (grads != apart) {      // other gradients than at the last step
      check_memory(&grads);
      apart = grads;
    }
    if (capturing) {
      captured = true;
      kept.insert(kept.end(), device_rates.begin(), device_rates.end());
    }
    described.read_on(stream, capturing);
    const void* groups_device = settle(now, stream, capturing);
    at::Tensor norm;
    if (need && given.defined()) norm = norm_scalar(given, dev);
    else if (need) out = at::empty({}, at::TensorOptions().dtype(at::kFloat).device(dev));
    const Workspace ws(dev, (int32_t)n, stream.stream());
    check(capi.adamw(table.data(), static_cast<const pde_amd_adamw_tensor*>(described.memory.const_data_ptr()), grads.data(), (int32_t)n,
                    static_cast<const pde_amd_adamw_group*>(groups_device), (int32_t)n_groups, lr.data(), (float)max_norm,
                    skip_nonfinite ? 1 : 0, norm.defined() ? norm.const_data_ptr<float>() : nullptr, out.defined() ? out.data_ptr<float>() : nullptr,
                    ws.data.get(), ws.bytes, stream.stream()),
          "multi_adamw");
    for (size_t i = 0; i < n; ++i) {
      if (grads[i]) written(params[i]);
    }
  }
};

const char* const PLAN = "pde_amd.AdamWPlan";

AdamWPlan* plan_of(PyObject* capsule) {
  void* p = PyCapsule_GetPointer(capsule, PLAN);
  if (!p) throw python_error();
  return static_cast<AdamWPlan*>(p);
}

void drop_plan(PyObject* capsule) { delete static_cast<AdamWPlan*>(PyCapsule_GetPointer(capsule, PLAN)); }

// adamw_plan(parameters, their groups, indices of those with state, exp_avg, exp_avg_sq, master, step of these) -> plan
PyObject* py_adamw_plan(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  need_args(n_args, 7);
  check_bound();
  std::vector<int64_t> ints[2];
  for (int k = 0; k < 2; ++k) {
    const Ref seq(PySequence_Fast(args[1 + k], "pde_amd: a list of numbers is needed"));
    if (!seq.o) throw python_error();
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq.o); ++i) ints[k].push_back(PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq.o, i)));
  }
  auto plan = std::make_unique<AdamWPlan>(TensorSeq(args[0], "parameters").all(), ints[0], ints[1], TensorSeq(args[3], "exp_avg").all(),
                                          TensorSeq(args[4], "exp_avg_sq").all(), TensorSeq(args[5], "master").all(), TensorSeq(args[6], "step").all());
  PyObject* capsule = PyCapsule_New(plan.get(), PLAN, drop_plan);
  if (capsule) plan.release();
  return capsule;
  END_HANDLE_TH_ERRORS
}

// adamw_step(plan, param_groups, max_norm or -1, skip_nonfinite, norm or None, state) -> the norm, or None where none was
// computed; False: the plan is not one of these parameters and this state; a list: the parameters with a gradient but
// without state (in both cases nothing was done)
PyObject* py_adamw_step(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  need_args(n_args, 6);
  at::NoGradGuard no_grad;
  AdamWPlan& plan = *plan_of(args[0]);
  TORCH_CHECK_TYPE(PyList_Check(args[1]), "pde_amd: param_groups must be a list");
  if (!plan.matches(args[1]) || !plan.matches_state(args[5], args[1])) Py_RETURN_FALSE;
  at::Tensor given, norm;
  if (args[4] != Py_None) given = tensor_of(args[4], "total_norm");
  std::vector<int64_t> missing;
  plan.run(args[1], number_of(args[2]), args[3] == Py_True, given, norm, missing);
  if (!missing.empty()) {
    PyObject* list = PyList_New((Py_ssize_t)missing.size());
    if (!list) throw python_error();
    for (size_t i = 0; i < missing.size(); ++i) PyList_SET_ITEM(list, (Py_ssize_t)i, PyLong_FromLongLong(missing[i]));
    return list;
  }
  if (norm.defined()) return THPVariable_Wrap(norm);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// adamw_captured(plan) -> whether a step with it was captured into a graph
PyObject* py_adamw_captured(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  HANDLE_TH_ERRORS
  need_args(n_args, 1);
  return PyBool_FromLong(plan_of(args[0])->captured);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"total_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_total_norm)), METH_FASTCALL, nullptr},
    {"clip_grad_norm_", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_clip_grad_norm)), METH_FASTCALL, nullptr},
    {"clip_grads_with_norm_", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_clip_grads_with_norm)), METH_FASTCALL, nullptr},
    {"adamw_plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_adamw_plan)), METH_FASTCALL, nullptr},
    {"adamw_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_adamw_step)), METH_FASTCALL, nullptr},
    {"adamw_captured", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_adamw_captured)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pde_amd_optim", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pde_amd_optim() { return PyModule_Create(&module); }

// Binds the C ABI of the kernel library at `path` (already loaded by the process or not); returns 0, or -1 with the
// reason in dlerror().
extern "C" int pde_amd_optim_bind(const char* path) {
  void* h = dlopen(path, RTLD_NOW | RTLD_GLOBAL);
  if (!h) return -1;
#define PDE_AMD_BIND(field, sym)                                        \
  capi.field = reinterpret_cast<decltype(capi.field)>(dlsym(h, #sym));    \
  if (!capi.field) return -1;
  PDE_AMD_BIND(workspace_bytes, pde_amd_multi_workspace_bytes)
  PDE_AMD_BIND(clip, pde_amd_multi_clip)
  PDE_AMD_BIND(norm_clip, pde_amd_multi_norm_clip)
  PDE_AMD_BIND(adamw_groups, pde_amd_multi_adamw_groups)
  PDE_AMD_BIND(adamw, pde_amd_multi_adamw)
  PDE_AMD_BIND(status_string, pde_amd_status_string)
  PDE_AMD_BIND(poison_lds, pde_amd_diag_poison_lds)
  PDE_AMD_BIND(norm, pde_amd_multi_norm)
#undef PDE_AMD_BIND
  return 0;
}
