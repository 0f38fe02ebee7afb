// Python side of the multi-tensor entry points: checks lists of tensors and turns them into the C
// ABI's arrays, and marks what is written for autograd.  A call over 65 tensors and four lists makes 1500
// attribute look-ups, 100 us in Python against 6 us on the GPU; here they take 6 us, the marks included.
// The C entries are given by address, so this module is bound to no particular shared library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cctype>
#include <cmath>
#include <deque>
#include <memory>
#include <optional>
#include <string>
#include <vector>

#include "../../include/flash_muon_b200.h"

namespace {

struct Refused {};  // a Python error is set

#define REQUIRE(cond, ...)                             \
  do {                                                 \
    if (!(cond)) {                                     \
      PyErr_Format(PyExc_AssertionError, __VA_ARGS__); \
      throw Refused{};                                 \
    }                                                  \
  } while (0)

// A list or tuple (or what becomes one) held for the call.
class Items {
 public:
  Items(PyObject* o, const char* name) : seq_(PySequence_Fast(o, "")) {
    if (!seq_) {
      PyErr_Format(PyExc_TypeError, "`%s` must be a sequence", name);
      throw Refused{};
    }
  }
  ~Items() { Py_DECREF(seq_); }
  Items(const Items&) = delete;
  Items& operator=(const Items&) = delete;
  Py_ssize_t size() const { return PySequence_Fast_GET_SIZE(seq_); }
  PyObject* operator[](Py_ssize_t i) const { return PySequence_Fast_GET_ITEM(seq_, i); }

 private:
  PyObject* seq_;
};

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "`%s` must be tensors", name);
    throw Refused{};
  }
  return THPVariable_Unpack(o);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return FM_BF16;
    case at::kHalf: return FM_F16;
    case at::kFloat: return FM_F32;
    default:
      PyErr_Format(PyExc_TypeError, "flash_muon_b200 supports bfloat16, float16 and float32, got torch.%s",
                   [&] { std::string s = c10::toString(t); for (char& c : s) c = (char)std::tolower(c); return s; }().c_str());
      throw Refused{};
  }
}

// One look at a tensor where all is well; what is wrong is found out apart.
[[gnu::noinline]] void refuse_place(const at::Tensor& t, const char* name) {
  REQUIRE(t.is_cuda(), "`%s` must be CUDA tensors", name);
  REQUIRE(t.layout() == at::kStrided && t.is_contiguous(), "`%s` must be contiguous", name);
  REQUIRE(false, "`%s` must be on the parameters' device", name);
}
void check_place(const at::Tensor& t, const char* name, int device) {
  const c10::TensorImpl* const x = t.unsafeGetTensorImpl();
  const c10::Device d = x->device();
  if (d.type() != at::kCUDA || d.index() != device || x->layout() != at::kStrided || !x->is_contiguous())
    refuse_place(t, name);
}

void* scalar(PyObject* o, const char* name, int device) {
  const at::Tensor& t = tensor(o, name);
  REQUIRE(t.is_cuda() && t.get_device() == device && t.numel() == 1 && t.scalar_type() == at::kFloat,
          "`%s` must be a float32 scalar on the parameters' CUDA device", name);
  return t.data_ptr();
}

double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw Refused{};
  return x;
}

// Tells autograd that a tensor was written: a backward pass that saved it is refused.
void mark_written(c10::TensorImpl* t) {
  if (!t->is_inference()) t->bump_version();
}

// One parameter group of a call, in arrays that live until the call returns: those of the library and the
// tensors that it writes.
struct Group {
  fm_adamw_group g;
  size_t count = 0, written = 0;
  void **params, **grads, **masters, **m, **v, **ms, **vs, **steps;
  int64_t* numels;
  uint32_t* seeds;
  c10::TensorImpl** marks;
  std::unique_ptr<void*[]> mem;

  Group(const fm_adamw_group& settings, size_t most, bool master) : g(settings) {
    const bool eight = g.state_bits == 8;
    mem.reset(new void*[most * (8 + 7 + 2 + 1)]);
    void** at = mem.get();
    auto take = [&](bool there) {
      void** const x = there ? at : nullptr;
      if (there) at += most;
      return x;
    };
    g.params = params = take(true);
    g.grads = grads = take(true);
    g.masters = masters = take(master);
    g.exp_avg = m = take(true);
    g.exp_avg_sq = v = take(true);
    g.exp_avg_scale = ms = take(eight);
    g.exp_avg_sq_scale = vs = take(eight);
    steps = take(true);
    g.steps = reinterpret_cast<float**>(steps);
    static_assert(sizeof(int64_t) == sizeof(void*));
    g.numels = numels = reinterpret_cast<int64_t*>(take(true));
    g.seeds = seeds = reinterpret_cast<uint32_t*>(take(eight));
    marks = reinterpret_cast<c10::TensorImpl**>(at);
  }
};

// What a parameter is stepped with; master, scales may be null.
struct Row {
  const at::Tensor *p, *grad, *master, *m, *v, *ms, *vs;
  void* step;               // the count, and the tensor that holds it
  const at::Tensor* count;
  uint32_t seed;
};

void* step_count(const at::Tensor& t, int device) {
  check_place(t, "steps", device);
  REQUIRE(t.scalar_type() == at::kFloat, "`steps` must be torch.float32");
  REQUIRE(t.numel() == 1, "`steps` must be scalars");
  return t.data_ptr();
}

// A tensor that goes element by element with a parameter has its shape; the order of the elements is as
// clear where one of the two is flat.
void check_sizes(const at::Tensor& t, const char* name, const at::Tensor& p) {
  REQUIRE(t.numel() == p.numel() && (p.dim() == 1 || t.dim() == 1 || t.sizes() == p.sizes()),
          "`%s` must have the parameters' sizes, or be flat", name);
}

// Takes the rows of one parameter group, checks them and sorts them by kind (types, masters, state bits).
class Builder {
 public:
  Builder(std::vector<Group>& out, int device, const fm_adamw_group& settings)
      : out_(out), first_(out.size()), device_(device), settings_(settings) {
    const fm_adamw_group& g = settings;
    REQUIRE(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0, "betas must lie in [0, 1)");
    REQUIRE(g.eps >= 0.0 && std::isfinite(g.eps), "eps must be finite and not negative");
    REQUIRE(std::isfinite(g.lr) && std::isfinite(g.weight_decay), "lr and weight_decay must be finite");
  }

  void add(const Row& r, size_t expected) {
    check_place(*r.p, "params", device_);
    check_place(*r.grad, "grads", device_);
    const int64_t n = r.p->numel(), blocks = (n + 31) / 32;
    check_sizes(*r.grad, "grads", *r.p);
    const int pd = dtype_code(r.p->scalar_type()), gd = dtype_code(r.grad->scalar_type());
    const bool eight = r.ms != nullptr;
    moment(*r.m, "exp_avgs", eight, *r.p, blocks);
    moment(*r.v, "exp_avg_sqs", eight, *r.p, blocks);
    if (eight) {
      scales(*r.ms, "exp_avg_scales", blocks);
      scales(*r.vs, "exp_avg_sq_scales", blocks);
    }
    if (r.master) {
      check_place(*r.master, "masters", device_);
      check_sizes(*r.master, "masters", *r.p);
      REQUIRE(r.master->scalar_type() == at::kFloat, "`masters` must be torch.float32");
      REQUIRE(pd != FM_F32, "float32 parameters have no master copies");
    }
    Group& x = group(pd, gd, eight, r.master != nullptr, expected);
    const size_t i = x.count++;
    auto put = [&](void** list, const at::Tensor& t) {
      list[i] = t.data_ptr();
      x.marks[x.written++] = t.unsafeGetTensorImpl();
    };
    x.numels[i] = n;
    x.grads[i] = r.grad->data_ptr();
    put(x.params, *r.p);
    put(x.m, *r.m);
    put(x.v, *r.v);
    if (r.master) put(x.masters, *r.master);
    if (eight) {
      put(x.ms, *r.ms);
      put(x.vs, *r.vs);
      x.seeds[i] = r.seed;
    }
    x.steps[i] = r.step;
    c10::TensorImpl* const count = r.count->unsafeGetTensorImpl();
    if (count != last_count_) x.marks[x.written++] = last_count_ = count;  // one tensor may hold them all
  }

 private:
  void moment(const at::Tensor& t, const char* name, bool eight, const at::Tensor& p, int64_t blocks) {
    check_place(t, name, device_);
    REQUIRE(t.scalar_type() == (eight ? at::kByte : at::kFloat), "`%s` must be torch.%s", name, eight ? "uint8" : "float32");
    if (eight) REQUIRE(t.numel() == blocks * 32, "`%s` must have one byte per element, padded to 32", name);
    else check_sizes(t, name, p);
  }
  void scales(const at::Tensor& t, const char* name, int64_t blocks) {
    check_place(t, name, device_);
    REQUIRE(t.scalar_type() == at::kByte, "`%s` must be torch.uint8", name);
    REQUIRE(t.numel() == blocks, "`%s` must have one byte per block of 32", name);
  }
  Group& group(int pd, int gd, bool eight, bool master, size_t expected) {
    for (size_t i = first_; i < out_.size(); ++i) {
      Group& x = out_[i];
      if (x.g.p_dtype == pd && x.g.g_dtype == gd && (x.g.state_bits == 8) == eight && (x.masters != nullptr) == master) return x;
    }
    fm_adamw_group g = settings_;
    g.p_dtype = pd;
    g.g_dtype = gd;
    g.state_bits = eight ? 8 : 32;
    return out_.emplace_back(g, expected, master);
  }

  std::vector<Group>& out_;
  const size_t first_;
  const int device_;
  const fm_adamw_group settings_;
  c10::TensorImpl* last_count_ = nullptr;
};

void learning_rate(PyObject* lr, int device, fm_adamw_group& g) {
  if (THPVariable_Check(lr)) g.lr_device = static_cast<const float*>(scalar(lr, "lr", device));
  else g.lr = number(lr);
}

uint32_t seed_of(PyObject* o) {
  const uint32_t s = (uint32_t)PyLong_AsUnsignedLongLongMask(o);
  if (PyErr_Occurred()) throw Refused{};
  return s;
}

// (params, grads, masters, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, steps, seeds, lr, beta1,
// beta2, eps, weight_decay); masters, scales and seeds may be None.  `keep` holds the tensors until the call
// returns.
void parse_group(PyObject* tuple, int& device, std::vector<Group>& out, std::deque<Items>& keep) {
  const Items f(tuple, "group");
  REQUIRE(f.size() == 14, "a group has 14 entries");
  const Items &params = keep.emplace_back(f[0], "params"), &grads = keep.emplace_back(f[1], "grads");
  const Py_ssize_t n = params.size();
  if (n == 0) return;
  const bool eight = f[5] != Py_None, master = f[2] != Py_None;
  const Items &m = keep.emplace_back(f[3], "exp_avgs"), &v = keep.emplace_back(f[4], "exp_avg_sqs");
  const Items *w = nullptr, *ms = nullptr, *vs = nullptr, *seeds = nullptr, *steps = nullptr;
  auto list = [&](const Items*& items, int k, const char* name) {
    items = &keep.emplace_back(f[k], name);
    return items->size() == n;
  };
  bool same = grads.size() == n && m.size() == n && v.size() == n;
  if (master) same = list(w, 2, "masters") && same;
  if (eight) same = list(ms, 5, "exp_avg_scales") && list(vs, 6, "exp_avg_sq_scales") && list(seeds, 8, "seeds") && same;
  float* counts = nullptr;
  if (!THPVariable_Check(f[7])) same = list(steps, 7, "steps") && same;
  REQUIRE(same, "lists must have one entry per parameter");
  const at::Tensor& p0 = tensor(params[0], "params");
  REQUIRE(p0.is_cuda(), "`params` must be CUDA tensors");
  if (device < 0) device = p0.get_device();
  if (!steps) {
    const at::Tensor& t = THPVariable_Unpack(f[7]);
    REQUIRE(t.dim() == 1 && t.numel() == n, "`steps` must have one count per parameter");
    check_place(t, "steps", device);
    REQUIRE(t.scalar_type() == at::kFloat, "`steps` must be torch.float32");
    counts = static_cast<float*>(t.data_ptr());
  }
  fm_adamw_group g = {};
  learning_rate(f[9], device, g);
  g.beta1 = number(f[10]);
  g.beta2 = number(f[11]);
  g.eps = number(f[12]);
  g.weight_decay = number(f[13]);
  Builder rows(out, device, g);
  for (Py_ssize_t i = 0; i < n; ++i) {
    Row r = {&tensor(params[i], "params"), &tensor(grads[i], "grads"), master ? &tensor((*w)[i], "masters") : nullptr,
             &tensor(m[i], "exp_avgs"), &tensor(v[i], "exp_avg_sqs"), nullptr, nullptr, nullptr, nullptr, 0};
    if (eight) {
      r.ms = &tensor((*ms)[i], "exp_avg_scales");
      r.vs = &tensor((*vs)[i], "exp_avg_sq_scales");
      r.seed = seed_of((*seeds)[i]);
    }
    r.count = steps ? &tensor((*steps)[i], "steps") : &THPVariable_Unpack(f[7]);
    r.step = steps ? step_count(*r.count, device) : counts + i;
    rows.add(r, n);
  }
}

template <typename Fn>
Fn entry(PyObject* address) {
  void* p = PyLong_AsVoidPtr(address);
  if (!p) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
    throw Refused{};
  }
  return reinterpret_cast<Fn>(p);
}

template <typename Body>
PyObject* guarded(Body body) {
  try {
    return body();
  } catch (const Refused&) {
  } catch (const std::exception&) {
    torch::translate_exception_to_python(std::current_exception());  // torch.OutOfMemoryError stays what it is
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

void need(Py_ssize_t have, Py_ssize_t want) {
  if (have == want) return;
  PyErr_Format(PyExc_TypeError, "%zd arguments, expected %zd", have, want);
  throw Refused{};
}

int launch(decltype(&fm_adamw_step) fn, std::vector<Group>& groups, int device, PyObject* grad_scale) {
  if (groups.empty()) return FM_OK;
  const float* scale = grad_scale == Py_None ? nullptr : static_cast<const float*>(scalar(grad_scale, "grad_scale", device));
  std::vector<fm_adamw_group> table;
  table.reserve(groups.size());
  for (Group& x : groups) {
    x.g.count = (int32_t)x.count;
    table.push_back(x.g);
  }
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  const int rc = fn(table.data(), (int)table.size(), scale, c10::cuda::getCurrentCUDAStream().stream());
  if (rc == FM_OK)
    for (const Group& x : groups)
      for (size_t i = 0; i < x.written; ++i) mark_written(x.marks[i]);
  return rc;
}

// adamw_step(fm_adamw_step, groups, grad_scale or None) -> status
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n, 3);
    const auto fn = entry<decltype(&fm_adamw_step)>(a[0]);
    const Items tuples(a[1], "groups");
    std::deque<Items> keep;
    std::vector<Group> groups;
    groups.reserve(tuples.size() + 4);
    int device = -1;
    for (Py_ssize_t i = 0; i < tuples.size(); ++i) parse_group(tuples[i], device, groups, keep);
    return PyLong_FromLong(launch(fn, groups, device, a[2]));
  });
}

// A dictionary's entry (borrowed), or null.
PyObject* entry_of(PyObject* dict, PyObject* key) {
  PyObject* x = PyDict_GetItemWithError(dict, key);
  if (!x && PyErr_Occurred()) throw Refused{};
  return x;
}

PyObject* setting(PyObject* dict, const char* name) {
  PyObject* x = PyDict_GetItemString(dict, name);
  if (!x) {
    PyErr_Format(PyExc_KeyError, "parameter group without `%s`", name);
    throw Refused{};
  }
  return x;
}

// optimizer_step(fm_adamw_step, param_groups, state, grad_scale or None) -> status, or the list of
// (parameter, group) that have a gradient and no state yet; nothing is launched then.
PyObject* optimizer_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n, 4);
    const auto fn = entry<decltype(&fm_adamw_step)>(a[0]);
    static PyObject* const k_m = PyUnicode_InternFromString("exp_avg");
    static PyObject* const k_v = PyUnicode_InternFromString("exp_avg_sq");
    static PyObject* const k_ms = PyUnicode_InternFromString("exp_avg_scale");
    static PyObject* const k_vs = PyUnicode_InternFromString("exp_avg_sq_scale");
    static PyObject* const k_step = PyUnicode_InternFromString("step");
    static PyObject* const k_master = PyUnicode_InternFromString("master");
    REQUIRE(PyDict_Check(a[2]), "`state` must be a dictionary");
    const Items param_groups(a[1], "param_groups");
    struct Missing {  // released on every way out
      PyObject* list = nullptr;
      ~Missing() { Py_XDECREF(list); }
    } missing;
    struct Device {
      int index;
      std::vector<Group> groups;
    };
    std::vector<Device> devices;
    int64_t index = 0;
    for (Py_ssize_t gi = 0; gi < param_groups.size(); ++gi) {
      PyObject* group = param_groups[gi];
      REQUIRE(PyDict_Check(group), "parameter groups must be dictionaries");
      const Items params(setting(group, "params"), "params");
      const Items betas(setting(group, "betas"), "betas");
      REQUIRE(betas.size() == 2, "`betas` must be a pair");
      fm_adamw_group g = {};
      g.beta1 = number(betas[0]);
      g.beta2 = number(betas[1]);
      g.eps = number(setting(group, "eps"));
      g.weight_decay = number(setting(group, "weight_decay"));
      PyObject* lr = setting(group, "lr");
      const uint32_t seed = seed_of(setting(group, "seed"));
      int builder_device = -1;
      std::optional<Builder> rows;
      for (Py_ssize_t i = 0; i < params.size(); ++i) {
        ++index;
        const at::Tensor& p = tensor(params[i], "params");
        const at::Tensor& grad = p.grad();
        if (!grad.defined()) continue;
        REQUIRE(p.is_cuda(), "`params` must be CUDA tensors");
        REQUIRE(grad.layout() == at::kStrided, "AdamW takes no sparse gradients");
        PyObject* state = entry_of(a[2], params[i]);
        if (!state || !PyDict_Check(state) || PyDict_GET_SIZE(state) == 0) {
          if (!missing.list) missing.list = PyList_New(0);
          PyObject* pair = missing.list ? PyTuple_Pack(2, params[i], group) : nullptr;
          const bool kept = pair && PyList_Append(missing.list, pair) == 0;
          Py_XDECREF(pair);
          if (!kept) throw Refused{};
          continue;
        }
        if (missing.list) continue;
        const int device = p.get_device();
        if (device != builder_device) {
          size_t d = 0;
          while (d < devices.size() && devices[d].index != device) ++d;
          if (d == devices.size()) {
            devices.push_back({device, {}});
            devices.back().groups.reserve(param_groups.size() * 2 + 4);
          }
          learning_rate(lr, device, g);
          rows.emplace(devices[d].groups, device, g);
          builder_device = device;
        }
        auto get = [&](PyObject* key, const char* name, bool needed) -> const at::Tensor* {
          PyObject* x = entry_of(state, key);
          REQUIRE(x || !needed, "state of a parameter without `%s`", name);
          return x ? &tensor(x, name) : nullptr;
        };
        Row r = {&p, &grad, get(k_master, "masters", false), get(k_m, "exp_avgs", true), get(k_v, "exp_avg_sqs", true),
                 get(k_ms, "exp_avg_scales", false), nullptr, nullptr, get(k_step, "steps", true),
                 (uint32_t)(seed + (uint32_t)index)};
        if (r.ms) r.vs = get(k_vs, "exp_avg_sq_scales", true);
        r.step = step_count(*r.count, device);
        rows->add(r, params.size());
      }
    }
    if (missing.list) {
      PyObject* list = missing.list;
      missing.list = nullptr;
      return list;
    }
    // refused, if at all, before the first device steps
    for (const Device& d : devices)
      if (a[3] != Py_None && !d.groups.empty()) scalar(a[3], "grad_scale", d.index);
    int rc = FM_OK;
    for (Device& d : devices) {
      rc = launch(fn, d.groups, d.index, a[3]);
      if (rc != FM_OK) break;
    }
    return PyLong_FromLong(rc);
  });
}

struct Gradients {
  int device = -1;
  std::vector<void*> at;
  std::vector<int64_t> numels;
  std::vector<int32_t> dtypes;
  explicit Gradients(const Items& grads) {
    REQUIRE(grads.size() > 0, "`grads` must not be empty");
    for (Py_ssize_t i = 0; i < grads.size(); ++i) {
      const at::Tensor& t = tensor(grads[i], "grads");
      if (device < 0 && t.is_cuda()) device = t.get_device();
      REQUIRE(t.is_cuda(), "`grads` must be CUDA tensors");
      REQUIRE(t.layout() == at::kStrided && t.is_contiguous(), "`grads` must be contiguous");
      REQUIRE(t.get_device() == device, "`grads` must be on one device");
      at.push_back(t.data_ptr());
      numels.push_back(t.numel());
      dtypes.push_back(dtype_code(t.scalar_type()));
    }
  }
};

// grad_norm(fm_grad_norm, fm_grad_norm_workspace_bytes, grads, max_norm) -> (status, norm, scale)
PyObject* grad_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n, 4);
    const auto fn = entry<decltype(&fm_grad_norm)>(a[0]);
    const auto bytes = entry<decltype(&fm_grad_norm_workspace_bytes)>(a[1]);
    const double max_norm = number(a[3]);
    REQUIRE(max_norm >= 0.0, "`max_norm` must not be negative");
    const Items grads(a[2], "grads");
    const Gradients g(grads);
    const int count = (int)g.at.size();
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)g.device);
    // the result and, behind it, the scratch; fresh memory for every call: calls on other streams, and
    // graphs captured apart, have their own
    const size_t scratch = bytes(count);
    const at::Tensor mem = at::empty({(int64_t)(4 + scratch / 4)}, at::TensorOptions().dtype(at::kFloat).device(at::kCUDA, g.device));
    float* at = static_cast<float*>(mem.data_ptr());
    const int rc = fn(const_cast<const void* const*>(g.at.data()), g.numels.data(), g.dtypes.data(), count, max_norm, at,
                      at + 4, scratch, c10::cuda::getCurrentCUDAStream().stream());
    return Py_BuildValue("iNN", rc, THPVariable_Wrap(mem.select(0, 0)), THPVariable_Wrap(mem.select(0, 1)));
  });
}

// scale(fm_scale_multi, grads, factor) -> status
PyObject* scale(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n, 3);
    const auto fn = entry<decltype(&fm_scale_multi)>(a[0]);
    const Items grads(a[1], "grads");
    const Gradients g(grads);
    const float* factor = static_cast<const float*>(scalar(a[2], "factor", g.device));
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)g.device);
    const int rc = fn(g.at.data(), g.numels.data(), g.dtypes.data(), (int)g.at.size(), factor,
                      c10::cuda::getCurrentCUDAStream().stream());
    if (rc == FM_OK)
      for (Py_ssize_t i = 0; i < grads.size(); ++i) mark_written(tensor(grads[i], "grads").unsafeGetTensorImpl());
    return PyLong_FromLong(rc);
  });
}

// adamw8_values(fm_adamw8_values, codes, scales, moment, numel or None, dtype) -> (status, values)
PyObject* adamw8_values(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n, 6);
    const auto fn = entry<decltype(&fm_adamw8_values)>(a[0]);
    const long moment = PyLong_AsLong(a[3]);
    if (PyErr_Occurred()) throw Refused{};
    REQUIRE(moment == 1 || moment == 2, "moment must be 1 (exp_avg) or 2 (exp_avg_sq)");
    const at::Tensor &codes = tensor(a[1], "codes"), &scales = tensor(a[2], "scales");
    REQUIRE(codes.is_cuda() && scales.is_cuda() && codes.device() == scales.device(),
            "states must be CUDA tensors on one device");
    REQUIRE(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, "states must be uint8");
    REQUIRE(codes.is_contiguous() && scales.is_contiguous(), "states must be contiguous");
    REQUIRE(codes.numel() == scales.numel() * 32, "states must have one scale per 32 codes");
    int64_t numel = codes.numel();
    if (a[4] != Py_None) {
      numel = PyLong_AsLongLong(a[4]);
      if (PyErr_Occurred()) throw Refused{};
      REQUIRE(numel >= 0 && numel <= codes.numel(), "`numel` exceeds the states");
    }
    REQUIRE(THPDtype_Check(a[5]), "`dtype` must be a torch.dtype");
    const at::ScalarType dtype = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
    const int code = dtype_code(dtype);
    const c10::cuda::CUDAGuard guard(codes.device());
    const at::Tensor out = at::empty({numel}, codes.options().dtype(dtype));
    const int rc = fn(codes.data_ptr(), scales.data_ptr(), numel, (int)moment, out.data_ptr(), code,
                      c10::cuda::getCurrentCUDAStream().stream());
    return Py_BuildValue("iN", rc, THPVariable_Wrap(out));
  });
}

PyMethodDef methods[] = {
    {"adamw_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw_step)), METH_FASTCALL, nullptr},
    {"optimizer_step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(optimizer_step)), METH_FASTCALL, nullptr},
    {"grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(grad_norm)), METH_FASTCALL, nullptr},
    {"scale", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scale)), METH_FASTCALL, nullptr},
    {"adamw8_values", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw8_values)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
