// Python side of the multi-tensor entry points: checks lists of tensors and turns them into the C
// ABI's arrays.  A call over 65 tensors and four lists makes 1500 attribute look-ups, 100 us in
// Python against 6 us on the GPU; here they take 3 us.
// The C entries are given by address, so this module is bound to no particular shared library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cctype>
#include <cmath>
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

void check_place(const at::Tensor& t, const char* name, int device) {
  REQUIRE(t.is_cuda(), "`%s` must be CUDA tensors", name);
  REQUIRE(t.layout() == at::kStrided && t.is_contiguous(), "`%s` must be contiguous", name);
  REQUIRE(t.get_device() == device, "`%s` must be on the parameters' device", name);
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

// Addresses of a list of tensors that go with the parameters: checked for place and, where given, for
// type and size (`per` elements of the parameter, rounded up to blocks of 32, per element here).
std::vector<void*> addresses(PyObject* list, const char* name, int device, const std::vector<int64_t>& numels,
                             std::optional<at::ScalarType> dtype, int per = 0) {
  const Items items(list, name);
  REQUIRE(items.size() == (Py_ssize_t)numels.size(), "lists must have one entry per parameter");
  std::vector<void*> out;
  out.reserve(numels.size());
  for (Py_ssize_t i = 0; i < items.size(); ++i) {
    const at::Tensor& t = tensor(items[i], name);
    check_place(t, name, device);
    if (per == 0) {
      REQUIRE(t.numel() == numels[i], "`%s` must have the parameters' sizes", name);
    }
    if (dtype) {
      REQUIRE(t.scalar_type() == *dtype, "`%s` must be torch.%s", name, *dtype == at::kFloat ? "float32" : "uint8");
    }
    if (per != 0) {
      const int64_t blocks = (numels[i] + 31) / 32;
      REQUIRE(t.numel() == (per == 1 ? blocks * 32 : blocks), "`%s` must have one byte per %s", name,
              per == 1 ? "element, padded to 32" : "block of 32");
    }
    out.push_back(t.data_ptr());
  }
  return out;
}

// One parameter group of a call, in arrays that live until the call returns.
struct Group {
  std::vector<int64_t> numels;
  std::vector<void*> params, grads, masters, m, v, ms, vs, steps;
  std::vector<uint32_t> seeds;
  fm_adamw_group g;
};

// (params, grads, masters, exp_avgs, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, steps, seeds, lr, beta1,
// beta2, eps, weight_decay); masters, scales and seeds may be None.  Appends one group per pair of types.
void parse_group(PyObject* tuple, int& device, std::vector<Group>& out) {
  const Items f(tuple, "group");
  REQUIRE(f.size() == 14, "a group has 14 entries");
  const Items params(f[0], "params"), grads(f[1], "grads");
  const size_t n = params.size();
  if (n == 0) return;
  REQUIRE((size_t)grads.size() == n, "lists must have one entry per parameter");
  std::vector<int64_t> numels(n);
  std::vector<uint8_t> kinds(n);  // pair of types
  std::vector<void*> ps(n), gs(n);
  bool one_kind = true, any_f32 = false;
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &p = tensor(params[i], "params"), &g = tensor(grads[i], "grads");
    if (device < 0 && p.is_cuda()) device = p.get_device();
    check_place(p, "params", device);
    check_place(g, "grads", device);
    REQUIRE(g.numel() == p.numel(), "`grads` must have the parameters' sizes");
    numels[i] = p.numel();
    const int pd = dtype_code(p.scalar_type());
    kinds[i] = (uint8_t)(pd * 4 + dtype_code(g.scalar_type()));
    one_kind = one_kind && kinds[i] == kinds[0];
    any_f32 = any_f32 || pd == FM_F32;
    ps[i] = p.data_ptr();
    gs[i] = g.data_ptr();
  }
  const bool eight = f[5] != Py_None;
  const auto state = eight ? at::kByte : at::kFloat;
  const int per = eight ? 1 : 0;
  std::vector<void*> m = addresses(f[3], "exp_avgs", device, numels, state, per);
  std::vector<void*> v = addresses(f[4], "exp_avg_sqs", device, numels, state, per);
  std::vector<void*> w, ms, vs;
  if (f[2] != Py_None) {
    w = addresses(f[2], "masters", device, numels, at::kFloat);
    REQUIRE(!any_f32, "float32 parameters have no master copies");
  }
  std::vector<uint32_t> seeds;
  if (eight) {
    ms = addresses(f[5], "exp_avg_scales", device, numels, at::kByte, 32);
    vs = addresses(f[6], "exp_avg_sq_scales", device, numels, at::kByte, 32);
    const Items s(f[8], "seeds");
    REQUIRE((size_t)s.size() == n, "lists must have one entry per parameter");
    seeds.resize(n);
    for (size_t i = 0; i < n; ++i) {
      seeds[i] = (uint32_t)PyLong_AsUnsignedLongLongMask(s[i]);
      if (PyErr_Occurred()) throw Refused{};
    }
  }
  std::vector<void*> steps(n);
  if (THPVariable_Check(f[7])) {
    const at::Tensor& t = THPVariable_Unpack(f[7]);
    REQUIRE(t.dim() == 1 && (size_t)t.numel() == n, "`steps` must have one count per parameter");
    check_place(t, "steps", device);
    REQUIRE(t.scalar_type() == at::kFloat, "`steps` must be torch.float32");
    for (size_t i = 0; i < n; ++i) steps[i] = static_cast<float*>(t.data_ptr()) + i;
  } else {
    const Items s(f[7], "steps");
    REQUIRE((size_t)s.size() == n, "lists must have one entry per parameter");
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor& t = tensor(s[i], "steps");
      check_place(t, "steps", device);
      REQUIRE(t.scalar_type() == at::kFloat, "`steps` must be torch.float32");
      REQUIRE(t.numel() == 1, "`steps` must be scalars");
      steps[i] = t.data_ptr();
    }
  }
  fm_adamw_group g = {};
  g.state_bits = eight ? 8 : 32;
  if (THPVariable_Check(f[9]))
    g.lr_device = static_cast<const float*>(scalar(f[9], "lr", device));
  else
    g.lr = number(f[9]);
  g.beta1 = number(f[10]);
  g.beta2 = number(f[11]);
  g.eps = number(f[12]);
  g.weight_decay = number(f[13]);
  REQUIRE(g.beta1 >= 0.0 && g.beta1 < 1.0 && g.beta2 >= 0.0 && g.beta2 < 1.0, "betas must lie in [0, 1)");
  REQUIRE(g.eps >= 0.0 && std::isfinite(g.eps), "eps must be finite and not negative");
  REQUIRE(std::isfinite(g.lr) && std::isfinite(g.weight_decay), "lr and weight_decay must be finite");

  auto add = [&](uint8_t kind, Group&& x) {
    x.g = g;
    x.g.p_dtype = kind / 4;
    x.g.g_dtype = kind % 4;
    x.g.count = (int32_t)x.numels.size();
    out.push_back(std::move(x));
  };
  if (one_kind) {
    Group x;
    x.numels = std::move(numels); x.params = std::move(ps); x.grads = std::move(gs); x.masters = std::move(w);
    x.m = std::move(m); x.v = std::move(v); x.ms = std::move(ms); x.vs = std::move(vs);
    x.steps = std::move(steps); x.seeds = std::move(seeds);
    add(kinds[0], std::move(x));
    return;
  }
  for (int kind = 0; kind < 12; ++kind) {
    Group x;
    for (size_t i = 0; i < n; ++i) {
      if (kinds[i] != kind) continue;
      x.numels.push_back(numels[i]);
      x.params.push_back(ps[i]);
      x.grads.push_back(gs[i]);
      x.m.push_back(m[i]);
      x.v.push_back(v[i]);
      x.steps.push_back(steps[i]);
      if (!w.empty()) x.masters.push_back(w[i]);
      if (eight) {
        x.ms.push_back(ms[i]);
        x.vs.push_back(vs[i]);
        x.seeds.push_back(seeds[i]);
      }
    }
    if (!x.numels.empty()) add((uint8_t)kind, std::move(x));
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
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
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

// adamw_step(fm_adamw_step, groups, grad_scale or None) -> status
PyObject* adamw_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n, 3);
    const auto fn = entry<decltype(&fm_adamw_step)>(a[0]);
    const Items tuples(a[1], "groups");
    std::vector<Group> groups;
    groups.reserve(tuples.size() + 4);
    int device = -1;
    for (Py_ssize_t i = 0; i < tuples.size(); ++i) parse_group(tuples[i], device, groups);
    if (groups.empty()) return PyLong_FromLong(FM_OK);
    const float* scale = a[2] == Py_None ? nullptr : static_cast<const float*>(scalar(a[2], "grad_scale", device));
    std::vector<fm_adamw_group> table;
    table.reserve(groups.size());
    for (Group& x : groups) {
      auto at = [](std::vector<void*>& p) { return p.empty() ? nullptr : p.data(); };
      x.g.params = at(x.params);
      x.g.grads = at(x.grads);
      x.g.masters = at(x.masters);
      x.g.exp_avg = at(x.m);
      x.g.exp_avg_sq = at(x.v);
      x.g.exp_avg_scale = at(x.ms);
      x.g.exp_avg_sq_scale = at(x.vs);
      x.g.steps = reinterpret_cast<float* const*>(at(x.steps));
      x.g.numels = x.numels.data();
      x.g.seeds = x.seeds.empty() ? nullptr : x.seeds.data();
      table.push_back(x.g);
    }
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    return PyLong_FromLong(fn(table.data(), (int)table.size(), scale, c10::cuda::getCurrentCUDAStream().stream()));
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
    return PyLong_FromLong(fn(g.at.data(), g.numels.data(), g.dtypes.data(), (int)g.at.size(), factor,
                              c10::cuda::getCurrentCUDAStream().stream()));
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
    {"grad_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(grad_norm)), METH_FASTCALL, nullptr},
    {"scale", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scale)), METH_FASTCALL, nullptr},
    {"adamw8_values", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(adamw8_values)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
