// coarse3d_amd._native -- the host side of the calls whose Python would take longer than their kernels.
//
// adamw, grad_norm: lists of torch tensors -> the host records (c3d_opt_tensor) of the many-tensor entry points, and their call.  A
// training step hands over hundreds of small tensors; reading one address, length and layout each through Python costs more host time
// (about 0.4 us a tensor) than the GPU needs for the whole step.
// group_norm, group_norm_bwd: checks, results and the call.  From Python one call cost 16 us of host time, and the kernel of a small
// image takes 4.
// Tensors that a call is about to write are marked as changed (autograd's version counters).  Nothing is kept from one call to the next.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <algorithm>
#include <cfloat>
#include <string>
#include <vector>

#include "../../include/coarse3d_hip.h"

namespace {

// ---------------------------------------------------------------- the library, refusals

#define C3D_CALLS(X) X(group_norm) X(group_norm_bwd) X(group_norm_ws_floats) X(grad_norm_partials) X(grad_norm) X(clip_grads) X(adamw_step) X(last_error)
struct Calls {
#define X(name) decltype(&c3d_##name) name = nullptr;
  C3D_CALLS(X)
#undef X
} lib;

// bind({name: address}): the entry points of the loaded library
PyObject* bind(PyObject*, PyObject* args) {
  PyObject* d;
  if (!PyArg_ParseTuple(args, "O!", &PyDict_Type, &d)) return nullptr;
#define X(name)                                                                                       \
  {                                                                                                   \
    PyObject* v = PyDict_GetItemString(d, "c3d_" #name);                                              \
    lib.name = v ? reinterpret_cast<decltype(lib.name)>(PyLong_AsUnsignedLongLong(v)) : nullptr;      \
    if (!lib.name || PyErr_Occurred()) {                                                              \
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_KeyError, "c3d_" #name);                           \
      return nullptr;                                                                                 \
    }                                                                                                 \
  }
  C3D_CALLS(X)
#undef X
  Py_RETURN_NONE;
}

PyObject* fail(PyObject* type, const std::string& what) {
  PyErr_SetString(type, what.c_str());
  return nullptr;
}
struct Refused {
  std::string what;
  bool type = false;            // TypeError instead of ValueError
};
void require(bool ok, const std::string& what) {
  if (!ok) throw Refused{what};
}
PyObject* failed(const char* name, int rc) {
  return fail(PyExc_RuntimeError, std::string(name) + " failed (rc=" + std::to_string(rc) + "): " + lib.last_error());
}
template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused& r) {
    return fail(r.type ? PyExc_TypeError : PyExc_ValueError, r.what);
  } catch (const std::exception& e) {
    return fail(PyExc_RuntimeError, e.what());
  }
}
std::string shape_of(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + (v.size() == 1 ? ",)" : ")");
}
// (a view that stands for the negative of what its memory holds is not)
bool own_memory(const at::Tensor& t) { return t.layout() == at::kStrided && !t.is_meta() && !t.is_quantized() && !t.is_neg(); }
std::string type_of(const at::Tensor& t) { return std::string("torch.") + c10::toString(t.scalar_type()); }

// ---------------------------------------------------------------- lists of tensors

constexpr int kSlots = 7;

struct Range {
  uintptr_t lo, hi;
  bool written;
};

bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  if (a.dim() != b.dim()) return false;
  const auto sa = a.sizes(), sb = b.sizes(), ta = a.strides(), tb = b.strides();
  for (int64_t d = 0; d < a.dim(); ++d)
    if (sa[d] != sb[d] || (sa[d] > 1 && ta[d] != tb[d])) return false;
  return true;
}

// The common case, in one pass: every list ascends in memory and no two lists interleave (`ends`: where each list's ranges end)
bool plainly_disjoint(const std::vector<Range>& r, const std::vector<size_t>& ends) {
  std::vector<Range> hull;
  size_t i = 0;
  for (size_t end : ends) {
    if (i == end) continue;
    for (size_t k = i + 1; k < end; ++k)
      if (r[k].lo < r[k - 1].hi) return false;
    hull.push_back({r[i].lo, r[end - 1].hi, true});
    i = end;
  }
  for (size_t a = 0; a < hull.size(); ++a)
    for (size_t b = a + 1; b < hull.size(); ++b)
      if (hull[a].lo < hull[b].hi && hull[b].lo < hull[a].hi) return false;
  return true;
}

// two ranges of which one is written share memory
bool overlapping(std::vector<Range>& r, const std::vector<size_t>& ends) {
  if (plainly_disjoint(r, ends)) return false;
  auto before = [](const Range& a, const Range& b) { return a.lo < b.lo; };
  if (!std::is_sorted(r.begin(), r.end(), before)) std::sort(r.begin(), r.end(), before);
  uintptr_t any = 0, written = 0;      // ends of what came before
  for (const Range& x : r) {
    if (x.lo < written || (x.written && x.lo < any)) return true;
    any = std::max(any, x.hi);
    if (x.written) written = std::max(written, x.hi);
  }
  return false;
}

// A call's lists as records.  lists: seven lists (or None), one for each slot of c3d_opt_tensor; kinds: seven letters: 'w' elementwise
// and written, 'r' elementwise and read, 's' block scales (written); names: seven words for messages
struct Lists {
  std::vector<c3d_opt_tensor> rec;
  at::ScalarType type[kSlots];
  bool have[kSlots] = {};
  c10::Device device = c10::kCPU;
  PyObject* seq[kSlots] = {};
  const char* kinds;

  Lists(const std::string& what, PyObject* const (&lists)[kSlots], const char* kinds_, const char* const (&names)[kSlots]) : kinds(kinds_) {
    int first = -1;
    Py_ssize_t count = 0;
    for (int s = 0; s < kSlots; ++s) {
      PyObject* l = lists[s];
      if (!l || l == Py_None) continue;
      if (!PyList_Check(l) && !PyTuple_Check(l)) throw Refused{what + names[s] + " is a list of tensors", true};
      seq[s] = l;
      have[s] = true;
      const Py_ssize_t k = PySequence_Fast_GET_SIZE(l);
      if (first < 0) {
        first = s;
        count = k;
      } else if (k != count) {
        throw Refused{what + names[s] + " has " + std::to_string(k) + " tensors, " + names[first] + " has " + std::to_string(count)};
      }
    }
    if (first < 0 || count == 0) throw Refused{what + "no tensors"};
    rec.assign(count, c3d_opt_tensor{});
    std::vector<Range> ranges;
    std::vector<size_t> ends;
    ranges.reserve((size_t)count * kSlots);
    bool seen = false;
    for (int s = 0; s < kSlots; ++s) {
      if (!seq[s]) continue;
      for (Py_ssize_t i = 0; i < count; ++i) {
        PyObject* o = PySequence_Fast_GET_ITEM(seq[s], i);
        auto need = [&](bool ok, const char* text) {
          if (!ok) throw Refused{what + names[s] + "[" + std::to_string(i) + "] " + text};
        };
        if (!THPVariable_Check(o)) throw Refused{what + names[s] + "[" + std::to_string(i) + "] is not a tensor", true};
        const at::Tensor& t = THPVariable_Unpack(o);
        need(own_memory(t), "is not a dense tensor with memory of its own");
        if (i == 0) type[s] = t.scalar_type();
        need(t.scalar_type() == type[s], "has another type than the first of its list");
        if (!seen) device = t.device();
        seen = true;
        need(t.device() == device, "is on another device than the others");
        const int64_t n = t.numel();
        if (s == first) rec[i].n = n;
        if (kinds[s] == 's') {
          need(n == (rec[i].n + C3D_ADAMW8_BLOCK - 1) / C3D_ADAMW8_BLOCK && t.is_contiguous(), "is not a contiguous tensor of one scale for each block");
        } else if (s == first) {
          need(n == 0 || t.is_non_overlapping_and_dense(), "is not dense: its elements have gaps or overlap");
        } else {
          const at::Tensor& r = THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq[first], i));
          if (n != rec[i].n || (n > 0 && !same_layout(t, r))) need(false, (std::string("differs in shape or strides from ") + names[first]).c_str());
        }
        if (n == 0) continue;
        rec[i].ptr[s] = t.data_ptr();
        const uintptr_t lo = reinterpret_cast<uintptr_t>(rec[i].ptr[s]);
        ranges.push_back({lo, lo + (uintptr_t)n * t.element_size(), kinds[s] != 'r'});
      }
      ends.push_back(ranges.size());
    }
    if (overlapping(ranges, ends)) throw Refused{what + "two tensors share memory"};
  }
  // the last of the checks
  void on_gpu(const std::string& what) const {
    if (!device.is_cuda()) throw Refused{what + "the tensors are on " + device.str() + ", not on a GPU"};
  }
  void mark_written() const {
    for (int s = 0; s < kSlots; ++s)
      for (size_t i = 0; seq[s] && kinds[s] != 'r' && i < rec.size(); ++i) {
        const at::Tensor& t = THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq[s], i));
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
      }
  }
  std::string type_name(int s) const { return have[s] ? std::string("torch.") + c10::toString(type[s]) : "None"; }
};

int type_code(at::ScalarType s) { return s == at::kFloat ? 0 : s == at::kBFloat16 ? 1 : s == at::kHalf ? 2 : -1; }

// a 0-dim fp32 device tensor, as lr, step and grad_scale may be
const float* scalar(const at::Tensor& t, const c10::Device& dev, const std::string& what) {
  if (t.numel() != 1 || t.scalar_type() != at::kFloat || t.device() != dev) throw Refused{what + " as a tensor is one fp32 value on the parameters' device"};
  return static_cast<const float*>(t.data_ptr());
}

// adamw(what, lists, bits, step, lr, beta1, beta2, eps, weight_decay, grad_scale, seed, stream): step and lr numbers or tensors
PyObject* adamw(PyObject*, PyObject* args) {
  const char* what_c;
  PyObject *lists_o, *step_o, *lr_o, *scale_o;
  int bits;
  double b1, b2, eps, wd;
  unsigned long long seed, stream;
  if (!PyArg_ParseTuple(args, "sO!iOOddddOKK", &what_c, &PyTuple_Type, &lists_o, &bits, &step_o, &lr_o, &b1, &b2, &eps, &wd, &scale_o, &seed, &stream))
    return nullptr;
  return guarded([&]() -> PyObject* {
    const std::string what = std::string(what_c) + ": ";
    const bool eight = bits == 8;
    PyObject* lists[kSlots];
    if (PyTuple_GET_SIZE(lists_o) != kSlots) throw Refused{what + "seven lists are expected"};
    for (int s = 0; s < kSlots; ++s) lists[s] = PyTuple_GET_ITEM(lists_o, s);
    static const char* const names32[kSlots] = {"params", "grads", "exp_avgs", "exp_avg_sqs", "", "", "masters"};
    static const char* const names8[kSlots] = {"params", "grads", "exp_avgs", "exp_avg_roots", "exp_avg_scales", "exp_avg_root_scales", "masters"};
    const Lists l(what, lists, "wrwwssw", eight ? names8 : names32);
    for (int s = 0; s < (eight ? 6 : 4); ++s)
      if (!l.have[s]) throw Refused{what + (eight ? names8 : names32)[s] + " is a list of tensors", true};
    require(type_code(l.type[0]) >= 0 && (l.type[1] == l.type[0] || l.type[1] == at::kFloat),
            what + "parameters are fp32, bf16 or fp16 and gradients of the same type or fp32, got " + l.type_name(0) + " and " + l.type_name(1));
    const auto want = eight ? at::kFloat8_e4m3fn : at::kFloat;
    require(l.type[2] == want && l.type[3] == want,
            what + "the states are torch." + c10::toString(want) + ", got " + l.type_name(2) + " and " + l.type_name(3));
    require(!eight || (l.type[4] == at::kFloat && l.type[5] == at::kFloat), what + "the states' scales are fp32");
    require(!l.have[6] || (l.type[6] == at::kFloat && l.type[0] != at::kFloat),
            what + "master copies are fp32, of 16-bit parameters; got " + l.type_name(6) + " of " + l.type_name(0));
    require(b1 >= 0.0 && b1 < 1.0 && b2 >= 0.0 && b2 < 1.0, what + "betas are in [0, 1), got (" + std::to_string(b1) + ", " + std::to_string(b2) + ")");
    require(eps == 0.0 || (float)eps >= FLT_MIN, what + "eps is 0 or at least 2^-126, got " + c10::str(eps));
    c3d_adamw_desc d{};
    if (THPVariable_Check(lr_o)) {
      d.lr_dev = scalar(THPVariable_Unpack(lr_o), l.device, what + "lr");
    } else {
      d.lr = PyFloat_AsDouble(lr_o);
      if (PyErr_Occurred()) return nullptr;
    }
    if (THPVariable_Check(step_o)) {
      d.step_dev = scalar(THPVariable_Unpack(step_o), l.device, what + "step");
    } else {
      d.step = PyLong_AsLongLong(step_o);
      if (PyErr_Occurred()) return nullptr;
      require(d.step >= 1, what + "step counts from 1, got " + std::to_string(d.step));
    }
    if (scale_o != Py_None) {
      if (!THPVariable_Check(scale_o)) throw Refused{what + "grad_scale is a tensor", true};
      d.grad_scale = scalar(THPVariable_Unpack(scale_o), l.device, what + "grad_scale");
    }
    l.on_gpu(what);
    d.beta1 = b1;
    d.beta2 = b2;
    d.eps = eps;
    d.weight_decay = wd;
    d.param_type = type_code(l.type[0]);
    d.grad_type = type_code(l.type[1]);
    d.state_bits = bits;
    d.has_master = l.have[6];
    d.seed = (uint32_t)seed;
    l.mark_written();
    const int rc = lib.adamw_step(l.rec.data(), (int)l.rec.size(), &d, reinterpret_cast<c3d_stream>(stream));
    if (rc) return failed("c3d_adamw_step", rc);
    Py_RETURN_NONE;
  });
}

// grads_of(params) -> (their gradients, None where there is none; a byte for each: its type, 255 without)
PyObject* grads_of(PyObject*, PyObject* params) {
  if (!PyList_Check(params) && !PyTuple_Check(params)) return fail(PyExc_TypeError, "grads_of: a list of tensors is expected");
  return guarded([&]() -> PyObject* {
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(params);
    std::string types((size_t)n, '\xff');
    THPObjectPtr out(PyList_New(n));
    if (!out) return nullptr;
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* o = PySequence_Fast_GET_ITEM(params, i);
      if (!THPVariable_Check(o)) throw Refused{"grads_of: a list of tensors is expected", true};
      const at::Tensor& g = THPVariable_Unpack(o).grad();
      if (g.defined()) types[(size_t)i] = (char)g.scalar_type();
      PyObject* w = THPVariable_Wrap(g);       // (None for an undefined one)
      if (!w) return nullptr;
      PyList_SET_ITEM(out.get(), i, w);
    }
    return Py_BuildValue("Ny#", out.release(), types.data(), n);
  });
}

// grad_norm(what, grads, max_norm, clip, stream) -> (norm, scale); clip: the gradients are scaled in place
PyObject* grad_norm(PyObject*, PyObject* args) {
  const char* what_c;
  PyObject* grads;
  double max_norm;
  int clip;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "sOdpK", &what_c, &grads, &max_norm, &clip, &stream)) return nullptr;
  return guarded([&]() -> PyObject* {
    const std::string what = std::string(what_c) + ": ";
    PyObject* const lists[kSlots] = {nullptr, grads};
    static const char* const names[kSlots] = {"", "grads", "", "", "", "", ""};
    const Lists l(what, lists, clip ? "wwwwssw" : "wrwwssw", names);
    if (!l.have[1]) throw Refused{what + "grads is a list of tensors", true};
    const int type = type_code(l.type[1]), n = (int)l.rec.size();
    require(type >= 0, what + "gradients are fp32, bf16 or fp16, got " + l.type_name(1));
    require(max_norm >= 0.0, what + "max_norm is not negative, got " + std::to_string(max_norm));
    l.on_gpu(what);
    const auto opt = at::TensorOptions().device(l.device).dtype(at::kFloat);
    const at::Tensor norm = at::empty({}, opt), scale = at::empty({}, opt);
    const at::Tensor part = at::empty({lib.grad_norm_partials(l.rec.data(), n, type)}, opt.dtype(at::kDouble));
    if (clip) l.mark_written();
    const int rc = (clip ? lib.clip_grads : lib.grad_norm)(l.rec.data(), n, type, max_norm, static_cast<double*>(part.data_ptr()),
                                                          static_cast<float*>(norm.data_ptr()), static_cast<float*>(scale.data_ptr()),
                                                          reinterpret_cast<c3d_stream>(stream));
    if (rc) return failed(clip ? "c3d_clip_grads" : "c3d_grad_norm", rc);
    return Py_BuildValue("NN", THPVariable_Wrap(norm), THPVariable_Wrap(scale));
  });
}

// ---------------------------------------------------------------- GroupNorm

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw Refused{std::string(what) + " is not a tensor", true};
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!own_memory(t)) throw Refused{std::string(what) + " is not a dense tensor with memory of its own"};
  return t;
}

struct Rows {
  int64_t n, hw, c, ns, ps;     // samples, pixels, channels; elements from sample to sample and from pixel to pixel
};
Rows rows_of(const at::Tensor& t, const char* what) {
  const int64_t dim = t.dim();
  if (dim < 2) throw Refused{std::string(what) + " is [N, ..., C], got " + shape_of(t.sizes())};
  Rows r{t.size(0), 1, t.size(dim - 1), 0, 0};
  if (t.numel() == 0) return {r.n, r.c && r.n ? 0 : 1, r.c, 0, r.c};
  if (t.is_contiguous()) {
    r.hw = t.numel() / (r.n * r.c);
    return {r.n, r.hw, r.c, r.hw * r.c, r.c};
  }
  bool ok = r.c == 1 || t.stride(dim - 1) == 1, first = true;
  for (int64_t d = dim - 2; d > 0; --d) {
    if (t.size(d) > 1) {
      if (first) r.ps = t.stride(d);
      first = false;
      ok = ok && t.stride(d) == r.ps * r.hw;
    }
    r.hw *= t.size(d);
  }
  if (first) r.ps = r.c;
  r.ns = r.n > 1 ? t.stride(0) : r.hw * r.ps;
  if (!ok || r.ps < r.c || (r.n > 1 && r.ns < (r.hw - 1) * r.ps + r.c))
    throw Refused{std::string(what) + ": the channels of a pixel have to lie side by side and the pixels one stride apart; got shape " +
                  shape_of(t.sizes()) + ", strides " + shape_of(t.strides()) + " (call .contiguous())"};
  return r;
}
int type_code(const at::Tensor& t, const char* what) {
  const int code = type_code(t.scalar_type());
  if (code < 0) throw Refused{std::string(what) + ": fp32, bf16 or fp16, got " + type_of(t)};
  return code;
}
int act_code(const char* act, double slope, const char* what) {
  const std::string a(act);
  if (a != "none" && a != "lrelu" && a != "silu") throw Refused{std::string(what) + ": act is one of ['lrelu', 'none', 'silu'], got '" + a + "'"};
  if (!(slope >= 0.0 && slope <= 1.0)) throw Refused{std::string(what) + ": slope is in [0, 1], got " + std::to_string(slope)};
  return a == "none" ? 0 : a == "lrelu" ? 1 : 2;
}
const float* affine(PyObject* o, int64_t c, const at::Device& dev, const char* name) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != c || !t.is_contiguous() || t.device() != dev)
    throw Refused{std::string("group_norm: ") + name + " is a contiguous fp32 tensor of " + std::to_string(c) + " values on " + dev.str()};
  return static_cast<const float*>(t.data_ptr());
}
void groups_divide(int64_t c, int64_t groups, const char* what) {
  if (groups < 1 || c < 1 || c % groups)
    throw Refused{std::string(what) + ": " + std::to_string(c) + " channels do not divide into " + std::to_string(groups) + " groups"};
}
void on_gpu(const at::Tensor& t, const char* what) {
  if (!t.is_cuda()) throw Refused{std::string(what) + ": the tensors are on " + t.device().str() + ", not on a GPU"};
}
void sizes_fit(const Rows& r, int64_t groups, const char* what) {
  if (r.n > INT32_MAX || r.c > INT32_MAX || groups > INT32_MAX) throw Refused{std::string(what) + ": too many samples or channels"};
}
PyObject* three(const at::Tensor& a, const at::Tensor& b, const at::Tensor& c) {
  auto wrap = [](const at::Tensor& t) {
    if (t.defined()) return THPVariable_Wrap(t);
    Py_INCREF(Py_None);
    return Py_None;
  };
  return Py_BuildValue("NNN", wrap(a), wrap(b), wrap(c));
}

// group_norm(x, groups, gamma, beta, eps, act, slope, stream) -> (y, mean, rstd)
PyObject* group_norm(PyObject*, PyObject* args) {
  PyObject *xo, *go, *bo;
  long long groups;
  double eps, slope;
  const char* act;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "OLOOdsdK", &xo, &groups, &go, &bo, &eps, &act, &slope, &stream)) return nullptr;
  return guarded([&]() -> PyObject* {
    constexpr const char* what = "group_norm";
    const at::Tensor& x = tensor(xo, "group_norm: x");
    const int type = type_code(x, what), code = act_code(act, slope, what);
    const Rows r = rows_of(x, "group_norm: x");
    groups_divide(r.c, groups, what);
    require(eps >= 0.0, "group_norm: eps is not negative, got " + std::to_string(eps));
    const float *ga = affine(go, r.c, x.device(), "gamma"), *be = affine(bo, r.c, x.device(), "beta");
    on_gpu(x, what);
    sizes_fit(r, groups, what);
    const auto opt = x.options().requires_grad(false).memory_format(c10::nullopt), f32 = opt.dtype(at::kFloat);
    const at::Tensor y = at::empty(x.sizes(), opt);
    if (r.n == 0 || r.hw == 0) return three(y, at::zeros({r.n, groups}, f32), at::zeros({r.n, groups}, f32));
    const at::Tensor mean = at::empty({r.n, groups}, f32), rstd = at::empty({r.n, groups}, f32);
    const int64_t floats = lib.group_norm_ws_floats((int)r.n, r.hw, (int)r.c, (int)groups, type);
    at::Tensor ws;
    if (floats) ws = at::empty({floats}, f32);
    const int rc = lib.group_norm(x.data_ptr(), r.ns, r.ps, (int)r.n, r.hw, (int)r.c, (int)groups, type, ga, be, (float)eps, code, (float)slope,
                                   y.data_ptr(), static_cast<float*>(mean.data_ptr()), static_cast<float*>(rstd.data_ptr()),
                                   floats ? static_cast<float*>(ws.data_ptr()) : nullptr, reinterpret_cast<c3d_stream>(stream));
    return rc ? failed("c3d_group_norm", rc) : three(y, mean, rstd);
  });
}

// group_norm_bwd(dy, x, mean, rstd, gamma, beta, act, slope, stream) -> (dx, dgamma, dbeta)
PyObject* group_norm_bwd(PyObject*, PyObject* args) {
  PyObject *dyo, *xo, *mo, *ro, *go, *bo;
  double slope;
  const char* act;
  unsigned long long stream;
  if (!PyArg_ParseTuple(args, "OOOOOOsdK", &dyo, &xo, &mo, &ro, &go, &bo, &act, &slope, &stream)) return nullptr;
  return guarded([&]() -> PyObject* {
    constexpr const char* what = "group_norm_bwd";
    const at::Tensor &dy = tensor(dyo, "group_norm_bwd: dy"), &x = tensor(xo, "group_norm_bwd: x"), &mean = tensor(mo, "group_norm_bwd: mean"),
                     &rstd = tensor(ro, "group_norm_bwd: rstd");
    const int type = type_code(x, what), code = act_code(act, slope, what);
    const Rows r = rows_of(x, "group_norm_bwd: x");
    require(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(),
            "group_norm_bwd: dy is " + shape_of(dy.sizes()) + " " + type_of(dy) + " on " + dy.device().str() + ", x is " + shape_of(x.sizes()) + " " +
                type_of(x) + " on " + x.device().str());
    const Rows d = rows_of(dy, "group_norm_bwd: dy");
    for (const at::Tensor* t : {&mean, &rstd})
      require(t->dim() == 2 && t->size(0) == r.n && t->sizes() == mean.sizes() && t->scalar_type() == at::kFloat && t->is_contiguous() &&
                  t->device() == x.device(),
              std::string("group_norm_bwd: ") + (t == &mean ? "mean" : "rstd") + " is the fp32 [N, groups] tensor that group_norm returned");
    const int64_t groups = mean.size(1);
    groups_divide(r.c, groups, what);
    const float *ga = affine(go, r.c, x.device(), "gamma"), *be = affine(bo, r.c, x.device(), "beta");
    on_gpu(x, what);
    sizes_fit(r, groups, what);
    const auto opt = x.options().requires_grad(false).memory_format(c10::nullopt), f32 = opt.dtype(at::kFloat);
    const at::Tensor dx = at::empty(x.sizes(), opt);
    const bool none = r.n == 0 || r.hw == 0;
    at::Tensor dgamma, dbeta, ws;
    if (ga || go != Py_None) dgamma = none ? at::zeros({r.c}, f32) : at::empty({r.c}, f32);
    if (be || bo != Py_None) dbeta = none ? at::zeros({r.c}, f32) : at::empty({r.c}, f32);
    if (none) return three(dx, dgamma, dbeta);
    const int64_t floats = lib.group_norm_ws_floats((int)r.n, r.hw, (int)r.c, (int)groups, type);
    if (floats) ws = at::empty({floats}, f32);
    auto f = [](const at::Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; };
    const int rc = lib.group_norm_bwd(dy.data_ptr(), d.ns, d.ps, x.data_ptr(), r.ns, r.ps, (int)r.n, r.hw, (int)r.c, (int)groups, type, f(mean), f(rstd),
                                       ga, be, code, (float)slope, dx.data_ptr(), f(dgamma), f(dbeta), f(ws), reinterpret_cast<c3d_stream>(stream));
    return rc ? failed("c3d_group_norm_bwd", rc) : three(dx, dgamma, dbeta);
  });
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "bind({name: address}): the entry points of the loaded library"},
                         {"adamw", adamw, METH_VARARGS,
                          "adamw(what, lists, bits, step, lr, beta1, beta2, eps, weight_decay, grad_scale, seed, stream)"},
                         {"grads_of", grads_of, METH_O, "grads_of(params) -> (gradients or None, a byte for each: its type)"},
                         {"grad_norm", grad_norm, METH_VARARGS, "grad_norm(what, grads, max_norm, clip, stream) -> (norm, scale)"},
                         {"group_norm", group_norm, METH_VARARGS, "group_norm(x, groups, gamma, beta, eps, act, slope, stream) -> (y, mean, rstd)"},
                         {"group_norm_bwd", group_norm_bwd, METH_VARARGS,
                          "group_norm_bwd(dy, x, mean, rstd, gamma, beta, act, slope, stream) -> (dx, dgamma, dbeta)"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "Host side of the calls whose Python would take longer than their kernels.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
