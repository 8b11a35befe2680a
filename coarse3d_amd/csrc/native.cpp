// coarse3d_amd._native -- the host side of the calls whose Python would take longer than their kernels.
//
// pack: lists of torch tensors -> the host records (c3d_opt_tensor) of the many-tensor entry points.  A training step hands over
// hundreds of small tensors; reading one address, length and layout each through Python costs more host time (about 0.4 us a tensor)
// than the GPU needs for the whole step.  It checks the lists, writes the records and marks the tensors that the call is about to
// write as changed (autograd's version counters).
// group_norm, group_norm_bwd: checks, results and the call of the C ABI.  From Python one call cost 16 us of host time, and the
// kernel of a small image takes 4.
// Nothing is kept from one call to the next.
#include <Python.h>
#include <ATen/ATen.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <string>
#include <vector>

#include "../../include/coarse3d_hip.h"

namespace {

constexpr int kSlots = 7;

struct Range {
  uintptr_t lo, hi;
  bool written;
};

PyObject* fail(PyObject* type, const std::string& what) {
  PyErr_SetString(type, what.c_str());
  return nullptr;
}

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

// pack(what, lists, kinds, names) -> (records, count, device index, dtypes)
// lists: a tuple of seven lists (or None), one for each slot of c3d_opt_tensor; kinds: seven letters: 'w' elementwise and written,
// 'r' elementwise and read, 's' block scales (written); names: seven words for messages
PyObject* pack_impl(PyObject* args) {
  const char *what_c, *kinds;
  PyObject *lists, *names;
  if (!PyArg_ParseTuple(args, "sO!sO!", &what_c, &PyTuple_Type, &lists, &kinds, &PyTuple_Type, &names)) return nullptr;
  const std::string what = std::string(what_c) + ": ";
  if (PyTuple_GET_SIZE(lists) != kSlots || PyTuple_GET_SIZE(names) != kSlots || std::string(kinds).size() != kSlots)
    return fail(PyExc_ValueError, what + "seven lists, kinds and names are expected");
  PyObject* seq[kSlots] = {};
  int first = -1;
  Py_ssize_t count = 0;
  std::string name[kSlots];
  for (int s = 0; s < kSlots; ++s) {
    PyObject* l = PyTuple_GET_ITEM(lists, s);
    const char* nm = PyUnicode_AsUTF8(PyTuple_GET_ITEM(names, s));
    if (!nm) return nullptr;
    name[s] = nm;
    if (l == Py_None) continue;
    if (!PyList_Check(l) && !PyTuple_Check(l)) return fail(PyExc_TypeError, what + name[s] + " is a list of tensors");
    seq[s] = l;
    const Py_ssize_t k = PySequence_Fast_GET_SIZE(l);
    if (first < 0) {
      first = s;
      count = k;
    } else if (k != count) {
      return fail(PyExc_ValueError, what + name[s] + " has " + std::to_string(k) + " tensors, " + name[first] + " has " + std::to_string(count));
    }
  }
  if (first < 0) return fail(PyExc_ValueError, what + "no tensors");
  PyObject* out = PyBytes_FromStringAndSize(nullptr, count * (Py_ssize_t)sizeof(c3d_opt_tensor));
  if (!out) return nullptr;
  c3d_opt_tensor* rec = reinterpret_cast<c3d_opt_tensor*>(PyBytes_AS_STRING(out));
  std::vector<Range> ranges;
  ranges.reserve((size_t)count * kSlots);
  std::vector<size_t> ends;
  at::ScalarType type[kSlots];
  c10::Device device(c10::kCPU);
  bool seen = false;
  std::string bad;
  PyObject* bad_type = PyExc_ValueError;
  for (int s = 0; s < kSlots && bad.empty(); ++s) {
    if (!seq[s]) {
      for (Py_ssize_t i = 0; i < count; ++i) rec[i].ptr[s] = nullptr;
      continue;
    }
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* o = PySequence_Fast_GET_ITEM(seq[s], i);
      const std::string* nm = &name[s];
      auto say = [&](const char* t) { bad = what + *nm + "[" + std::to_string(i) + "] " + t; };
      if (!THPVariable_Check(o)) {
        say("is not a tensor");
        bad_type = PyExc_TypeError;
        break;
      }
      const at::Tensor& t = THPVariable_Unpack(o);
      if (t.layout() != at::kStrided || t.is_meta() || t.is_quantized()) {
        say("is not a dense tensor with memory of its own");
        break;
      }
      if (i == 0) type[s] = t.scalar_type();
      else if (t.scalar_type() != type[s]) {
        say("has another type than the first of its list");
        break;
      }
      if (!seen) {
        device = t.device();
        seen = true;
      } else if (t.device() != device) {
        say("is on another device than the others");
        break;
      }
      const int64_t n = t.numel();
      if (s == first) rec[i].n = n;
      if (kinds[s] == 's') {
        if (n != (rec[i].n + C3D_ADAMW8_BLOCK - 1) / C3D_ADAMW8_BLOCK || !t.is_contiguous()) {
          say("is not a contiguous tensor of one scale for each block");
          break;
        }
      } else if (s == first) {
        if (n > 0 && !t.is_non_overlapping_and_dense()) {
          say("is not dense: its elements have gaps or overlap");
          break;
        }
      } else {
        const at::Tensor& r = THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq[first], i));
        if (n != rec[i].n || (n > 0 && !same_layout(t, r))) {
          say(("differs in shape or strides from " + name[first]).c_str());
          break;
        }
      }
      rec[i].ptr[s] = n > 0 ? t.data_ptr() : nullptr;
      if (n > 0) {
        const uintptr_t lo = reinterpret_cast<uintptr_t>(rec[i].ptr[s]);
        ranges.push_back({lo, lo + (uintptr_t)n * t.element_size(), kinds[s] != 'r'});
      }
    }
    ends.push_back(ranges.size());
  }
  if (bad.empty() && overlapping(ranges, ends)) bad = what + "two tensors share memory";
  if (bad.empty() && count > 0 && !device.is_cuda()) bad = what + "the tensors are on " + device.str() + ", not on a GPU";
  if (!bad.empty()) {
    Py_DECREF(out);
    return fail(bad_type, bad);
  }
  for (int s = 0; s < kSlots; ++s)
    for (Py_ssize_t i = 0; seq[s] && kinds[s] != 'r' && i < count; ++i) {
      const at::Tensor& t = THPVariable_Unpack(PySequence_Fast_GET_ITEM(seq[s], i));
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    }
  PyObject* types = PyTuple_New(kSlots);
  if (!types) {
    Py_DECREF(out);
    return nullptr;
  }
  for (int s = 0; s < kSlots; ++s) {
    PyObject* d = seq[s] && count > 0 ? reinterpret_cast<PyObject*>(torch::getTHPDtype(type[s])) : Py_None;
    Py_INCREF(d);
    PyTuple_SET_ITEM(types, s, d);
  }
  return Py_BuildValue("NniN", out, count, seen ? (int)device.index() : -1, types);
}

// ---------------------------------------------------------------- GroupNorm

decltype(&c3d_group_norm) call_group_norm = nullptr;
decltype(&c3d_group_norm_bwd) call_group_norm_bwd = nullptr;
decltype(&c3d_group_norm_ws_floats) call_ws_floats = nullptr;
decltype(&c3d_last_error) call_last_error = nullptr;

// bind(group_norm, group_norm_bwd, group_norm_ws_floats, last_error): addresses in the loaded library
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a, b, c, d;
  if (!PyArg_ParseTuple(args, "KKKK", &a, &b, &c, &d)) return nullptr;
  call_group_norm = reinterpret_cast<decltype(call_group_norm)>(a);
  call_group_norm_bwd = reinterpret_cast<decltype(call_group_norm_bwd)>(b);
  call_ws_floats = reinterpret_cast<decltype(call_ws_floats)>(c);
  call_last_error = reinterpret_cast<decltype(call_last_error)>(d);
  Py_RETURN_NONE;
}

std::string shape_of(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + (v.size() == 1 ? ",)" : ")");
}
std::string type_of(const at::Tensor& t) { return std::string("torch.") + c10::toString(t.scalar_type()); }

struct Refused {
  std::string what;
};
void require(bool ok, const std::string& what) {
  if (!ok) throw Refused{what};
}
const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw Refused{std::string(what) + " is not a tensor"};
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.layout() != at::kStrided || t.is_meta()) throw Refused{std::string(what) + " is not a dense tensor with memory of its own"};
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
  const auto s = t.scalar_type();
  if (s != at::kFloat && s != at::kBFloat16 && s != at::kHalf) throw Refused{std::string(what) + ": fp32, bf16 or fp16, got " + type_of(t)};
  return s == at::kFloat ? 0 : s == at::kBFloat16 ? 1 : 2;
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
PyObject* failed(const char* name, int rc) {
  return fail(PyExc_RuntimeError, std::string(name) + " failed (rc=" + std::to_string(rc) + "): " + call_last_error());
}
template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused& r) {
    return fail(PyExc_ValueError, r.what);
  } catch (const std::exception& e) {
    return fail(PyExc_RuntimeError, e.what());
  }
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
    const int64_t floats = call_ws_floats((int)r.n, r.hw, (int)r.c, (int)groups, type);
    at::Tensor ws;
    if (floats) ws = at::empty({floats}, f32);
    const int rc = call_group_norm(x.data_ptr(), r.ns, r.ps, (int)r.n, r.hw, (int)r.c, (int)groups, type, ga, be, (float)eps, code, (float)slope,
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
    const int64_t floats = call_ws_floats((int)r.n, r.hw, (int)r.c, (int)groups, type);
    if (floats) ws = at::empty({floats}, f32);
    auto f = [](const at::Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; };
    const int rc = call_group_norm_bwd(dy.data_ptr(), d.ns, d.ps, x.data_ptr(), r.ns, r.ps, (int)r.n, r.hw, (int)r.c, (int)groups, type, f(mean), f(rstd),
                                       ga, be, code, (float)slope, dx.data_ptr(), f(dgamma), f(dbeta), f(ws), reinterpret_cast<c3d_stream>(stream));
    return rc ? failed("c3d_group_norm_bwd", rc) : three(dx, dgamma, dbeta);
  });
}

PyObject* pack(PyObject*, PyObject* args) {
  try {
    return pack_impl(args);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {{"pack", pack, METH_VARARGS, "pack(what, lists, kinds, names) -> (records, count, device index, dtypes)"},
                         {"bind", bind, METH_VARARGS, "bind(group_norm, group_norm_bwd, group_norm_ws_floats, last_error): addresses"},
                         {"group_norm", group_norm, METH_VARARGS, "group_norm(x, groups, gamma, beta, eps, act, slope, stream) -> (y, mean, rstd)"},
                         {"group_norm_bwd", group_norm_bwd, METH_VARARGS,
                          "group_norm_bwd(dy, x, mean, rstd, gamma, beta, act, slope, stream) -> (dx, dgamma, dbeta)"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "Host side of the calls whose Python would take longer than their kernels.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
