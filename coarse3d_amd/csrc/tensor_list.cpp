// coarse3d_amd._tensor_list -- lists of torch tensors -> the host records (c3d_opt_tensor) of the many-tensor entry points.
//
// A training step hands over hundreds of small tensors; reading one address, length and layout each through Python costs more
// host time (about 0.4 us a tensor) than the GPU needs for the whole step.  This module does nothing else: it checks the lists,
// writes the records and marks the tensors that the call is about to write as changed (autograd's version counters).  It launches
// nothing and keeps nothing.
#include <Python.h>
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

PyObject* pack(PyObject*, PyObject* args) {
  try {
    return pack_impl(args);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {{"pack", pack, METH_VARARGS, "pack(what, lists, kinds, names) -> (records, count, device index, dtypes)"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensor_list", "Lists of tensors -> host records of the many-tensor entry points.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__tensor_list(void) { return PyModule_Create(&module); }
