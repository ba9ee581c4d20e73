// lists.cpp -- what is quicker asked of torch's tensors from here than from Python (an extension, sdmchat_amd/lib/_lists.so,
// loaded by sdmchat_amd/_lib.py): lists of tensors as the sdm_rt_tensor array that a training step's calls take, and several
// small outputs at once.
//
// A step over a model asks five things of each of some 700 tensors: asked from Python they take longer than the step itself
// (182 tensors with two moments each: 230 us of host time, from here 20).
#include <Python.h>
#include <ATen/Functions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdint>
#include <vector>

#include "sdm_rt.h"

namespace {

constexpr int64_t kBlock = 128, kBlockBytes = 264;   // of 8-bit moments

enum Role { kParams, kGrads, kExpAvgs, kExpAvgSqs, kRoles };

struct Span {
  uintptr_t begin, end;
  bool written;
};

// no two of the spans overlap of which one is written
bool apart(std::vector<Span>& spans) {
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;   // the furthest ends so far
  for (const Span& s : spans) {
    if (s.begin < (s.written ? any : written)) return false;
    any = std::max(any, s.end);
    if (s.written) written = std::max(written, s.end);
  }
  return true;
}

int64_t code_of(at::ScalarType t) {
  return t == at::kFloat ? SDM_RT_F32 : t == at::kBFloat16 ? SDM_RT_BF16 : -1;
}

// pack(params, grads, exp_avgs, exp_avg_sqs, eight, reading): each a list of tensors or None.  The table as bytes and the
// index of the GPU, where all of it is plain: lists of equal length of torch.Tensor or Parameter, contiguous, on one GPU, of
// the dtypes and sizes that belong together; else None (the caller finds out why, or sets it right).  ValueError where two
// tensors overlap of which one is written.  eight: exp_avgs hold both moments in 8 bits; reading: they are read, params and
// exp_avg_sqs written.
PyObject* pack(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6) {
    PyErr_SetString(PyExc_TypeError, "pack: 6 arguments");
    return nullptr;
  }
  const bool eight = args[4] == Py_True, reading = args[5] == Py_True;
  Py_ssize_t n = -1;
  for (int r = 0; r < kRoles; ++r) {
    if (args[r] == Py_None) continue;
    if (!PyList_CheckExact(args[r]) || (n >= 0 && PyList_GET_SIZE(args[r]) != n)) Py_RETURN_NONE;
    n = PyList_GET_SIZE(args[r]);
  }
  if (n <= 0) Py_RETURN_NONE;
  try {
    std::vector<Span> spans;
    const bool written[kRoles] = {true, false, !reading, true};
    PyObject* bytes = PyBytes_FromStringAndSize(nullptr, n * static_cast<Py_ssize_t>(sizeof(sdm_rt_tensor)));
    if (!bytes) return nullptr;
    struct Hold {
      PyObject* o;
      ~Hold() { Py_XDECREF(o); }
    } hold{bytes};
    sdm_rt_tensor* table = reinterpret_cast<sdm_rt_tensor*>(PyBytes_AS_STRING(bytes));
    spans.reserve(static_cast<size_t>(n) * kRoles);
    int device = -1;
    const int leader = args[kParams] == Py_None ? kGrads : kParams;
    for (Py_ssize_t i = 0; i < n; ++i) {
      void* at[kRoles] = {};
      const at::Tensor* first = nullptr;
      int64_t numel = 0, code = 0;
      for (int k = 0; k < kRoles; ++k) {
        const int r = k == 0 ? leader : k == leader ? 0 : k;   // the one that the others are compared with comes first
        if (args[r] == Py_None) continue;
        PyObject* o = PyList_GET_ITEM(args[r], i);
        if (!THPVariable_CheckExact(o)) Py_RETURN_NONE;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!t.defined() || t.layout() != at::kStrided || !t.is_cuda() || !t.is_contiguous() || t.is_neg()) Py_RETURN_NONE;
        if (device < 0) device = t.get_device();
        if (t.get_device() != device) Py_RETURN_NONE;
        if (!first) {
          first = &t;
          numel = t.numel();
          code = code_of(t.scalar_type());
          if (code < 0) Py_RETURN_NONE;
        } else if (r == kExpAvgs && eight) {
          if (t.scalar_type() != at::kByte || t.dim() != 2 || t.size(0) != (numel + kBlock - 1) / kBlock ||
              t.size(1) != kBlockBytes)
            Py_RETURN_NONE;
        } else if (r == kGrads || reading) {
          if (t.scalar_type() != first->scalar_type() || t.sizes() != first->sizes()) Py_RETURN_NONE;
        } else if (t.scalar_type() != at::kFloat || t.sizes() != first->sizes()) {
          Py_RETURN_NONE;
        }
        at[r] = t.data_ptr();
        if (t.numel()) {
          const uintptr_t begin = reinterpret_cast<uintptr_t>(at[r]);
          spans.push_back(Span{begin, begin + t.nbytes(), written[r]});
        }
      }
      table[i] = sdm_rt_tensor{at[kParams], at[kGrads], at[kExpAvgs], at[kExpAvgSqs], numel, code};
    }
    if (leader == kParams && !apart(spans)) {
      PyErr_SetString(PyExc_ValueError, "two of the tensors overlap, and one of them is written");
      return nullptr;
    }
    return Py_BuildValue("(Oi)", bytes, device);
  } catch (const std::exception&) {   // a tensor without storage of its own, or no memory
    Py_RETURN_NONE;
  }
}

// written(list, ...): counts up the versions of tensors that a kernel has written (inference tensors have none)
PyObject* written(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  try {
    for (Py_ssize_t a = 0; a < nargs; ++a) {
      for (Py_ssize_t i = 0; i < PyList_GET_SIZE(args[a]); ++i) {
        const at::Tensor& t = THPVariable_Unpack(PyList_GET_ITEM(args[a], i));
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
      }
    }
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  Py_RETURN_NONE;
}

// new_rows(like, n, k, kinds): uninitialised tensors on the GPU of the tensor `like`, one for each letter of kinds: f float32
// [n], F float32 [n][k], I int64 [n][k]; None for any other.  (Half the time of as many calls from Python: a decode step's token
// waits for them.)
PyObject* new_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4 || !THPVariable_Check(args[0]) || !PyUnicode_Check(args[3])) {
    PyErr_SetString(PyExc_TypeError, "new_rows: a tensor, two numbers and the kinds");
    return nullptr;
  }
  const int64_t n = PyLong_AsLongLong(args[1]), k = PyLong_AsLongLong(args[2]);
  Py_ssize_t count = 0;
  const char* kinds = PyUnicode_AsUTF8AndSize(args[3], &count);
  if (!kinds || PyErr_Occurred()) return nullptr;
  PyObject* out = PyTuple_New(count);
  if (!out) return nullptr;
  try {
    const at::TensorOptions on = THPVariable_Unpack(args[0]).options().requires_grad(false);
    for (Py_ssize_t i = 0; i < count; ++i) {
      PyObject* t;
      if (kinds[i] == 'f') {
        t = THPVariable_Wrap(at::empty({n}, on.dtype(at::kFloat)));
      } else if (kinds[i] == 'F') {
        t = THPVariable_Wrap(at::empty({n, k}, on.dtype(at::kFloat)));
      } else if (kinds[i] == 'I') {
        t = THPVariable_Wrap(at::empty({n, k}, on.dtype(at::kLong)));
      } else {
        t = Py_None;
        Py_INCREF(t);
      }
      if (!t) {
        Py_DECREF(out);
        return nullptr;
      }
      PyTuple_SET_ITEM(out, i, t);
    }
  } catch (const std::exception& e) {   // no memory
    Py_DECREF(out);
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  return out;
}

PyMethodDef methods[] = {
    {"pack", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pack)), METH_FASTCALL,
     "pack(params, grads, exp_avgs, exp_avg_sqs, eight, reading) -> (table, GPU) or None"},
    {"written", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(written)), METH_FASTCALL,
     "written(list of tensors, ...)"},
    {"new_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(new_rows)), METH_FASTCALL,
     "new_rows(like, n, k, kinds) -> tensors"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lists", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__lists() { return PyModule_Create(&module); }
