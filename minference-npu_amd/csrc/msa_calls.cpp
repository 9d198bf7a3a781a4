// The cache operators' calls from Python in one step: descriptors of the
// tensors, outputs, workspace, device and stream, then the C ABI (include/msa.h).
// A CPython module, bound to the loaded libmsa by the addresses of its functions.
//
// Through ctypes a call of two launches costs 21 to 27 us of host time, of which
// the launches are 7; many calls of these operators (a token of a few sequences)
// take the GPU less than that.  Through this module it is 12 to 15 us.
//
// Nothing here decides what is valid: the library does.  A function returns its
// outputs, or the library's status (an int) when nothing was launched or the
// launch failed, or None for tensors it has no descriptor for; the Python side
// then explains or falls back to copies the library takes.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>

#include "../../include/msa.h"

namespace {

struct Library {
  decltype(&msa_shared_prefix_workspace_bytes) prefix_ws;
  decltype(&msa_shared_prefix_attention) prefix;
  decltype(&msa_decode_accumulate_workspace_bytes) accumulate_ws;
  decltype(&msa_decode_accumulate) accumulate;
  decltype(&msa_attention_weight_sums_workspace_bytes) sums_ws;
  decltype(&msa_attention_weight_sums) sums;
  decltype(&msa_cache_evict_workspace_bytes) evict_ws;
  decltype(&msa_cache_evict) evict;
} lib;

// bind(addresses of the functions above, in order)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* p[8];
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "bind takes 8 addresses");
    return nullptr;
  }
  for (int i = 0; i < 8; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  lib.prefix_ws = reinterpret_cast<decltype(lib.prefix_ws)>(p[0]);
  lib.prefix = reinterpret_cast<decltype(lib.prefix)>(p[1]);
  lib.accumulate_ws = reinterpret_cast<decltype(lib.accumulate_ws)>(p[2]);
  lib.accumulate = reinterpret_cast<decltype(lib.accumulate)>(p[3]);
  lib.sums_ws = reinterpret_cast<decltype(lib.sums_ws)>(p[4]);
  lib.sums = reinterpret_cast<decltype(lib.sums)>(p[5]);
  lib.evict_ws = reinterpret_cast<decltype(lib.evict_ws)>(p[6]);
  lib.evict = reinterpret_cast<decltype(lib.evict)>(p[7]);
  Py_RETURN_NONE;
}

const at::Tensor* tensor(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}

// [B, H, S, D], or [B, H, S] as [B, H, S, 1], on GPU `device`.
bool describe(const at::Tensor* t, c10::DeviceIndex device, msa_tensor4& d) {
  if (!t || !t->is_cuda() || t->get_device() != device || t->layout() != at::kStrided) return false;
  const auto size = t->sizes(), stride = t->strides();
  if (size.size() != 3 && size.size() != 4) return false;
  switch (t->scalar_type()) {
    case at::kBFloat16: d.dtype = MSA_DTYPE_BF16; break;
    case at::kHalf: d.dtype = MSA_DTYPE_FP16; break;
    case at::kFloat: d.dtype = MSA_DTYPE_FP32; break;
    default: return false;
  }
  d.size[3] = d.stride[3] = 1;
  for (size_t i = 0; i < size.size(); ++i) {
    d.size[i] = size[i];
    d.stride[i] = stride[i];
  }
  d.data = t->data_ptr();
  d.reserved = 0;
  return true;
}

// lens: None or int32 [batch], contiguous, on the device.
bool lens_of(PyObject* o, int64_t batch, c10::DeviceIndex device, const int32_t*& p) {
  p = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (!t || !t->is_cuda() || t->get_device() != device || t->scalar_type() != at::kInt ||
      t->dim() != 1 || t->size(0) != batch || !t->is_contiguous())
    return false;
  p = static_cast<const int32_t*>(t->data_ptr());
  return true;
}

// The device of a call is current while it lasts.
struct Call {
  c10::Device device;
  c10::DeviceGuard guard;
  at::Tensor workspace;
  explicit Call(const at::Tensor& t) : device(t.device()), guard(device) {}
  msa_stream_t stream() const {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream();
  }
  at::Tensor empty(at::IntArrayRef size, at::ScalarType type) const {
    return at::empty(size, at::TensorOptions().device(device).dtype(type));
  }
  void* room(size_t bytes) {
    if (bytes == 0) return nullptr;
    workspace = empty({int64_t(bytes)}, at::kByte);
    return workspace.data_ptr();
  }
};

PyObject* status(int st) { return PyLong_FromLong(st); }

// shared_prefix(q, k_prefix, v_prefix, k, v, out or None, lens or None, scale)
PyObject* shared_prefix(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* q = n == 8 ? tensor(a[0]) : nullptr;
  if (!q || !q->is_cuda() || q->dim() != 4 || q->numel() == 0) Py_RETURN_NONE;
  const auto dev = q->get_device();
  msa_tensor4 d[6];
  for (int i = 0; i < 5; ++i)
    if (!describe(tensor(a[i]), dev, d[i])) Py_RETURN_NONE;
  const int32_t* lens;
  if (!lens_of(a[6], q->size(0), dev, lens)) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[7]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  Call call(*q);
  const at::Tensor out = a[5] == Py_None ? call.empty(q->sizes(), q->scalar_type())
                                         : THPVariable_Check(a[5]) ? THPVariable_Unpack(a[5]) : at::Tensor();
  if (!out.defined() || !describe(&out, dev, d[5])) Py_RETURN_NONE;
  const size_t bytes = lib.prefix_ws(&d[0], &d[1], &d[2], &d[3], &d[4]);
  const int st = lib.prefix(&d[0], &d[1], &d[2], &d[3], &d[4], &d[5], lens, float(scale),
                            call.room(bytes), bytes, call.stream());
  return st == MSA_OK ? THPVariable_Wrap(out) : status(st);
  END_HANDLE_TH_ERRORS
}

// decode_accumulate(q, k, v, out or None, lens or None, scores, scores_out, scale)
PyObject* decode_accumulate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* q = n == 8 ? tensor(a[0]) : nullptr;
  if (!q || !q->is_cuda() || q->dim() != 4 || q->numel() == 0) Py_RETURN_NONE;
  const auto dev = q->get_device();
  msa_tensor4 d[6];
  const int at_arg[5] = {0, 1, 2, 5, 6};
  for (int i = 0; i < 5; ++i)
    if (!describe(tensor(a[at_arg[i]]), dev, d[i])) Py_RETURN_NONE;
  const int32_t* lens;
  if (!lens_of(a[4], q->size(0), dev, lens)) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[7]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  Call call(*q);
  const at::Tensor out = a[3] == Py_None ? call.empty(q->sizes(), q->scalar_type())
                                         : THPVariable_Check(a[3]) ? THPVariable_Unpack(a[3]) : at::Tensor();
  if (!out.defined() || !describe(&out, dev, d[5])) Py_RETURN_NONE;
  const size_t bytes = lib.accumulate_ws(&d[0], &d[1], &d[2]);
  const int st = lib.accumulate(&d[0], &d[1], &d[2], &d[5], lens, &d[3], &d[4], float(scale),
                                call.room(bytes), bytes, call.stream());
  return st == MSA_OK ? THPVariable_Wrap(out) : status(st);
  END_HANDLE_TH_ERRORS
}

// weight_sums(q, k, sums or None, scale): sums given are added to
PyObject* weight_sums(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* q = n == 4 ? tensor(a[0]) : nullptr;
  const at::Tensor* k = n == 4 ? tensor(a[1]) : nullptr;
  if (!q || !k || !q->is_cuda() || q->dim() != 4 || k->dim() != 4 || q->numel() == 0) Py_RETURN_NONE;
  const auto dev = q->get_device();
  msa_tensor4 d[3];
  if (!describe(q, dev, d[0]) || !describe(k, dev, d[1])) Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(a[3]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  Call call(*q);
  const bool add = a[2] != Py_None;
  const at::Tensor sums = add ? THPVariable_Check(a[2]) ? THPVariable_Unpack(a[2]) : at::Tensor()
                              : call.empty(k->sizes().slice(0, 3), at::kFloat);
  if (!sums.defined() || !describe(&sums, dev, d[2])) Py_RETURN_NONE;
  const size_t bytes = lib.sums_ws(&d[0], &d[1]);
  const int st = lib.sums(&d[0], &d[1], &d[2], add, float(scale), call.room(bytes), bytes, call.stream());
  return st == MSA_OK ? THPVariable_Wrap(sums) : status(st);
  END_HANDLE_TH_ERRORS
}

// evict(k, v, scores, lens or None, keep, recent, sinks, k_out, v_out, scores_out or three times None)
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* k = n == 10 ? tensor(a[0]) : nullptr;
  if (!k || !k->is_cuda() || k->dim() != 4 || k->numel() == 0) Py_RETURN_NONE;
  const auto dev = k->get_device();
  msa_tensor4 d[6];
  for (int i = 0; i < 3; ++i)
    if (!describe(tensor(a[i]), dev, d[i])) Py_RETURN_NONE;
  const int32_t* lens;
  if (!lens_of(a[3], k->size(0), dev, lens)) Py_RETURN_NONE;
  long long count[3];
  for (int i = 0; i < 3; ++i) {
    count[i] = PyLong_AsLongLong(a[4 + i]);
    if (count[i] == -1 && PyErr_Occurred()) return nullptr;
  }
  const int64_t keep = count[0];
  if (keep < 1 || keep > k->size(2)) return status(MSA_E_TOPK);
  Call call(*k);
  const int64_t B = k->size(0), H = k->size(1);
  at::Tensor out[3];
  for (int i = 0; i < 3; ++i) {
    if (a[7 + i] == Py_None)
      out[i] = i < 2 ? call.empty({B, H, keep, k->size(3)}, k->scalar_type())
                     : call.empty({B, H, keep}, at::kFloat);
    else if (THPVariable_Check(a[7 + i]))
      out[i] = THPVariable_Unpack(a[7 + i]);
    if (!out[i].defined() || !describe(&out[i], dev, d[3 + i])) Py_RETURN_NONE;
  }
  const at::Tensor pos = call.empty({B, H, keep}, at::kInt), new_lens = call.empty({B}, at::kInt);
  const size_t bytes = lib.evict_ws(B, H, k->size(2));
  const int st = lib.evict(&d[0], &d[1], &d[2], lens, keep, count[1], count[2], &d[3], &d[4], &d[5],
                           static_cast<int32_t*>(pos.data_ptr()),
                           static_cast<int32_t*>(new_lens.data_ptr()), call.room(bytes), bytes,
                           call.stream());
  if (st != MSA_OK) return status(st);
  const at::Tensor* all[5] = {&out[0], &out[1], &out[2], &pos, &new_lens};
  PyObject* r = PyTuple_New(5);
  if (!r) return nullptr;
  for (int i = 0; i < 5; ++i) {
    PyObject* o = THPVariable_Wrap(*all[i]);
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i, o);
  }
  return r;
  END_HANDLE_TH_ERRORS
}

#define MSA_CALL(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MSA_CALL(bind),        MSA_CALL(shared_prefix), MSA_CALL(decode_accumulate),
                         MSA_CALL(weight_sums), MSA_CALL(evict),         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_msa_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__msa_calls() { return PyModule_Create(&module); }
