// What the Python calls of the operators share: tensors as they are seen through the DLPack C exchange interface or their
// attributes, arguments by position or name, streams and status codes.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "../../include/laya_b200.h"

namespace laya_python {

using ErrorFn = const char* (*)(laya_engine*);
using DeviceFn = int (*)(int*);

// ---------------------------------------------------------------------------------------------
// Tensors
// ---------------------------------------------------------------------------------------------

// The parts of the DLPack standard (version 1) that are used: a borrowed view of a tensor, and the table of functions
// that a tensor type offers in the capsule `__dlpack_c_exchange_api__`.
struct DLTensor {
  void* data;
  int32_t device_type, device_id;
  int32_t ndim;
  uint8_t code, bits;
  uint16_t lanes;
  int64_t* shape;
  int64_t* strides;  // elements; null: contiguous
  uint64_t byte_offset;
};
struct DLExchange {
  uint32_t major, minor;
  void* previous;
  void *allocate, *managed_from_object, *managed_to_object;
  int (*tensor_from_object)(void* object, DLTensor* out);  // no reference is kept, nothing is synchronised; may be null
  int (*current_stream)(int32_t device_type, int32_t device_id, void** out);  // may be null
};
enum { kDLCuda = 2, kDLCudaManaged = 13, kDLInt = 0, kDLFloat = 2, kDLBfloat = 4 };

constexpr int kInt32 = 100, kInt64 = 101;  // dtypes beside LAYA_DTYPE_*
constexpr int kMostDims = 8;

struct View {
  void* data;
  int ndim;
  int64_t shape[kMostDims], strides[kMostDims];
  int device;  // index of the CUDA device, -1: not on one
  int dtype;   // LAYA_DTYPE_*, kInt32, kInt64, or -1 for others
  int64_t item, numel;
  bool contiguous;
};

enum Name { DATA_PTR, SHAPE, STRIDE, DTYPE, GET_DEVICE, ELEMENT_SIZE, EXCHANGE, NAMES };
inline PyObject* g_names[NAMES];  // filled when the module is made
constexpr const char* kNames[NAMES] = {"data_ptr", "shape", "stride", "dtype", "get_device", "element_size",
                                       "__dlpack_c_exchange_api__"};

inline bool failed(long long n) { return n == -1 && PyErr_Occurred(); }

// The result of a method without arguments as an integer; -1 with an exception set on failure.
inline long long method(PyObject* o, Name name) {
  PyObject* value = PyObject_CallMethodNoArgs(o, g_names[name]);
  if (!value) return -1;
  const long long n = PyLong_AsLongLong(value);
  Py_DECREF(value);
  return n;
}

// A tuple of integers (taken over) into out; their number, -1 on failure.
inline int integers(PyObject* tuple, int64_t* out) {
  if (!tuple) return -1;
  int n = -1;
  PyObject* items = PySequence_Fast(tuple, "a tensor's shape and stride are sequences");
  Py_DECREF(tuple);
  if (!items) return -1;
  if (PySequence_Fast_GET_SIZE(items) > kMostDims) {
    PyErr_Format(PyExc_ValueError, "a tensor of %zd dimensions", PySequence_Fast_GET_SIZE(items));
  } else {
    n = (int)PySequence_Fast_GET_SIZE(items);
    for (int i = 0; i < n; ++i) {
      out[i] = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(items, i));
      if (failed(out[i])) {
        n = -1;
        break;
      }
    }
  }
  Py_DECREF(items);
  return n;
}

inline void settle(View* v) {
  v->numel = 1;
  v->contiguous = true;
  for (int i = v->ndim - 1; i >= 0; --i) {
    if (v->shape[i] != 1 && v->strides[i] != v->numel) v->contiguous = false;
    v->numel *= v->shape[i];
  }
  if (!v->numel) v->contiguous = true;
}

// The exchange table of a tensor's type (kept as long as its framework is loaded); null where it has none.  Types are
// looked at once (and kept).
inline const DLExchange* exchange_of(PyTypeObject* type) {
  static struct {
    PyTypeObject* type;
    const DLExchange* table;
  } known[16];
  static int count = 0;
  for (int i = 0; i < count; ++i)
    if (known[i].type == type) return known[i].table;
  const DLExchange* table = nullptr;
  PyObject* capsule = PyObject_GetAttr(reinterpret_cast<PyObject*>(type), g_names[EXCHANGE]);
  if (capsule && PyCapsule_IsValid(capsule, "dlpack_exchange_api")) {
    const DLExchange* api = static_cast<const DLExchange*>(PyCapsule_GetPointer(capsule, "dlpack_exchange_api"));
    if (api->major == 1) table = api;
  }
  Py_XDECREF(capsule);
  PyErr_Clear();
  if (count < 16) {
    Py_INCREF(type);
    known[count++] = {type, table};
  }
  return table;
}

// A tensor's attributes; false with an exception set where one is missing or fails.
inline bool view_attributes(PyObject* o, View* v) {
  v->ndim = integers(PyObject_GetAttr(o, g_names[SHAPE]), v->shape);
  if (v->ndim < 0) return false;
  const int n = integers(PyObject_CallMethodNoArgs(o, g_names[STRIDE]), v->strides);
  if (n < 0) return false;
  if (n != v->ndim) {
    PyErr_SetString(PyExc_ValueError, "a tensor's shape and stride differ in length");
    return false;
  }
  v->item = method(o, ELEMENT_SIZE);
  if (failed(v->item)) return false;
  const long long device = method(o, GET_DEVICE);
  if (failed(device)) return false;
  v->device = device < 0 ? -1 : (int)device;
  const long long data = method(o, DATA_PTR);
  if (failed(data)) return false;
  v->data = reinterpret_cast<void*>(data);
  PyObject* d = PyObject_GetAttr(o, g_names[DTYPE]);
  PyObject* s = d ? PyObject_Str(d) : nullptr;
  Py_XDECREF(d);
  const char* text = s ? PyUnicode_AsUTF8(s) : nullptr;
  if (text)
    v->dtype = !strcmp(text, "torch.float32") ? LAYA_DTYPE_F32 : !strcmp(text, "torch.float16") ? LAYA_DTYPE_F16
               : !strcmp(text, "torch.bfloat16") ? LAYA_DTYPE_BF16 : !strcmp(text, "torch.int32") ? kInt32
               : !strcmp(text, "torch.int64") ? kInt64 : -1;
  Py_XDECREF(s);
  if (!text) return false;
  settle(v);
  return true;
}

inline bool view(PyObject* o, View* v) {
  const DLExchange* table = exchange_of(Py_TYPE(o));
  DLTensor t;
  if (!table || !table->tensor_from_object) return view_attributes(o, v);
  // Refused by the type (a tensor that requires a gradient, say): its attributes tell the same.
  if (table->tensor_from_object(o, &t) != 0 || t.ndim > kMostDims || t.lanes != 1 || t.bits % 8) {
    PyErr_Clear();
    return view_attributes(o, v);
  }
  v->data = static_cast<char*>(t.data) + t.byte_offset;
  v->ndim = t.ndim;
  int64_t next = 1;
  for (int i = t.ndim - 1; i >= 0; --i) {
    v->shape[i] = t.shape[i];
    v->strides[i] = t.strides ? t.strides[i] : next;
    next *= t.shape[i];
  }
  v->device = t.device_type == kDLCuda || t.device_type == kDLCudaManaged ? t.device_id : -1;
  v->dtype = t.code == kDLFloat && t.bits == 32 ? LAYA_DTYPE_F32 : t.code == kDLFloat && t.bits == 16 ? LAYA_DTYPE_F16
             : t.code == kDLBfloat && t.bits == 16 ? LAYA_DTYPE_BF16 : t.code == kDLInt && t.bits == 32 ? kInt32
             : t.code == kDLInt && t.bits == 64 ? kInt64 : -1;
  v->item = t.bits / 8;
  settle(v);
  return true;
}

// Raises ValueError with a tensor's shape at the end.
inline void refuse_shape(const char* what, const View& v, const char* format, long long rows, long long cols) {
  char shape[128] = "(", wanted[160];
  size_t at = 1;
  for (int i = 0; i < v.ndim && at < 100; ++i)
    at += (size_t)snprintf(shape + at, sizeof shape - at, i ? ", %lld" : "%lld", (long long)v.shape[i]);
  snprintf(shape + at, sizeof shape - at, v.ndim == 1 ? ",)" : ")");
  snprintf(wanted, sizeof wanted, format, rows, cols);
  PyErr_Format(PyExc_ValueError, "%s %s, got %s", what, wanted, shape);
}

// ---------------------------------------------------------------------------------------------
// Arguments: positional or by name, `required` of them at least; the others keep what `out` holds.
// ---------------------------------------------------------------------------------------------
template <size_t N>
struct Signature {
  const char* function;
  const char* names[N];
  PyObject* keys[N];  // the names interned, as call sites hold them
};

template <size_t N>
bool parse(Signature<N>& sig, size_t required, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames, PyObject* (&out)[N]) {
  if (nargs > (Py_ssize_t)N) {
    PyErr_Format(PyExc_TypeError, "%s() takes at most %zu arguments (%zd given)", sig.function, N, nargs);
    return false;
  }
  for (Py_ssize_t i = 0; i < nargs; ++i) out[i] = args[i];
  const Py_ssize_t nkw = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
  for (size_t i = 0; nkw && i < N; ++i)
    if (!sig.keys[i] && !(sig.keys[i] = PyUnicode_InternFromString(sig.names[i]))) return false;
  for (Py_ssize_t k = 0; k < nkw; ++k) {
    PyObject* key = PyTuple_GET_ITEM(kwnames, k);
    size_t at = 0;
    while (at < N && key != sig.keys[at]) ++at;
    if (at == N)
      for (at = 0; at < N && PyUnicode_CompareWithASCIIString(key, sig.names[at]) != 0;) ++at;
    if (at == N) {
      PyErr_Format(PyExc_TypeError, "%s() got an unexpected keyword argument '%U'", sig.function, key);
      return false;
    }
    if ((Py_ssize_t)at < nargs) {
      PyErr_Format(PyExc_TypeError, "%s() got multiple values for argument '%s'", sig.function, sig.names[at]);
      return false;
    }
    out[at] = args[nargs + k];
  }
  for (size_t i = 0; i < required; ++i)
    if (!out[i]) {
      PyErr_Format(PyExc_TypeError, "%s() missing required argument '%s'", sig.function, sig.names[i]);
      return false;
    }
  return true;
}

inline bool to_int(PyObject* o, const char* what, int* out) {
  const long long n = PyLong_AsLongLong(o);
  if (failed(n)) return false;
  if (n < -2147483647 || n > 2147483647) {
    PyErr_Format(PyExc_ValueError, "%s = %lld is out of range", what, n);
    return false;
  }
  *out = (int)n;
  return true;
}

// A stream given as an integer; without one, the stream on which the framework of `tensor` works on `device` now, or, where
// its type does not tell, the legacy default stream.
inline bool to_stream(PyObject* o, PyObject* tensor, int device, void** out) {
  *out = nullptr;
  if (!o || o == Py_None) {
    const DLExchange* table = exchange_of(Py_TYPE(tensor));
    if (!table || !table->current_stream || table->current_stream(kDLCuda, device, out) == 0) return true;
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "no current stream on CUDA device %d", device);
    return false;
  }
  const unsigned long long n = PyLong_AsUnsignedLongLong(o);
  if (n == (unsigned long long)-1 && PyErr_Occurred()) return false;
  *out = reinterpret_cast<void*>(n);
  return true;
}

// ---------------------------------------------------------------------------------------------
// Tensors and statuses of the calls
// ---------------------------------------------------------------------------------------------
// `n` contiguous float32 values on `device`; null where `t` is absent or None.
inline bool take_vector(const char* name, PyObject* t, int n, int device, const float** out) {
  *out = nullptr;
  if (!t || t == Py_None) return true;
  View v;
  if (!view(t, &v)) return false;
  if (v.ndim != 1 || v.shape[0] != n || v.dtype != LAYA_DTYPE_F32 || !v.contiguous || v.device != device) {
    PyErr_Format(PyExc_ValueError, "%s must be %d contiguous float32 values on CUDA device %d", name, n, device);
    return false;
  }
  *out = static_cast<const float*>(v.data);
  return true;
}

// Refuses buffers on another device than the one that the call would launch on.  (Without a current device the
// library's call says what is wrong.)
inline bool on_current_device(const char* what, int device, DeviceFn current_device) {
  int current;
  if (current_device(&current) == LAYA_OK && current != device) {
    PyErr_Format(PyExc_ValueError, "%s on CUDA device %d, the current device is %d", what, device, current);
    return false;
  }
  return true;
}

// ValueError for refused arguments, RuntimeError for the rest, with the library's message.
inline PyObject* finish(int status, ErrorFn last_error) {
  if (status == LAYA_OK) Py_RETURN_NONE;
  const char* text = last_error(nullptr);
  PyErr_SetString(status == LAYA_ERR_INVALID ? PyExc_ValueError : PyExc_RuntimeError, text ? text : "");
  return nullptr;
}

}  // namespace laya_python
