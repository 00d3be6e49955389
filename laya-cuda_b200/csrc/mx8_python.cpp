// laya_cuda._mx8: the Python calls of the MX8 operators as a CPython extension.
//
// A single token's call spends its time on the host: through ctypes a linear layer's arguments took 4-6 us to
// check and convert beside the 2.1 us of the kernel's launch, and the device waited.  Here a tensor is looked
// at through the DLPack C exchange interface of its type (one call, no Python objects), or, where its type has
// none, through the attributes of torch's tensors: `data_ptr`, `shape`, `stride`, `dtype`, `element_size` and
// `get_device`.  torch is not linked or imported.  The library's functions come by address from
// laya_cuda._lib (`bind`), which loads it on the first call.
#include "python_tensors.h"

#include <structmember.h>

#include <cstddef>

// The calls of laya_cuda.attention, in the same extension (attention_python.cpp).
PyMethodDef* attention_methods();

namespace {

using namespace laya_python;

using ConvertFn = int (*)(const laya_mx8_convert*, void*);
using NormFn = int (*)(const laya_rms_norm_mx8*, void*);
using LinearFn = int (*)(const laya_mx8_linear*, int*, void*);

struct Library {
  ConvertFn quantize, dequantize;
  NormFn rms_norm;
  LinearFn linear;
  ErrorFn last_error;
  DeviceFn current_device;
} g_lib = {};
PyObject* g_loader = nullptr;  // called before the first operator: it calls bind()

long long scale_bytes(long long rows, long long cols) { return (rows + 127) / 128 * ((cols + 127) / 128) * 512; }

// ---------------------------------------------------------------------------------------------
// Matrix
// ---------------------------------------------------------------------------------------------
struct Matrix {
  PyObject_HEAD
  PyObject* values;
  PyObject* scales;
  int rows, cols;
};

// Where a matrix's buffers are.  Looked at anew by each call (0.1 us): a tensor's storage can be moved or resized
// after a Matrix of it was made.
struct Operand {
  void *values, *scales;
  long long ld;  // bytes from one row of values to the next
  int device;
};

PyTypeObject MatrixType = {PyVarObject_HEAD_INIT(nullptr, 0)};

bool look(PyObject* values, PyObject* scales, int rows, int cols, Operand* m) {
  if (rows < 0 || cols < 1) {
    PyErr_Format(PyExc_ValueError, "bad shape %d x %d: rows may be 0, columns may not", rows, cols);
    return false;
  }
  const long long room = ((long long)cols + 15) / 16 * 16, need = scale_bytes(rows, cols);
  View v, s;
  if (!view(values, &v) || !view(scales, &s)) return false;
  m->ld = room;
  if (!v.contiguous || v.numel * v.item != rows * room) {
    // Rows further apart than they need to be, of one-byte elements.
    if (v.ndim != 2 || v.shape[0] != rows || v.shape[1] < room || v.strides[1] != 1 || v.item != 1) {
      refuse_shape("values", v, "of a %lld x %lld matrix must be bytes in as many contiguous rows, with room for a multiple of 16", rows, cols);
      return false;
    }
    if (rows > 1) m->ld = v.strides[0];  // the stride of a single row says nothing
  }
  if (!s.contiguous || s.numel * s.item < need) {
    PyErr_Format(PyExc_ValueError, "scales of a %d x %d matrix need %lld contiguous bytes", rows, cols, need);
    return false;
  }
  if (v.device < 0 || s.device != v.device) {
    PyErr_SetString(PyExc_ValueError, "values and scales must be on the same CUDA device");
    return false;
  }
  m->device = v.device;
  m->values = v.data;
  m->scales = s.data;
  return true;
}
bool look(const Matrix* m, Operand* out) { return look(m->values, m->scales, m->rows, m->cols, out); }

PyObject* matrix_make(PyTypeObject* type, PyObject* (&given)[4]) {
  int rows, cols;
  if (!to_int(given[2], "rows", &rows) || !to_int(given[3], "cols", &cols)) return nullptr;
  Operand checked;
  if (!look(given[0], given[1], rows, cols, &checked)) return nullptr;
  Matrix* m = reinterpret_cast<Matrix*>(type->tp_alloc(type, 0));
  if (!m) return nullptr;
  Py_INCREF(given[0]);
  Py_INCREF(given[1]);
  m->values = given[0];
  m->scales = given[1];
  m->rows = rows;
  m->cols = cols;
  return reinterpret_cast<PyObject*>(m);
}

Signature<4> g_matrix_args = {"Matrix", {"values", "scales", "rows", "cols"}, {}};

PyObject* matrix_call(PyObject* type, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
  PyObject* given[4] = {};
  if (!parse(g_matrix_args, 4, args, PyVectorcall_NARGS(nargsf), kwnames, given)) return nullptr;
  return matrix_make(reinterpret_cast<PyTypeObject*>(type), given);
}

void matrix_dealloc(PyObject* self) {
  Matrix* m = reinterpret_cast<Matrix*>(self);
  Py_XDECREF(m->values);
  Py_XDECREF(m->scales);
  Py_TYPE(self)->tp_free(self);
}

PyObject* matrix_empty(PyObject* type, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  static Signature<3> sig = {"empty", {"like", "rows", "cols"}, {}};
  PyObject* given[3] = {};
  int rows, cols;
  if (!parse(sig, 3, args, nargs, kwnames, given) || !to_int(given[1], "rows", &rows) || !to_int(given[2], "cols", &cols))
    return nullptr;
  if (rows < 0 || cols < 1) {
    PyErr_Format(PyExc_ValueError, "bad shape %d x %d: rows may be 0, columns may not", rows, cols);
    return nullptr;
  }
  // like.new_zeros(n, dtype=torch.uint8).  `like` is torch's, so torch has been imported.
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* uint8 = torch ? PyObject_GetAttrString(torch, "uint8") : nullptr;
  PyObject* dtype = uint8 ? Py_BuildValue("{s:O}", "dtype", uint8) : nullptr;
  Py_XDECREF(torch);
  Py_XDECREF(uint8);
  if (!dtype) return nullptr;
  auto bytes = [&](long long n) -> PyObject* {
    PyObject* method = PyObject_GetAttrString(given[0], "new_zeros");
    PyObject* args = method ? Py_BuildValue("(L)", n) : nullptr;
    PyObject* made = args ? PyObject_Call(method, args, dtype) : nullptr;
    Py_XDECREF(method);
    Py_XDECREF(args);
    return made;
  };
  const long long room = ((long long)cols + 15) / 16 * 16;
  PyObject* flat = bytes(rows * room);
  PyObject* values = flat ? PyObject_CallMethod(flat, "view", "LL", (long long)rows, room) : nullptr;
  PyObject* scales = values ? bytes(scale_bytes(rows, cols)) : nullptr;
  PyObject* made = nullptr;
  if (scales) {
    PyObject* parts[4] = {values, scales, given[1], given[2]};
    made = matrix_make(reinterpret_cast<PyTypeObject*>(type), parts);
  }
  Py_DECREF(dtype);
  Py_XDECREF(flat);
  Py_XDECREF(values);
  Py_XDECREF(scales);
  return made;
}

PyMemberDef matrix_members[] = {
    {"values", T_OBJECT_EX, offsetof(Matrix, values), READONLY, nullptr},
    {"scales", T_OBJECT_EX, offsetof(Matrix, scales), READONLY, nullptr},
    {"rows", T_INT, offsetof(Matrix, rows), READONLY, nullptr},
    {"cols", T_INT, offsetof(Matrix, cols), READONLY, nullptr},
    {nullptr, 0, 0, 0, nullptr}};

PyObject* matrix_ld(PyObject* self, void*) {
  Operand m;
  return look(reinterpret_cast<Matrix*>(self), &m) ? PyLong_FromLongLong(m.ld) : nullptr;
}
PyObject* matrix_device(PyObject* self, void*) {
  Operand m;
  return look(reinterpret_cast<Matrix*>(self), &m) ? PyLong_FromLong(m.device) : nullptr;
}
PyGetSetDef matrix_getset[] = {{"ld", matrix_ld, nullptr, "bytes from one row of values to the next", nullptr},
                               {"device", matrix_device, nullptr, "index of the CUDA device", nullptr},
                               {nullptr, nullptr, nullptr, nullptr, nullptr}};

PyMethodDef matrix_methods[] = {
    {"empty", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(matrix_empty)), METH_FASTCALL | METH_KEYWORDS | METH_CLASS,
     "empty(like, rows, cols)\n--\n\nBuffers for a matrix on the device of the torch tensor `like` (uint8, cleared)."},
    {nullptr, nullptr, 0, nullptr}};

// ---------------------------------------------------------------------------------------------
// Tensors beside a matrix
// ---------------------------------------------------------------------------------------------
struct Rows {
  void* ptr;
  long long ld;
  int dtype;
};

// A [rows][cols] tensor of 16- or 32-bit floats with contiguous rows, on `device`.
bool take_rows(const char* name, PyObject* t, int rows, int cols, int device, Rows* out) {
  View v;
  if (!view(t, &v)) return false;
  if (v.ndim != 2 || v.shape[0] != rows || v.shape[1] != cols) {
    refuse_shape(name, v, "must be [%lld][%lld]", rows, cols);
    return false;
  }
  if (cols > 1 && v.strides[1] != 1 && !v.contiguous) {
    PyErr_Format(PyExc_ValueError, "%s: the values of a row must be contiguous", name);
    return false;
  }
  if (v.dtype < 0 || v.dtype >= kInt32) {
    PyErr_Format(PyExc_ValueError, "%s is not float32, float16 or bfloat16", name);
    return false;
  }
  if (v.device != device) {
    PyErr_Format(PyExc_ValueError, "%s is not on CUDA device %d, where the matrix is", name, device);
    return false;
  }
  out->ptr = v.data;
  out->ld = rows > 1 && !v.contiguous ? v.strides[0] : cols;
  out->dtype = v.dtype;
  return true;
}

// A Matrix and where its buffers are now; null with an exception set where it is none or they no longer hold it.
const Matrix* take_matrix(const char* name, PyObject* o, Operand* at) {
  if (Py_TYPE(o) != &MatrixType) {
    PyErr_Format(PyExc_TypeError, "%s must be a Matrix, not %s", name, Py_TYPE(o)->tp_name);
    return nullptr;
  }
  const Matrix* m = reinterpret_cast<const Matrix*>(o);
  return look(m, at) ? m : nullptr;
}

bool ready() {
  if (g_lib.linear) return true;
  if (!g_loader) {
    PyErr_SetString(PyExc_RuntimeError, "laya_cuda._mx8 is used through laya_cuda.mx8");
    return false;
  }
  PyObject* r = PyObject_CallNoArgs(g_loader);
  Py_XDECREF(r);
  if (r && !g_lib.linear) PyErr_SetString(PyExc_RuntimeError, "the library was not bound");
  return r && g_lib.linear;
}

// Binds the library, and refuses buffers on another device than the one that the call would launch on; without rows the
// call needs none.
bool ready_on(int device, int rows) {
  return ready() && (!rows || on_current_device("the matrix is", device, g_lib.current_device));
}

// ---------------------------------------------------------------------------------------------
// Operators
// ---------------------------------------------------------------------------------------------
PyObject* convert(const char* tensor, const char* matrix, PyObject* o, PyObject* t, PyObject* stream, ConvertFn Library::*call) {
  Operand at;
  const Matrix* m = take_matrix(matrix, o, &at);
  if (!m) return nullptr;
  Rows data;
  void* st;
  if (!take_rows(tensor, t, m->rows, m->cols, at.device, &data) || !to_stream(stream, m->values, at.device, &st) || !ready_on(at.device, m->rows)) return nullptr;
  laya_mx8_convert a{};
  a.rows = m->rows; a.cols = m->cols; a.dtype = data.dtype;
  a.values = at.values; a.scales = at.scales; a.ldv = at.ld;
  a.data = data.ptr; a.ld = data.ld;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = (g_lib.*call)(&a, st);
  Py_END_ALLOW_THREADS
  return finish(status, g_lib.last_error);
}

Signature<3> g_quantize_args = {"quantize", {"x", "out", "stream"}, {}};
Signature<3> g_dequantize_args = {"dequantize", {"x", "out", "stream"}, {}};

PyObject* quantize(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  PyObject* g[3] = {};
  if (!parse(g_quantize_args, 2, args, nargs, kwnames, g)) return nullptr;
  return convert("x", "out", g[1], g[0], g[2], &Library::quantize);
}

PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  PyObject* g[3] = {};
  if (!parse(g_dequantize_args, 2, args, nargs, kwnames, g)) return nullptr;
  return convert("out", "x", g[0], g[1], g[2], &Library::dequantize);
}

PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  static Signature<7> sig = {"rms_norm", {"x", "weight", "out", "residual", "sum_out", "eps", "stream"}, {}};
  PyObject* g[7] = {};
  if (!parse(sig, 3, args, nargs, kwnames, g)) return nullptr;
  Operand at;
  const Matrix* m = take_matrix("out", g[2], &at);
  if (!m) return nullptr;
  laya_rms_norm_mx8 a{};
  Rows x, r = {}, s = {};
  void* st;
  if (!take_rows("x", g[0], m->rows, m->cols, at.device, &x)) return nullptr;
  a.residual_dtype = x.dtype;
  const bool residual = g[3] && g[3] != Py_None, sum = g[4] && g[4] != Py_None;
  if (residual) {
    if (!take_rows("residual", g[3], m->rows, m->cols, at.device, &r)) return nullptr;
    a.residual_dtype = r.dtype;
  }
  if (sum) {
    if (!take_rows("sum_out", g[4], m->rows, m->cols, at.device, &s)) return nullptr;
    if (residual && s.dtype != r.dtype) {
      PyErr_SetString(PyExc_ValueError, "sum_out must have the residual's type");
      return nullptr;
    }
    a.residual_dtype = s.dtype;
  }
  if (g[1] == Py_None) {
    PyErr_SetString(PyExc_ValueError, "weight must be a tensor");
    return nullptr;
  }
  if (!take_vector("weight", g[1], m->cols, at.device, &a.weight)) return nullptr;
  a.eps = 1e-6f;
  if (g[5]) {
    const double eps = PyFloat_AsDouble(g[5]);
    if (eps == -1.0 && PyErr_Occurred()) return nullptr;
    a.eps = (float)eps;
  }
  if (!to_stream(g[6], m->values, at.device, &st) || !ready_on(at.device, m->rows)) return nullptr;
  a.rows = m->rows; a.cols = m->cols; a.dtype = x.dtype;
  a.x = x.ptr; a.ldx = x.ld; a.residual = r.ptr; a.ldr = r.ld; a.sum_out = s.ptr; a.lds = s.ld;
  a.values = at.values; a.scales = at.scales; a.ldv = at.ld;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_lib.rms_norm(&a, st);
  Py_END_ALLOW_THREADS
  return finish(status, g_lib.last_error);
}

// LAYA_ACT_* of a name; -1 with an exception set for others.
int activation(PyObject* o) {
  if (!o) return LAYA_ACT_NONE;
  if (PyUnicode_Check(o)) {
    static constexpr const char* kActs[] = {"none", "relu", "gelu", "silu"};
    for (int i = 0; i < 4; ++i)
      if (PyUnicode_CompareWithASCIIString(o, kActs[i]) == 0) return i;
  }
  PyErr_Format(PyExc_ValueError, "activation %R is not one of none, relu, gelu, silu", o);
  return -1;
}

PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  static Signature<10> sig = {"linear", {"x", "w", "out", "bias", "gate", "gate_bias", "activation", "residual", "err", "stream"}, {}};
  PyObject* g[10] = {};
  if (!parse(sig, 3, args, nargs, kwnames, g)) return nullptr;
  Operand x_at, w_at;
  const Matrix *x = take_matrix("x", g[0], &x_at), *w = x ? take_matrix("w", g[1], &w_at) : nullptr;
  if (!w) return nullptr;
  const int rows = x->rows, cols = x->cols, n = w->rows, device = x_at.device;
  if (w->cols != cols || w_at.device != device) {
    PyErr_Format(PyExc_ValueError, "w is %d x %d on device %d, x has %d columns on device %d", n, w->cols, w_at.device, cols, device);
    return nullptr;
  }
  laya_mx8_linear a{};
  a.rows = rows; a.features = n; a.cols = cols;
  a.activation = activation(g[6]);
  if (a.activation < 0) return nullptr;
  a.x = x_at.values; a.x_scales = x_at.scales; a.ldx = x_at.ld;
  a.w = w_at.values; a.w_scales = w_at.scales; a.ldw = w_at.ld;
  if (g[4] && g[4] != Py_None) {
    Operand at;
    const Matrix* gate = take_matrix("gate", g[4], &at);
    if (!gate) return nullptr;
    if (gate->rows != n || gate->cols != cols || at.device != device) {
      PyErr_Format(PyExc_ValueError, "gate is %d x %d, w %d x %d", gate->rows, gate->cols, n, cols);
      return nullptr;
    }
    a.gate = at.values; a.gate_scales = at.scales; a.ldg = at.ld;
  }
  if (!take_vector("bias", g[3], n, device, &a.bias) || !take_vector("gate_bias", g[5], n, device, &a.gate_bias)) return nullptr;
  Rows t;
  if (g[7] && g[7] != Py_None) {
    if (!take_rows("residual", g[7], rows, n, device, &t)) return nullptr;
    a.residual = t.ptr; a.ldr = t.ld; a.residual_dtype = t.dtype;
  }
  if (Py_TYPE(g[2]) == &MatrixType) {
    Operand at;
    const Matrix* out = take_matrix("out", g[2], &at);
    if (!out) return nullptr;
    if (out->rows != rows || out->cols != n || at.device != device) {
      PyErr_Format(PyExc_ValueError, "out is %d x %d, the result %d x %d", out->rows, out->cols, rows, n);
      return nullptr;
    }
    a.out = at.values; a.out_scales = at.scales; a.ldo = at.ld;
    a.out_dtype = LAYA_DTYPE_MX8;
  } else {
    if (!take_rows("out", g[2], rows, n, device, &t)) return nullptr;
    a.out = t.ptr; a.ldo = t.ld; a.out_dtype = t.dtype;
  }
  int* err = nullptr;
  if (g[8] && g[8] != Py_None) {
    View v;
    if (!view(g[8], &v)) return nullptr;
    if (v.dtype != kInt32 || v.device != device || v.numel < 1) {
      PyErr_Format(PyExc_ValueError, "err must be int32 on CUDA device %d", device);
      return nullptr;
    }
    err = static_cast<int*>(v.data);
  }
  void* st;
  if (!to_stream(g[9], x->values, device, &st) || !ready_on(device, rows)) return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_lib.linear(&a, err, st);
  Py_END_ALLOW_THREADS
  return finish(status, g_lib.last_error);
}

PyObject* py_scale_bytes(PyObject*, PyObject* args) {
  int rows, cols;
  if (!PyArg_ParseTuple(args, "ii", &rows, &cols)) return nullptr;
  if (rows < 0 || cols < 1) {
    PyErr_Format(PyExc_ValueError, "bad shape %d x %d: rows may be 0, columns may not", rows, cols);
    return nullptr;
  }
  return PyLong_FromLongLong(scale_bytes(rows, cols));
}

PyObject* set_loader(PyObject*, PyObject* loader) {
  Py_INCREF(loader);
  Py_XSETREF(g_loader, loader);
  Py_RETURN_NONE;
}

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long q, d, n, l, e, c;
  if (!PyArg_ParseTuple(args, "KKKKKK", &q, &d, &n, &l, &e, &c)) return nullptr;
  g_lib = {reinterpret_cast<ConvertFn>(q), reinterpret_cast<ConvertFn>(d), reinterpret_cast<NormFn>(n),
           reinterpret_cast<LinearFn>(l), reinterpret_cast<ErrorFn>(e), reinterpret_cast<DeviceFn>(c)};
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL | METH_KEYWORDS
PyMethodDef methods[] = {
    {"quantize", FAST(quantize), "quantize(x, out, stream=None)\n--\n\nx [rows][cols] in 16 or 32 bits -> the Matrix `out`."},
    {"dequantize", FAST(dequantize), "dequantize(x, out, stream=None)\n--\n\nThe Matrix `x` -> out [rows][cols] in 16 or 32 bits."},
    {"rms_norm", FAST(rms_norm),
     "rms_norm(x, weight, out, residual=None, sum_out=None, eps=1e-6, stream=None)\n--\n\n"
     "h = x + residual; sum_out = h; out = h / sqrt(mean(h^2) + eps) * weight, in MX8.\n\n"
     "`residual` and `sum_out` are optional, of one type, and may be the same tensor."},
    {"linear", FAST(linear),
     "linear(x, w, out, bias=None, gate=None, gate_bias=None, activation='none', residual=None, err=None, stream=None)\n--\n\n"
     "out = act(x w^T + bias) + residual, or, with a `gate` matrix,\n"
     "out = act(x gate^T + gate_bias) * (x w^T + bias) + residual.\n\n"
     "x: Matrix [rows][cols]; w, gate: Matrix [features][cols]; out: a Matrix or a tensor\n"
     "[rows][features].  bias, gate_bias: float32 [features].  residual: [rows][features] in 16 or 32\n"
     "bits, added before the one rounding; it may be `out` itself.  activation: 'none', 'relu', 'gelu' (erf)\n"
     "or 'silu'.  err: an int32 tensor, zero on entry, that receives a device error."},
    {"scale_bytes", py_scale_bytes, METH_VARARGS,
     "scale_bytes(rows, cols)\n--\n\nBytes of the scales of an MX8 matrix (tiles of 128 rows x 128 columns, 512 bytes each)."},
    {"set_loader", set_loader, METH_O, "set_loader(f)\n--\n\nf() is called before the first operator and calls bind()."},
    {"bind", bind, METH_VARARGS, "bind(quantize, dequantize, rms_norm, linear, last_error, current_device)\n--\n\nAddresses of the library's functions."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mx8", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__mx8() {
  for (int i = 0; i < NAMES; ++i)
    if (!(g_names[i] = PyUnicode_InternFromString(kNames[i]))) return nullptr;
  MatrixType.tp_name = "laya_cuda.mx8.Matrix";
  MatrixType.tp_basicsize = sizeof(Matrix);
  MatrixType.tp_flags = Py_TPFLAGS_DEFAULT;
  MatrixType.tp_doc =
      "Matrix(values, scales, rows, cols)\n--\n\n"
      "An MX8 matrix [rows][cols]: `values`, bytes in `rows` rows of cols rounded up to a multiple of\n"
      "16, and `scales`, `scale_bytes(rows, cols)` bytes.  Both are contiguous, of any type of that many\n"
      "bytes; two-dimensional values of one-byte elements may have a larger row stride.  Holds\n"
      "references to both tensors; each call looks anew at where their storage is.";
  MatrixType.tp_dealloc = matrix_dealloc;
  MatrixType.tp_vectorcall = matrix_call;
  MatrixType.tp_members = matrix_members;
  MatrixType.tp_getset = matrix_getset;
  MatrixType.tp_methods = matrix_methods;
  if (PyType_Ready(&MatrixType) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module);
  if (!m) return nullptr;
  Py_INCREF(&MatrixType);
  if (PyModule_AddObject(m, "Matrix", reinterpret_cast<PyObject*>(&MatrixType)) < 0 || PyModule_AddFunctions(m, attention_methods()) < 0) {
    Py_DECREF(&MatrixType);
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
