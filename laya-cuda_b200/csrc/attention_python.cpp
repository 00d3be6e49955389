// The Python calls of laya_cuda.attention: rotary positions and attention over packed sequences.  They live in the
// extension laya_cuda._mx8, beside the operators of 8-bit linear layers.
#include "python_tensors.h"

#include <cmath>
#include <limits>

namespace {

using namespace laya_python;

using RotaryFn = int (*)(const laya_rotary*, void*);
using AttendFn = int (*)(const laya_attend*, int*, void*);

struct Library {
  RotaryFn rotary;
  AttendFn attend;
  ErrorFn last_error;
  DeviceFn current_device;
} g_lib = {};
PyObject* g_loader = nullptr;  // called before the first operator: it calls bind_attention()

bool ready() {
  if (g_lib.attend) return true;
  if (!g_loader) {
    PyErr_SetString(PyExc_RuntimeError, "these calls are used through laya_cuda.attention");
    return false;
  }
  PyObject* r = PyObject_CallNoArgs(g_loader);
  Py_XDECREF(r);
  if (r && !g_lib.attend) PyErr_SetString(PyExc_RuntimeError, "the library was not bound");
  return r && g_lib.attend;
}

bool given(PyObject* o) { return o && o != Py_None; }

// A [tokens][heads][dim] tensor whose heads' values are contiguous.
struct Heads {
  void* ptr;
  int64_t token, head;  // strides in elements
  int tokens, heads, dim, dtype, device;
};

bool take_heads(const char* name, PyObject* t, Heads* out) {
  View v;
  if (!view(t, &v)) return false;
  if (v.ndim != 3) {
    PyErr_Format(PyExc_ValueError, "%s must be [tokens][heads][head_dim], got %d dimensions", name, v.ndim);
    return false;
  }
  for (int i = 0; i < 3; ++i)
    if (v.shape[i] > 2147483647) {
      PyErr_Format(PyExc_ValueError, "%s is too large", name);
      return false;
    }
  if (v.shape[2] > 1 && v.strides[2] != 1) {
    PyErr_Format(PyExc_ValueError, "%s: the values of a head must be contiguous", name);
    return false;
  }
  if (v.dtype < 0 || v.dtype >= kInt32) {
    PyErr_Format(PyExc_ValueError, "%s is not float32, float16 or bfloat16", name);
    return false;
  }
  if (v.device < 0) {
    PyErr_Format(PyExc_ValueError, "%s is not on a CUDA device", name);
    return false;
  }
  // The stride of a dimension of one says nothing.
  const int64_t head = v.shape[1] > 1 ? v.strides[1] : v.shape[2];
  *out = {v.data, v.shape[0] > 1 ? v.strides[0] : v.shape[1] * head, head, (int)v.shape[0], (int)v.shape[1], (int)v.shape[2], v.dtype, v.device};
  return true;
}

// The same, of the shape, type and device of `like` but for `heads`.
bool take_heads_like(const char* name, PyObject* t, const Heads& like, int tokens, int heads, Heads* out) {
  if (!take_heads(name, t, out)) return false;
  if (out->tokens != tokens || out->heads != heads || out->dim != like.dim) {
    PyErr_Format(PyExc_ValueError, "%s must be [%d][%d][%d], got [%d][%d][%d]", name, tokens, heads, like.dim, out->tokens, out->heads, out->dim);
    return false;
  }
  if (out->dtype != like.dtype || out->device != like.device) {
    PyErr_Format(PyExc_ValueError, "%s must have the type and device of the other tensors", name);
    return false;
  }
  return true;
}

// `n` contiguous int32 values on `device`; null where `t` is absent or None.
bool take_ints(const char* name, PyObject* t, int n, int device, const int32_t** out) {
  *out = nullptr;
  if (!given(t)) return true;
  View v;
  if (!view(t, &v)) return false;
  if (v.ndim != 1 || v.shape[0] != n || v.dtype != kInt32 || !v.contiguous || v.device != device) {
    PyErr_Format(PyExc_ValueError, "%s must be %d contiguous int32 values on CUDA device %d", name, n, device);
    return false;
  }
  *out = static_cast<const int32_t*>(v.data);
  return true;
}

bool to_double(PyObject* o, double* out) {
  if (!given(o)) return true;
  const double d = PyFloat_AsDouble(o);
  if (d == -1.0 && PyErr_Occurred()) return false;
  *out = d;
  return true;
}

bool to_truth(PyObject* o, int32_t* out) {
  if (!o) return true;
  const int truth = PyObject_IsTrue(o);
  if (truth < 0) return false;
  *out = truth;
  return true;
}

PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { X, POSITIONS, OUT, K, K_OUT, DIMS, INTERLEAVED, THETA, SCALING, FACTOR, LENGTH, LOW, HIGH, MAGNITUDE, BACKWARD, STREAM, COUNT };
  static Signature<COUNT> sig = {"rotary", {"x", "positions", "out", "k", "k_out", "dims", "interleaved", "theta", "scaling", "factor",
                                            "length", "low", "high", "magnitude", "backward", "stream"}, {}};
  PyObject* g[COUNT] = {};
  if (!parse(sig, 3, args, nargs, kwnames, g)) return nullptr;
  Heads x, out;
  if (!take_heads("x", g[X], &x) || !take_heads_like("out", g[OUT], x, x.tokens, x.heads, &out)) return nullptr;
  laya_rotary a{};
  a.tokens = x.tokens; a.head_dim = x.dim; a.dims = x.dim; a.dtype = x.dtype;
  a.part[0] = {x.ptr, x.token, x.head, out.ptr, out.token, out.head, x.heads, 0};
  if (given(g[K]) != given(g[K_OUT])) {
    PyErr_SetString(PyExc_ValueError, "k and k_out go together");
    return nullptr;
  }
  if (given(g[K])) {
    Heads k, k_out;
    if (!take_heads("k", g[K], &k) || !take_heads_like("k", g[K], x, x.tokens, k.heads, &k) ||
        !take_heads_like("k_out", g[K_OUT], x, x.tokens, k.heads, &k_out))
      return nullptr;
    a.part[1] = {k.ptr, k.token, k.head, k_out.ptr, k_out.token, k_out.head, k.heads, 0};
  }
  View p;
  if (!view(g[POSITIONS], &p)) return nullptr;
  if (p.ndim != 1 || p.shape[0] != x.tokens || (p.dtype != kInt32 && p.dtype != kInt64) || !p.contiguous || p.device != x.device) {
    PyErr_Format(PyExc_ValueError, "positions must be %d contiguous int32 or int64 values on CUDA device %d", x.tokens, x.device);
    return nullptr;
  }
  a.positions = p.data;
  a.positions_64 = p.dtype == kInt64;
  if (given(g[DIMS]) && !to_int(g[DIMS], "dims", &a.dims)) return nullptr;
  if (given(g[SCALING])) {
    static constexpr const char* kNames[] = {"none", "linear", "ntk", "parts"};
    int at = 0;
    while (at < 4 && !(PyUnicode_Check(g[SCALING]) && PyUnicode_CompareWithASCIIString(g[SCALING], kNames[at]) == 0)) ++at;
    if (at == 4) {
      PyErr_Format(PyExc_ValueError, "scaling %R is not one of none, linear, ntk, parts", g[SCALING]);
      return nullptr;
    }
    a.scaling = at;
  }
  a.theta = 10000.0; a.factor = 1.0; a.low = 1.0; a.high = 32.0;
  double magnitude = 1.0;
  if (!to_truth(g[INTERLEAVED], &a.interleaved) || !to_truth(g[BACKWARD], &a.backward) || !to_double(g[THETA], &a.theta) ||
      !to_double(g[FACTOR], &a.factor) || !to_double(g[LENGTH], &a.length) || !to_double(g[LOW], &a.low) ||
      !to_double(g[HIGH], &a.high) || !to_double(g[MAGNITUDE], &magnitude))
    return nullptr;
  a.magnitude = (float)magnitude;
  void* st;
  if (!to_stream(g[STREAM], g[X], x.device, &st) || !ready() || (x.tokens && !on_current_device("x is", x.device, g_lib.current_device)))
    return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_lib.rotary(&a, st);
  Py_END_ALLOW_THREADS
  return finish(status, g_lib.last_error);
}

// None, n (n to both sides) or (left, right).
bool to_window(PyObject* o, int32_t* left, int32_t* right) {
  *left = *right = -1;
  if (!given(o)) return true;
  if (PyLong_Check(o)) {
    if (!to_int(o, "window", left)) return false;
    *right = *left;
    return true;
  }
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) {
    PyErr_SetString(PyExc_ValueError, "window must be a number or a pair (left, right)");
    return false;
  }
  return to_int(PyTuple_GET_ITEM(o, 0), "window", left) && to_int(PyTuple_GET_ITEM(o, 1), "window", right);
}

PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  enum { Q, K, V, OUT, STARTS, LENGTHS, K_STARTS, K_LENGTHS, MAX_QUERIES, MAX_KEYS, SCALE, CAP, CAUSAL, WINDOW, PREFIX, DOCUMENTS,
         K_DOCUMENTS, SLOPES, DISTANCE_BIAS, LSE, ERR, STREAM, COUNT };
  static Signature<COUNT> sig = {"attend", {"q", "k", "v", "out", "starts", "lengths", "k_starts", "k_lengths", "max_queries", "max_keys",
                                            "scale", "cap", "causal", "window", "prefix", "documents", "k_documents", "slopes",
                                            "distance_bias", "lse", "err", "stream"}, {}};
  PyObject* g[COUNT] = {};
  if (!parse(sig, 6, args, nargs, kwnames, g)) return nullptr;
  Heads q, k, v, out;
  if (!take_heads("q", g[Q], &q) || !take_heads("k", g[K], &k)) return nullptr;
  if (!take_heads_like("k", g[K], q, k.tokens, k.heads, &k) || !take_heads_like("v", g[V], q, k.tokens, k.heads, &v) ||
      !take_heads_like("out", g[OUT], q, q.tokens, q.heads, &out))
    return nullptr;
  laya_attend a{};
  a.heads = q.heads; a.kv_heads = k.heads; a.head_dim = q.dim; a.dtype = q.dtype;
  a.q_tokens = q.tokens; a.k_tokens = k.tokens; a.max_queries = q.tokens; a.max_keys = k.tokens;
  a.q = q.ptr; a.q_token = q.token; a.q_head = q.head;
  a.k = k.ptr; a.k_token = k.token; a.k_head = k.head;
  a.v = v.ptr; a.v_token = v.token; a.v_head = v.head;
  a.out = out.ptr; a.out_token = out.token; a.out_head = out.head;
  View starts;
  if (!view(g[STARTS], &starts)) return nullptr;
  if (starts.ndim != 1 || starts.shape[0] > 65535) {
    PyErr_SetString(PyExc_ValueError, "starts must be one int32 value for each of at most 65535 sequences");
    return nullptr;
  }
  const int n = (int)starts.shape[0], device = q.device;
  a.sequences = n;
  if (!given(g[LENGTHS])) {
    PyErr_SetString(PyExc_ValueError, "lengths must be a tensor");
    return nullptr;
  }
  if (given(g[K_STARTS]) != given(g[K_LENGTHS])) {
    PyErr_SetString(PyExc_ValueError, "k_starts and k_lengths go together");
    return nullptr;
  }
  if (!take_ints("starts", g[STARTS], n, device, &a.starts) || !take_ints("lengths", g[LENGTHS], n, device, &a.lengths) ||
      !take_ints("k_starts", g[K_STARTS], n, device, &a.k_starts) || !take_ints("k_lengths", g[K_LENGTHS], n, device, &a.k_lengths) ||
      !take_ints("prefix", g[PREFIX], n, device, &a.prefix) || !take_ints("documents", g[DOCUMENTS], q.tokens, device, &a.documents) ||
      !take_ints("k_documents", g[K_DOCUMENTS], k.tokens, device, &a.k_documents))
    return nullptr;
  if (a.documents && !given(g[K_DOCUMENTS])) {  // self-attention: the queries' are the keys'
    if (k.tokens != q.tokens) {
      PyErr_SetString(PyExc_ValueError, "k_documents is needed where the keys are not the queries' tokens");
      return nullptr;
    }
    a.k_documents = a.documents;
  }
  if (given(g[MAX_QUERIES]) && !to_int(g[MAX_QUERIES], "max_queries", &a.max_queries)) return nullptr;
  if (given(g[MAX_KEYS]) && !to_int(g[MAX_KEYS], "max_keys", &a.max_keys)) return nullptr;
  double scale = 1 / std::sqrt((double)(q.dim ? q.dim : 1)), cap = 0;
  if (!to_double(g[SCALE], &scale) || !to_double(g[CAP], &cap) || !to_truth(g[CAUSAL], &a.causal) ||
      !to_window(g[WINDOW], &a.window_left, &a.window_right))
    return nullptr;
  a.scale = (float)scale;
  a.cap = (float)cap;
  if (cap > 0 && a.cap == 0) a.cap = std::numeric_limits<float>::denorm_min();  // 0 would be no cap
  if (!take_vector("slopes", g[SLOPES], q.heads, device, &a.slopes)) return nullptr;
  if (given(g[DISTANCE_BIAS])) {
    View t;
    if (!view(g[DISTANCE_BIAS], &t)) return nullptr;
    if (t.ndim != 2 || t.shape[0] != q.heads || t.shape[1] % 2 != 1 || t.shape[1] > 2147483647 || t.dtype != LAYA_DTYPE_F32 ||
        !t.contiguous || t.device != device) {
      PyErr_Format(PyExc_ValueError, "distance_bias must be [%d][2 reach + 1] contiguous float32 on CUDA device %d", q.heads, device);
      return nullptr;
    }
    a.distance_bias = static_cast<const float*>(t.data);
    a.reach = (int)(t.shape[1] / 2);
  }
  if (given(g[LSE])) {
    View t;
    if (!view(g[LSE], &t)) return nullptr;
    if (t.ndim != 2 || t.shape[0] != q.tokens || t.shape[1] != q.heads || t.dtype != LAYA_DTYPE_F32 || !t.contiguous || t.device != device) {
      PyErr_Format(PyExc_ValueError, "lse must be [%d][%d] contiguous float32 on CUDA device %d", q.tokens, q.heads, device);
      return nullptr;
    }
    a.lse = static_cast<float*>(t.data);
  }
  int* err = nullptr;
  if (given(g[ERR])) {
    View t;
    if (!view(g[ERR], &t)) return nullptr;
    if (t.dtype != kInt32 || t.device != device || t.numel < 1) {
      PyErr_Format(PyExc_ValueError, "err must be int32 on CUDA device %d", device);
      return nullptr;
    }
    err = static_cast<int*>(t.data);
  }
  void* st;
  if (!to_stream(g[STREAM], g[Q], device, &st) || !ready() || (q.tokens && !on_current_device("q is", device, g_lib.current_device)))
    return nullptr;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = g_lib.attend(&a, err, st);
  Py_END_ALLOW_THREADS
  return finish(status, g_lib.last_error);
}

PyObject* set_loader(PyObject*, PyObject* loader) {
  Py_INCREF(loader);
  Py_XSETREF(g_loader, loader);
  Py_RETURN_NONE;
}

PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long r, a, e, c;
  if (!PyArg_ParseTuple(args, "KKKK", &r, &a, &e, &c)) return nullptr;
  g_lib = {reinterpret_cast<RotaryFn>(r), reinterpret_cast<AttendFn>(a), reinterpret_cast<ErrorFn>(e), reinterpret_cast<DeviceFn>(c)};
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL | METH_KEYWORDS
PyMethodDef methods[] = {
    {"rotary", FAST(rotary),
     "rotary(x, positions, out, k=None, k_out=None, dims=None, interleaved=False, theta=10000.0, scaling='none', factor=1.0,\n"
     "       length=0.0, low=1.0, high=32.0, magnitude=1.0, backward=False, stream=None)\n--\n\n"
     "Turns the first `dims` values (all, without it) of each head of x [tokens][heads][head_dim] in pairs\n"
     "by position * f_k, f_k = theta^(-2k / dims), and copies the rest; k [tokens][kv heads][head_dim]\n"
     "likewise, in the same launch.  out may be x, k_out may be k.  16 or 32 bits.\n\n"
     "Pairs are (2k, 2k + 1) interleaved, (k, k + dims / 2) otherwise.  positions: int32 or int64 [tokens].\n"
     "scaling: 'linear' (f_k / factor), 'ntk' (theta * factor^(dims / (dims - 2))) or 'parts' (f_k where it turns\n"
     "`high` times or more over `length` positions, f_k / factor where `low` times or fewer, linear between).\n"
     "magnitude multiplies the turned values.  backward: the transposed map, for gradients."},
    {"attend", FAST(attend),
     "attend(q, k, v, out, starts, lengths, k_starts=None, k_lengths=None, max_queries=None, max_keys=None, scale=None,\n"
     "       cap=0.0, causal=False, window=None, prefix=None, documents=None, k_documents=None, slopes=None,\n"
     "       distance_bias=None, lse=None, err=None, stream=None)\n--\n\n"
     "Attention of packed sequences: out = softmax(s) v over the visible keys, zeros where there are none.\n\n"
     "q, out [q tokens][heads][head_dim]; k, v [k tokens][kv heads][head_dim], in float16 or bfloat16.  Sequence b\n"
     "has lengths[b] queries from row starts[b] on, and k_lengths[b] keys from k_starts[b] on (as the queries, without\n"
     "them); query i is at p = i + keys - queries.  s = scale q . k (1 / sqrt(head_dim)); s = cap tanh(s / cap);\n"
     "s -= slopes[head] |p - j|, or s += distance_bias[head][clamp(j - p, -reach, reach) + reach].\n"
     "Key j is visible where j < prefix[b], or where documents[query] == k_documents[key], causal implies\n"
     "j <= p, and p - left <= j <= p + right (window; -1: no bound).  max_queries, max_keys: bounds on the lengths\n"
     "(the tensors' rows, without them): each sequence is launched for max_queries, so give it where there are several\n"
     "(64 x 1024 tokens, 12 heads of 64: 0.34 ms, 2.2 without).  lse: float32 [q tokens][heads], receives the\n"
     "logarithm of the sum of exp(s).  err: an int32 tensor, zero on entry, that receives a device error."},
    {"set_attention_loader", set_loader, METH_O, "set_attention_loader(f)\n--\n\nf() is called before the first operator and calls bind_attention()."},
    {"bind_attention", bind, METH_VARARGS, "bind_attention(rotary, attend, last_error, current_device)\n--\n\nAddresses of the library's functions."},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

PyMethodDef* attention_methods() { return methods; }
