// moe_python.cpp -- the Python calls of the mixture-of-experts operators: reads and checks the tensors'
// attributes and calls the C-ABI (include/grouped_gemm_b200.h). A decoding step makes some ten such calls, each of a
// few microseconds on the GPU; with the checks in Python and the call through ctypes a call took 6.1 us on the
// host, of which the launch is 2.9. The module knows a tensor only by its Python attributes (dtype, shape,
// stride(), get_device(), data_ptr()), so it is not tied to a version of torch.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <climits>
#include <cstdint>

#include "grouped_gemm_b200.h"

namespace {

// Interned attribute names, and torch's dtype objects (fetched on the first call).
PyObject *n_dtype, *n_shape, *n_stride, *n_get_device, *n_data_ptr, *n_is_contiguous, *n_numel, *n_cuda_stream, *n_element_size;
PyObject *t_f32, *t_f16, *t_bf16, *t_i32, *t_u8, *t_bool;

bool load_types() {
  if (t_bool) return true;
  PyObject* torch = PyImport_ImportModule("torch");
  if (!torch) return false;
  t_f32 = PyObject_GetAttrString(torch, "float32");
  t_f16 = PyObject_GetAttrString(torch, "float16");
  t_bf16 = PyObject_GetAttrString(torch, "bfloat16");
  t_i32 = PyObject_GetAttrString(torch, "int32");
  t_u8 = PyObject_GetAttrString(torch, "uint8");
  t_bool = t_f32 && t_f16 && t_bf16 && t_i32 && t_u8 ? PyObject_GetAttrString(torch, "bool") : nullptr;
  Py_DECREF(torch);
  return t_bool != nullptr;
}

// An attribute that the caller only compares (dtypes and truth values outlive the reference).
PyObject* peek(PyObject* t, PyObject* name) {
  PyObject* v = PyObject_GetAttr(t, name);
  Py_XDECREF(v);
  return v;
}

bool call_int(PyObject* t, PyObject* name, int64_t* out) {
  PyObject* v = PyObject_CallMethodNoArgs(t, name);
  if (!v) return false;
  *out = static_cast<int64_t>(PyLong_AsLongLong(v));
  Py_DECREF(v);
  return !(*out == -1 && PyErr_Occurred());
}

// Whether a tensor is on the current device, which the call's launch goes to (-1 of get_device(): on none). Each call
// looks the device up once, and leaves it negative where there is none.
bool on_device(PyObject* t, int device, bool* is) {
  int64_t of = 0;
  if (!call_int(t, n_get_device, &of)) return false;
  *is = of >= 0 && of == device;
  return true;
}

int current_device() {
  int device = -1;
  return gg_current_device(&device) == 0 ? device : -1;
}

bool pointer_of(PyObject* t, void** out) {
  PyObject* v = PyObject_CallMethodNoArgs(t, n_data_ptr);
  if (!v) return false;
  *out = PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  return !(*out == nullptr && PyErr_Occurred());
}

// Two numbers of a tuple (shape or stride()), which is released.
bool two_of(PyObject* tuple, const char* what, int64_t* a, int64_t* b) {
  if (!tuple) return false;
  bool ok = PyTuple_Check(tuple) && PyTuple_GET_SIZE(tuple) == 2;
  if (!ok) {
    PyErr_Format(PyExc_ValueError, "%s: two dimensions expected", what);
  } else {
    *a = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, 0));
    *b = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, 1));
    ok = !PyErr_Occurred();
    if (ok && (*a > INT_MAX || *b > INT_MAX)) {
      PyErr_Format(PyExc_ValueError, "%s: sizes and pitches below 2^31 expected", what);
      ok = false;
    }
  }
  Py_DECREF(tuple);
  return ok;
}

struct Matrix {
  PyObject* dtype;
  void* data;
  int rows, cols, ld;
};

// A rows x cols tensor of the device with contiguous columns and rows that do not overlap; rows or cols < 0: any.
bool matrix(PyObject* t, const char* what, int device, int64_t rows, int64_t cols, Matrix* m) {
  int64_t r, c, sr, sc;
  if (!two_of(PyObject_GetAttr(t, n_shape), what, &r, &c)) return false;
  if ((rows >= 0 && r != rows) || (cols >= 0 && c != cols)) {
    PyErr_Format(PyExc_ValueError, "%s: shape (%lld, %lld) expected, got (%lld, %lld)", what,
                 static_cast<long long>(rows < 0 ? r : rows), static_cast<long long>(cols < 0 ? c : cols),
                 static_cast<long long>(r), static_cast<long long>(c));
    return false;
  }
  if (!two_of(PyObject_CallMethodNoArgs(t, n_stride), what, &sr, &sc)) return false;
  bool here;
  if (!on_device(t, device, &here)) return false;
  if ((sc != 1 && c > 1) || (sr < c && r > 1) || !here) {
    PyErr_Format(PyExc_ValueError,
                 "%s: a tensor on the current CUDA device (%d) with contiguous columns and rows that do not overlap expected", what, device);
    return false;
  }
  m->dtype = peek(t, n_dtype);
  m->rows = static_cast<int>(r);
  m->cols = static_cast<int>(c);
  m->ld = static_cast<int>(sr >= c && sr > 0 ? sr : c > 1 ? c : 1);
  return m->dtype && pointer_of(t, &m->data);
}

// A contiguous tensor of the device, of `count` elements of a dtype (or of `other`).
bool flat(PyObject* t, const char* what, int device, int64_t count, PyObject* dtype, void** data, PyObject* other = nullptr) {
  PyObject* is = peek(t, n_dtype);
  if (!is) return false;
  int64_t have = 0;
  if (!call_int(t, n_numel, &have)) return false;
  PyObject* cont = PyObject_CallMethodNoArgs(t, n_is_contiguous);
  if (!cont) return false;
  Py_DECREF(cont);
  bool here;
  if (!on_device(t, device, &here)) return false;
  if ((is != dtype && is != other) || have != count || cont != Py_True || !here) {
    PyErr_Format(PyExc_ValueError,
                 "%s: a contiguous tensor on the current CUDA device (%d) of %lld elements of %R expected, got %lld of %R", what, device,
                 static_cast<long long>(count), dtype, static_cast<long long>(have), is);
    return false;
  }
  return pointer_of(t, data);
}

// The same, or NULL for None.
template <typename T>
bool flat_or_none(PyObject* t, const char* what, int device, int64_t count, PyObject* dtype, T** data, PyObject* other = nullptr) {
  void* p = nullptr;
  if (t != Py_None && !flat(t, what, device, count, dtype, &p, other)) return false;
  *data = static_cast<T*>(p);
  return true;
}
template <typename T>
bool flat_into(PyObject* t, const char* what, int device, int64_t count, PyObject* dtype, T** data) {
  void* p = nullptr;
  if (!flat(t, what, device, count, dtype, &p)) return false;
  *data = static_cast<T*>(p);
  return true;
}

bool output_type(PyObject* dtype, const char* what, int* type) {
  if (dtype == t_f32) *type = GG_OUTPUT_F32;
  else if (dtype == t_f16) *type = GG_OUTPUT_F16;
  else if (dtype == t_bf16) *type = GG_OUTPUT_BF16;
  else {
    PyErr_Format(PyExc_ValueError, "%s: float32, float16 or bfloat16 expected, got %R", what, dtype);
    return false;
  }
  return true;
}

// None (the legacy default stream), a handle, or an object with cuda_stream.
bool stream_of(PyObject* s, void** out) {
  *out = nullptr;
  if (s == Py_None) return true;
  if (PyLong_Check(s)) {
    *out = PyLong_AsVoidPtr(s);
    return !PyErr_Occurred();
  }
  PyObject* v = PyObject_GetAttr(s, n_cuda_stream);
  if (!v) return false;
  *out = PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  return !PyErr_Occurred();
}

bool arguments(Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return load_types();
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, got);
  return false;
}

template <typename F>
PyObject* status_of(F call) {  // the C-ABI throws nothing; a full launch queue may block
  int st;
  Py_BEGIN_ALLOW_THREADS st = call();
  Py_END_ALLOW_THREADS return PyLong_FromLong(st);
}

bool router_logits(PyObject* t, PyObject* type, int experts, const char* what, int device, Matrix* m) {
  int is;
  if (!matrix(t, what, device, -1, experts, m) || !output_type(m->dtype, what, &is)) return false;
  if (is == PyLong_AsLong(type)) return true;
  PyErr_Format(PyExc_ValueError, "%s: the router was made for another type than %R", what, m->dtype);
  return false;
}

// (handle, experts, top_k, logit_type, logits, indices, weights, positions, rows, losses, row_tokens, lse, prob_mean,
//  token_mask, stream)
PyObject* router_run(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 15)) return nullptr;
  const int device = current_device();
  gg_router* router = static_cast<gg_router*>(PyLong_AsVoidPtr(a[0]));
  const int experts = static_cast<int>(PyLong_AsLong(a[1])), top_k = static_cast<int>(PyLong_AsLong(a[2]));
  Matrix l;
  if (PyErr_Occurred() || !router_logits(a[4], a[3], experts, "logits", device, &l)) return nullptr;
  const int64_t slots = static_cast<int64_t>(l.rows) * top_k;
  gg_route q{};
  void* mask = nullptr;
  void* stream;
  if (!flat_into(a[5], "indices", device, slots, t_i32, &q.indices) || !flat_into(a[6], "weights", device, slots, t_f32, &q.weights) ||
      !flat_into(a[7], "positions", device, slots, t_i32, &q.positions) || !flat_into(a[8], "rows", device, experts, t_i32, &q.rows) ||
      !flat_into(a[9], "losses", device, 3, t_f32, &q.losses) || !flat_or_none(a[10], "row_tokens", device, slots, t_i32, &q.row_tokens) ||
      !flat_or_none(a[11], "lse", device, l.rows, t_f32, &q.lse) || !flat_or_none(a[12], "prob_mean", device, experts, t_f32, &q.prob_mean) ||
      !flat_or_none(a[13], "token_mask", device, l.rows, t_u8, &mask, t_bool) || !stream_of(a[14], &stream))
    return nullptr;
  q.logits = l.data;
  q.token_mask = static_cast<const unsigned char*>(mask);
  q.tokens = l.rows;
  q.ld = l.ld;
  return status_of([&] { return gg_router_run(router, &q, stream); });
}

// (handle, experts, top_k, logit_type, logits, indices, weights, rows, losses, lse, grad_weights, grad_losses,
//  grad_logits, stream)
PyObject* router_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 14)) return nullptr;
  const int device = current_device();
  const gg_router* router = static_cast<const gg_router*>(PyLong_AsVoidPtr(a[0]));
  const int experts = static_cast<int>(PyLong_AsLong(a[1])), top_k = static_cast<int>(PyLong_AsLong(a[2]));
  Matrix l, g;
  if (PyErr_Occurred() || !router_logits(a[4], a[3], experts, "logits", device, &l) ||
      !router_logits(a[12], a[3], experts, "grad_logits", device, &g))
    return nullptr;
  if (g.rows != l.rows) {
    PyErr_SetString(PyExc_ValueError, "grad_logits: the shape of logits expected");
    return nullptr;
  }
  const int64_t slots = static_cast<int64_t>(l.rows) * top_k;
  int *indices, *rows;
  float *weights, *losses, *lse, *grad_weights, *grad_losses;
  void* stream;
  if (!flat_into(a[5], "indices", device, slots, t_i32, &indices) || !flat_into(a[6], "weights", device, slots, t_f32, &weights) ||
      !flat_into(a[7], "rows", device, experts, t_i32, &rows) || !flat_into(a[8], "losses", device, 3, t_f32, &losses) ||
      !flat_into(a[9], "lse", device, l.rows, t_f32, &lse) || !flat_or_none(a[10], "grad_weights", device, slots, t_f32, &grad_weights) ||
      !flat_or_none(a[11], "grad_losses", device, 2, t_f32, &grad_losses) || !stream_of(a[13], &stream))
    return nullptr;
  const gg_route_gradient q{l.data, indices, weights, rows, losses, lse, grad_weights, grad_losses, g.data, l.rows, l.ld, g.ld};
  return status_of([&] { return gg_router_backward(router, &q, stream); });
}

// positions (tokens, top_k), contiguous.
bool positions_of(PyObject* t, int device, int tokens, int* top_k, int** data) {
  int64_t r, c;
  if (!two_of(PyObject_GetAttr(t, n_shape), "positions", &r, &c)) return false;
  if (r != tokens) {
    PyErr_Format(PyExc_ValueError, "positions: (%d, top_k) expected, got (%lld, %lld)", tokens, static_cast<long long>(r),
                 static_cast<long long>(c));
    return false;
  }
  *top_k = static_cast<int>(c);
  return flat_into(t, "positions", device, r * c, t_i32, data);
}

bool same_dtype(const Matrix& x, const Matrix& y, const char* what) {
  if (x.dtype == y.dtype) return true;
  PyErr_Format(PyExc_ValueError, "%s: one dtype expected, got %R and %R", what, x.dtype, y.dtype);
  return false;
}

// (x, positions, packed, stream)
PyObject* dispatch(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const int device = current_device();
  Matrix x, p;
  int k, *pos;
  int64_t bytes;
  void* stream;
  if (!arguments(n, 4) || !matrix(a[0], "x", device, -1, -1, &x) || !matrix(a[2], "packed", device, -1, x.cols, &p) ||
      !same_dtype(x, p, "x, packed") || !positions_of(a[1], device, x.rows, &k, &pos) || !call_int(a[0], n_element_size, &bytes) ||
      !stream_of(a[3], &stream))
    return nullptr;
  return status_of([&] {
    return gg_moe_dispatch(x.data, x.ld, pos, x.rows, k, x.cols, static_cast<int>(bytes), p.data, p.rows, p.ld, stream);
  });
}

// (packed, positions, out, weights, stream)
PyObject* combine(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const int device = current_device();
  Matrix p, o;
  int k, *pos, pt, ot;
  float* weights;
  void* stream;
  if (!arguments(n, 5) || !matrix(a[2], "out", device, -1, -1, &o) || !matrix(a[0], "packed", device, -1, o.cols, &p) ||
      !output_type(p.dtype, "packed", &pt) || !output_type(o.dtype, "out", &ot) || !positions_of(a[1], device, o.rows, &k, &pos) ||
      !flat_or_none(a[3], "weights", device, static_cast<int64_t>(o.rows) * k, t_f32, &weights) || !stream_of(a[4], &stream))
    return nullptr;
  return status_of([&] {
    return gg_moe_combine(p.data, pt, p.rows, p.ld, pos, weights, o.rows, k, o.cols, o.data, ot, o.ld, stream);
  });
}

// (grad_out, packed, positions, weights, grad_packed, grad_weights, stream)
PyObject* combine_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  const int device = current_device();
  Matrix g, p, gp;
  int k, *pos, pt, ot;
  float *weights, *grad_weights;
  void* stream;
  if (!arguments(n, 7) || !matrix(a[0], "grad_out", device, -1, -1, &g) || !matrix(a[1], "packed", device, -1, g.cols, &p) ||
      !matrix(a[4], "grad_packed", device, p.rows, g.cols, &gp) || !same_dtype(p, gp, "packed, grad_packed") ||
      !output_type(g.dtype, "grad_out", &ot) || !output_type(p.dtype, "packed", &pt) || !positions_of(a[2], device, g.rows, &k, &pos))
    return nullptr;
  const int64_t slots = static_cast<int64_t>(g.rows) * k;
  if (!flat_into(a[3], "weights", device, slots, t_f32, &weights) || !flat_into(a[5], "grad_weights", device, slots, t_f32, &grad_weights) ||
      !stream_of(a[6], &stream))
    return nullptr;
  return status_of([&] {
    return gg_moe_combine_backward(g.data, ot, g.ld, p.data, pt, p.rows, p.ld, pos, weights, g.rows, k, g.cols, gp.data, gp.ld,
                                   grad_weights, stream);
  });
}

// (handle, experts, n, k, input_type, output_type, a, rows, d, row_tokens, stream)
PyObject* q4_run(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 11)) return nullptr;
  const int device = current_device();
  gg_q4_plan* plan = static_cast<gg_q4_plan*>(PyLong_AsVoidPtr(a[0]));
  const long experts = PyLong_AsLong(a[1]), cols = PyLong_AsLong(a[2]), k = PyLong_AsLong(a[3]), in = PyLong_AsLong(a[4]),
             out = PyLong_AsLong(a[5]);
  Matrix x, d;
  int dt, *rows, *row_tokens;
  void* stream;
  if (PyErr_Occurred() || !matrix(a[6], "a", device, -1, k, &x) || !matrix(a[8], "d", device, -1, cols, &d) || !output_type(d.dtype, "d", &dt))
    return nullptr;
  if (x.dtype != (in == GG_INPUT_F16 ? t_f16 : t_bf16) || dt != out) {
    PyErr_Format(PyExc_ValueError, "a, d: the plan was made for other types than %R, %R", x.dtype, d.dtype);
    return nullptr;
  }
  if (!flat_or_none(a[7], "rows", device, experts, t_i32, &rows) || !flat_or_none(a[9], "row_tokens", device, d.rows, t_i32, &row_tokens) ||
      !stream_of(a[10], &stream))
    return nullptr;
  return status_of([&] { return gg_q4_plan_run(plan, x.data, x.ld, x.rows, row_tokens, rows, d.data, d.ld, d.rows, stream); });
}

#define GG_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {GG_METHOD(router_run), GG_METHOD(router_backward),  GG_METHOD(dispatch), GG_METHOD(combine),
                         GG_METHOD(combine_backward), GG_METHOD(q4_run), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_moe_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__moe_native() {
  struct {
    PyObject** to;
    const char* name;
  } names[] = {{&n_dtype, "dtype"}, {&n_shape, "shape"}, {&n_stride, "stride"}, {&n_get_device, "get_device"}, {&n_data_ptr, "data_ptr"},
               {&n_is_contiguous, "is_contiguous"}, {&n_numel, "numel"}, {&n_cuda_stream, "cuda_stream"},
               {&n_element_size, "element_size"}};
  for (auto& n : names)
    if (!(*n.to = PyUnicode_InternFromString(n.name))) return nullptr;
  return PyModule_Create(&module);
}
