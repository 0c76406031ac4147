// The short way from Python into the calls that are made once per layer, some of them for a single row: tensors are read
// through torch's C++ interface and the kernels' library is called directly. Through ctypes and Python's tensor attributes a
// quantisation of one row takes 6.7 us, a linear layer 12 and a head norm 8.6; this way 2.9, 6.5 to 7.1 and 2.9, of which
// 2.3, 4.5 and 2.3 are the launches. (A rotation of one row
// 8.1, a block end 11.4: 3.3 and 3.8.)
//
// Every function takes what its namesake in ops.py takes and returns the library's status, or None for anything that is
// not plain (a wrong type, shape, stride or device, a subclass, no memory): the caller then goes the long way, which has
// the checks with their messages and switches devices.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>

#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <algorithm>
#include <climits>
#include <cstring>

#include "foidfinder_b200.h"

namespace {

struct {
  decltype(&ff_quantize_fp4) quantize;
  decltype(&ff_dequantize_fp4) dequantize;
  decltype(&ff_linear_fp4_workspace_bytes) workspace;
  decltype(&ff_linear_fp4) linear;
  decltype(&ff_qk_norm_rope) qk_norm_rope;
  decltype(&ff_rope) rope;
  decltype(&ff_norm_residual) norm_residual;
  decltype(&ff_cross_attention_workspace_bytes) cross_workspace;
  decltype(&ff_cross_attention) cross_attention;
} lib;

const at::Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == c10::kStrided ? &t : nullptr;
}

struct Matrix {
  void* data;
  int type, rows, cols, device;
  int64_t ld;
};
// A 2-D tensor of a floating type whose columns are contiguous.
bool matrix(PyObject* o, Matrix* m) {
  const at::Tensor* t = tensor(o);
  if (t == nullptr || t->dim() != 2) return false;
  switch (t->scalar_type()) {
    case at::kHalf: m->type = FF_F16; break;
    case at::kBFloat16: m->type = FF_BF16; break;
    case at::kFloat: m->type = FF_F32; break;
    default: return false;
  }
  const int64_t rows = t->size(0), cols = t->size(1);
  if (rows > (1 << 30) || cols > INT_MAX || (cols > 1 && t->stride(1) != 1)) return false;
  m->rows = static_cast<int>(rows);
  m->cols = static_cast<int>(cols);
  m->ld = rows > 1 ? t->stride(0) : std::max(t->stride(0), cols);
  m->device = t->get_device();
  m->data = t->data_ptr();
  return true;
}
// An optional f32 parameter of n values.
bool vector(PyObject* o, int64_t n, int device, float** p) {
  *p = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (t == nullptr || t->scalar_type() != at::kFloat || t->numel() != n || !t->is_contiguous() || t->get_device() != device) return false;
  *p = static_cast<float*>(t->data_ptr());
  return true;
}
bool buffer(PyObject* o, int64_t bytes, int device, uint8_t** p) {
  const at::Tensor* t = tensor(o);
  if (t == nullptr || t->scalar_type() != at::kByte || t->numel() < bytes || !t->is_contiguous() || t->get_device() != device) return false;
  *p = static_cast<uint8_t*>(t->data_ptr());
  return true;
}
struct Operand {
  uint8_t *codes, *scales;
  float* row_scale;
};
bool operand(PyObject* const* a, int rows, int cols, int fmt, int device, Operand* q) {
  const int64_t code_bytes = static_cast<int64_t>(rows) * ((static_cast<int64_t>(cols) + 31) / 32 * 16);
  const int64_t scale_bytes = static_cast<int64_t>((rows + 127) / 128) * ((static_cast<int64_t>(cols) + 255) / 256 * (fmt == FF_FP4_NV ? 2048 : 1024));
  q->row_scale = nullptr;
  return buffer(a[0], code_bytes, device, &q->codes) && buffer(a[1], scale_bytes, device, &q->scales) &&
         (fmt != FF_FP4_NV || (a[2] != Py_None && vector(a[2], rows, device, &q->row_scale)));
}

bool integer(PyObject* o, int* v) {
  if (!PyLong_Check(o)) return false;
  int overflow = 0;
  const long l = PyLong_AsLongAndOverflow(o, &overflow);
  *v = static_cast<int>(l);
  return overflow == 0 && l >= INT_MIN && l <= INT_MAX;
}
bool number(PyObject* o, float* v) {
  if (PyFloat_Check(o))
    *v = static_cast<float>(PyFloat_AS_DOUBLE(o));
  else
    return false;
  return true;
}
// The addresses of a prepared epilogue's tensors (its attribute `tensors`: bias, q weight, q bias, k weight, k bias, cos,
// sin) into its fields. One that was filled in by hand has none.
bool address(PyObject* o, int N, int device, ff_fp4_epilogue* e) {
  static PyObject* const name = PyUnicode_InternFromString("tensors");
  PyObject* const ts = name != nullptr ? PyObject_GetAttr(o, name) : nullptr;
  if (ts == nullptr || ts == Py_None) {
    PyErr_Clear();
    Py_XDECREF(ts);
    return name != nullptr;
  }
  const bool qkv = e->kind == FF_EPI_QKV_NORM_ROPE;
  float* p[7] = {};
  bool ok = PyTuple_Check(ts) && PyTuple_GET_SIZE(ts) == 7 && (!qkv || e->tokens >= 1);
  for (int i = 0; ok && i < (qkv ? 7 : 1); ++i)
    ok = vector(PyTuple_GET_ITEM(ts, i), i == 0 ? N : i < 5 ? 64 : 32 * static_cast<int64_t>(e->tokens), device, &p[i]);
  Py_DECREF(ts);
  e->bias = p[0];
  e->q_w = p[1];
  e->q_b = p[2];
  e->k_w = p[3];
  e->k_b = p[4];
  e->rope_cos = p[5];
  e->rope_sin = p[6];
  return ok;
}

bool current(int device) { return c10::cuda::current_device() == device; }
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

// f() with the interpreter unlocked (a launch waits while its stream's queue is full).
template <class F>
PyObject* status(F f) {
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS rc = f();
  Py_END_ALLOW_THREADS return PyLong_FromLong(rc);
}
// Anything thrown is left to the long way, and so is a Python error.
template <class F>
PyObject* guarded(F f) {
  try {
    PyObject* r = f();
    if (r != nullptr) return r;
  } catch (...) {
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

// quantize(x, codes, scales, row_scale, fmt, gamma, beta, eps)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix x;
    Operand q;
    int fmt;
    float *gamma, *beta, eps;
    if (n != 8 || !matrix(a[0], &x) || !integer(a[4], &fmt) || !operand(a + 1, x.rows, x.cols, fmt, x.device, &q) ||
        !vector(a[5], x.cols, x.device, &gamma) || !vector(a[6], x.cols, x.device, &beta) || !number(a[7], &eps) || !current(x.device))
      return nullptr;
    void* const s = stream_of(x.device);
    return status([&] { return lib.quantize(x.data, x.type, x.ld, gamma, beta, eps, x.rows, x.cols, fmt, q.codes, q.scales, q.row_scale, s); });
  });
}

// dequantize(codes, scales, row_scale, out, fmt)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix out;
    Operand q;
    int fmt;
    if (n != 5 || !matrix(a[3], &out) || !integer(a[4], &fmt) || !operand(a, out.rows, out.cols, fmt, out.device, &q) || !current(out.device))
      return nullptr;
    void* const s = stream_of(out.device);
    return status([&] { return lib.dequantize(q.codes, q.scales, q.row_scale, out.rows, out.cols, fmt, out.data, out.type, out.ld, s); });
  });
}

// linear(x, (codes, scales, row_scale) of the weight, fmt, N, K, gamma, beta, eps, epilogue, out, residual)
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix x, out;
    int fmt, N, K;
    float eps;
    float *gamma, *beta;
    Operand w;
    if (n != 11 || !matrix(a[0], &x) || !PyTuple_Check(a[1]) || PyTuple_GET_SIZE(a[1]) != 3 || !integer(a[2], &fmt) || !integer(a[3], &N) ||
        !integer(a[4], &K) || N < 1 || K < 1)
      return nullptr;
    PyObject* const wt[3] = {PyTuple_GET_ITEM(a[1], 0), PyTuple_GET_ITEM(a[1], 1), PyTuple_GET_ITEM(a[1], 2)};
    if (!operand(wt, N, K, fmt, x.device, &w) || !vector(a[5], K, x.device, &gamma) || !vector(a[6], K, x.device, &beta) || !number(a[7], &eps) ||
        !matrix(a[9], &out))
      return nullptr;
    ff_fp4_epilogue e;
    Py_buffer view;
    if (PyObject_GetBuffer(a[8], &view, PyBUF_SIMPLE) != 0) return nullptr;
    const bool fits = view.len == static_cast<Py_ssize_t>(sizeof e);
    if (fits) std::memcpy(&e, view.buf, sizeof e);
    PyBuffer_Release(&view);
    if (!fits || !address(a[8], N, x.device, &e) || x.rows == 0 || x.cols != K || out.rows != x.rows || out.device != x.device ||
        (e.kind == FF_EPI_SWIGLU ? out.cols < 1 || out.cols > N / 2 : out.cols != N) || !current(x.device))
      return nullptr;
    e.out_dtype = out.type;
    e.out = out.data;
    e.ldo = out.ld;
    e.out_cols = out.cols;
    if (e.kind == FF_EPI_RESIDUAL) {
      Matrix r;
      if (!matrix(a[10], &r) || r.type != out.type || r.rows != out.rows || r.cols != out.cols || r.device != out.device) return nullptr;
      e.residual = r.data;
      e.ldr = r.ld;
    }
    const int64_t bytes = lib.workspace(x.rows, K, fmt);
    if (bytes <= 0) return nullptr;
    const auto s = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(x.device)).stream();
    // from torch's stream-ordered cache: free for the stream's next use as soon as the call has returned
    void* const ws = c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(static_cast<size_t>(bytes), s);
    PyObject* const rc = status([&] {
      return lib.linear(x.data, x.type, x.ld, gamma, beta, eps, w.codes, w.scales, w.row_scale, fmt, x.rows, N, K, &e, ws, bytes, s);
    });
    c10::cuda::CUDACachingAllocator::raw_delete(ws);
    return rc;
  });
}

// qk_norm_rope(x, out, q_heads, k_heads, head_dim, norm, q_weight, q_bias, k_weight, k_bias, eps, cos, sin, pairing)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix x, out;
    int qh, kh, d, norm, pairing;
    float eps, *p[4], *cos, *sin;
    if (n != 14 || !matrix(a[0], &x) || !matrix(a[1], &out) || !integer(a[2], &qh) || !integer(a[3], &kh) || !integer(a[4], &d) ||
        !integer(a[5], &norm) || !number(a[10], &eps) || !integer(a[13], &pairing))
      return nullptr;
    if (qh < 0 || kh < 0 || qh > (1 << 16) || kh > (1 << 16) || d < 2 || d > 256) return nullptr;
    const int64_t cols = static_cast<int64_t>(qh + kh) * d;
    if (x.type == FF_F32 || out.type != x.type || x.cols < cols || out.cols < cols || out.rows != x.rows || out.device != x.device) return nullptr;
    for (int i = 0; i < 4; ++i)
      if (!vector(a[6 + i], d, x.device, &p[i])) return nullptr;
    const at::Tensor *c = tensor(a[11]), *s = tensor(a[12]);
    if (c == nullptr || s == nullptr || c->dim() != 2 || c->size(0) != d / 2 || c->size(1) < 1 || c->size(1) > INT_MAX || c->sizes() != s->sizes() ||
        !vector(a[11], c->numel(), x.device, &cos) || !vector(a[12], c->numel(), x.device, &sin) || !current(x.device))
      return nullptr;
    const int tokens = static_cast<int>(c->size(1));
    void* const st = stream_of(x.device);
    return status([&] {
      return lib.qk_norm_rope(x.data, x.type, x.ld, out.data, out.ld, x.rows, qh, kh, d, norm, p[0], p[1], p[2], p[3], eps, cos, sin, tokens, pairing, st);
    });
  });
}

// rope(x, out, positions, frequencies, heads, head_dim, start, pairing, scale)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix x, out;
    int heads, dim, start, pairing;
    float scale;
    if (n != 9 || !matrix(a[0], &x) || !matrix(a[1], &out) || !integer(a[4], &heads) || !integer(a[5], &dim) || !integer(a[6], &start) ||
        !integer(a[7], &pairing) || !number(a[8], &scale) || heads < 0 || heads > (1 << 16) || dim < 1 || dim > (1 << 16))
      return nullptr;
    const at::Tensor *p = tensor(a[2]), *f = tensor(a[3]);
    const int64_t cols = static_cast<int64_t>(heads) * dim;
    if (p == nullptr || f == nullptr || out.type != x.type || x.cols < cols || out.cols < cols || out.rows != x.rows || out.device != x.device) return nullptr;
    const bool wide_p = p->scalar_type() == at::kLong, wide_f = f->scalar_type() == at::kDouble;
    if ((!wide_p && p->scalar_type() != at::kInt) || (!wide_f && f->scalar_type() != at::kFloat) || p->dim() < 1 || p->dim() > 2 || f->dim() != 1 ||
        p->size(0) != x.rows || !p->is_contiguous() || !f->is_contiguous() || p->get_device() != x.device || f->get_device() != x.device ||
        f->size(0) > (1 << 16) || !current(x.device))
      return nullptr;
    const int64_t axes = p->dim() == 1 ? 1 : p->size(1);
    if (axes < 1 || axes > (1 << 16)) return nullptr;
    const void *positions = p->data_ptr(), *frequencies = f->data_ptr();
    const int rotary = 2 * static_cast<int>(f->size(0));
    void* const s = stream_of(x.device);
    return status([&] {
      return lib.rope(x.data, x.type, x.ld, out.data, out.ld, x.rows, heads, dim, start, rotary, pairing, positions, wide_p ? 8 : 4, static_cast<int>(axes),
                      frequencies, wide_f ? 8 : 4, scale, s);
    });
  });
}

// norm_residual(x, y, out, normed, alpha, post, post_weight, post_bias, gate, gate_act, gate_rows, scale, pre, pre_weight, pre_bias, eps, pre_eps)
PyObject* norm_residual(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix x, y, out, normed{}, gate{};
    ff_norm_residual_args r{};
    int gate_rows;
    float* p[5];
    if (n != 17 || !matrix(a[0], &x) || !matrix(a[1], &y) || !matrix(a[2], &out) || !number(a[4], &r.alpha) || !integer(a[5], &r.post) ||
        !integer(a[9], &r.gate_act) || !integer(a[10], &gate_rows) || !integer(a[12], &r.pre) || !number(a[15], &r.post_eps) || !number(a[16], &r.pre_eps))
      return nullptr;
    auto like = [&](const Matrix& m, int type) { return m.type == type && m.rows == x.rows && m.cols == x.cols && m.device == x.device; };
    if (!like(y, y.type) || !like(out, x.type) || (x.type != y.type && x.type != FF_F32)) return nullptr;
    if ((a[3] == Py_None) != (r.pre == FF_NORM_NONE) || (a[3] != Py_None && (!matrix(a[3], &normed) || !like(normed, y.type)))) return nullptr;
    PyObject* const params[5] = {a[6], a[7], a[11], a[13], a[14]};
    for (int i = 0; i < 5; ++i)
      if (!vector(params[i], x.cols, x.device, &p[i])) return nullptr;
    if (a[8] != Py_None) {
      if (!matrix(a[8], &gate) || gate.device != x.device || (gate.cols != 1 && gate.cols != x.cols) || (gate.type != FF_F32 && gate.type != y.type) ||
          gate_rows < 1 || static_cast<int64_t>(gate.rows) * gate_rows < x.rows || x.rows == 0)
        return nullptr;
      r.gate = gate.data;
      r.ldg = gate.ld;
      r.gate_type = gate.type;
      r.gate_cols = gate.cols;
      r.gate_rows = gate_rows;
    }
    if (!current(x.device)) return nullptr;
    r.x = x.data;
    r.ldx = x.ld;
    r.y = y.data;
    r.ldy = y.ld;
    r.out = out.data;
    r.ldo = out.ld;
    r.normed = normed.data;
    r.ldn = normed.ld;
    r.x_type = x.type;
    r.y_type = y.type;
    r.rows = x.rows;
    r.cols = x.cols;
    r.post_w = p[0];
    r.post_b = p[1];
    r.scale = p[2];
    r.pre_w = p[3];
    r.pre_b = p[4];
    void* const s = stream_of(x.device);
    return status([&] { return lib.norm_residual(&r, s); });
  });
}

// An optional tensor of n int32 values.
bool starts(PyObject* o, int64_t n, int device, const int32_t** p) {
  *p = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o);
  if (t == nullptr || t->scalar_type() != at::kInt || t->numel() != n || !t->is_contiguous() || t->get_device() != device) return false;
  *p = static_cast<const int32_t*>(t->data_ptr());
  return true;
}

// cross_attention(q, k, v, out, heads, kv_heads, head_dim, sequences, q_start, k_start, k_len, mask, scale)
PyObject* cross_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Matrix q, k, v, out;
    int heads, kv_heads, dim, sequences;
    float scale;
    const int32_t *q_start, *k_start, *k_len;
    const uint8_t* mask = nullptr;
    if (n != 13 || !matrix(a[0], &q) || !matrix(a[1], &k) || !matrix(a[2], &v) || !matrix(a[3], &out) || !integer(a[4], &heads) || !integer(a[5], &kv_heads) ||
        !integer(a[6], &dim) || !integer(a[7], &sequences) || !number(a[12], &scale) || heads < 1 || heads > 1024 || kv_heads < 1 || dim < 1 || dim > 128 ||
        heads % kv_heads != 0 || sequences < 1)
      return nullptr;
    if (q.type == FF_F32 || k.type != q.type || v.type != q.type || out.type != q.type || q.cols != heads * dim || out.cols != q.cols || k.cols != kv_heads * dim ||
        v.cols != k.cols || out.rows != q.rows || v.rows != k.rows || k.device != q.device || v.device != q.device || out.device != q.device || q.rows < 1)
      return nullptr;
    if (!starts(a[8], static_cast<int64_t>(sequences) + 1, q.device, &q_start) || !starts(a[9], static_cast<int64_t>(sequences) + 1, q.device, &k_start) ||
        !starts(a[10], sequences, q.device, &k_len))
      return nullptr;
    if (a[11] != Py_None) {
      const at::Tensor* t = tensor(a[11]);
      if (t == nullptr || (t->scalar_type() != at::kBool && t->scalar_type() != at::kByte) || t->numel() != k.rows || !t->is_contiguous() ||
          t->get_device() != q.device)
        return nullptr;
      mask = static_cast<const uint8_t*>(t->data_ptr());
    }
    if (!current(q.device)) return nullptr;
    const int64_t bytes = lib.cross_workspace(q.rows, k.rows, sequences, heads, kv_heads, dim);
    const auto s = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(q.device)).stream();
    void* const ws = bytes > 0 ? c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(static_cast<size_t>(bytes), s) : nullptr;
    PyObject* const rc = status([&] {
      return lib.cross_attention(q.data, q.ld, k.data, k.ld, v.data, v.ld, out.data, out.ld, q.type, q.rows, k.rows, sequences, q_start, k_start, k_len, mask, heads,
                                 kv_heads, dim, scale, ws, bytes, s);
    });
    if (ws != nullptr) c10::cuda::CUDACachingAllocator::raw_delete(ws);
    return rc;
  });
}

// bind(addresses of the functions of the kernels' library, in the order of `lib`)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int kFunctions = 9;
  void* f[kFunctions];
  static_assert(sizeof f == sizeof lib, "one address each");
  if (n != kFunctions) {
    PyErr_SetString(PyExc_TypeError, "bind takes nine addresses");
    return nullptr;
  }
  for (int i = 0; i < kFunctions; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (f[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "bind takes nine addresses");
      return nullptr;
    }
  }
  std::memcpy(&lib, f, sizeof lib);
  Py_RETURN_NONE;
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),         METHOD(quantize), METHOD(dequantize),    METHOD(linear),
                         METHOD(qk_norm_rope), METHOD(rope),     METHOD(norm_residual), METHOD(cross_attention),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  PyObject* const m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", FF_TORCH_VERSION) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
