// Native host path of the torch wrappers.
//
// A decode step calls its norms, projections and attention on tensors so small
// that the call is bound by the host: checking the arguments in Python,
// allocating through torch's Python bindings and building ctypes arguments
// took 8-15 us per call, against 3-4 us for the launch itself.  The functions
// here do the same for the usual case of each op -- plain GPU tensors on the
// current device in layouts that need no copy or cast -- and return None for
// anything else (other layouts, dtypes or devices, tensor subclasses, function
// modes, wrong arguments), which the wrapper then serves or rejects in Python.
// The kernels and their arguments are those of the Python path, but for a
// softmax of a single row (see there).
// add_rms_norm bf16 (8, 4096) 15.1 -> 5.65 us per call, silu of a few rows 7.1
// -> 4.4, softmax 10.7 -> 4.6.
//
// Entry points of the kernel library are handed over by address (init), so
// both paths call the one loaded library.
#include <Python.h>

#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/DispatchKeySet.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "../../../include/ntops_amd.h"

namespace {

decltype(&ntops_unary) f_unary;
decltype(&ntops_softmax) f_softmax;
decltype(&ntops_rms_norm) f_rms_norm;
decltype(&ntops_layer_norm) f_layer_norm;
decltype(&ntops_add_rms_norm) f_add_rms_norm;
decltype(&ntops_rope_qk) f_rope_qk;
decltype(&ntops_gemm_ws) f_gemm_ws;
decltype(&ntops_gemm_workspace) f_gemm_workspace;
decltype(&ntops_sdpa_ws) f_sdpa_ws;
decltype(&ntops_sdpa_workspace) f_sdpa_workspace;
decltype(&ntops_copy2) f_copy2;
decltype(&ntops_quantize_mxfp4) f_quantize_mxfp4;
decltype(&ntops_dequantize_mxfp4) f_dequantize_mxfp4;
decltype(&ntops_mxfp4_mm) f_mxfp4_mm;
decltype(&ntops_mxfp4_mm_workspace) f_mxfp4_mm_workspace;
decltype(&ntops_mxfp4_linear) f_mxfp4_linear;
decltype(&ntops_mxfp4_linear_workspace) f_mxfp4_linear_workspace;
decltype(&ntops_store_kv_cache) f_store_kv_cache;
decltype(&ntops_kv_cache_attention) f_kv_cache_attention;
decltype(&ntops_kv_cache_attention_workspace) f_kv_cache_attention_workspace;
decltype(&ntops_sliding_window_attention) f_sliding_window_attention;
decltype(&ntops_sliding_window_attention_workspace) f_sliding_window_attention_workspace;
decltype(&ntops_shared_prefix_attention) f_shared_prefix_attention;
decltype(&ntops_shared_prefix_attention_workspace) f_shared_prefix_attention_workspace;
decltype(&ntops_rope_axes_qk) f_rope_axes_qk;
bool ready = false;
PyObject* get_device = nullptr;  // torch._C._cuda_getDevice
PyObject* get_stream = nullptr;  // torch._C._cuda_getCurrentRawStream

// The dtype's code in the C ABI (F32 / F16 / BF16), else -1.
int code16_32(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return NTOPS_F32;
    case at::kHalf: return NTOPS_F16;
    case at::kBFloat16: return NTOPS_BF16;
    default: return -1;
  }
}

// The tensor of a torch.Tensor or Parameter that is an ordinary dense GPU
// tensor -- no subclass, wrapper of a transform, or lazily applied operation;
// else null.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  static const uint64_t allowed =
      c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::ADInplaceOrView, c10::DispatchKey::AutogradCUDA,
                           c10::DispatchKey::AutocastCUDA})
          .raw_repr();
  if (!t.defined() || !t.is_cuda() || (t.key_set().raw_repr() & ~allowed) != 0) return nullptr;
  return &t;
}

// Current device and its current stream; false on any error (cleared).
bool current(int64_t& device, void*& stream) {
  PyObject* d = PyObject_CallNoArgs(get_device);
  if (!d) {
    PyErr_Clear();
    return false;
  }
  PyObject* s = PyObject_CallOneArg(get_stream, d);
  device = PyLong_AsLongLong(d);
  Py_DECREF(d);
  if (!s) {
    PyErr_Clear();
    return false;
  }
  stream = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool usable() { return ready && at::impl::PythonTorchFunctionTLS::stack_len() == 0; }

bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }

at::Tensor new_like(const at::Tensor& t, c10::IntArrayRef sizes) {
  return at::empty(sizes, at::TensorOptions().dtype(t.dtype()).device(t.device()));
}
at::Tensor workspace(const at::Tensor& t, int64_t bytes) {
  return at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(t.device()));
}

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrap2(const at::Tensor& a, const at::Tensor& b) {
  PyObject* x = wrap(a);
  PyObject* y = x ? wrap(b) : nullptr;
  PyObject* r = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return r;
}
PyObject* none() { Py_RETURN_NONE; }

// The interpreter is free while a call allocates and launches (either may wait
// for the device), as it is in torch's own allocations and in ctypes calls;
// no Python object is touched inside.
class NoGil {
 public:
  NoGil() : state_(PyEval_SaveThread()) {}
  ~NoGil() { PyEval_RestoreThread(state_); }
  NoGil(const NoGil&) = delete;
  NoGil& operator=(const NoGil&) = delete;

 private:
  PyThreadState* state_;
};

// A Python float or int (not a bool) as a double.
bool number(PyObject* o, double& v) {
  if (PyFloat_CheckExact(o)) {
    v = PyFloat_AS_DOUBLE(o);
    return true;
  }
  if (PyLong_CheckExact(o)) {
    v = PyLong_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
    return true;
  }
  return false;
}

// Elements of the normalized dims when `shape` (an int, or a tuple or list of
// ints) names the input's last dims; else -1.
int64_t norm_cols(const at::Tensor& x, PyObject* shape) {
  const auto sizes = x.sizes();
  const int64_t nd = static_cast<int64_t>(sizes.size());
  if (PyLong_CheckExact(shape)) {
    const int64_t n = PyLong_AsLongLong(shape);
    if (n == -1 && PyErr_Occurred()) PyErr_Clear();
    return nd >= 1 && sizes[nd - 1] == n ? n : -1;
  }
  if (!PyTuple_Check(shape) && !PyList_CheckExact(shape)) return -1;
  const Py_ssize_t k = PySequence_Fast_GET_SIZE(shape);
  if (k < 1 || k > nd) return -1;
  int64_t cols = 1;
  for (Py_ssize_t i = 0; i < k; ++i) {
    PyObject* v = PySequence_Fast_GET_ITEM(shape, i);
    if (!PyLong_CheckExact(v)) return -1;
    const int64_t n = PyLong_AsLongLong(v);
    if (n == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return -1;
    }
    if (sizes[nd - k + i] != n) return -1;
    cols *= n;
  }
  return cols;
}

// A norm's weight or bias as one contiguous row of the normalized dims, of the
// input's dtype or fp32; `o` None leaves p null.  False: the Python path.
bool norm_param(PyObject* o, const at::Tensor& x, int64_t cols, int dev, const at::Tensor*& p) {
  p = nullptr;
  if (o == Py_None) return true;
  p = plain(o);
  if (!p || p->get_device() != dev || !p->is_contiguous() || p->numel() != cols) return false;
  if (p->scalar_type() != x.scalar_type() && p->scalar_type() != at::kFloat) return false;
  const auto ps = p->sizes(), xs = x.sizes();
  if (ps.size() > xs.size()) return false;
  for (size_t i = 0; i < ps.size(); ++i)
    if (ps[i] != xs[xs.size() - ps.size() + i]) return false;
  return true;
}

// Whatever goes wrong (out of memory, say) is left to the Python path, which
// meets it again and raises what it always has.
#define NTOPS_TRY try {
#define NTOPS_END       \
  }                     \
  catch (...) {         \
    PyErr_Clear();      \
    return none();      \
  }

// unary(op, input): a contiguous floating input into empty_like(input)
PyObject* unary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  if (n != 2 || !usable()) return none();
  const at::Tensor* x = plain(a[1]);
  int64_t dev;
  void* st;
  if (!x || code16_32(*x) < 0 || !x->is_contiguous() || x->dim() > 16 || !current(dev, st) || x->get_device() != dev)
    return none();
  const int op = static_cast<int>(PyLong_AsLong(a[0]));
  at::Tensor y;
  int rc;
  {
    NoGil free;
    y = at::empty_like(*x);
    rc = f_unary(op, code16_32(*x), static_cast<int>(x->dim()), x->sizes().data(), x->data_ptr(), x->strides().data(),
                 y.data_ptr(), y.strides().data(), st);
  }
  return rc == NTOPS_OK ? wrap(y) : none();
  NTOPS_END
}

// softmax(input, dim).  A single row has its length as the row stride here,
// where the Python path's merged strides give 1: it takes the row kernels (bf16
// (1, 131072) 70.6 -> 18.6 us), whose sums round in another order.
PyObject* softmax(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  if (n != 2 || !usable() || !PyLong_CheckExact(a[1])) return none();
  const at::Tensor* x = plain(a[0]);
  int64_t dev;
  void* st;
  if (!x || code16_32(*x) < 0 || !x->is_contiguous() || x->dim() < 1 || !current(dev, st) || x->get_device() != dev)
    return none();
  int64_t dim = PyLong_AsLongLong(a[1]);
  if (dim == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (dim < -x->dim() || dim >= x->dim()) return none();
  if (dim < 0) dim += x->dim();
  int64_t outer = 1, inner = 1;
  for (int64_t i = 0; i < dim; ++i) outer *= x->size(i);
  for (int64_t i = dim + 1; i < x->dim(); ++i) inner *= x->size(i);
  const int64_t size = x->size(dim);
  const int64_t strides[3] = {size * inner, inner, 1};
  at::Tensor y;
  int rc;
  {
    NoGil free;
    y = new_like(*x, x->sizes());
    rc = f_softmax(code16_32(*x), code16_32(*x), outer, size, inner, x->data_ptr(), strides, y.data_ptr(), strides, st);
  }
  return rc == NTOPS_OK ? wrap(y) : none();
  NTOPS_END
}

// rms_norm(input, normalized_shape, weight, eps)
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  double eps;
  if (n != 4 || !usable() || !number(a[3], eps)) return none();
  const at::Tensor* x = plain(a[0]);
  const at::Tensor* w;
  int64_t dev;
  void* st;
  if (!x || code16_32(*x) < 0 || !x->is_contiguous() || !aligned16(*x) || x->numel() == 0 || !current(dev, st) ||
      x->get_device() != dev)
    return none();
  const int64_t cols = norm_cols(*x, a[1]);
  if (cols <= 0 || !norm_param(a[2], *x, cols, static_cast<int>(dev), w)) return none();
  at::Tensor y;
  int rc;
  {
    NoGil free;
    y = new_like(*x, x->sizes());
    rc = f_rms_norm(code16_32(*x), x->numel() / cols, cols, x->data_ptr(), cols, w ? w->data_ptr() : nullptr, 0,
                    w ? code16_32(*w) : code16_32(*x), eps, y.data_ptr(), cols, st);
  }
  return rc == NTOPS_OK ? wrap(y) : none();
  NTOPS_END
}

// layer_norm(input, normalized_shape, weight, bias, eps)
PyObject* layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  double eps;
  if (n != 5 || !usable() || !number(a[4], eps)) return none();
  const at::Tensor* x = plain(a[0]);
  const at::Tensor *w, *b;
  int64_t dev;
  void* st;
  if (!x || code16_32(*x) < 0 || !x->is_contiguous() || !aligned16(*x) || x->numel() == 0 || !current(dev, st) ||
      x->get_device() != dev)
    return none();
  const int64_t cols = norm_cols(*x, a[1]);
  if (cols <= 0 || !norm_param(a[2], *x, cols, static_cast<int>(dev), w) ||
      !norm_param(a[3], *x, cols, static_cast<int>(dev), b))
    return none();
  int code = code16_32(*x);
  if (w) code = code16_32(*w);
  if (b) {
    if (w && b->scalar_type() != w->scalar_type()) return none();
    code = code16_32(*b);
  }
  at::Tensor y;
  int rc;
  {
    NoGil free;
    y = new_like(*x, x->sizes());
    rc = f_layer_norm(code16_32(*x), x->numel() / cols, cols, x->data_ptr(), cols, w ? w->data_ptr() : nullptr,
                      b ? b->data_ptr() : nullptr, 0, code, eps, y.data_ptr(), cols, st);
  }
  return rc == NTOPS_OK ? wrap(y) : none();
  NTOPS_END
}

// add_rms_norm(input, residual, normalized_shape, weight, eps)
PyObject* add_rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  double eps;
  if (n != 5 || !usable() || !number(a[4], eps)) return none();
  const at::Tensor *x = plain(a[0]), *r = plain(a[1]);
  const at::Tensor* w;
  int64_t dev;
  void* st;
  if (!x || !r || code16_32(*x) < 0 || !x->is_contiguous() || !r->is_contiguous() || !aligned16(*x) || !aligned16(*r) ||
      x->numel() == 0 || r->scalar_type() != x->scalar_type() || r->sizes() != x->sizes() || !current(dev, st) ||
      x->get_device() != dev || r->get_device() != dev)
    return none();
  const int64_t cols = norm_cols(*x, a[2]);
  if (cols <= 0 || !norm_param(a[3], *x, cols, static_cast<int>(dev), w)) return none();
  at::Tensor y, h;
  int rc;
  {
    NoGil free;
    y = new_like(*x, x->sizes());
    h = new_like(*x, x->sizes());
    rc = f_add_rms_norm(code16_32(*x), x->numel() / cols, cols, x->data_ptr(), cols, r->data_ptr(), cols,
                        w ? w->data_ptr() : nullptr, 0, w ? code16_32(*w) : code16_32(*x), eps, y.data_ptr(), cols,
                        h.data_ptr(), cols, st);
  }
  return rc == NTOPS_OK ? wrap2(y, h) : none();
  NTOPS_END
}

// rope_qk(q, k, sin, cos, interleaved)
PyObject* rope_qk(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  if (n != 5 || !usable() || !PyBool_Check(a[4])) return none();
  const at::Tensor* t[4];
  int64_t dev;
  void* st;
  if (!current(dev, st)) return none();
  for (int i = 0; i < 4; ++i) {
    t[i] = plain(a[i]);
    if (!t[i] || t[i]->get_device() != dev || t[i]->dim() != (i < 2 ? 4 : 2) ||
        t[i]->scalar_type() != t[0]->scalar_type())
      return none();
  }
  const at::Tensor &q = *t[0], &k = *t[1], &sn = *t[2], &cs = *t[3];
  const int64_t B = q.size(0), S = q.size(1), D = q.size(3), tw = sn.size(1);
  if (code16_32(q) < 0 || k.size(0) != B || k.size(1) != S || k.size(3) != D || D % 2 != 0 || sn.size(0) < S ||
      cs.size(0) < S || (tw != D && tw != D / 2) || cs.size(1) != tw || sn.stride(1) != 1 || cs.stride(1) != 1 ||
      sn.stride(0) != cs.stride(0))
    return none();
  const int interleaved = a[4] == Py_True ? 1 : 0;
  at::Tensor qo, ko;
  int rc;
  {
    NoGil free;
    qo = at::empty_like(q);
    ko = at::empty_like(k);
    rc = f_rope_qk(code16_32(q), B, S, q.size(2), k.size(2), D, q.data_ptr(), q.strides().data(), k.data_ptr(),
                   k.strides().data(), sn.data_ptr(), cs.data_ptr(), sn.stride(0), tw, interleaved, qo.data_ptr(),
                   qo.strides().data(), ko.data_ptr(), ko.strides().data(), st);
  }
  return rc == NTOPS_OK ? wrap2(qo, ko) : none();
  NTOPS_END
}

// mm(a, b) / addmm(c, a, b, beta, alpha): a K-major, b N- or K-major, both in
// 16-byte rows (what the matrix-core kernels read in place)
PyObject* gemm(const at::Tensor* c, PyObject* pa, PyObject* pb, double beta, double alpha) {
  const at::Tensor *x = plain(pa), *w = plain(pb);
  int64_t dev;
  void* st;
  if (!x || !w || code16_32(*x) < 0 || x->dim() != 2 || w->dim() != 2 || w->scalar_type() != x->scalar_type() ||
      x->size(1) != w->size(0) || !aligned16(*x) || !aligned16(*w) || !current(dev, st) || x->get_device() != dev ||
      w->get_device() != dev)
    return none();
  const int64_t M = x->size(0), K = x->size(1), N = w->size(1);
  const int64_t unit = x->scalar_type() == at::kFloat ? 4 : 8;
  if (M <= 0 || N <= unit || K <= 0 || K % unit != 0 || x->stride(1) != 1 || x->stride(0) % unit != 0) return none();
  const bool n_major = w->stride(1) == 1 && w->stride(0) % unit == 0 && N % unit == 0;
  const bool k_major = w->stride(0) == 1 && w->stride(1) != 1 && w->stride(1) % unit == 0;
  if (!n_major && !k_major) return none();
  int64_t cst[3] = {0, 0, 0};
  if (c) {
    if (c->scalar_type() != x->scalar_type() || c->get_device() != dev || c->dim() < 1 || c->dim() > 2) return none();
    const int64_t cn = c->size(c->dim() - 1), cm = c->dim() == 2 ? c->size(0) : 1;
    if ((cn != N && cn != 1) || (cm != M && cm != 1)) return none();
    cst[2] = cn == 1 && N != 1 ? 0 : c->stride(c->dim() - 1);
    cst[1] = cm == 1 && M != 1 ? 0 : c->dim() == 2 ? c->stride(0) : 0;
  }
  const int code = code16_32(*x);
  const int64_t ast[3] = {0, x->stride(0), 1}, bst[3] = {0, w->stride(0), w->stride(1)}, dst[3] = {0, N, 1};
  at::Tensor out;
  int rc;
  {
    NoGil free;
    out = new_like(*x, {M, N});
    const int64_t bytes = f_gemm_workspace(code, 1, M, N, K);
    at::Tensor ws;
    if (bytes > 0) ws = workspace(*x, bytes);
    rc = f_gemm_ws(code, 1, M, N, K, x->data_ptr(), ast, w->data_ptr(), bst, c ? c->data_ptr() : nullptr,
                   c ? cst : nullptr, alpha, beta, out.data_ptr(), dst, bytes > 0 ? ws.data_ptr() : nullptr, bytes, st);
  }
  return rc == NTOPS_OK ? wrap(out) : none();
}
PyObject* mm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  if (n != 2 || !usable()) return none();
  return gemm(nullptr, a[0], a[1], 0.0, 1.0);
  NTOPS_END
}
PyObject* addmm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  double beta, alpha;
  if (n != 5 || !usable() || !number(a[3], beta) || !number(a[4], alpha) || beta == 0.0) return none();
  const at::Tensor* c = plain(a[0]);
  return c ? gemm(c, a[1], a[2], beta, alpha) : none();
  NTOPS_END
}

// sdpa(q, k, v, mask, causal mode, scale (None: 1 / sqrt(D)), gqa, present_key,
// present_value, present_key_slot, present_value_slot)
PyObject* sdpa(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  if (n != 11 || !usable() || !PyLong_CheckExact(a[4]) || !PyBool_Check(a[6])) return none();
  const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]);
  int64_t dev;
  void* st;
  if (!q || !k || !v || q->dim() != 4 || k->dim() != 4 || v->dim() != 4 || code16_32(*q) < 0 ||
      k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || !current(dev, st) ||
      q->get_device() != dev || k->get_device() != dev || v->get_device() != dev)
    return none();
  const int64_t B = q->size(0), Hq = q->size(1), Sq = q->size(2), D = q->size(3), Hk = k->size(1), Sk = k->size(2);
  if (k->size(0) != B || v->size(0) != B || v->size(1) != Hk || v->size(2) != Sk || k->size(3) != D ||
      v->size(3) != D || D <= 0 || Hk <= 0 || (a[6] == Py_True ? Hq % Hk != 0 : Hq != Hk))
    return none();
  double scale;
  if (a[5] == Py_None)
    scale = 1.0 / std::sqrt(static_cast<double>(D));
  else if (!number(a[5], scale))
    return none();
  const at::Tensor* m = nullptr;
  int64_t mst[4] = {0, 0, 0, 0};
  int mcode = 0;
  if (a[3] != Py_None) {
    m = plain(a[3]);
    if (!m || m->get_device() != dev || m->dim() < 1 || m->dim() > 4) return none();
    mcode = m->scalar_type() == at::kBool ? NTOPS_BOOL : code16_32(*m);
    if (mcode < 0) return none();
    const int64_t full[4] = {B, Hq, Sq, Sk};
    for (int64_t i = 0; i < m->dim(); ++i) {
      const int64_t d = 4 - m->dim() + i;
      if (m->size(i) != full[d] && m->size(i) != 1) return none();
      mst[d] = m->size(i) == 1 && full[d] != 1 ? 0 : m->stride(i);
    }
  }
  const int causal = static_cast<int>(PyLong_AsLong(a[4]));
  const at::Tensor* p[4] = {};
  if (a[7] != Py_None) {
    for (int i = 0; i < 4; ++i) {  // key, value, key slot, value slot
      p[i] = plain(a[7 + i]);
      if (!p[i] || p[i]->get_device() != dev || p[i]->scalar_type() != p[0]->scalar_type() || p[i]->dim() > 16 ||
          code16_32(*p[i]) < 0 || p[i]->sizes() != p[0]->sizes())
        return none();
    }
  }
  const int code = code16_32(*q);
  at::Tensor out;
  int rc = NTOPS_OK;
  {
    NoGil free;
    if (p[0])
      rc = f_copy2(code16_32(*p[0]), static_cast<int>(p[0]->dim()), p[0]->sizes().data(), p[0]->data_ptr(),
                   p[0]->strides().data(), p[2]->data_ptr(), p[2]->strides().data(), p[1]->data_ptr(),
                   p[1]->strides().data(), p[3]->data_ptr(), p[3]->strides().data(), st);
    if (rc == NTOPS_OK) {
      out = new_like(*q, q->sizes());
      int64_t bytes = 0;
      at::Tensor ws;
      if (!m && Sq <= 16) bytes = f_sdpa_workspace(code, B, Hq, Hk, Sq, Sk, D, 0);
      if (bytes > 0) ws = workspace(*q, bytes);
      rc = f_sdpa_ws(code, B, Hq, Hk, Sq, Sk, D, q->data_ptr(), q->strides().data(), k->data_ptr(), k->strides().data(),
                     v->data_ptr(), v->strides().data(), m ? m->data_ptr() : nullptr, mcode, m ? mst : nullptr, causal,
                     scale, out.data_ptr(), out.strides().data(), bytes > 0 ? ws.data_ptr() : nullptr, bytes, st);
    }
  }
  return rc == NTOPS_OK ? wrap(out) : none();
  NTOPS_END
}

// A torch.dtype's code in the C ABI (F32 / F16 / BF16) and scalar type.
bool float_dtype(PyObject* o, int& code, at::ScalarType& type) {
  if (!THPDtype_Check(o)) return false;
  type = reinterpret_cast<THPDtype*>(o)->scalar_type;
  code = type == at::kFloat ? NTOPS_F32 : type == at::kHalf ? NTOPS_F16 : type == at::kBFloat16 ? NTOPS_BF16 : -1;
  return code >= 0;
}

at::Tensor bytes_like(const at::Tensor& t, c10::IntArrayRef sizes) {
  return at::empty(sizes, at::TensorOptions().dtype(at::kByte).device(t.device()));
}

// quantize_mxfp4(input): a contiguous input
PyObject* quantize_mxfp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  if (n != 1 || !usable()) return none();
  const at::Tensor* x = plain(a[0]);
  int64_t dev;
  void* st;
  if (!x || code16_32(*x) < 0 || x->dim() < 1 || !x->is_contiguous() || x->numel() == 0 || !current(dev, st) ||
      x->get_device() != dev)
    return none();
  const int64_t cols = x->size(-1), rows = x->numel() / cols, blocks = (cols + 31) / 32;
  auto sizes = x->sizes().vec();
  at::Tensor codes, scales;
  int rc;
  {
    NoGil free;
    sizes.back() = 16 * blocks;
    codes = bytes_like(*x, sizes);
    sizes.back() = blocks;
    scales = bytes_like(*x, sizes);
    rc = f_quantize_mxfp4(code16_32(*x), rows, cols, x->data_ptr(), cols, codes.data_ptr(), scales.data_ptr(), st);
  }
  return rc == NTOPS_OK ? wrap2(codes, scales) : none();
  NTOPS_END
}

// Blocks along the last dim of an MXFP4 pair on `dev`; -1: the Python path.
int64_t mx4_blocks(const at::Tensor* codes, const at::Tensor* scales, int64_t dev) {
  if (!codes || !scales || codes->scalar_type() != at::kByte || scales->scalar_type() != at::kByte || codes->dim() < 1 ||
      scales->dim() != codes->dim() || codes->get_device() != dev || scales->get_device() != dev)
    return -1;
  for (int64_t i = 0; i + 1 < codes->dim(); ++i)
    if (codes->size(i) != scales->size(i)) return -1;
  return codes->size(-1) == 16 * scales->size(-1) ? scales->size(-1) : -1;
}

// dequantize_mxfp4(codes, scales, size, dtype): contiguous codes and scales
PyObject* dequantize_mxfp4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  int code;
  at::ScalarType type;
  int64_t dev;
  void* st;
  if (n != 4 || !usable() || !float_dtype(a[3], code, type) || !current(dev, st)) return none();
  const at::Tensor *codes = plain(a[0]), *scales = plain(a[1]);
  const int64_t blocks = mx4_blocks(codes, scales, dev);
  if (blocks <= 0 || !codes->is_contiguous() || !scales->is_contiguous() || codes->numel() == 0 ||
      (reinterpret_cast<uintptr_t>(codes->data_ptr()) & 3u) != 0)
    return none();
  int64_t cols = 32 * blocks;
  if (a[2] != Py_None) {
    if (!PyLong_CheckExact(a[2])) return none();
    cols = PyLong_AsLongLong(a[2]);
    if (cols == -1 && PyErr_Occurred()) PyErr_Clear();
    if (cols <= 0 || (cols + 31) / 32 != blocks) return none();
  }
  auto sizes = codes->sizes().vec();
  sizes.back() = cols;
  at::Tensor y;
  int rc;
  {
    NoGil free;
    y = at::empty(sizes, at::TensorOptions().dtype(type).device(codes->device()));
    rc = f_dequantize_mxfp4(code, scales->numel() / blocks, cols, codes->data_ptr(), 16 * blocks, scales->data_ptr(), blocks,
                            y.data_ptr(), st);
  }
  return rc == NTOPS_OK ? wrap(y) : none();
  NTOPS_END
}

// mxfp4_mm(input, input_scale or None, mat2, mat2_scale, bias or None, dtype):
// code rows the kernels read in place; a float input contiguous.
PyObject* mxfp4_mm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  int code;
  at::ScalarType type;
  int64_t dev;
  void* st;
  if (n != 6 || !usable() || !float_dtype(a[5], code, type) || !current(dev, st)) return none();
  const at::Tensor *x = plain(a[0]), *w = plain(a[2]), *ws = plain(a[3]);
  const int64_t blocks = mx4_blocks(w, ws, dev);
  if (!x || x->dim() != 2 || x->get_device() != dev || blocks <= 0 || w->dim() != 2) return none();
  const auto rows16 = [](const at::Tensor& t) { return t.stride(1) == 1 && t.stride(0) >= 0 && t.stride(0) % 16 == 0 && aligned16(t); };
  const auto rows1 = [](const at::Tensor& t) { return t.stride(1) == 1 && t.stride(0) >= 0; };
  const int64_t M = x->size(0), N = w->size(0), K = 32 * blocks;
  if (M <= 0 || N <= 0 || !rows16(*w) || !rows1(*ws)) return none();
  const at::Tensor* xs = nullptr;
  if (a[1] != Py_None) {
    xs = plain(a[1]);
    if (mx4_blocks(x, xs, dev) != blocks || !rows16(*x) || !rows1(*xs)) return none();
  } else if (code16_32(*x) < 0 || !x->is_contiguous() || (x->size(1) + 31) / 32 != blocks) {
    return none();
  }
  const at::Tensor* bias = nullptr;
  if (a[4] != Py_None) {
    bias = plain(a[4]);
    if (!bias || bias->get_device() != dev || bias->scalar_type() != type || bias->dim() != 1 || bias->size(0) != N ||
        !bias->is_contiguous())
      return none();
  }
  at::Tensor out;
  int rc;
  {
    NoGil free;
    out = at::empty({M, N}, at::TensorOptions().dtype(type).device(x->device()));
    const int64_t cols = x->size(1);
    const int64_t bytes = xs ? f_mxfp4_mm_workspace(M, N, K)
                             : f_mxfp4_linear_workspace(code16_32(*x), M, N, cols, x->data_ptr(), cols);
    at::Tensor tmp;
    if (bytes > 0) tmp = workspace(*x, bytes);
    void* at = bytes > 0 ? tmp.data_ptr() : nullptr;
    const void* b = bias ? bias->data_ptr() : nullptr;
    rc = xs ? f_mxfp4_mm(code, M, N, K, x->data_ptr(), x->stride(0), xs->data_ptr(), xs->stride(0), w->data_ptr(), w->stride(0),
                         ws->data_ptr(), ws->stride(0), b, out.data_ptr(), N, at, bytes, st)
            : f_mxfp4_linear(code16_32(*x), code, M, N, cols, x->data_ptr(), cols, w->data_ptr(), w->stride(0), ws->data_ptr(),
                             ws->stride(0), b, out.data_ptr(), N, at, bytes, st);
  }
  return rc == NTOPS_OK ? wrap(out) : none();
  NTOPS_END
}

// A cache (key_cache, value_cache, key_scale, value_scale) at a[0 ..] in layouts
// that need no copy.
struct Cache {
  const at::Tensor* t[4];
  int64_t B, H, C, D;
  bool read(PyObject* const* a, int64_t block, int64_t dev) {
    if (block < 16 || (block & (block - 1)) != 0) return false;
    for (int i = 0; i < 4; ++i) {
      t[i] = plain(a[i]);
      if (!t[i] || t[i]->get_device() != dev || t[i]->scalar_type() != (i < 2 ? at::kFloat8_e4m3fn : at::kFloat) ||
          t[i]->dim() != (i < 2 ? 4 : 3) || t[i]->numel() == 0 || t[i]->stride(-1) != 1)
        return false;
      for (int64_t d = 0; d < t[i]->dim(); ++d)
        if (t[i]->stride(d) == 0 && t[i]->size(d) > 1) return false;
    }
    B = t[0]->size(0);
    H = t[0]->size(1);
    C = t[0]->size(2);
    D = t[0]->size(3);
    const int64_t s[3] = {B, H, (C + block - 1) / block};
    return t[1]->sizes() == t[0]->sizes() && t[2]->sizes() == c10::IntArrayRef(s, 3) && t[3]->sizes() == t[2]->sizes();
  }
};

// A block size given as an int; -1, which no cache has, if it is past 64 bits.
int64_t block_of(PyObject* o) {
  const int64_t block = PyLong_AsLongLong(o);
  if (block == -1 && PyErr_Occurred()) PyErr_Clear();
  return block;
}

// An index vector (batch,) or None; false: the Python path.
bool index_vector(PyObject* o, int64_t batch, int64_t dev, const at::Tensor*& t, int& code) {
  t = nullptr;
  code = 0;
  if (o == Py_None) return true;
  t = plain(o);
  if (!t || t->get_device() != dev || t->dim() != 1 || t->size(0) != batch || !t->is_contiguous()) return false;
  code = t->scalar_type() == at::kInt ? NTOPS_I32 : t->scalar_type() == at::kLong ? NTOPS_I64 : -1;
  return code >= 0;
}

// store_kv_cache(key, value, key_cache, value_cache, key_scale, value_scale,
// positions (int or tensor), lengths or None, block_size): True when stored
PyObject* store_kv_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  int64_t dev;
  void* st;
  if (n != 9 || !usable() || !PyLong_CheckExact(a[8]) || !current(dev, st)) return none();
  const int64_t block = block_of(a[8]);
  Cache c;
  const at::Tensor *k = plain(a[0]), *v = plain(a[1]), *pos = nullptr, *len = nullptr;
  if (!k || !v || !c.read(a + 2, block, dev) || k->dim() != 4 || v->sizes() != k->sizes() || code16_32(*k) < 0 ||
      v->scalar_type() != k->scalar_type() || k->get_device() != dev || v->get_device() != dev || k->size(0) != c.B ||
      k->size(1) != c.H || k->size(2) <= 0 || k->size(3) != c.D || k->stride(3) != 1 || v->stride(3) != 1)
    return none();
  int64_t position = 0;
  int pcode = 0, lcode;
  if (PyLong_CheckExact(a[6])) {
    position = PyLong_AsLongLong(a[6]);
    if (position == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return none();
    }
  } else if (a[6] == Py_None || !index_vector(a[6], c.B, dev, pos, pcode)) {
    return none();
  }
  if (!index_vector(a[7], c.B, dev, len, lcode)) return none();
  int rc;
  {
    NoGil free;
    rc = f_store_kv_cache(code16_32(*k), c.B, c.H, k->size(2), c.D, c.C, block, k->data_ptr(), k->strides().data(), v->data_ptr(),
                          v->strides().data(), c.t[0]->data_ptr(), c.t[0]->strides().data(), c.t[1]->data_ptr(),
                          c.t[1]->strides().data(), static_cast<float*>(c.t[2]->data_ptr()), c.t[2]->strides().data(),
                          static_cast<float*>(c.t[3]->data_ptr()), c.t[3]->strides().data(), pos ? pos->data_ptr() : nullptr,
                          pcode, position, len ? len->data_ptr() : nullptr, lcode, st);
  }
  if (rc != NTOPS_OK) return none();
  Py_RETURN_TRUE;
  NTOPS_END
}

// kv_cache_attention(query, key_cache, value_cache, key_scale, value_scale,
// lengths or None, is_causal, scale (None: 1 / sqrt(D)), block_size)
PyObject* kv_cache_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  int64_t dev;
  void* st;
  if (n != 9 || !usable() || !PyBool_Check(a[6]) || !PyLong_CheckExact(a[8]) || !current(dev, st)) return none();
  const int64_t block = block_of(a[8]);
  Cache c;
  const at::Tensor *q = plain(a[0]), *len = nullptr;
  int lcode;
  if (!q || !c.read(a + 1, block, dev) || q->dim() != 4 || code16_32(*q) < 0 || q->get_device() != dev || q->numel() == 0 ||
      q->size(0) != c.B || q->size(3) != c.D || q->stride(3) != 1 || q->size(1) % c.H != 0 ||
      !index_vector(a[5], c.B, dev, len, lcode))
    return none();
  double scale;
  if (a[7] == Py_None)
    scale = 1.0 / std::sqrt(static_cast<double>(c.D));
  else if (!number(a[7], scale))
    return none();
  const int code = code16_32(*q);
  const int64_t Hq = q->size(1), Sq = q->size(2);
  at::Tensor out;
  int rc;
  {
    NoGil free;
    out = new_like(*q, q->sizes());
    const int64_t bytes = f_kv_cache_attention_workspace(code, c.B, Hq, c.H, Sq, c.C, c.D);
    at::Tensor ws;
    if (bytes > 0) ws = workspace(*q, bytes);
    rc = f_kv_cache_attention(code, c.B, Hq, c.H, Sq, c.C, c.D, block, q->data_ptr(), q->strides().data(), c.t[0]->data_ptr(),
                              c.t[0]->strides().data(), c.t[1]->data_ptr(), c.t[1]->strides().data(),
                              static_cast<const float*>(c.t[2]->data_ptr()), c.t[2]->strides().data(),
                              static_cast<const float*>(c.t[3]->data_ptr()), c.t[3]->strides().data(),
                              len ? len->data_ptr() : nullptr, lcode, a[6] == Py_True ? 1 : 0, scale, out.data_ptr(),
                              out.strides().data(), bytes > 0 ? ws.data_ptr() : nullptr, bytes, st);
  }
  return rc == NTOPS_OK ? wrap(out) : none();
  NTOPS_END
}

// A Python int (not a bool); false: the Python path, as for one past 64 bits.
bool integer(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// Query, key and value (a[0], a[i], a[i + 1]) of attention in one type, with unit strides
// along the head dim.
struct Attention {
  const at::Tensor *q, *k, *v;
  int64_t B, Hq, H, Sq, C, D;
  int code;
  bool read(PyObject* const* a, int i, int64_t dev) {
    q = plain(a[0]);
    k = plain(a[i]);
    v = plain(a[i + 1]);
    if (!q || !k || !v || q->dim() != 4 || k->dim() != 4 || v->sizes() != k->sizes() || (code = code16_32(*q)) < 0 ||
        q->numel() == 0 || k->numel() == 0 || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() ||
        q->get_device() != dev || k->get_device() != dev || v->get_device() != dev || q->stride(3) != 1)
      return false;
    B = q->size(0);
    Hq = q->size(1);
    Sq = q->size(2);
    D = q->size(3);
    H = k->size(1);
    C = k->size(2);
    return k->size(0) == B && k->size(3) == D && Hq % H == 0;
  }
  bool scale(PyObject* o, double& s) const {
    if (o != Py_None) return number(o, s);
    s = 1.0 / std::sqrt(static_cast<double>(D));
    return true;
  }
};

// sliding_window_attention(query, key, value, window, sinks, lengths or None, scale or None)
PyObject* sliding_window_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  int64_t dev, window, sinks;
  void* st;
  if (n != 7 || !usable() || !integer(a[3], window) || !integer(a[4], sinks) || window < 1 || sinks < 0 || !current(dev, st))
    return none();
  Attention t;
  const at::Tensor* len;
  int lcode;
  double scale;
  if (!t.read(a, 1, dev) || !index_vector(a[5], t.B, dev, len, lcode) || !t.scale(a[6], scale)) return none();
  at::Tensor out;
  int rc;
  {
    NoGil free;
    out = new_like(*t.q, t.q->sizes());
    const int64_t bytes = f_sliding_window_attention_workspace(t.code, t.B, t.Hq, t.H, t.Sq, t.C, t.D, window, sinks);
    at::Tensor ws;
    if (bytes > 0) ws = workspace(*t.q, bytes);
    rc = f_sliding_window_attention(t.code, t.B, t.Hq, t.H, t.Sq, t.C, t.D, t.q->data_ptr(), t.q->strides().data(), t.k->data_ptr(),
                                    t.k->strides().data(), t.v->data_ptr(), t.v->strides().data(), len ? len->data_ptr() : nullptr,
                                    lcode, window, sinks, scale, out.data_ptr(), out.strides().data(),
                                    bytes > 0 ? ws.data_ptr() : nullptr, bytes, st);
  }
  return rc == NTOPS_OK ? wrap(out) : none();
  NTOPS_END
}

// shared_prefix_attention(query, prefix_key, prefix_value, key, value, prefix_lengths or
// None, lengths or None, scale or None)
PyObject* shared_prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  int64_t dev;
  void* st;
  if (n != 8 || !usable() || !current(dev, st)) return none();
  Attention t;
  const at::Tensor *pk = plain(a[1]), *pv = plain(a[2]), *plen, *len;
  int pcode, lcode;
  double scale;
  if (!pk || !pv || !t.read(a, 3, dev) || pk->dim() != 4 || pv->sizes() != pk->sizes() || pk->numel() == 0 ||
      pk->scalar_type() != t.q->scalar_type() || pv->scalar_type() != t.q->scalar_type() || pk->get_device() != dev ||
      pv->get_device() != dev || pk->size(1) != t.H || pk->size(3) != t.D || t.B % pk->size(0) != 0 ||
      !index_vector(a[5], pk->size(0), dev, plen, pcode) || !index_vector(a[6], t.B, dev, len, lcode) || !t.scale(a[7], scale))
    return none();
  const int64_t G = pk->size(0), P = pk->size(2);
  at::Tensor out;
  int rc;
  {
    NoGil free;
    out = new_like(*t.q, t.q->sizes());
    const int64_t bytes = f_shared_prefix_attention_workspace(t.code, G, t.B, t.Hq, t.H, t.Sq, P, t.C, t.D);
    at::Tensor ws;
    if (bytes > 0) ws = workspace(*t.q, bytes);
    rc = f_shared_prefix_attention(t.code, G, t.B, t.Hq, t.H, t.Sq, P, t.C, t.D, t.q->data_ptr(), t.q->strides().data(),
                                   pk->data_ptr(), pk->strides().data(), pv->data_ptr(), pv->strides().data(),
                                   plen ? plen->data_ptr() : nullptr, pcode, t.k->data_ptr(), t.k->strides().data(), t.v->data_ptr(),
                                   t.v->strides().data(), len ? len->data_ptr() : nullptr, lcode, scale, out.data_ptr(),
                                   out.strides().data(), bytes > 0 ? ws.data_ptr() : nullptr, bytes, st);
  }
  return rc == NTOPS_OK ? wrap(out) : none();
  NTOPS_END
}

// rope_axes_qk(q, k, sin, cos, positions, sections (a list or tuple of ints), interleaved, inplace = False)
PyObject* rope_axes_qk(PyObject*, PyObject* const* a, Py_ssize_t n) {
  NTOPS_TRY
  if ((n != 7 && n != 8) || !usable() || !PyBool_Check(a[6]) || (n == 8 && !PyBool_Check(a[7])) || (!PyTuple_CheckExact(a[5]) && !PyList_CheckExact(a[5]))) return none();
  const at::Tensor* t[5];
  int64_t dev;
  void* st;
  if (!current(dev, st)) return none();
  for (int i = 0; i < 5; ++i) {
    t[i] = plain(a[i]);
    if (!t[i] || t[i]->get_device() != dev || t[i]->dim() != (i < 2 ? 4 : i < 4 ? 2 : 3) || t[i]->numel() == 0) return none();
  }
  const at::Tensor &q = *t[0], &k = *t[1], &sn = *t[2], &cs = *t[3], &pos = *t[4];
  const int64_t B = q.size(0), S = q.size(1), D = q.size(3), tw = sn.size(1);
  const int code = code16_32(q), tcode = code16_32(sn);
  const int pcode = pos.scalar_type() == at::kInt ? NTOPS_I32 : pos.scalar_type() == at::kLong ? NTOPS_I64 : -1;
  if (code < 0 || k.scalar_type() != q.scalar_type() || k.size(0) != B || k.size(1) != S || k.size(3) != D || D % 2 != 0 ||
      cs.sizes() != sn.sizes() || cs.scalar_type() != sn.scalar_type() || (tcode != NTOPS_F32 && tcode != code) ||
      (tw != D && tw != D / 2) || sn.stride(1) != 1 || cs.stride(1) != 1 || pcode < 0 || pos.size(1) != B || pos.size(2) != S)
    return none();
  int64_t sections[256];
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(a[5]);
  if (count > 256) return none();
  for (Py_ssize_t i = 0; i < count; ++i)
    if (!integer(PySequence_Fast_GET_ITEM(a[5], i), sections[i])) return none();
  const bool inplace = n == 8 && a[7] == Py_True;
  at::Tensor qo, ko;
  int rc;
  {
    NoGil free;
    qo = inplace ? q : new_like(q, q.sizes());
    ko = inplace ? k : new_like(k, k.sizes());
    rc = f_rope_axes_qk(code, B, S, q.size(2), k.size(2), D, q.data_ptr(), q.strides().data(), k.data_ptr(), k.strides().data(), tcode,
                        sn.data_ptr(), sn.stride(0), cs.data_ptr(), cs.stride(0), sn.size(0), tw, pos.size(0), pos.data_ptr(), pcode,
                        pos.strides().data(), count, sections, a[6] == Py_True ? 1 : 0, qo.data_ptr(), qo.strides().data(),
                        ko.data_ptr(), ko.strides().data(), st);
  }
  return rc == NTOPS_OK ? wrap2(qo, ko) : none();
  NTOPS_END
}

// init({name: address}, get_device, get_stream)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3 || !PyDict_Check(a[0])) {
    PyErr_SetString(PyExc_TypeError, "init(addresses, get_device, get_stream)");
    return nullptr;
  }
  ready = false;
  const auto set = [&](const char* name, auto& fn) {
    PyObject* v = PyDict_GetItemString(a[0], name);
    void* p = v ? PyLong_AsVoidPtr(v) : nullptr;
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(p);
    return p != nullptr;
  };
  const bool all = set("ntops_unary", f_unary) & set("ntops_softmax", f_softmax) & set("ntops_rms_norm", f_rms_norm) &
                   set("ntops_layer_norm", f_layer_norm) & set("ntops_add_rms_norm", f_add_rms_norm) &
                   set("ntops_rope_qk", f_rope_qk) & set("ntops_gemm_ws", f_gemm_ws) &
                   set("ntops_gemm_workspace", f_gemm_workspace) & set("ntops_sdpa_ws", f_sdpa_ws) &
                   set("ntops_sdpa_workspace", f_sdpa_workspace) & set("ntops_copy2", f_copy2) &
                   set("ntops_quantize_mxfp4", f_quantize_mxfp4) & set("ntops_dequantize_mxfp4", f_dequantize_mxfp4) &
                   set("ntops_mxfp4_mm", f_mxfp4_mm) & set("ntops_mxfp4_mm_workspace", f_mxfp4_mm_workspace) &
                   set("ntops_mxfp4_linear", f_mxfp4_linear) & set("ntops_mxfp4_linear_workspace", f_mxfp4_linear_workspace) &
                   set("ntops_store_kv_cache", f_store_kv_cache) & set("ntops_kv_cache_attention", f_kv_cache_attention) &
                   set("ntops_kv_cache_attention_workspace", f_kv_cache_attention_workspace) &
                   set("ntops_sliding_window_attention", f_sliding_window_attention) &
                   set("ntops_sliding_window_attention_workspace", f_sliding_window_attention_workspace) &
                   set("ntops_shared_prefix_attention", f_shared_prefix_attention) &
                   set("ntops_shared_prefix_attention_workspace", f_shared_prefix_attention_workspace) &
                   set("ntops_rope_axes_qk", f_rope_axes_qk);
  if (PyErr_Occurred()) return nullptr;
  Py_INCREF(a[1]);
  Py_INCREF(a[2]);
  Py_XDECREF(get_device);
  Py_XDECREF(get_stream);
  get_device = a[1];
  get_stream = a[2];
  ready = all;
  return PyBool_FromLong(all);
}

#define NTOPS_M(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {NTOPS_M(init),         NTOPS_M(unary),   NTOPS_M(softmax), NTOPS_M(rms_norm), NTOPS_M(layer_norm),
                         NTOPS_M(add_rms_norm), NTOPS_M(rope_qk), NTOPS_M(mm),      NTOPS_M(addmm),    NTOPS_M(sdpa),
                         NTOPS_M(quantize_mxfp4), NTOPS_M(dequantize_mxfp4), NTOPS_M(mxfp4_mm), NTOPS_M(store_kv_cache),
                         NTOPS_M(kv_cache_attention), NTOPS_M(sliding_window_attention), NTOPS_M(shared_prefix_attention),
                         NTOPS_M(rope_axes_qk), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fast", "native host path of the torch wrappers", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fast(void) { return PyModule_Create(&module); }
