// The Python package's calls, from tensors to the C ABI, in native code.
//
// A decode step is a dozen launches of a few microseconds and the attention calls of an image model are not much
// longer: reading shapes and strides through Python objects, packing a descriptor and converting a dozen arguments
// for ctypes costs 6 to 12 us a call, more than such a kernel runs.  Each function here does for well-formed
// arguments exactly what its Python twin in __init__.py does.  Whatever it does not recognise at once (another type
// than a plain CUDA tensor, shapes or strides that the twin would refuse, scratch that has to be allocated) it
// answers with None and leaves to the twin, which also words the errors.  Nothing is kept from one call to the next.
#include <Python.h>

#include <ATen/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DispatchKeySet.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "ixk.h"

namespace {

decltype(&ixk_gemm) g_gemm;
decltype(&ixk_gemm_fp8) g_gemm_fp8;
decltype(&ixk_gemm_workspace_bytes) g_gemm_bytes;
decltype(&ixk_gemm_geglu) g_geglu;
decltype(&ixk_fmha_fwd) g_fwd;
decltype(&ixk_fmha_fwd_workspace_bytes) g_fwd_bytes;
decltype(&ixk_fmha_bwd) g_bwd;
decltype(&ixk_fmha_bwd_workspace_bytes) g_bwd_bytes;
decltype(&ixk_row_norm) g_row_norm;
decltype(&ixk_row_norm_gain) g_row_norm_gain;
decltype(&ixk_rotary_interleaved) g_rotary, g_rotary_half;
decltype(&ixk_kv_append) g_kv_append;
decltype(&ixk_residual_add) g_residual_add;
decltype(&ixk_row_norm_fwd) g_norm_fwd;
decltype(&ixk_row_norm_bwd) g_norm_bwd;
decltype(&ixk_row_norm_bwd_workspace_bytes) g_norm_bwd_bytes;
decltype(&ixk_linear_xent_fwd) g_xent_fwd;
decltype(&ixk_linear_xent_bwd) g_xent_bwd;
decltype(&ixk_linear_distill_fwd) g_distill_fwd;
decltype(&ixk_linear_distill_bwd) g_distill_bwd;
decltype(&ixk_linear_loss_workspace_bytes) g_loss_bytes;
decltype(&ixk_paged_extend) g_extend;
decltype(&ixk_paged_keep) g_keep;
decltype(&ixk_qk_norm_rotary_fwd) g_qk_fwd;
decltype(&ixk_qk_norm_rotary_bwd) g_qk_bwd;
decltype(&ixk_qk_norm_rotary_bwd_workspace_bytes) g_qk_bwd_bytes;
decltype(&ixk_fmha_paged_fwd) g_paged_fwd;
decltype(&ixk_fmha_paged_fwd_workspace_bytes) g_paged_fwd_bytes;

// A plain CUDA tensor, nullptr for anything else (None included; see `optional`).
const at::Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  constexpr c10::DispatchKeySet special({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                         c10::DispatchKey::Functionalize, c10::DispatchKey::Python, c10::DispatchKey::Conjugate,
                                         c10::DispatchKey::Negative, c10::DispatchKey::ZeroTensor});
  if (!t.defined() || !t.is_cuda() || t.layout() != c10::kStrided || t.key_set().has_any(special) ||
      t.unsafeGetTensorImpl()->has_symbolic_sizes_strides())
    return nullptr;
  return &t;
}
// An argument that may be None: false if it is neither None nor a plain CUDA tensor.
bool optional(PyObject* o, const at::Tensor** t) {
  *t = nullptr;
  return o == Py_None || (*t = tensor(o)) != nullptr;
}
void* ptr(const at::Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }
size_t size_of(const at::Tensor* t) { return t == nullptr ? 0 : t->nbytes(); }

int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return IXK_BF16;
    case at::kHalf: return IXK_F16;
    case at::kFloat: return IXK_F32;
    case at::kFloat8_e4m3fn: return IXK_F8E4M3;
    case at::kFloat8_e5m2: return IXK_F8E5M2;
    case at::kChar: return IXK_S8;
    case at::kInt: return IXK_S32;
    default: return -1;
  }
}

// A stream object, or None for torch's current stream on the current device.
bool stream_arg(PyObject* o, void** s) {
  if (o == Py_None) {
    *s = c10::cuda::getCurrentCUDAStream().stream();
    return true;
  }
  PyObject* handle = PyObject_GetAttrString(o, "cuda_stream");
  *s = handle != nullptr ? PyLong_AsVoidPtr(handle) : nullptr;
  Py_XDECREF(handle);
  if (PyErr_Occurred() == nullptr) return true;
  PyErr_Clear();
  return false;
}
bool number(PyObject* o, double* v) {
  if (PyFloat_CheckExact(o)) *v = PyFloat_AS_DOUBLE(o);
  else if (PyLong_CheckExact(o)) *v = PyLong_AsDouble(o);
  else return false;
  if (PyErr_Occurred() == nullptr) return true;
  PyErr_Clear();
  return false;
}
bool integer(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (PyErr_Occurred() == nullptr) return true;
  PyErr_Clear();
  return false;
}

template <typename Call>
int unlocked(const Call& call) {   // the library's calls run without the interpreter's lock, as under ctypes
  int st;
  Py_BEGIN_ALLOW_THREADS
  st = call();
  Py_END_ALLOW_THREADS
  return st;
}
PyObject* status(int st) { return PyLong_FromLong(st); }
// The result tensor, or the status where it is not OK.
PyObject* result(int st, PyObject* given, const at::Tensor& made) {
  if (st != IXK_OK) return status(st);
  if (given == Py_None) return THPVariable_Wrap(made);
  Py_INCREF(given);
  return given;
}

// _matrix_layout: whichever of the last two dimensions has stride 1 decides the order.
bool layout(const at::Tensor& t, ixk_matrix_layout* l) {
  const int64_t d = t.dim();
  if (d != 2 && d != 3) return false;
  const int64_t rows = t.size(d - 2), cols = t.size(d - 1), sr = t.stride(d - 2), sc = t.stride(d - 1);
  if (sc == 1 && (sr >= cols || rows == 1)) {
    l->order = IXK_ROW_MAJOR;
    l->leading_dim_stride = rows > 1 ? sr : std::max(sr, cols);
  } else if (sr == 1 && (sc >= rows || cols == 1)) {
    l->order = IXK_COL_MAJOR;
    l->leading_dim_stride = cols > 1 ? sc : std::max(sc, rows);
  } else {
    return false;
  }
  l->dtype = dtype_of(t);
  l->num_rows = rows;
  l->num_cols = cols;
  l->batch_stride = d == 3 ? t.stride(0) : rows * cols;
  return l->dtype >= 0;
}

// _require_c: C lies in memory as the result does, dimensions of one entry aside.
bool lies_alike(const at::Tensor& c, const at::Tensor& out) {
  if (c.scalar_type() != out.scalar_type() || c.numel() != out.numel()) return false;
  int64_t i = 0, j = 0;
  for (;; ++i, ++j) {
    while (i < c.dim() && c.size(i) == 1) ++i;
    while (j < out.dim() && out.size(j) == 1) ++j;
    if (i == c.dim() || j == out.dim()) break;
    if (c.size(i) != out.size(j) || c.stride(i) != out.stride(j)) break;
  }
  if (i == c.dim() && j == out.dim()) return true;
  return c.is_contiguous() && out.is_contiguous() && (c.dim() < 2 || c.size(c.dim() - 1) == out.size(out.dim() - 1));
}

#define IXK_PY_FUNCTION(name, count)                             \
  PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n) {  \
    HANDLE_TH_ERRORS                                             \
    if (n != (count)) Py_RETURN_NONE;
#define IXK_PY_END     \
  END_HANDLE_TH_ERRORS \
  }

// lhs, rhs, bias, c, out, out dtype, alpha, beta, epilogue, workspace, stream, inv_scale_a, inv_scale_b
IXK_PY_FUNCTION(py_gemm, 13)
  const at::Tensor *lhs = tensor(a[0]), *rhs = tensor(a[1]), *bias, *c, *out, *ws;
  double alpha, beta;
  int64_t epilogue;
  void* stream;
  if (lhs == nullptr || rhs == nullptr || !optional(a[2], &bias) || !optional(a[3], &c) || !optional(a[4], &out) ||
      !number(a[6], &alpha) || !number(a[7], &beta) || !integer(a[8], &epilogue) || !optional(a[9], &ws) || !stream_arg(a[10], &stream))
    Py_RETURN_NONE;
  double sa = 1.0, sb = 1.0;
  const bool fp8 = a[11] != Py_None || a[12] != Py_None;
  if (fp8 && (!number(a[11], &sa) || !number(a[12], &sb) || (out == nullptr && a[5] == Py_None))) Py_RETURN_NONE;
  ixk_gemm_desc d{};
  if (!layout(*lhs, &d.lhs) || !layout(*rhs, &d.rhs)) Py_RETURN_NONE;
  at::Tensor made;
  if (out == nullptr) {
    at::ScalarType type = lhs->scalar_type();
    if (a[5] != Py_None) {
      if (!THPDtype_Check(a[5])) Py_RETURN_NONE;
      type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
    }
    c10::SmallVector<int64_t, 3> shape(lhs->sizes().begin(), lhs->sizes().end());
    shape.back() = rhs->size(rhs->dim() - 1);
    made = at::empty(shape, at::TensorOptions().device(lhs->device()).dtype(type));
    out = &made;
  }
  if (!layout(*out, &d.output)) Py_RETURN_NONE;
  d.batch_size = out->dim() == 3 ? out->size(0) : 1;
  d.alpha = static_cast<float>(alpha);
  d.beta = static_cast<float>(beta);
  d.epilogue = static_cast<int32_t>(epilogue);
  if (c != nullptr && d.beta != 0.0f && !lies_alike(*c, *out)) Py_RETURN_NONE;
  // An fp8 call that makes its own result takes the scratch it can use as well, from the pool of the stream it was given
  // (where that is not the current one the twin does).
  at::Tensor own;
  if (fp8 && ws == nullptr && a[4] == Py_None) {
    if (const size_t need = g_gemm_bytes(&d)) {
      if (a[10] != Py_None) Py_RETURN_NONE;
      try {
        own = at::empty({static_cast<int64_t>(need)}, at::TensorOptions().device(lhs->device()).dtype(at::kByte));
        ws = &own;
      } catch (const c10::OutOfMemoryError&) {   // it runs without
      }
    }
  }
  const size_t bytes = size_of(ws);
  void *pa = ptr(lhs), *pb = ptr(rhs), *pc = ptr(c), *pbias = ptr(bias), *pd = ptr(out), *pw = ptr(ws);
  const int st = unlocked([&] {
    return fp8 ? g_gemm_fp8(&d, pa, pb, pc, pbias, pd, static_cast<float>(sa), static_cast<float>(sb), pw, bytes, stream)
               : g_gemm(&d, pa, pb, pc, pbias, pd, pw, bytes, stream);
  });
  return result(st, a[4], made);
IXK_PY_END

// x, w_gate_up, out, workspace, stream
IXK_PY_FUNCTION(py_geglu, 5)
  const at::Tensor *x = tensor(a[0]), *w = tensor(a[1]), *out, *ws = tensor(a[3]);
  void* stream;
  if (x == nullptr || w == nullptr || !optional(a[2], &out) || ws == nullptr || !stream_arg(a[4], &stream)) Py_RETURN_NONE;
  ixk_gemm_desc d{};
  if (!layout(*x, &d.lhs) || !layout(*w, &d.rhs)) Py_RETURN_NONE;
  const int64_t m = x->size(x->dim() - 2), n2 = w->size(w->dim() - 1);
  at::Tensor made;
  if (out == nullptr) {
    made = at::empty({m, n2 / 2}, at::TensorOptions().device(x->device()).dtype(x->scalar_type()));
    out = &made;
  } else if (out->dim() < 2) {
    Py_RETURN_NONE;
  }
  d.output = ixk_matrix_layout{IXK_ROW_MAJOR, d.lhs.dtype, m, n2, m * n2, n2};
  d.batch_size = 1;
  d.alpha = 1.0f;
  void *px = ptr(x), *pw = ptr(w), *po = ptr(out), *scratch = ptr(ws);
  const int64_t ld = out->stride(out->dim() - 2);
  const size_t bytes = ws->nbytes();
  const int st = unlocked([&] { return g_geglu(&d, px, pw, po, ld, scratch, bytes, stream); });
  return result(st, a[2], made);
IXK_PY_END

// _fmha_desc
bool fmha_desc(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor* bias, const at::Tensor& out, double scale,
               bool causal, ixk_fmha_desc* d) {
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || out.dim() != 4) return false;
  const int64_t B = q.size(0), N = q.size(1), F = q.size(2), H = q.size(3), T = k.size(2);
  if (k.size(0) != B || k.size(1) != N || k.size(3) != H || v.sizes() != k.sizes() || out.sizes() != q.sizes()) return false;
  if (B > INT32_MAX || N > INT32_MAX || F > INT32_MAX || T > INT32_MAX || H > INT32_MAX) return false;
  const at::ScalarType type = q.scalar_type();
  if (k.scalar_type() != type || v.scalar_type() != type || out.scalar_type() != type) return false;
  if (H > 1 && (q.stride(3) != 1 || k.stride(3) != 1 || v.stride(3) != 1 || out.stride(3) != 1)) return false;
  *d = ixk_fmha_desc{};
  if (bias != nullptr) {
    if (bias->scalar_type() != type || bias->dim() != 4 || bias->size(3) != T || bias->size(2) != F || bias->stride(3) != 1) return false;
    d->bias_strides[0] = bias->size(0) > 1 ? bias->stride(0) : 0;
    d->bias_strides[1] = bias->size(1) > 1 ? bias->stride(1) : 0;
    d->bias_strides[2] = bias->stride(2);
  }
  d->dtype = dtype_of(q);
  if (d->dtype < 0) return false;
  d->causal = causal ? 1 : 0;
  d->num_batches = static_cast<int32_t>(B);
  d->num_heads = static_cast<int32_t>(N);
  d->head_size = static_cast<int32_t>(H);
  d->num_queries = static_cast<int32_t>(F);
  d->num_keys = static_cast<int32_t>(T);
  d->head_scale = static_cast<float>(scale);
  for (int i = 0; i < 3; ++i) {
    d->q_strides[i] = q.stride(i);
    d->k_strides[i] = k.stride(i);
    d->v_strides[i] = v.stride(i);
    d->o_strides[i] = out.stride(i);
  }
  return true;
}

// q, k, v, bias, out, log-sum-exp rows, scale, causal, workspace, stream
IXK_PY_FUNCTION(py_fmha_forward, 10)
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *bias, *out = tensor(a[4]), *lse, *ws;
  double scale;
  void* stream;
  ixk_fmha_desc d;
  if (q == nullptr || k == nullptr || v == nullptr || !optional(a[3], &bias) || out == nullptr || !optional(a[5], &lse) ||
      !number(a[6], &scale) || !PyBool_Check(a[7]) || !optional(a[8], &ws) || !stream_arg(a[9], &stream) ||
      !fmha_desc(*q, *k, *v, bias, *out, scale, a[7] == Py_True, &d))
    Py_RETURN_NONE;
  const size_t bytes = size_of(ws);
  if (g_fwd_bytes(&d) > bytes) Py_RETURN_NONE;   // (the twin allocates)
  void *pq = ptr(q), *pk = ptr(k), *pv = ptr(v), *pb = ptr(bias), *po = ptr(out), *pl = ptr(lse), *pw = ptr(ws);
  return status(unlocked([&] { return g_fwd(&d, pq, pk, pv, pb, po, static_cast<float*>(pl), pw, bytes, stream); }));
IXK_PY_END

// q, k, v, out, bias, grad_out, log-sum-exp rows, dq, dk, dv, scale, causal, workspace, stream
IXK_PY_FUNCTION(py_fmha_backward, 14)
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *out = tensor(a[3]), *bias, *go = tensor(a[5]),
                   *lse = tensor(a[6]), *dq = tensor(a[7]), *dk = tensor(a[8]), *dv = tensor(a[9]), *ws = tensor(a[12]);
  double scale;
  void* stream;
  ixk_fmha_bwd_desc d{};
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || !optional(a[4], &bias) || go == nullptr || lse == nullptr ||
      dq == nullptr || dk == nullptr || dv == nullptr || !number(a[10], &scale) || !PyBool_Check(a[11]) || ws == nullptr ||
      !stream_arg(a[13], &stream) || !fmha_desc(*q, *k, *v, bias, *out, scale, a[11] == Py_True, &d.fwd))
    Py_RETURN_NONE;
  if (lse->scalar_type() != at::kFloat || !lse->is_contiguous() || lse->dim() != 3 || lse->sizes() != q->sizes().slice(0, 3)) Py_RETURN_NONE;
  const at::Tensor* grads[4] = {go, dq, dk, dv};
  const at::Tensor* like[4] = {q, q, k, v};
  int64_t* strides[4] = {d.do_strides, d.dq_strides, d.dk_strides, d.dv_strides};
  for (int i = 0; i < 4; ++i) {
    const at::Tensor& t = *grads[i];
    if (t.sizes() != like[i]->sizes() || t.scalar_type() != like[i]->scalar_type() || (t.stride(3) != 1 && t.size(3) > 1)) Py_RETURN_NONE;
    for (int j = 0; j < 3; ++j) strides[i][j] = t.stride(j);
  }
  const size_t bytes = ws->nbytes();
  if (g_bwd_bytes(&d) > bytes) Py_RETURN_NONE;
  void *pq = ptr(q), *pk = ptr(k), *pv = ptr(v), *po = ptr(out), *pb = ptr(bias), *pg = ptr(go), *pl = ptr(lse), *pdq = ptr(dq),
       *pdk = ptr(dk), *pdv = ptr(dv), *pw = ptr(ws);
  return status(unlocked([&] {
    return g_bwd(&d, pq, pk, pv, po, pb, pg, static_cast<const float*>(pl), pdq, pdk, pdv, pw, bytes, stream);
  }));
IXK_PY_END

// x, kind, eps, out, gain, gain_offset, stream
IXK_PY_FUNCTION(py_row_norm, 7)
  const at::Tensor *x = tensor(a[0]), *out, *gain;
  int64_t kind;
  double eps, offset;
  void* stream;
  if (x == nullptr || !integer(a[1], &kind) || !number(a[2], &eps) || !optional(a[3], &out) || !optional(a[4], &gain) ||
      !number(a[5], &offset) || !stream_arg(a[6], &stream) || x->dim() < 1 || !x->is_contiguous() || dtype_of(*x) < 0)
    Py_RETURN_NONE;
  const int64_t cols = x->size(x->dim() - 1), rows = cols != 0 ? x->numel() / cols : 0;
  if (gain != nullptr && (gain->dim() != 1 || gain->size(0) != cols || gain->scalar_type() != x->scalar_type() || !gain->is_contiguous()))
    Py_RETURN_NONE;
  at::Tensor made;
  if (out == nullptr) {
    made = at::empty(x->sizes(), at::TensorOptions().device(x->device()).dtype(x->scalar_type()));
    out = &made;
  } else if (out->sizes() != x->sizes() || out->scalar_type() != x->scalar_type() || !out->is_contiguous()) {
    Py_RETURN_NONE;
  }
  void *px = ptr(x), *pg = ptr(gain), *po = ptr(out);
  const int type = dtype_of(*x), k = static_cast<int>(kind);
  const float e = static_cast<float>(eps), off = static_cast<float>(offset);
  const int st = unlocked([&] {
    return gain != nullptr ? g_row_norm_gain(type, k, rows, cols, px, cols, pg, off, po, cols, e, stream)
                           : g_row_norm(type, k, rows, cols, px, cols, po, cols, e, stream);
  });
  return result(st, a[3], made);
IXK_PY_END

// x, cos, sin, seq_len, rotary_dim, half_split, stream
IXK_PY_FUNCTION(py_rotary, 7)
  const at::Tensor *x = tensor(a[0]), *cos = tensor(a[1]), *sin = tensor(a[2]);
  int64_t seq_len, dim;
  void* stream;
  if (x == nullptr || cos == nullptr || sin == nullptr || !integer(a[3], &seq_len) || !integer(a[4], &dim) || !PyBool_Check(a[5]) ||
      !stream_arg(a[6], &stream) || x->dim() != 3 || x->stride(2) != 1 || cos->scalar_type() != at::kFloat ||
      sin->scalar_type() != at::kFloat || !cos->is_contiguous() || !sin->is_contiguous() || cos->dim() != 2 ||
      cos->size(0) != seq_len || cos->size(1) != dim / 2 || sin->sizes() != cos->sizes() || dim > x->size(2) || dim < 0 || dtype_of(*x) < 0)
    Py_RETURN_NONE;
  void *px = ptr(x), *pc = ptr(cos), *ps = ptr(sin);
  const auto fn = a[5] == Py_True ? g_rotary_half : g_rotary;
  const int type = dtype_of(*x);
  const int64_t tokens = x->size(0), heads = x->size(1), s0 = x->stride(0), s1 = x->stride(1);
  return status(unlocked([&] {
    return fn(type, px, tokens, seq_len, heads, dim, s0, s1, static_cast<const float*>(pc), static_cast<const float*>(ps), stream);
  }));
IXK_PY_END

// k_cache, v_cache, k_new, v_new, position, stream
IXK_PY_FUNCTION(py_kv_append, 6)
  const at::Tensor *kc = tensor(a[0]), *vc = tensor(a[1]), *kn = tensor(a[2]), *vn = tensor(a[3]);
  int64_t position;
  void* stream;
  if (kc == nullptr || vc == nullptr || kn == nullptr || vn == nullptr || !integer(a[4], &position) || !stream_arg(a[5], &stream) ||
      kc->dim() != 4 || kn->dim() != 3 || dtype_of(*kc) < 0)
    Py_RETURN_NONE;
  const int64_t B = kc->size(0), T = kc->size(1), N = kc->size(2), H = kc->size(3);
  if (vc->sizes() != kc->sizes() || vc->strides() != kc->strides() || kn->size(0) != B || kn->size(1) != N || kn->size(2) != H ||
      vn->sizes() != kn->sizes() || vn->strides() != kn->strides() || kc->stride(3) != 1 || kn->stride(2) != 1 || position < 0 || position >= T)
    Py_RETURN_NONE;
  void *pkn = ptr(kn), *pvn = ptr(vn), *pkc = ptr(kc), *pvc = ptr(vc);
  const int type = dtype_of(*kc);
  const int64_t n0 = kn->stride(0), n1 = kn->stride(1), c0 = kc->stride(0), c1 = kc->stride(1), c2 = kc->stride(2);
  return status(unlocked([&] { return g_kv_append(type, B, N, H, pkn, pvn, n0, n1, pkc, pvc, c0, c1, c2, position, stream); }));
IXK_PY_END

// x, partial, bias, out, stream
IXK_PY_FUNCTION(py_residual_add, 5)
  const at::Tensor *x = tensor(a[0]), *p = tensor(a[1]), *bias, *out;
  void* stream;
  if (x == nullptr || p == nullptr || !optional(a[2], &bias) || !optional(a[3], &out) || !stream_arg(a[4], &stream) || x->dim() < 1 ||
      !x->is_contiguous() || !p->is_contiguous() || p->numel() != x->numel() || p->scalar_type() != x->scalar_type() || dtype_of(*x) < 0)
    Py_RETURN_NONE;
  const int64_t cols = x->size(x->dim() - 1), rows = cols != 0 ? x->numel() / cols : 0;
  if (bias != nullptr && (bias->dim() != 1 || bias->size(0) != cols || bias->scalar_type() != x->scalar_type() || !bias->is_contiguous()))
    Py_RETURN_NONE;
  at::Tensor made;
  if (out == nullptr) {
    made = at::empty(x->sizes(), at::TensorOptions().device(x->device()).dtype(x->scalar_type()));
    out = &made;
  } else if (out->numel() != x->numel() || out->scalar_type() != x->scalar_type() || !out->is_contiguous()) {
    Py_RETURN_NONE;
  }
  void *px = ptr(x), *pp = ptr(p), *pb = ptr(bias), *po = ptr(out);
  const int type = dtype_of(*x);
  const int st = unlocked([&] { return g_residual_add(type, rows, cols, px, pp, pb, po, stream); });
  return result(st, a[3], made);
IXK_PY_END

// bind(name -> address): the entry points of the library that the package has loaded
// ------------------------------------------------------------------------------------------------ training

at::Tensor like(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  return at::empty(sizes, at::TensorOptions().device(t.device()).dtype(type));
}
PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
// (given or made, ...); the status where it is not OK.
PyObject* results(int st, std::initializer_list<std::pair<PyObject*, const at::Tensor*>> items) {
  if (st != IXK_OK) return status(st);
  PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
  Py_ssize_t i = 0;
  for (const auto& [given, made] : items) {
    PyObject* o = given;
    if (o != nullptr) Py_INCREF(o);
    else o = wrap(*made);
    if (o == nullptr) {
      Py_DECREF(t);
      return nullptr;
    }
    PyTuple_SET_ITEM(t, i++, o);
  }
  return t;
}
// _row_pitch
bool row_pitch(const at::Tensor& t, int64_t* pitch) {
  const int64_t d = t.dim();
  if (d < 1) return false;
  if (t.is_contiguous()) *pitch = t.size(d - 1);
  else if (d == 2 && (t.stride(1) == 1 || t.size(1) == 1) && t.stride(0) >= t.size(1)) *pitch = t.stride(0);
  else return false;
  return true;
}
bool param(const at::Tensor* p, int64_t cols, const at::Tensor& x) {
  return p == nullptr || (p->dim() == 1 && p->size(0) == cols && p->is_contiguous() && (p->scalar_type() == x.scalar_type() || p->scalar_type() == at::kFloat));
}
bool float_type(const at::Tensor& t, bool with_fp32) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || (with_fp32 && t.scalar_type() == at::kFloat);
}

// _row_norm_desc
bool norm_desc(const at::Tensor& x, int64_t kind, const at::Tensor* gain, double offset, const at::Tensor* shift, double eps, ixk_row_norm_desc* d) {
  if (x.dim() < 1 || x.size(x.dim() - 1) < 1 || !float_type(x, true)) return false;
  const int64_t cols = x.size(x.dim() - 1);
  if (!param(gain, cols, x) || !param(shift, cols, x) || (gain != nullptr && shift != nullptr && gain->scalar_type() != shift->scalar_type())) return false;
  *d = ixk_row_norm_desc{};
  d->dtype = dtype_of(x);
  d->param_dtype = dtype_of(gain != nullptr ? *gain : shift != nullptr ? *shift : x);
  d->kind = static_cast<int32_t>(kind);
  d->eps = static_cast<float>(eps);
  d->gain_offset = static_cast<float>(offset);
  d->rows = x.numel() / cols;
  d->cols = cols;
  if (!row_pitch(x, &d->x_stride)) return false;
  d->y_stride = d->grad_y_stride = d->dx_stride = d->x_stride;
  return true;
}

// x, kind, eps, gain, gain_offset, shift, out, stream
IXK_PY_FUNCTION(py_row_norm_forward, 8)
  const at::Tensor *x = tensor(a[0]), *gain, *shift, *out;
  int64_t kind;
  double eps, offset;
  void* stream;
  ixk_row_norm_desc d;
  if (x == nullptr || !integer(a[1], &kind) || !number(a[2], &eps) || !optional(a[3], &gain) || !number(a[4], &offset) ||
      !optional(a[5], &shift) || !optional(a[6], &out) || !stream_arg(a[7], &stream) || (kind != IXK_NORM_LAYER && kind != IXK_NORM_RMS) ||
      !norm_desc(*x, kind, gain, offset, shift, eps, &d))
    Py_RETURN_NONE;
  if (out != nullptr && (out->sizes() != x->sizes() || out->scalar_type() != x->scalar_type() || !row_pitch(*out, &d.y_stride))) Py_RETURN_NONE;
  at::Tensor made, mean, rstd = like(*x, x->sizes().slice(0, x->dim() - 1), at::kFloat);
  if (out == nullptr) {
    made = like(*x, x->sizes(), x->scalar_type());
    out = &made;
    d.y_stride = d.cols;
  }
  if (kind == IXK_NORM_LAYER) mean = like(*x, x->sizes().slice(0, x->dim() - 1), at::kFloat);
  void *px = ptr(x), *pg = ptr(gain), *ps = ptr(shift), *po = ptr(out), *pr = ptr(&rstd), *pm = mean.defined() ? ptr(&mean) : nullptr;
  const int st = unlocked([&] { return g_norm_fwd(&d, px, pg, ps, po, static_cast<float*>(pm), static_cast<float*>(pr), stream); });
  return results(st, {{a[6] == Py_None ? nullptr : a[6], &made}, {nullptr, &mean}, {nullptr, &rstd}});
IXK_PY_END

// grad_out, x, mean, rstd, kind, gain, gain_offset, with_shift, grad_x, workspace, stream
IXK_PY_FUNCTION(py_row_norm_backward, 11)
  const at::Tensor *gy = tensor(a[0]), *x = tensor(a[1]), *mean, *rstd = tensor(a[3]), *gain, *dx, *ws;
  int64_t kind;
  double offset;
  void* stream;
  ixk_row_norm_desc d;
  if (gy == nullptr || x == nullptr || !optional(a[2], &mean) || rstd == nullptr || !integer(a[4], &kind) || !optional(a[5], &gain) ||
      !number(a[6], &offset) || !PyBool_Check(a[7]) || !optional(a[8], &dx) || !optional(a[9], &ws) || !stream_arg(a[10], &stream) ||
      (kind != IXK_NORM_LAYER && kind != IXK_NORM_RMS) || !norm_desc(*x, kind, gain, offset, nullptr, 0.0, &d))
    Py_RETURN_NONE;
  const at::IntArrayRef rows = x->sizes().slice(0, x->dim() - 1);
  auto stats = [&](const at::Tensor* t) { return t != nullptr && t->scalar_type() == at::kFloat && t->sizes() == rows && t->is_contiguous(); };
  if (!stats(rstd) || (kind == IXK_NORM_LAYER && !stats(mean))) Py_RETURN_NONE;
  auto fits = [&](const at::Tensor& t, int64_t* pitch) { return t.sizes() == x->sizes() && t.scalar_type() == x->scalar_type() && row_pitch(t, pitch); };
  if (!fits(*gy, &d.grad_y_stride) || (dx != nullptr && !fits(*dx, &d.dx_stride))) Py_RETURN_NONE;
  const bool with_shift = a[7] == Py_True;
  if (ws == nullptr && (gain != nullptr || with_shift) && a[10] != Py_None) Py_RETURN_NONE;   // (the twin allocates in that stream's pool)
  at::Tensor made, dgain, dshift, scratch;
  if (dx == nullptr) {
    made = like(*x, x->sizes(), x->scalar_type());
    dx = &made;
    d.dx_stride = d.cols;
  }
  const at::ScalarType type = gain != nullptr ? gain->scalar_type() : x->scalar_type();
  if (gain != nullptr) dgain = like(*x, {d.cols}, type);
  if (with_shift) dshift = like(*x, {d.cols}, type);
  if (ws == nullptr && (gain != nullptr || with_shift)) {
    scratch = like(*x, {static_cast<int64_t>(g_norm_bwd_bytes(&d))}, at::kByte);
    ws = &scratch;
  }
  void *pgy = ptr(gy), *px = ptr(x), *pg = ptr(gain), *pm = ptr(mean), *pr = ptr(rstd), *pdx = ptr(dx), *pw = ptr(ws);
  void *pdg = dgain.defined() ? ptr(&dgain) : nullptr, *pds = dshift.defined() ? ptr(&dshift) : nullptr;
  const size_t bytes = size_of(ws);
  const int st = unlocked([&] {
    return g_norm_bwd(&d, pgy, px, pg, static_cast<float*>(pm), static_cast<float*>(pr), pdx, pdg, pds, pw, bytes, stream);
  });
  return results(st, {{a[8] == Py_None ? nullptr : a[8], &made}, {nullptr, &dgain}, {nullptr, &dshift}});
IXK_PY_END

// _linear_loss_desc
bool loss_desc(const at::Tensor& x, const at::Tensor& w, const at::Tensor* bias, const at::Tensor& index, const at::Tensor* teacher, double scale,
               int64_t ignore, ixk_linear_loss_desc* d) {
  if (x.dim() != 2 || w.dim() != 2 || w.size(1) != x.size(1) || !float_type(x, false) || w.scalar_type() != x.scalar_type()) return false;
  const int64_t rows = x.size(0), hidden = x.size(1), vocab = w.size(0);
  if (hidden > 1 && x.stride(1) != 1) return false;
  if (bias != nullptr && (bias->scalar_type() != x.scalar_type() || bias->dim() != 1 || bias->size(0) != vocab || !bias->is_contiguous())) return false;
  if (index.scalar_type() != at::kInt && index.scalar_type() != at::kLong) return false;
  *d = ixk_linear_loss_desc{};
  if (teacher == nullptr) {
    if (index.dim() != 1 || index.size(0) != rows || !index.is_contiguous()) return false;
  } else {
    if (index.dim() != 2 || index.size(0) != rows || teacher->sizes() != index.sizes() || index.size(1) < 1 || index.size(1) > INT32_MAX ||
        !float_type(*teacher, true) || !row_pitch(index, &d->index_stride) || !row_pitch(*teacher, &d->teacher_stride))
      return false;
    d->entries = static_cast<int32_t>(index.size(1));
    d->teacher_dtype = dtype_of(*teacher);
  }
  ixk_matrix_layout l;
  if (!layout(w, &l)) return false;
  d->dtype = dtype_of(x);
  d->index_bytes = index.scalar_type() == at::kLong ? 8 : 4;
  d->scale = static_cast<float>(scale);
  d->ignore_index = ignore;
  d->rows = rows;
  d->hidden = hidden;
  d->vocab = vocab;
  d->x_stride = rows > 1 ? x.stride(0) : std::max(x.stride(0), (hidden + 7) / 8 * 8);
  d->w_order = d->dw_order = l.order;
  d->w_stride = d->dw_stride = l.leading_dim_stride;
  d->dx_stride = hidden;
  return true;
}

// x, weight, bias, labels or index, None or teacher, scale, ignore_index, workspace, stream
IXK_PY_FUNCTION(py_linear_loss_forward, 9)
  const at::Tensor *x = tensor(a[0]), *w = tensor(a[1]), *bias, *index = tensor(a[3]), *teacher, *ws;
  double scale;
  int64_t ignore;
  void* stream;
  ixk_linear_loss_desc d;
  if (x == nullptr || w == nullptr || !optional(a[2], &bias) || index == nullptr || !optional(a[4], &teacher) || !number(a[5], &scale) ||
      !integer(a[6], &ignore) || !optional(a[7], &ws) || !stream_arg(a[8], &stream) || !loss_desc(*x, *w, bias, *index, teacher, scale, ignore, &d))
    Py_RETURN_NONE;
  if (ws == nullptr && a[8] != Py_None) Py_RETURN_NONE;
  at::Tensor loss = like(*x, {d.rows}, at::kFloat), lse = like(*x, {d.rows}, at::kFloat), scratch;
  if (ws == nullptr) {
    scratch = like(*x, {static_cast<int64_t>(g_loss_bytes(&d, 0))}, at::kByte);
    ws = &scratch;
  }
  void *px = ptr(x), *pw = ptr(w), *pb = ptr(bias), *pi = ptr(index), *pt = ptr(teacher), *pws = ptr(ws);
  float *pl = static_cast<float*>(ptr(&loss)), *pe = static_cast<float*>(ptr(&lse));
  const size_t bytes = size_of(ws);
  const int st = unlocked([&] {
    return teacher == nullptr ? g_xent_fwd(&d, px, pw, pb, pi, pl, pe, pws, bytes, stream)
                              : g_distill_fwd(&d, px, pw, pb, pi, pt, pl, pe, pws, bytes, stream);
  });
  return results(st, {{nullptr, &loss}, {nullptr, &lse}});
IXK_PY_END

// x, weight, bias, labels or index, None or teacher, lse, grad_loss, scale, ignore_index, grad_x, grad_weight, weight_grad, workspace, stream
IXK_PY_FUNCTION(py_linear_loss_backward, 14)
  const at::Tensor *x = tensor(a[0]), *w = tensor(a[1]), *bias, *index = tensor(a[3]), *teacher, *lse = tensor(a[5]), *g = tensor(a[6]), *dx, *dw, *ws;
  double scale;
  int64_t ignore;
  void* stream;
  ixk_linear_loss_desc d;
  if (x == nullptr || w == nullptr || !optional(a[2], &bias) || index == nullptr || !optional(a[4], &teacher) || lse == nullptr || g == nullptr ||
      !number(a[7], &scale) || !integer(a[8], &ignore) || !optional(a[9], &dx) || !optional(a[10], &dw) || !PyBool_Check(a[11]) ||
      !optional(a[12], &ws) || !stream_arg(a[13], &stream) || !loss_desc(*x, *w, bias, *index, teacher, scale, ignore, &d))
    Py_RETURN_NONE;
  if (lse->dim() != 1 || lse->size(0) != d.rows || lse->scalar_type() != at::kFloat || !lse->is_contiguous()) Py_RETURN_NONE;
  if (g->scalar_type() != at::kFloat || g->dim() > 1 || (g->dim() == 1 && g->size(0) != d.rows)) Py_RETURN_NONE;
  if (ws == nullptr && a[13] != Py_None) Py_RETURN_NONE;
  d.grad_loss_stride = g->dim() == 1 ? g->stride(0) : 0;
  if (dx != nullptr && (dx->sizes() != x->sizes() || dx->scalar_type() != x->scalar_type() || !row_pitch(*dx, &d.dx_stride))) Py_RETURN_NONE;
  if (dw != nullptr) {
    ixk_matrix_layout l;
    if (dw->sizes() != w->sizes() || dw->scalar_type() != x->scalar_type() || !layout(*dw, &l)) Py_RETURN_NONE;
    d.dw_order = l.order;
    d.dw_stride = l.leading_dim_stride;
  }
  const bool weight_grad = a[11] == Py_True;
  at::Tensor made_dx, made_dw, dbias, scratch;
  if (dx == nullptr) {
    made_dx = like(*x, {d.rows, d.hidden}, x->scalar_type());
    dx = &made_dx;
  }
  if (dw == nullptr && weight_grad) {
    made_dw = d.w_order == IXK_ROW_MAJOR ? like(*x, {d.vocab, d.hidden}, x->scalar_type()) : like(*x, {d.hidden, d.vocab}, x->scalar_type()).t();
    dw = &made_dw;
    ixk_matrix_layout l;
    if (!layout(made_dw, &l)) Py_RETURN_NONE;
    d.dw_order = l.order;
    d.dw_stride = l.leading_dim_stride;
  }
  if (bias != nullptr && weight_grad) dbias = like(*x, {d.vocab}, x->scalar_type());
  if (ws == nullptr) {
    scratch = like(*x, {static_cast<int64_t>(g_loss_bytes(&d, 1))}, at::kByte);
    ws = &scratch;
  }
  void *px = ptr(x), *pw = ptr(w), *pb = ptr(bias), *pi = ptr(index), *pt = ptr(teacher), *pws = ptr(ws), *pdx = ptr(dx), *pdw = ptr(dw);
  void* pdb = dbias.defined() ? ptr(&dbias) : nullptr;
  const float *pe = static_cast<const float*>(ptr(lse)), *pg = static_cast<const float*>(ptr(g));
  const size_t bytes = size_of(ws);
  const int st = unlocked([&] {
    return teacher == nullptr ? g_xent_bwd(&d, px, pw, pb, pi, pe, pg, pdx, pdw, pdb, pws, bytes, stream)
                              : g_distill_bwd(&d, px, pw, pb, pi, pt, pe, pg, pdx, pdw, pdb, pws, bytes, stream);
  });
  return results(st, {{a[9] == Py_None ? nullptr : a[9], &made_dx}, {a[10] == Py_None ? nullptr : a[10], &made_dw}, {nullptr, &dbias}});
IXK_PY_END

// ------------------------------------------------------------------------------------------------ a paged cache

// A new dense tensor on the current device (on which `here` has found the operands), from the same pool as any other's, without the way
// through the dispatcher, which costs half as much as the launch.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type) {
  return at::Tensor(at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt));
}
// A vector of `n` elements from element `at` of a tensor's memory on.
at::Tensor piece(const at::Tensor& whole, int64_t at, int64_t n) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}
// _require_here: given tensors are on the current device.
bool here(std::initializer_list<const at::Tensor*> tensors) {
  const at::Tensor* one = nullptr;
  for (const at::Tensor* t : tensors) {
    if (t == nullptr) continue;
    if (one == nullptr && t->device().index() != c10::cuda::current_device()) return false;
    if (one != nullptr && t->device() != one->device()) return false;
    one = t;
  }
  return true;      // (also where none is on a GPU: asking for the current device would be an error of its own)
}
// _int32
bool ints(const at::Tensor* t, int64_t n) {
  return t != nullptr && t->scalar_type() == at::kInt && t->is_contiguous() && (n == 1 ? t->numel() == 1 : t->dim() == 1 && t->size(0) == n);
}
int32_t* ip(const at::Tensor* t) { return static_cast<int32_t*>(ptr(t)); }
bool int_rows(const at::Tensor* t) { return t != nullptr && t->dim() == 2 && t->scalar_type() == at::kInt && (t->size(1) <= 1 || t->stride(1) == 1); }

// _page_pool
bool page_pool(const at::Tensor* table, const at::Tensor* lengths, const at::Tensor* free_pages, const at::Tensor* free_count, int64_t page_size,
               ixk_page_pool* d) {
  if (!int_rows(table) || free_pages == nullptr || free_pages->dim() != 1) return false;
  const int64_t B = table->size(0), columns = table->size(1), pages = free_pages->size(0);
  if (B > INT32_MAX || columns > INT32_MAX || pages > INT32_MAX || page_size > INT32_MAX || page_size < 1) return false;
  *d = ixk_page_pool{static_cast<int32_t>(page_size), static_cast<int32_t>(pages), static_cast<int32_t>(B), static_cast<int32_t>(columns), table->stride(0)};
  return ints(lengths, B) && ints(free_pages, pages) && ints(free_count, 1);
}

// _paged_cache
bool paged_cache(const at::Tensor* k, const at::Tensor* v, bool layers, ixk_paged_cache* c) {
  if (k == nullptr || v == nullptr) return false;
  const int64_t dims = k->dim();
  if ((dims != 4 && !(layers && dims == 5)) || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type() || !float_type(*k, false) ||
      k->numel() == 0 || k->stride(dims - 1) != 1 || v->stride(dims - 1) != 1)
    return false;
  const int64_t at = dims - 4;
  for (int64_t i = 0; i < dims; ++i)
    if (k->size(i) > INT32_MAX) return false;
  c->dtype = dtype_of(*k);
  c->pages = static_cast<int32_t>(k->size(at));
  c->page_size = static_cast<int32_t>(k->size(at + 1));
  c->heads = static_cast<int32_t>(k->size(at + 2));
  c->head_size = static_cast<int32_t>(k->size(at + 3));
  c->layers = at == 1 ? static_cast<int32_t>(k->size(0)) : 1;
  for (int i = 0; i < 4; ++i) {
    const int64_t dim = i - 1 + at;
    const bool used = dim >= 0 && k->size(dim) != 1;
    c->k_strides[i] = used ? k->stride(dim) : 0;
    c->v_strides[i] = used ? v->stride(dim) : 0;
  }
  return true;
}

// page_table, lengths, new_tokens, free_pages, free_count, rows, page_size, out, stream
IXK_PY_FUNCTION(py_paged_extend, 9)
  const at::Tensor *table = tensor(a[0]), *lengths = tensor(a[1]), *added = tensor(a[2]), *pages = tensor(a[3]), *count = tensor(a[4]);
  int64_t rows, page_size;
  void* stream;
  ixk_page_pool d;
  if (table == nullptr || !integer(a[5], &rows) || !integer(a[6], &page_size) || rows < 0 || !stream_arg(a[8], &stream) ||
      !page_pool(table, lengths, pages, count, page_size, &d) || !ints(added, d.requests) || !here({table, lengths, added, pages, count}))
    Py_RETURN_NONE;
  const int64_t shapes[6] = {d.requests + 1, d.requests, rows, rows, rows, 1};
  at::Tensor made[6], whole;
  const at::Tensor* o[6];
  PyObject* given[6] = {nullptr, nullptr, nullptr, nullptr, nullptr, nullptr};
  if (a[7] == Py_None) {
    if (a[8] != Py_None) Py_RETURN_NONE;    // (the twin allocates in that stream's pool)
    // six small results in one piece of memory, each from a 256-byte boundary on: six allocations would cost more than the kernel
    int64_t at[7] = {0};
    for (int i = 0; i < 6; ++i) at[i + 1] = at[i] + (shapes[i] + 63) / 64 * 64;
    whole = fresh({at[6]}, at::kInt);
    for (int i = 0; i < 6; ++i) {
      made[i] = piece(whole, at[i], shapes[i]);
      o[i] = &made[i];
    }
  } else {
    if (!PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 6) Py_RETURN_NONE;
    for (int i = 0; i < 6; ++i) {
      given[i] = PyTuple_GET_ITEM(a[7], i);
      o[i] = tensor(given[i]);
      if (!ints(o[i], shapes[i]) || !here({o[i]})) Py_RETURN_NONE;
    }
  }
  int32_t *pt = ip(table), *pl = ip(lengths), *pn = ip(added), *pp = ip(pages), *pc = ip(count), *r[6];
  for (int i = 0; i < 6; ++i) r[i] = ip(o[i]);
  const int st = unlocked([&] { return g_extend(&d, pl, pn, pt, pp, pc, r[5], r[1], r[0], rows, r[2], r[3], r[4], stream); });
  return results(st, {{given[0], &made[0]}, {given[1], &made[1]}, {given[2], &made[2]}, {given[3], &made[3]}, {given[4], &made[4]}, {given[5], &made[5]}});
IXK_PY_END

// page_table, lengths, granted, kept, free_pages, free_count, page_size, path, k_pages, v_pages, lengths_out, free_count_out, stream
IXK_PY_FUNCTION(py_paged_keep, 13)
  const at::Tensor *table = tensor(a[0]), *lengths = tensor(a[1]), *granted = tensor(a[2]), *kept = tensor(a[3]), *pages = tensor(a[4]),
                   *count = tensor(a[5]), *path, *k, *v, *lengths_out, *count_out;
  int64_t page_size;
  void* stream;
  ixk_page_pool d;
  ixk_paged_cache c;
  if (table == nullptr || !integer(a[6], &page_size) || !optional(a[7], &path) || !optional(a[8], &k) || !optional(a[9], &v) || !optional(a[10], &lengths_out) ||
      !optional(a[11], &count_out) || !stream_arg(a[12], &stream) || !page_pool(table, lengths, pages, count, page_size, &d) ||
      !ints(granted, d.requests) || !ints(kept, d.requests) ||
      !here({table, lengths, granted, kept, pages, count, path, k, v, lengths_out, count_out}))
    Py_RETURN_NONE;
  if (path != nullptr ? !int_rows(path) || path->size(0) != d.requests || !paged_cache(k, v, true, &c) : k != nullptr || v != nullptr) Py_RETURN_NONE;
  if ((lengths_out == nullptr || count_out == nullptr) && a[12] != Py_None) Py_RETURN_NONE;
  at::Tensor made_lengths, made_count;
  if (lengths_out == nullptr || count_out == nullptr) {      // in one piece of memory, as extend's
    const int64_t own = lengths_out == nullptr ? (d.requests + 63) / 64 * 64 : 0;
    const at::Tensor whole = fresh({own + (count_out == nullptr ? 1 : 0)}, at::kInt);
    if (lengths_out == nullptr) {
      made_lengths = piece(whole, 0, d.requests);
      lengths_out = &made_lengths;
    }
    if (count_out == nullptr) {
      made_count = piece(whole, own, 1);
      count_out = &made_count;
    }
  }
  if (!ints(lengths_out, d.requests) || !ints(count_out, 1)) Py_RETURN_NONE;
  int32_t *pt = ip(table), *pl = ip(lengths), *pg = ip(granted), *pk = ip(kept), *pp = ip(pages), *pc = ip(count), *ppath = ip(path),
          *plo = ip(lengths_out), *pco = ip(count_out);
  void *kp = ptr(k), *vp = ptr(v);
  const int64_t columns = path != nullptr ? path->size(1) : 0, stride = path != nullptr ? path->stride(0) : 0;
  const ixk_paged_cache* cache = path != nullptr ? &c : nullptr;
  const int st = unlocked([&] { return g_keep(&d, pl, pg, pk, ppath, columns, stride, pt, pp, pc, pco, plo, cache, kp, vp, stream); });
  return results(st, {{a[10] == Py_None ? nullptr : a[10], &made_lengths}, {a[11] == Py_None ? nullptr : a[11], &made_count}});
IXK_PY_END

// _heads_view
bool heads_view(const at::Tensor* t, at::IntArrayRef sizes, at::ScalarType type, int64_t* strides) {
  if (t == nullptr || t->dim() != 3 || t->sizes() != sizes || t->scalar_type() != type || (t->size(2) > 1 && t->stride(2) != 1)) return false;
  for (int i = 0; i < 2; ++i) strides[i] = t->size(i) == 1 ? 0 : t->stride(i);
  return true;
}
// _qk_desc
bool qk_desc(const at::Tensor* q, const at::Tensor* k, const at::Tensor* q_gain, const at::Tensor* k_gain, double offset, double eps,
             const at::Tensor* cos, const at::Tensor* sin, const at::Tensor* positions, bool half_split, ixk_qk_desc* d) {
  if (q == nullptr || k == nullptr || cos == nullptr || sin == nullptr || q->dim() != 3 || k->dim() != 3 || k->size(0) != q->size(0) ||
      k->size(2) != q->size(2) || !float_type(*q, true) || q->size(1) > INT32_MAX || k->size(1) > INT32_MAX || q->size(2) > INT32_MAX)
    return false;
  *d = ixk_qk_desc{};
  if (!heads_view(q, q->sizes(), q->scalar_type(), d->q_strides) || !heads_view(k, k->sizes(), q->scalar_type(), d->k_strides)) return false;
  if (!param(q_gain, q->size(2), *q) || !param(k_gain, q->size(2), *q) ||
      (q_gain != nullptr && k_gain != nullptr && q_gain->scalar_type() != k_gain->scalar_type()))
    return false;
  for (const at::Tensor* t : {cos, sin})
    if (t->dim() != 2 || t->scalar_type() != at::kFloat || t->sizes() != cos->sizes() || !t->is_contiguous() || t->size(1) > INT32_MAX / 2) return false;
  if (positions != nullptr && ((positions->scalar_type() != at::kInt && positions->scalar_type() != at::kLong) || positions->dim() != 1 ||
                               positions->size(0) != q->size(0) || !positions->is_contiguous()))
    return false;
  const at::Tensor& gained = q_gain != nullptr ? *q_gain : k_gain != nullptr ? *k_gain : *q;
  d->dtype = dtype_of(*q);
  d->param_dtype = dtype_of(gained);
  d->tokens = q->size(0);
  d->heads = static_cast<int32_t>(q->size(1));
  d->kv_heads = static_cast<int32_t>(k->size(1));
  d->head_size = static_cast<int32_t>(q->size(2));
  d->rotary_dim = static_cast<int32_t>(2 * cos->size(1));
  d->places = cos->size(0);
  d->interleaved = half_split ? 0 : 1;
  d->position_bytes = positions != nullptr && positions->scalar_type() == at::kLong ? 8 : 4;
  d->eps = static_cast<float>(eps);
  d->gain_offset = static_cast<float>(offset);
  return true;
}

// q, k, q_gain, k_gain, gain_offset, eps, cos, sin, positions, half_split, v, slots, k_pages, v_pages, q_out, k_out, stream
IXK_PY_FUNCTION(py_qk_forward, 17)
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *qg, *kg, *cos = tensor(a[6]), *sin = tensor(a[7]), *pos, *v, *slots, *kp, *vp, *qo, *ko;
  double offset, eps;
  void* stream;
  ixk_qk_desc d;
  ixk_paged_cache c;
  if (q == nullptr || !optional(a[2], &qg) || !optional(a[3], &kg) || !number(a[4], &offset) || !number(a[5], &eps) || !optional(a[8], &pos) ||
      !PyBool_Check(a[9]) || !optional(a[10], &v) || !optional(a[11], &slots) || !optional(a[12], &kp) || !optional(a[13], &vp) ||
      !optional(a[14], &qo) || !optional(a[15], &ko) || !stream_arg(a[16], &stream) ||
      !qk_desc(q, k, qg, kg, offset, eps, cos, sin, pos, a[9] == Py_True, &d) || !here({q, k, qg, kg, cos, sin, pos, v, slots, kp, vp, qo, ko}))
    Py_RETURN_NONE;
  const bool paged = v != nullptr || slots != nullptr || kp != nullptr || vp != nullptr;
  if (paged && (ko != nullptr || !ints(slots, d.tokens) || !heads_view(v, k->sizes(), q->scalar_type(), d.v_strides) || !paged_cache(kp, vp, false, &c)))
    Py_RETURN_NONE;
  if (a[16] != Py_None && (qo == nullptr || (!paged && ko == nullptr))) Py_RETURN_NONE;
  at::Tensor made_q, made_k;
  if (qo == nullptr) {
    made_q = fresh(q->sizes(), q->scalar_type());
    qo = &made_q;
  }
  if (!paged && ko == nullptr) {
    made_k = fresh(k->sizes(), k->scalar_type());
    ko = &made_k;
  }
  if (!heads_view(qo, q->sizes(), q->scalar_type(), d.q_out_strides) || (ko != nullptr && !heads_view(ko, k->sizes(), q->scalar_type(), d.k_out_strides)))
    Py_RETURN_NONE;
  void *pq = ptr(q), *pk = ptr(k), *pv = ptr(v), *pqg = ptr(qg), *pkg = ptr(kg), *ppos = ptr(pos), *pqo = ptr(qo), *pko = ptr(ko), *pkp = ptr(kp),
       *pvp = ptr(vp);
  const float *pc = static_cast<const float*>(ptr(cos)), *ps = static_cast<const float*>(ptr(sin));
  const int32_t* psl = ip(slots);
  const int st = unlocked([&] { return g_qk_fwd(&d, pq, pk, pv, pqg, pkg, pc, ps, ppos, pqo, pko, paged ? &c : nullptr, psl, pkp, pvp, stream); });
  return results(st, {{a[14] == Py_None ? nullptr : a[14], &made_q}, {a[15] == Py_None ? nullptr : a[15], &made_k}});
IXK_PY_END

// grad_q, grad_k, q, k, q_gain, k_gain, gain_offset, eps, cos, sin, positions, half_split, dq, dk, workspace, stream
IXK_PY_FUNCTION(py_qk_backward, 16)
  const at::Tensor *gq = tensor(a[0]), *gk = tensor(a[1]), *q = tensor(a[2]), *k = tensor(a[3]), *qg, *kg, *cos = tensor(a[8]), *sin = tensor(a[9]),
                   *pos, *dq, *dk, *ws;
  double offset, eps;
  void* stream;
  ixk_qk_desc d;
  if (q == nullptr || !optional(a[4], &qg) || !optional(a[5], &kg) || !number(a[6], &offset) || !number(a[7], &eps) || !optional(a[10], &pos) ||
      !PyBool_Check(a[11]) || !optional(a[12], &dq) || !optional(a[13], &dk) || !optional(a[14], &ws) || !stream_arg(a[15], &stream) ||
      !qk_desc(q, k, qg, kg, offset, eps, cos, sin, pos, a[11] == Py_True, &d) || !heads_view(gq, q->sizes(), q->scalar_type(), d.gq_strides) ||
      !heads_view(gk, k->sizes(), q->scalar_type(), d.gk_strides) || !here({gq, gk, q, k, qg, kg, cos, sin, pos, dq, dk, ws}))
    Py_RETURN_NONE;
  const bool gains = qg != nullptr || kg != nullptr;
  if (a[15] != Py_None && (dq == nullptr || dk == nullptr || gains)) Py_RETURN_NONE;
  at::Tensor made_q, made_k, dqg, dkg, scratch;
  if (dq == nullptr) {
    made_q = fresh(q->sizes(), q->scalar_type());
    dq = &made_q;
  }
  if (dk == nullptr) {
    made_k = fresh(k->sizes(), k->scalar_type());
    dk = &made_k;
  }
  if (!heads_view(dq, q->sizes(), q->scalar_type(), d.q_out_strides) || !heads_view(dk, k->sizes(), q->scalar_type(), d.k_out_strides)) Py_RETURN_NONE;
  if (gains) {      // (both in one piece of memory, 16-byte boundaries for heads of any size)
    const int64_t n = (q->size(2) + 7) / 8 * 8;
    const at::Tensor both = fresh({2 * n}, (qg != nullptr ? qg : kg)->scalar_type());
    if (qg != nullptr) dqg = piece(both, 0, q->size(2));
    if (kg != nullptr) dkg = piece(both, n, q->size(2));
  }
  if (gains && ws == nullptr) {
    scratch = fresh({static_cast<int64_t>(g_qk_bwd_bytes(&d))}, at::kByte);
    ws = &scratch;
  }
  void *pgq = ptr(gq), *pgk = ptr(gk), *pq = ptr(q), *pk = ptr(k), *pqg = ptr(qg), *pkg = ptr(kg), *ppos = ptr(pos), *pdq = ptr(dq), *pdk = ptr(dk),
       *pw = ptr(ws), *pdqg = dqg.defined() ? ptr(&dqg) : nullptr, *pdkg = dkg.defined() ? ptr(&dkg) : nullptr;
  const float *pc = static_cast<const float*>(ptr(cos)), *ps = static_cast<const float*>(ptr(sin));
  const size_t bytes = size_of(ws);
  const int st = unlocked([&] { return g_qk_bwd(&d, pgq, pgk, pq, pk, pqg, pkg, pc, ps, ppos, pdq, pdk, pdqg, pdkg, pw, bytes, stream); });
  return results(st, {{a[12] == Py_None ? nullptr : a[12], &made_q}, {a[13] == Py_None ? nullptr : a[13], &made_k}, {nullptr, &dqg}, {nullptr, &dkg}});
IXK_PY_END

// q, k_pages, v_pages, page_table, lengths, row_start, granted, scale, mask, out, lse, with_lse, workspace, stream
IXK_PY_FUNCTION(py_fmha_paged, 14)
  const at::Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *table = tensor(a[3]), *lengths = tensor(a[4]), *start = tensor(a[5]),
                   *granted = tensor(a[6]), *mask, *out, *lse, *ws;
  double scale;
  void* stream;
  ixk_fmha_paged_desc d{};
  ixk_paged_cache c;
  if (q == nullptr || !number(a[7], &scale) || !optional(a[8], &mask) || !optional(a[9], &out) || !optional(a[10], &lse) || !PyBool_Check(a[11]) ||
      !optional(a[12], &ws) || !stream_arg(a[13], &stream) || !paged_cache(k, v, false, &c) || !int_rows(table) ||
      !here({q, k, v, table, lengths, start, granted, mask, out, lse, ws}))
    Py_RETURN_NONE;
  const int64_t B = table->size(0);
  if (q->dim() != 3 || q->scalar_type() != k->scalar_type() || q->size(2) != c.head_size || q->size(1) > INT32_MAX || B > INT32_MAX - 1 ||
      table->size(1) > INT32_MAX || !ints(lengths, B) || !ints(start, B + 1) || !ints(granted, B) ||
      (mask != nullptr && (!int_rows(mask) || mask->size(0) != q->size(0) || mask->size(1) < 1 || mask->size(1) > INT32_MAX)))
    Py_RETURN_NONE;
  const bool want_lse = lse != nullptr || a[11] == Py_True;
  if (a[13] != Py_None && (out == nullptr || (want_lse && lse == nullptr) || ws == nullptr)) Py_RETURN_NONE;
  at::Tensor made, made_lse, scratch;
  if (out == nullptr) {
    made = fresh(q->sizes(), q->scalar_type());
    out = &made;
  }
  d.rows = q->size(0);
  d.heads = static_cast<int32_t>(q->size(1));
  d.requests = static_cast<int32_t>(B);
  d.columns = static_cast<int32_t>(table->size(1));
  d.table_stride = table->stride(0);
  d.head_scale = static_cast<float>(scale);
  if (mask != nullptr) {
    d.mask_words = static_cast<int32_t>(mask->size(1));
    d.mask_stride = mask->stride(0);
  }
  if (!heads_view(q, q->sizes(), q->scalar_type(), d.q_strides) || !heads_view(out, q->sizes(), q->scalar_type(), d.o_strides)) Py_RETURN_NONE;
  if (lse == nullptr && want_lse) {
    made_lse = fresh({d.rows, q->size(1)}, at::kFloat);
    lse = &made_lse;
  }
  if (lse != nullptr && (lse->scalar_type() != at::kFloat || lse->sizes() != q->sizes().slice(0, 2) || !lse->is_contiguous())) Py_RETURN_NONE;
  if (ws == nullptr) {
    scratch = fresh({static_cast<int64_t>(g_paged_fwd_bytes(&d, &c))}, at::kByte);
    ws = &scratch;
  }
  void *pq = ptr(q), *pk = ptr(k), *pv = ptr(v), *po = ptr(out), *pw = ptr(ws);
  int32_t *pt = ip(table), *pl = ip(lengths), *ps = ip(start), *pg = ip(granted), *pm = ip(mask);
  float* ple = static_cast<float*>(ptr(lse));
  const size_t bytes = size_of(ws);
  const int st = unlocked([&] { return g_paged_fwd(&d, &c, pq, pk, pv, pt, pl, ps, pg, pm, po, ple, pw, bytes, stream); });
  return results(st, {{a[9] == Py_None ? nullptr : a[9], &made}, {a[10] == Py_None ? nullptr : a[10], &made_lse}});
IXK_PY_END

PyObject* py_bind(PyObject*, PyObject* table) {
  struct Entry {
    const char* name;
    void** slot;
  };
  const Entry entries[] = {
      {"ixk_gemm", reinterpret_cast<void**>(&g_gemm)},
      {"ixk_gemm_fp8", reinterpret_cast<void**>(&g_gemm_fp8)},
      {"ixk_gemm_workspace_bytes", reinterpret_cast<void**>(&g_gemm_bytes)},
      {"ixk_gemm_geglu", reinterpret_cast<void**>(&g_geglu)},
      {"ixk_fmha_fwd", reinterpret_cast<void**>(&g_fwd)},
      {"ixk_fmha_fwd_workspace_bytes", reinterpret_cast<void**>(&g_fwd_bytes)},
      {"ixk_fmha_bwd", reinterpret_cast<void**>(&g_bwd)},
      {"ixk_fmha_bwd_workspace_bytes", reinterpret_cast<void**>(&g_bwd_bytes)},
      {"ixk_row_norm", reinterpret_cast<void**>(&g_row_norm)},
      {"ixk_row_norm_gain", reinterpret_cast<void**>(&g_row_norm_gain)},
      {"ixk_rotary_interleaved", reinterpret_cast<void**>(&g_rotary)},
      {"ixk_rotary_half", reinterpret_cast<void**>(&g_rotary_half)},
      {"ixk_kv_append", reinterpret_cast<void**>(&g_kv_append)},
      {"ixk_residual_add", reinterpret_cast<void**>(&g_residual_add)},
      {"ixk_row_norm_fwd", reinterpret_cast<void**>(&g_norm_fwd)},
      {"ixk_row_norm_bwd", reinterpret_cast<void**>(&g_norm_bwd)},
      {"ixk_row_norm_bwd_workspace_bytes", reinterpret_cast<void**>(&g_norm_bwd_bytes)},
      {"ixk_linear_xent_fwd", reinterpret_cast<void**>(&g_xent_fwd)},
      {"ixk_linear_xent_bwd", reinterpret_cast<void**>(&g_xent_bwd)},
      {"ixk_linear_distill_fwd", reinterpret_cast<void**>(&g_distill_fwd)},
      {"ixk_linear_distill_bwd", reinterpret_cast<void**>(&g_distill_bwd)},
      {"ixk_linear_loss_workspace_bytes", reinterpret_cast<void**>(&g_loss_bytes)},
      {"ixk_paged_extend", reinterpret_cast<void**>(&g_extend)},
      {"ixk_paged_keep", reinterpret_cast<void**>(&g_keep)},
      {"ixk_qk_norm_rotary_fwd", reinterpret_cast<void**>(&g_qk_fwd)},
      {"ixk_qk_norm_rotary_bwd", reinterpret_cast<void**>(&g_qk_bwd)},
      {"ixk_qk_norm_rotary_bwd_workspace_bytes", reinterpret_cast<void**>(&g_qk_bwd_bytes)},
      {"ixk_fmha_paged_fwd", reinterpret_cast<void**>(&g_paged_fwd)},
      {"ixk_fmha_paged_fwd_workspace_bytes", reinterpret_cast<void**>(&g_paged_fwd_bytes)},
  };
  for (const Entry& e : entries) {
    PyObject* address = PyDict_GetItemString(table, e.name);   // borrowed
    if (address == nullptr) {
      PyErr_SetString(PyExc_KeyError, e.name);
      return nullptr;
    }
    *e.slot = PyLong_AsVoidPtr(address);
    if (PyErr_Occurred() != nullptr) return nullptr;
  }
  Py_RETURN_NONE;
}

#define IXK_METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    {"bind", py_bind, METH_O, nullptr},
    IXK_METHOD("gemm", py_gemm),
    IXK_METHOD("geglu", py_geglu),
    IXK_METHOD("fmha_forward", py_fmha_forward),
    IXK_METHOD("fmha_backward", py_fmha_backward),
    IXK_METHOD("row_norm", py_row_norm),
    IXK_METHOD("rotary", py_rotary),
    IXK_METHOD("kv_append", py_kv_append),
    IXK_METHOD("residual_add", py_residual_add),
    IXK_METHOD("row_norm_forward", py_row_norm_forward),
    IXK_METHOD("row_norm_backward", py_row_norm_backward),
    IXK_METHOD("linear_loss_forward", py_linear_loss_forward),
    IXK_METHOD("linear_loss_backward", py_linear_loss_backward),
    IXK_METHOD("paged_extend", py_paged_extend),
    IXK_METHOD("paged_keep", py_paged_keep),
    IXK_METHOD("qk_forward", py_qk_forward),
    IXK_METHOD("qk_backward", py_qk_backward),
    IXK_METHOD("fmha_paged", py_fmha_paged),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ixk_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ixk_calls() { return PyModule_Create(&module); }
