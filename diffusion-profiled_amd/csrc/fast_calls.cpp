// The conditioning and MXFP4 operators' Python calls where nothing has to be converted: checks, allocation and
// the C entry in one native call. An eager call on small operands waits for its host side, of which
// Python code and its arguments' conversion were two thirds: 4 x 1 queries over 77 keys 9.6 us in
// Python, 3.4 us of it the launch.
//
// Every function returns None for a call that it does not take -- operands that need a copy, are
// refused, or are anything but plain strided GPU tensors; conditioning.py and mxfp4.py then go the general way,
// which copies or raises. A module of the CPython API; the kernels' library is not linked but handed
// over as addresses (init).
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/dpa_fp8.h"

namespace {

decltype(&dpa_cross_attention_fwd) attn_fwd;
decltype(&dpa_cross_attention_fwd_workspace_bytes) attn_fwd_bytes;
decltype(&dpa_cross_attention_bwd) attn_bwd;
decltype(&dpa_cross_attention_bwd_workspace_bytes) attn_bwd_bytes;
decltype(&dpa_dropout) drop;
decltype(&dpa_embedding_fwd) emb_fwd;
decltype(&dpa_embedding_bwd) emb_bwd;
decltype(&dpa_embedding_bwd_workspace_bytes) emb_bwd_bytes;
decltype(&dpa_mxfp4_quantize) mx_quant;
decltype(&dpa_mxfp4_dequantize) mx_dequant;
decltype(&dpa_mxfp4_operand_bytes) mx_operand_bytes;
decltype(&dpa_mxfp4_operands) mx_operands;
decltype(&dpa_mxfp4_gemm) mx_gemm;
decltype(&dpa_mxfp4_gemm_workspace_bytes) mx_gemm_bytes;
decltype(&dpa_mxfp4_gemm_plan) mx_plan;
decltype(&dpa_mxfp4_linear) mx_linear;
decltype(&dpa_mxfp4_linear_workspace_bytes) mx_linear_bytes;
decltype(&dpa_column_sum) column_sum;
decltype(&dpa_column_sum_workspace_bytes) column_sum_bytes;
decltype(&dpa_cross_attention_mxfp4) mx_attn;
decltype(&dpa_cross_attention_mxfp4_workspace_bytes) mx_attn_bytes;
decltype(&dpa_status_string) status_string;

// A plain strided tensor on a GPU (device: the first one's), or null
const at::Tensor* plain(PyObject* o, int* device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_conj() || t.is_neg())
    return nullptr;
  const int d = t.get_device();
  if (*device < 0) *device = d;
  return d == *device ? &t : nullptr;
}

// None (*out stays null) or a plain tensor; false for anything else
bool maybe(PyObject* o, int* device, const at::Tensor** out) {
  *out = nullptr;
  return o == Py_None || (*out = plain(o, device)) != nullptr;
}

int dtype_of(at::ScalarType t) {
  return t == at::kBFloat16 ? DPA_DTYPE_BF16 : t == at::kFloat ? DPA_DTYPE_F32 : t == at::kHalf ? DPA_DTYPE_F16 : -1;
}

void* stream_of(int device) { return c10::hip::getCurrentHIPStream(device).stream(); }

PyObject* failed(const char* what, int status) {
  PyErr_Format(PyExc_RuntimeError, "%s failed: %s (status %d)", what, status_string(status), status);
  return nullptr;
}

PyObject* none() { Py_RETURN_NONE; }

bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// Strides of a [batch, tokens, heads, head_dim] operand as the kernels read it
bool strides_of(const at::Tensor& t, int64_t* s) {
  if (t.stride(3) != 1) return false;
  for (int i = 0; i < 3; ++i) {
    s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    if (s[i] % 8) return false;
  }
  return aligned16(t);
}

// What a call over keys of any kind describes: queries, masks over lk keys, the scale. Sizes past 32 bits and
// the rest that the entries refuse are left to them, and so to the general way's message.
bool describe_queries(DpaCrossAttention& a, const at::Tensor& q, int64_t lk, const at::Tensor* lengths,
                      const at::Tensor* mask, PyObject* scale) {
  const int64_t b = q.size(0), lq = q.size(1), h = q.size(2), d = q.size(3), most = INT32_MAX;
  if ((q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf) || b <= 0 || lq <= 0 || h <= 0 || b > most ||
      lq > most || h > most)
    return false;
  if (lengths && (lengths->dim() != 1 || lengths->size(0) != b || lengths->scalar_type() != at::kInt || !lengths->is_contiguous()))
    return false;
  if (mask && (mask->dim() != 2 || mask->size(0) != b || mask->size(1) != lk || (lk > 1 && mask->stride(1) != 1) ||
               (mask->scalar_type() != at::kBool && mask->scalar_type() != at::kByte)))
    return false;
  if (scale == Py_None) {
    a.scale = (float)(1.0 / std::sqrt((double)d));
  } else if (PyFloat_CheckExact(scale)) {
    const double s = PyFloat_AS_DOUBLE(scale);
    if (!(s > 0.0 && s < 2.3e38)) return false;
    a.scale = (float)s;
  } else {
    return false;
  }
  if (!strides_of(q, a.q_stride)) return false;
  a.q = q.data_ptr();
  a.key_lengths = lengths ? (const int32_t*)lengths->data_ptr() : nullptr;
  a.key_mask = mask ? (const uint8_t*)mask->data_ptr() : nullptr;
  a.mask_stride = mask ? mask->stride(0) : 0;
  a.dtype = dtype_of(q.scalar_type());
  a.batch = (int32_t)b, a.q_len = (int32_t)lq, a.heads = (int32_t)h;
  return true;
}

// What forward and backward describe alike
bool describe(DpaCrossAttention& a, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
              const at::Tensor* lengths, const at::Tensor* mask, PyObject* scale) {
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || q.scalar_type() != k.scalar_type() ||
      q.scalar_type() != v.scalar_type() || k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
    return false;
  const int64_t h = q.size(2), d = q.size(3), lk = k.size(1), g = k.size(2), most = INT32_MAX;
  if (lk <= 0 || g <= 0 || d <= 0 || d % 8 || d > 128 || h % g || lk > most) return false;
  if (!describe_queries(a, q, lk, lengths, mask, scale) || !strides_of(k, a.k_stride) || !strides_of(v, a.v_stride)) return false;
  a.k = k.data_ptr(), a.v = v.data_ptr();
  a.kv_len = (int32_t)lk, a.kv_heads = (int32_t)g, a.head_dim = (int32_t)d;
  return true;
}

// (q, k, v, key_lengths, key_mask, scale) -> (out, lse)
PyObject* attention_fwd(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return none();
  int device = -1;
  const at::Tensor *q = plain(o[0], &device), *k = plain(o[1], &device), *v = plain(o[2], &device), *lengths, *mask;
  DpaCrossAttention a{};
  if (!q || !k || !v || !maybe(o[3], &device, &lengths) || !maybe(o[4], &device, &mask) ||
      !describe(a, *q, *k, *v, lengths, mask, o[5]))
    return none();
  at::Tensor out = at::empty(q->sizes(), q->options());
  at::Tensor lse = at::empty({q->size(0), q->size(2), q->size(1)}, q->options().dtype(at::kFloat)), ws;
  a.out = out.data_ptr(), a.lse = (float*)lse.data_ptr();
  const int64_t bytes = attn_fwd_bytes(&a);
  if (bytes) ws = at::empty({bytes}, q->options().dtype(at::kByte));
  const int status = attn_fwd(&a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(device));
  if (status) return failed("dpa_cross_attention_fwd", status);
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(out)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(lse)));
  return r;
  END_HANDLE_TH_ERRORS
}

// (dout, q, k, v, out, lse, key_lengths, key_mask, scale, dk, dv) -> (dq, dk, dv); dk and dv: None
// (not formed), True (a new dense tensor) or where to write them
PyObject* attention_bwd(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return none();
  int device = -1;
  const at::Tensor *g = plain(o[0], &device), *q = plain(o[1], &device), *k = plain(o[2], &device),
                   *v = plain(o[3], &device), *out = plain(o[4], &device), *lse = plain(o[5], &device), *lengths, *mask;
  DpaCrossAttention a{};
  if (!g || !q || !k || !v || !out || !lse || !maybe(o[6], &device, &lengths) || !maybe(o[7], &device, &mask) ||
      !describe(a, *q, *k, *v, lengths, mask, o[8]))
    return none();
  if (g->sizes() != q->sizes() || g->scalar_type() != q->scalar_type() || !strides_of(*g, a.dout_stride) ||
      out->sizes() != q->sizes() || out->scalar_type() != q->scalar_type() || !out->is_contiguous() || !aligned16(*out) ||
      lse->dim() != 3 || lse->size(0) != q->size(0) || lse->size(1) != q->size(2) || lse->size(2) != q->size(1) ||
      lse->scalar_type() != at::kFloat || !lse->is_contiguous())
    return none();
  const at::Tensor* given[2] = {nullptr, nullptr};
  at::Tensor made[2];
  if (o[9] == Py_True && o[10] == Py_True) {
    for (at::Tensor& t : made) t = at::empty(k->sizes(), k->options());
    given[0] = &made[0], given[1] = &made[1];
  } else if (o[9] != Py_None || o[10] != Py_None) {
    for (int i = 0; i < 2; ++i) {
      given[i] = plain(o[9 + i], &device);
      if (!given[i] || given[i]->sizes() != k->sizes() || given[i]->scalar_type() != k->scalar_type()) return none();
    }
  }
  if (given[0]) {
    if (!strides_of(*given[0], a.dk_stride) || !strides_of(*given[1], a.dv_stride)) return none();
    a.dk = given[0]->data_ptr(), a.dv = given[1]->data_ptr();
  }
  at::Tensor dq = at::empty(q->sizes(), q->options()), ws;
  a.dout = g->data_ptr(), a.out = out->data_ptr(), a.lse = (float*)lse->data_ptr(), a.dq = dq.data_ptr();
  const int64_t bytes = attn_bwd_bytes(&a);
  if (bytes) ws = at::empty({bytes}, q->options().dtype(at::kByte));
  const int status = attn_bwd(&a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(device));
  if (status) return failed("dpa_cross_attention_bwd", status);
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(dq)));
  for (int i = 0; i < 2; ++i) {
    PyObject* x = o[9 + i];
    if (made[i].defined()) x = THPVariable_Wrap(std::move(made[i]));
    else Py_INCREF(x);
    PyTuple_SET_ITEM(r, 1 + i, x);
  }
  return r;
  END_HANDLE_TH_ERRORS
}

// p as a Python float in [0, 1), in fp32 too
bool drop_p(PyObject* o, float* p) {
  if (!PyFloat_CheckExact(o)) return false;
  const double x = PyFloat_AS_DOUBLE(o);
  *p = (float)x;
  return x >= 0.0 && x < 1.0 && *p < 1.0f;
}

bool seed_ok(const at::Tensor* s) { return s && s->scalar_type() == at::kLong && s->numel() == 1; }

// (x, p, seed, residual) -> y
PyObject* dropout(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) return none();
  int device = -1;
  float p;
  const at::Tensor *x = plain(o[0], &device), *seed = plain(o[2], &device), *r;
  if (!x || !seed_ok(seed) || !maybe(o[3], &device, &r) || !drop_p(o[1], &p)) return none();
  const int dtype = dtype_of(x->scalar_type());
  if (dtype < 0 || !x->is_non_overlapping_and_dense()) return none();
  if (!x->is_contiguous() && !(x->dim() == 4 && x->is_contiguous(at::MemoryFormat::ChannelsLast))) return none();
  if (r && (r->scalar_type() != x->scalar_type() || r->sizes() != x->sizes() || r->strides() != x->strides())) return none();
  at::Tensor y = at::empty_like(*x);
  const int status = drop(x->data_ptr(), r ? r->data_ptr() : nullptr, y.data_ptr(), dtype, x->numel(), seed->data_ptr(), p,
                          stream_of(device));
  if (status) return failed("dpa_dropout", status);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// the dropout of an embedding: p as above, and with p > 0 a seed
bool embed_drop(PyObject* po, PyObject* so, int* device, float* p, const at::Tensor** seed) {
  if (!drop_p(po, p) || !maybe(so, device, seed)) return false;
  if (*p == 0.0f) *seed = nullptr;
  return *p == 0.0f || seed_ok(*seed);
}

bool tokens_ok(const at::Tensor& t) {
  return (t.scalar_type() == at::kLong || t.scalar_type() == at::kInt) && t.is_contiguous();
}

bool dtype_arg(PyObject* o, at::ScalarType* t) {
  if (o == Py_None) return true;
  if (!THPDtype_Check(o)) return false;
  *t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  return true;
}

// (tokens, weight, scale, p, seed, out_dtype) -> out
PyObject* embedding_fwd(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return none();
  int device = -1;
  const at::Tensor *t = plain(o[0], &device), *w = plain(o[1], &device), *seed;
  float p;
  if (!t || !w || !tokens_ok(*t) || w->dim() != 2 || w->numel() == 0 || w->size(1) > 1 << 20 || !w->is_contiguous() || !PyFloat_CheckExact(o[2]) ||
      !embed_drop(o[3], o[4], &device, &p, &seed))
    return none();
  at::ScalarType type = w->scalar_type();
  if (dtype_of(type) < 0 || !dtype_arg(o[5], &type) || dtype_of(type) < 0) return none();
  at::DimVector shape(t->sizes().begin(), t->sizes().end());
  shape.push_back(w->size(1));
  at::Tensor out = at::empty(shape, w->options().dtype(type));
  const int status = emb_fwd(t->data_ptr(), (int)t->element_size(), w->data_ptr(), dtype_of(w->scalar_type()), out.data_ptr(),
                             dtype_of(type), t->numel(), w->size(0), (int)w->size(1), (float)PyFloat_AS_DOUBLE(o[2]),
                             seed ? seed->data_ptr() : nullptr, p, stream_of(device));
  if (status) return failed("dpa_embedding_fwd", status);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (dout, tokens, num_embeddings, scale, padding_idx or None, p, seed, dtype) -> dweight
PyObject* embedding_bwd(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return none();
  int device = -1;
  const at::Tensor *g = plain(o[0], &device), *t = plain(o[1], &device), *seed;
  float p;
  if (!g || !t || !tokens_ok(*t) || !g->is_contiguous() || g->dim() != t->dim() + 1 || !PyLong_CheckExact(o[2]) ||
      !PyFloat_CheckExact(o[3]) || (o[4] != Py_None && !PyLong_CheckExact(o[4])) || !embed_drop(o[5], o[6], &device, &p, &seed))
    return none();
  at::ScalarType type = g->scalar_type();
  if (dtype_of(type) < 0 || !dtype_arg(o[7], &type) || dtype_of(type) < 0) return none();
  const int64_t v = PyLong_AsLongLong(o[2]), pad = o[4] == Py_None ? -1 : PyLong_AsLongLong(o[4]), c = g->size(-1);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (v <= 0 || (o[4] != Py_None && pad < 0) || pad >= v || c <= 0 || c > 1 << 20 || t->numel() == 0 || g->sizes().slice(0, t->dim()) != t->sizes())
    return none();
  at::Tensor dw = at::empty({v, c}, g->options().dtype(type));
  const int64_t bytes = emb_bwd_bytes(t->numel(), (int)c);
  at::Tensor ws = at::empty({bytes}, g->options().dtype(at::kByte));
  const int status = emb_bwd(g->data_ptr(), dtype_of(g->scalar_type()), t->data_ptr(), (int)t->element_size(), dw.data_ptr(),
                             dtype_of(type), t->numel(), v, (int)c, (float)PyFloat_AS_DOUBLE(o[3]), pad,
                             seed ? seed->data_ptr() : nullptr, p, ws.data_ptr(), bytes, stream_of(device));
  if (status) return failed("dpa_embedding_bwd", status);
  return THPVariable_Wrap(std::move(dw));
  END_HANDLE_TH_ERRORS
}

// ---- MXFP4 (mxfp4.py) ----
// A plain tensor on the current device (the general way makes another one current first)
const at::Tensor* local(PyObject* o, int* device) {
  const at::Tensor* t = plain(o, device);
  return t && *device == c10::hip::current_device() ? t : nullptr;
}

at::Tensor bytes_like(const at::Tensor& t, int64_t n) { return at::empty({n}, t.options().dtype(at::kByte)); }

// the 16-B aligned beginning of the next part of a workspace
int64_t round256(int64_t n) { return (n + 255) & ~255ll; }

PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    if (t.defined()) {
      PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
    } else {
      Py_INCREF(Py_None);
      PyTuple_SET_ITEM(r, i++, Py_None);
    }
  }
  return r;
}

// x -> (data, scales)
PyObject* mxfp4_quantize(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 1) return none();
  int device = -1;
  const at::Tensor* x = local(o[0], &device);
  if (!x || dtype_of(x->scalar_type()) < 0 || x->dim() < 1 || x->numel() == 0 || x->size(-1) % 32 || !x->is_contiguous() ||
      !aligned16(*x))
    return none();
  at::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = x->size(-1) / 2;
  at::Tensor data = at::empty(shape, x->options().dtype(at::kByte));
  shape.back() = x->size(-1) / 32;
  at::Tensor scales = at::empty(shape, x->options().dtype(at::kByte));
  const int status = mx_quant(x->data_ptr(), dtype_of(x->scalar_type()), x->numel(), data.data_ptr(), scales.data_ptr(),
                              stream_of(device));
  if (status) return failed("dpa_mxfp4_quantize", status);
  return tuple_of({data, scales});
  END_HANDLE_TH_ERRORS
}

bool mxfp4_ok(const at::Tensor& d, const at::Tensor& s) {
  const int64_t k = d.dim();
  return d.scalar_type() == at::kByte && s.scalar_type() == at::kByte && k >= 1 && s.dim() == k &&
         d.sizes().slice(0, k - 1) == s.sizes().slice(0, k - 1) && d.size(-1) == 16 * s.size(-1);
}

// (data, scales, dtype) -> y
PyObject* mxfp4_dequantize(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) return none();
  int device = -1;
  const at::Tensor *d = local(o[0], &device), *s = local(o[1], &device);
  at::ScalarType type = at::kBFloat16;
  if (!d || !s || !mxfp4_ok(*d, *s) || !dtype_arg(o[2], &type) || dtype_of(type) < 0 || d->numel() == 0 || !d->is_contiguous() ||
      !s->is_contiguous() || !aligned16(*d))
    return none();
  at::DimVector shape(d->sizes().begin(), d->sizes().end());
  shape.back() *= 2;
  at::Tensor y = at::empty(shape, d->options().dtype(type));
  const int status = mx_dequant(d->data_ptr(), s->data_ptr(), y.data_ptr(), dtype_of(type), y.numel(), stream_of(device));
  if (status) return failed("dpa_mxfp4_dequantize", status);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// x [..., K] as a matrix of dense rows; its rows
bool matrix_of(const at::Tensor& x, int64_t k, int64_t* rows) {
  if (dtype_of(x.scalar_type()) < 0 || x.dim() < 1 || k <= 0 || x.size(-1) != k || x.numel() == 0 || !x.is_contiguous()) return false;
  *rows = x.numel() / k;
  return true;
}

bool bias_ok(const at::Tensor* b, int64_t n) {
  return !b || (b->scalar_type() == at::kFloat && b->dim() == 1 && b->size(0) == n && b->is_contiguous());
}

// (x, operand, rows, cols, bias, out_dtype) -> y
PyObject* mxfp4_linear(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 6 || !PyLong_CheckExact(o[2]) || !PyLong_CheckExact(o[3])) return none();
  int device = -1;
  const at::Tensor *x = local(o[0], &device), *w = local(o[1], &device), *bias;
  if (!x || !w || !maybe(o[4], &device, &bias)) return none();
  const int64_t n = PyLong_AsLongLong(o[2]), k = PyLong_AsLongLong(o[3]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  int64_t m;
  at::ScalarType type = x->scalar_type();
  if (!dtype_arg(o[5], &type) || dtype_of(type) < 0 || n <= 0 || !matrix_of(*x, k, &m) || !bias_ok(bias, n) ||
      w->scalar_type() != at::kByte || !w->is_contiguous() || !aligned16(*w) || w->numel() != mx_operand_bytes(n, k))
    return none();
  const int64_t bytes = mx_linear_bytes(x->data_ptr(), dtype_of(x->scalar_type()), k, m, n, k);
  at::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = n;
  at::Tensor y = at::empty(shape, x->options().dtype(type)), ws;
  if (bytes) ws = bytes_like(*x, bytes);
  const int status = mx_linear(x->data_ptr(), dtype_of(x->scalar_type()), k, w->data_ptr(),
                               bias ? (const float*)bias->data_ptr() : nullptr, y.data_ptr(), dtype_of(type), m, n, k,
                               bytes ? ws.data_ptr() : nullptr, bytes, stream_of(device));
  if (status) return failed("dpa_mxfp4_linear", status);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// (x, weight, bias, out_dtype) -> (y, operand of x^T, operand of weight^T)
PyObject* mxfp4_train_fwd(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 4) return none();
  int device = -1;
  const at::Tensor *x = local(o[0], &device), *w = local(o[1], &device), *bias;
  if (!x || !w || !maybe(o[2], &device, &bias) || w->dim() != 2) return none();
  const int64_t n = w->size(0), k = w->size(1);
  int64_t m, rows;
  at::ScalarType type = x->scalar_type();
  if (!dtype_arg(o[3], &type) || dtype_of(type) < 0 || n <= 0 || !matrix_of(*x, k, &m) || !matrix_of(*w, k, &rows) ||
      !bias_ok(bias, n))
    return none();
  const int64_t xr = mx_operand_bytes(m, k), xc = mx_operand_bytes(k, m), wr = mx_operand_bytes(n, k), wc = mx_operand_bytes(k, n);
  // (of the gradients' products too: sizes that one of them does not take are refused before a launch)
  if (!xr || !xc || !wr || !wc || mx_plan(m, n, k, DPA_DTYPE_F32, nullptr) || mx_plan(m, k, n, DPA_DTYPE_F32, nullptr) ||
      mx_plan(n, k, m, DPA_DTYPE_F32, nullptr))
    return none();
  const int64_t gemm = mx_gemm_bytes(m, n, k), at_w = round256(xr), at_ws = at_w + round256(wr);
  at::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = n;
  at::Tensor y = at::empty(shape, x->options().dtype(type)), xo = bytes_like(*x, xc), wo = bytes_like(*x, wc),
             ws = bytes_like(*x, at_ws + gemm);
  uint8_t* p = (uint8_t*)ws.data_ptr();
  void* s = stream_of(device);
  int status = mx_operands(x->data_ptr(), dtype_of(x->scalar_type()), m, k, k, p, xo.data_ptr(), nullptr, nullptr, s);
  if (!status) status = mx_operands(w->data_ptr(), dtype_of(w->scalar_type()), n, k, k, p + at_w, wo.data_ptr(), nullptr, nullptr, s);
  if (status) return failed("dpa_mxfp4_operands", status);
  status = mx_gemm(p, p + at_w, bias ? (const float*)bias->data_ptr() : nullptr, y.data_ptr(), dtype_of(type), m, n, k, p + at_ws,
                   gemm, s);
  if (status) return failed("dpa_mxfp4_gemm", status);
  return tuple_of({y, xo, wo});
  END_HANDLE_TH_ERRORS
}

// (dy, operand of x^T, operand of weight^T, n, k, dx dtype, dw dtype, whether dbias, seed) -> (dx, dw, db)
PyObject* mxfp4_bwd(PyObject*, PyObject* const* o, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 9 || !PyLong_CheckExact(o[3]) || !PyLong_CheckExact(o[4])) return none();
  int device = -1;
  const at::Tensor *dy = local(o[0], &device), *xo = local(o[1], &device), *wo = local(o[2], &device), *seed;
  if (!dy || !xo || !wo || !maybe(o[8], &device, &seed) || (seed && !seed_ok(seed))) return none();
  const int64_t n = PyLong_AsLongLong(o[3]), k = PyLong_AsLongLong(o[4]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  int64_t m;
  at::ScalarType dxt = at::kFloat, dwt = at::kFloat;
  if (o[5] == Py_None || o[6] == Py_None || !dtype_arg(o[5], &dxt) || !dtype_arg(o[6], &dwt) || dtype_of(dxt) < 0 ||
      dtype_of(dwt) < 0 || !matrix_of(*dy, n, &m))
    return none();
  const int64_t xc = mx_operand_bytes(k, m), wc = mx_operand_bytes(k, n), dr = mx_operand_bytes(m, n), dc = mx_operand_bytes(n, m);
  if (!xc || !wc || !dr || !dc || xo->numel() != xc || wo->numel() != wc || xo->scalar_type() != at::kByte ||
      wo->scalar_type() != at::kByte || !xo->is_contiguous() || !wo->is_contiguous() || !aligned16(*xo) || !aligned16(*wo))
    return none();
  const bool bias = o[7] == Py_True;
  const int64_t g1 = mx_gemm_bytes(m, k, n), g2 = mx_gemm_bytes(n, k, m);
  const int64_t pieces = (m + 63) / 64, part = bias ? round256(pieces * n * 4) : 0, sums = bias ? column_sum_bytes(pieces, n) : 0;
  const int64_t at_c = round256(dr), at_ws = at_c + round256(dc), most = std::max(std::max(g1, g2), part + sums);
  at::DimVector shape(dy->sizes().begin(), dy->sizes().end());
  shape.back() = k;
  at::Tensor dx = at::empty(shape, dy->options().dtype(dxt)), dw = at::empty({n, k}, dy->options().dtype(dwt)), db,
             ws = bytes_like(*dy, at_ws + most);
  if (bias) db = at::empty({n}, dy->options().dtype(at::kFloat));
  uint8_t* p = (uint8_t*)ws.data_ptr();
  void* s = stream_of(device);
  const int type = dtype_of(dy->scalar_type());
  int status = mx_operands(dy->data_ptr(), type, m, n, n, p, p + at_c, bias ? (float*)(p + at_ws) : nullptr,
                           seed ? seed->data_ptr() : nullptr, s);
  if (status) return failed("dpa_mxfp4_operands", status);
  if (bias) status = column_sum(p + at_ws, DPA_DTYPE_F32, pieces, n, n, db.data_ptr(), p + at_ws + part, sums, s);
  if (status) return failed("dpa_column_sum", status);
  status = mx_gemm(p, wo->data_ptr(), nullptr, dx.data_ptr(), dtype_of(dxt), m, k, n, p + at_ws, g1, s);
  if (!status) status = mx_gemm(p + at_c, xo->data_ptr(), nullptr, dw.data_ptr(), dtype_of(dwt), n, k, m, p + at_ws, g2, s);
  if (status) return failed("dpa_mxfp4_gemm", status);
  return tuple_of({dx, dw, db});
  END_HANDLE_TH_ERRORS
}

// Byte strides of a cache's part [batch, tokens, 2, heads, width] in the order batch, token, head
void part_strides(const at::Tensor& t, int64_t* s) {
  s[0] = t.size(0) > 1 ? t.stride(0) : 0, s[1] = t.size(1) > 1 ? t.stride(1) : 0, s[2] = t.size(3) > 1 ? t.stride(3) : 0;
}

// (q, data, scales, key_lengths, key_mask, scale) -> (out, lse)
PyObject* mxfp4_attention(PyObject*, PyObject* const* o, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return none();
  int device = -1;
  const at::Tensor *q = local(o[0], &device), *d = local(o[1], &device), *x = local(o[2], &device), *lengths, *mask;
  if (!q || !d || !x || !maybe(o[3], &device, &lengths) || !maybe(o[4], &device, &mask)) return none();
  if (q->dim() != 4 || d->dim() != 5 || !mxfp4_ok(*d, *x) || d->size(2) != 2 || d->stride(4) != 1 ||
      (x->stride(4) != 1 && x->size(4) > 1) || !aligned16(*d) || d->stride(2) % 16 || d->size(4) * 2 % 32)
    return none();
  // (shapes, masks and the scale as over keys of that shape: strides of k and v are those of q there)
  DpaCrossAttention c{};
  const int64_t b = q->size(0), lk = d->size(1), g = d->size(3), dim = 2 * d->size(4), most = INT32_MAX;
  if (d->size(0) != b || q->size(3) != dim || g <= 0 || lk <= 0 || lk > most || g > most || q->size(2) % g || dim > 128 || dim <= 0 ||
      !describe_queries(c, *q, lk, lengths, mask, o[5]))
    return none();
  DpaCrossAttentionMxfp4 a{};
  part_strides(*d, a.k_data_stride), part_strides(*x, a.k_scale_stride);
  for (int i = 0; i < 3; ++i) {
    if (a.k_data_stride[i] % 16) return none();
    a.q_stride[i] = c.q_stride[i], a.v_data_stride[i] = a.k_data_stride[i], a.v_scale_stride[i] = a.k_scale_stride[i];
  }
  at::Tensor out = at::empty(q->sizes(), q->options());
  at::Tensor lse = at::empty({b, q->size(2), q->size(1)}, q->options().dtype(at::kFloat)), ws;
  a.q = c.q, a.key_lengths = c.key_lengths, a.key_mask = c.key_mask, a.mask_stride = c.mask_stride;
  a.k_data = d->data_ptr(), a.v_data = (uint8_t*)d->data_ptr() + d->stride(2);
  a.k_scales = x->data_ptr(), a.v_scales = (uint8_t*)x->data_ptr() + x->stride(2);
  a.out = out.data_ptr(), a.lse = (float*)lse.data_ptr();
  a.dtype = c.dtype, a.batch = c.batch, a.q_len = c.q_len, a.kv_len = (int32_t)lk;
  a.heads = c.heads, a.kv_heads = (int32_t)g, a.head_dim = (int32_t)dim, a.scale = c.scale;
  const int64_t bytes = mx_attn_bytes(&a);
  if (bytes) ws = bytes_like(*q, bytes);
  const int status = mx_attn(&a, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(device));
  if (status) return failed("dpa_cross_attention_mxfp4", status);
  return tuple_of({out, lse});
  END_HANDLE_TH_ERRORS
}

// init(addresses of the library's entries, in this order)
PyObject* init(PyObject*, PyObject* const* o, Py_ssize_t n) {
  void** const to[] = {(void**)&attn_fwd, (void**)&attn_fwd_bytes, (void**)&attn_bwd, (void**)&attn_bwd_bytes, (void**)&drop,
                       (void**)&emb_fwd, (void**)&emb_bwd, (void**)&emb_bwd_bytes, (void**)&status_string,
                       (void**)&mx_quant, (void**)&mx_dequant, (void**)&mx_operand_bytes, (void**)&mx_operands,
                       (void**)&mx_gemm, (void**)&mx_gemm_bytes, (void**)&mx_plan, (void**)&mx_linear, (void**)&mx_linear_bytes,
                       (void**)&column_sum, (void**)&column_sum_bytes, (void**)&mx_attn, (void**)&mx_attn_bytes};
  if (n != (Py_ssize_t)(sizeof(to) / sizeof(to[0]))) {
    PyErr_Format(PyExc_TypeError, "init takes %d addresses, got %d", (int)(sizeof(to) / sizeof(to[0])), (int)n);
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    void* const address = PyLong_AsVoidPtr(o[i]);
    if (PyErr_Occurred()) return nullptr;
    *to[i] = address;
  }
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(init), FAST(attention_fwd), FAST(attention_bwd), FAST(dropout),
                         FAST(embedding_fwd), FAST(embedding_bwd), FAST(mxfp4_quantize),
                         FAST(mxfp4_dequantize), FAST(mxfp4_linear), FAST(mxfp4_train_fwd), FAST(mxfp4_bwd),
                         FAST(mxfp4_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "dpa_fast_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dpa_fast_calls() { return PyModule_Create(&module); }
