// The conditioning operators' Python calls where nothing has to be converted: checks, allocation and
// the C entry in one native call. An eager call on small operands waits for its host side, of which
// Python code and its arguments' conversion were two thirds: 4 x 1 queries over 77 keys 9.6 us in
// Python, 3.4 us of it the launch.
//
// Every function returns None for a call that it does not take -- operands that need a copy, are
// refused, or are anything but plain strided GPU tensors; conditioning.py then goes the general way,
// which copies or raises. A module of the CPython API; the kernels' library is not linked but handed
// over as addresses (init).
#include <Python.h>

#include <ATen/ATen.h>
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

// What forward and backward describe alike. Sizes past 32 bits and the rest that the entry refuses
// are left to it, and so to the general way's message.
bool describe(DpaCrossAttention& a, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
              const at::Tensor* lengths, const at::Tensor* mask, PyObject* scale) {
  if (q.dim() != 4 || k.dim() != 4 || v.dim() != 4 || q.scalar_type() != k.scalar_type() ||
      q.scalar_type() != v.scalar_type() || (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf) ||
      k.sizes() != v.sizes() || k.size(0) != q.size(0) || k.size(3) != q.size(3))
    return false;
  const int64_t b = q.size(0), lq = q.size(1), h = q.size(2), d = q.size(3), lk = k.size(1), g = k.size(2);
  const int64_t most = INT32_MAX;
  if (b <= 0 || lq <= 0 || lk <= 0 || h <= 0 || g <= 0 || d <= 0 || d % 8 || d > 128 || h % g || b > most || lq > most ||
      lk > most || h > most)
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
  if (!strides_of(q, a.q_stride) || !strides_of(k, a.k_stride) || !strides_of(v, a.v_stride)) return false;
  a.q = q.data_ptr(), a.k = k.data_ptr(), a.v = v.data_ptr();
  a.key_lengths = lengths ? (const int32_t*)lengths->data_ptr() : nullptr;
  a.key_mask = mask ? (const uint8_t*)mask->data_ptr() : nullptr;
  a.mask_stride = mask ? mask->stride(0) : 0;
  a.dtype = dtype_of(q.scalar_type());
  a.batch = (int32_t)b, a.q_len = (int32_t)lq, a.kv_len = (int32_t)lk;
  a.heads = (int32_t)h, a.kv_heads = (int32_t)g, a.head_dim = (int32_t)d;
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

// init(addresses of the library's entries, in the order of the pointers above)
PyObject* init(PyObject*, PyObject* args) {
  unsigned long long f[9];
  if (!PyArg_ParseTuple(args, "KKKKKKKKK", f, f + 1, f + 2, f + 3, f + 4, f + 5, f + 6, f + 7, f + 8)) return nullptr;
  attn_fwd = reinterpret_cast<decltype(attn_fwd)>(f[0]);
  attn_fwd_bytes = reinterpret_cast<decltype(attn_fwd_bytes)>(f[1]);
  attn_bwd = reinterpret_cast<decltype(attn_bwd)>(f[2]);
  attn_bwd_bytes = reinterpret_cast<decltype(attn_bwd_bytes)>(f[3]);
  drop = reinterpret_cast<decltype(drop)>(f[4]);
  emb_fwd = reinterpret_cast<decltype(emb_fwd)>(f[5]);
  emb_bwd = reinterpret_cast<decltype(emb_bwd)>(f[6]);
  emb_bwd_bytes = reinterpret_cast<decltype(emb_bwd_bytes)>(f[7]);
  status_string = reinterpret_cast<decltype(status_string)>(f[8]);
  Py_RETURN_NONE;
}

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"init", init, METH_VARARGS, nullptr}, FAST(attention_fwd), FAST(attention_bwd), FAST(dropout),
                         FAST(embedding_fwd), FAST(embedding_bwd), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "dpa_fast_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_dpa_fast_calls() { return PyModule_Create(&module); }
