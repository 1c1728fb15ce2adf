// srw_host.cpp -- the Python side of the paged cache's calls, and of sampling, in
// native code.
//
// For single tokens the kernels take a few microseconds, and checking a call's
// tensors and describing it from Python takes more than that.  Here a call whose
// tensors are as the C entry points take them is described and made in about a
// microsecond beside its launch.  Anything else -- another type, shape, stride or
// alignment, whether an error or a case that kv.py prepares first -- gives None
// (False), and kv.py (sampling.py) goes through its own checks, which say what is wrong.
//
// Tensors are looked at, nothing is kept of them; the current stream is the
// caller's last argument.

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cfloat>
#include <cmath>

#include "srw_amd.h"

namespace {

constexpr int64_t kMost = 0x7fffffff;

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool plain(const at::Tensor* t, at::ScalarType type, int64_t dims, int device) {
  return t && t->scalar_type() == type && t->dim() == dims && t->is_cuda() && t->get_device() == device;
}

// The calls have no derivatives: kv.py refuses tensors that want them, of either mode.
bool wants_grad(const at::Tensor* t) {
  return (t->requires_grad() && c10::GradMode::is_enabled()) || t->_fw_grad(/*level=*/0).defined();
}

bool i64(PyObject* o, int64_t* v) {
  if (!PyLong_Check(o)) return false;
  *v = PyLong_AsLongLong(o);
  return !(*v == -1 && PyErr_Occurred());
}

PyObject* none() {
  PyErr_Clear();
  Py_RETURN_NONE;
}

// The pages of a KvPages: the tensors k, v, k_scale, v_scale, looked at anew in
// every call (their memory can be another's by then), and, behind them, what
// host_pages gave for them, which still has to be so (kv.py refuses others).
bool pages_of(PyObject* o, srw_kv_t* c, int* device) {
  if (!PyTuple_CheckExact(o) || (PyTuple_GET_SIZE(o) != 4 && PyTuple_GET_SIZE(o) != 10)) return false;
  const at::Tensor *k = tensor(PyTuple_GET_ITEM(o, 0)), *v = tensor(PyTuple_GET_ITEM(o, 1));
  if (!k || !v || k->dim() != 4 || v->dim() != 4 || !k->is_cuda()) return false;
  *device = static_cast<int>(k->get_device());
  const auto type = k->scalar_type();
  const int kind = type == at::kBFloat16 ? SRW_KV_BF16 : type == at::kChar ? SRW_KV_INT8
                   : type == at::kFloat8_e4m3fn                            ? SRW_KV_FP8
                                                                           : -1;
  const int64_t N = k->size(0), H = k->size(1), P = k->size(2), D = k->size(3);
  if (kind < 0 || !plain(v, type, 4, *device) || v->size(0) != N || v->size(1) != H || v->size(2) != D ||
      v->size(3) != P || !k->is_contiguous() || !v->is_contiguous() || H > kMost || P > kMost || D > kMost ||
      wants_grad(k) || wants_grad(v))
    return false;
  float* scale[2] = {nullptr, nullptr};
  for (int i = 0; i < 2; ++i) {
    PyObject* so = PyTuple_GET_ITEM(o, 2 + i);
    if (kind == SRW_KV_BF16) {
      if (so != Py_None) return false;
      continue;
    }
    const at::Tensor* s = tensor(so);
    if (!plain(s, at::kFloat, 3, *device) || s->size(0) != N || s->size(1) != H || s->size(2) != P ||
        !s->is_contiguous() || wants_grad(s))
      return false;
    scale[i] = static_cast<float*>(s->data_ptr());
  }
  if (PyTuple_GET_SIZE(o) == 10) {
    const int64_t now[6] = {N, H, P, D, kind, *device};
    for (int i = 0; i < 6; ++i) {
      int64_t then;
      if (!i64(PyTuple_GET_ITEM(o, 4 + i), &then) || then != now[i]) return false;
    }
  }
  c->k = k->data_ptr();
  c->v = v->data_ptr();
  c->k_scale = scale[0];
  c->v_scale = scale[1];
  c->n_pages = N;
  c->n_kv_heads = static_cast<int32_t>(H);
  c->page_size = static_cast<int32_t>(P);
  c->head_dim = static_cast<int32_t>(D);
  c->kind = kind;
  return true;
}

// table, lens, cu (a tensor or None) of T tokens.
bool sequences(PyObject* table, PyObject* lens, PyObject* cu, int64_t T, int device, srw_kv_t* c) {
  const at::Tensor *t = tensor(table), *l = tensor(lens), *u = cu == Py_None ? nullptr : tensor(cu);
  if (!plain(t, at::kInt, 2, device) || !plain(l, at::kInt, 1, device)) return false;
  c->B = l->size(0);
  c->T = T;
  if (!l->is_contiguous() || t->size(0) != c->B || t->stride(1) != 1 || t->stride(0) < t->size(1)) return false;
  if (cu == Py_None ? T != c->B : !plain(u, at::kInt, 1, device) || u->size(0) != c->B + 1 || !u->is_contiguous())
    return false;
  c->table = static_cast<const int32_t*>(t->data_ptr());
  c->lens = static_cast<const int32_t*>(l->data_ptr());
  c->cu = u ? static_cast<const int32_t*>(u->data_ptr()) : nullptr;
  c->table_width = t->size(1);
  c->table_stride = t->stride(0);
  return true;
}

// Rows [T, heads, head_dim] as the kernels read them, unit elements at a time, and
// their strides (that of a single token or head is never used, and may be anything).
bool rows(const at::Tensor* t, int64_t unit, int32_t head_dim, int64_t* token, int64_t* head) {
  *head = t->size(1) == 1 ? head_dim : t->stride(1);
  *token = t->size(0) == 1 ? t->size(1) * head_dim : t->stride(0);
  return t->size(2) == head_dim && t->stride(2) == 1 && *token % unit == 0 && *head % unit == 0 &&
         reinterpret_cast<uintptr_t>(t->data_ptr()) % (unit * t->element_size()) == 0;
}

// pages((k, v, k_scale, v_scale)) -> (n_pages, heads, page_size, head_dim, kind, device), or None
PyObject* host_pages(PyObject* const* a, Py_ssize_t n) {
  srw_kv_t c{};
  int device;
  if (n != 1 || !pages_of(a[0], &c, &device)) return none();
  return Py_BuildValue("(Liiiii)", static_cast<long long>(c.n_pages), c.n_kv_heads, c.page_size, c.head_dim, c.kind,
                       device);
}

// write(pages, k, v, table, lens, cu, stream) -> status, or None
PyObject* host_write(PyObject* const* a, Py_ssize_t n) {
  srw_kv_t c{};
  int device;
  int64_t stream;
  if (n != 7 || !pages_of(a[0], &c, &device) || !i64(a[6], &stream)) return none();
  const at::Tensor *k = tensor(a[1]), *v = tensor(a[2]);
  if (!k || !v || k->dim() != 3) return none();
  const auto type = k->scalar_type();
  if ((type != at::kBFloat16 && type != at::kFloat) || !plain(k, type, 3, device) || !plain(v, type, 3, device) ||
      wants_grad(k) || wants_grad(v))
    return none();
  const int64_t T = k->size(0);
  srw_kv_rows_t r{k->data_ptr(), v->data_ptr(), 0, 0, 0, 0};
  if (v->size(0) != T || k->size(1) != c.n_kv_heads || v->size(1) != c.n_kv_heads ||
      !rows(k, 4, c.head_dim, &r.k_token_stride, &r.k_head_stride) ||
      !rows(v, 4, c.head_dim, &r.v_token_stride, &r.v_head_stride) || !sequences(a[3], a[4], a[5], T, device, &c))
    return none();
  const int status = srw_kv_write(&c, &r, type == at::kFloat ? SRW_F32 : SRW_BF16, reinterpret_cast<void*>(stream));
  for (int i = 0; i < 4; ++i) {  // written in place
    const at::Tensor* t = tensor(PyTuple_GET_ITEM(a[0], i));
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  }
  return PyLong_FromLong(status);
}

// read(pages, table, lens, cu, T, float32, stream) -> (k, v), or None
PyObject* host_read(PyObject* const* a, Py_ssize_t n) {
  srw_kv_t c{};
  int device;
  int64_t T, f32, stream;
  if (n != 7 || !pages_of(a[0], &c, &device) || !i64(a[4], &T) || !i64(a[5], &f32) || !i64(a[6], &stream)) return none();
  if (T < 0 || !sequences(a[1], a[2], a[3], T, device, &c)) return none();
  const auto opt = at::TensorOptions().dtype(f32 ? at::kFloat : at::kBFloat16).device(at::kCUDA, device);
  const int64_t H = c.n_kv_heads, D = c.head_dim;
  at::Tensor k = at::empty({T, H, D}, opt), v = at::empty({T, H, D}, opt);
  const srw_kv_rows_t r{k.data_ptr(), v.data_ptr(), H * D, D, H * D, D};
  const int status = srw_kv_read(&c, &r, f32 ? SRW_F32 : SRW_BF16, reinterpret_cast<void*>(stream));
  if (status != SRW_OK) return none();  // (the general path says what is wrong)
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(v)));
  return out;
}

// attention(pages, q, table, lens, cu, max_new, scale, window, sinks, stream) -> out, or None
PyObject* host_attention(PyObject* const* a, Py_ssize_t n) {
  srw_attention_t s{};
  int device;
  int64_t most, window, sinks, stream;
  if (n != 10 || !pages_of(a[0], &s.kv, &device) || !i64(a[5], &most) || !i64(a[7], &window) || !i64(a[8], &sinks) ||
      !i64(a[9], &stream) || !PyFloat_Check(a[6]))
    return none();
  const at::Tensor* q = tensor(a[1]);
  if (!plain(q, at::kBFloat16, 3, device) || wants_grad(q) ||
      !rows(q, 8, s.kv.head_dim, &s.q_token_stride, &s.q_head_stride))
    return none();
  if (most < 0 || most > kMost || window < 0 || window > kMost || sinks < 0 || sinks > kMost || q->size(1) > kMost)
    return none();
  const int64_t T = q->size(0);
  if (T == 0 || !sequences(a[2], a[3], a[4], T, device, &s.kv)) return none();
  s.q = q->data_ptr();
  s.n_heads = static_cast<int32_t>(q->size(1));
  s.max_new = static_cast<int32_t>(most);
  s.window = static_cast<int32_t>(window);
  s.sinks = static_cast<int32_t>(sinks);
  s.scale = static_cast<float>(PyFloat_AS_DOUBLE(a[6]));
  size_t need = 0;
  if (srw_attention_workspace_size(&s, &need) != SRW_OK) return none();
  const auto opt = at::TensorOptions().device(at::kCUDA, device);
  at::Tensor out = at::empty({T, q->size(1), s.kv.head_dim}, opt.dtype(at::kBFloat16)), ws;
  if (need) ws = at::empty({static_cast<int64_t>(need)}, opt.dtype(at::kByte));
  s.out = out.data_ptr();
  if (srw_attention(&s, need ? ws.data_ptr() : nullptr, need, reinterpret_cast<void*>(stream)) != SRW_OK) return none();
  return THPVariable_Wrap(std::move(out));
}

// The index of pages of c: (codes, scale).
bool index_of(PyObject* o, const srw_kv_t& c, int device, srw_kv_index_t* x) {
  if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 2) return false;
  const at::Tensor *codes = tensor(PyTuple_GET_ITEM(o, 0)), *scale = tensor(PyTuple_GET_ITEM(o, 1));
  if (!plain(codes, at::kChar, 3, device) || !plain(scale, at::kFloat, 2, device) || !codes->is_contiguous() ||
      !scale->is_contiguous() || wants_grad(scale) || codes->size(0) != c.n_pages || codes->size(1) != c.n_kv_heads ||
      codes->size(2) != c.head_dim || scale->size(0) != c.n_pages || scale->size(1) != c.n_kv_heads)
    return false;
  x->codes = static_cast<int8_t*>(codes->data_ptr());
  x->scale = static_cast<float*>(scale->data_ptr());
  return true;
}

// index_pair((codes, scale)) -> whether they are an index of some pages
PyObject* host_index_pair(PyObject* const* a, Py_ssize_t n) {
  if (n != 1 || !PyTuple_CheckExact(a[0]) || PyTuple_GET_SIZE(a[0]) != 2) Py_RETURN_FALSE;
  const at::Tensor* codes = tensor(PyTuple_GET_ITEM(a[0], 0));
  if (!codes || !codes->is_cuda() || codes->dim() != 3) Py_RETURN_FALSE;
  srw_kv_t c{};
  srw_kv_index_t x{};
  c.n_pages = codes->size(0);
  c.n_kv_heads = static_cast<int32_t>(codes->size(1));
  c.head_dim = static_cast<int32_t>(codes->size(2));
  if (index_of(a[0], c, static_cast<int>(codes->get_device()), &x)) Py_RETURN_TRUE;
  Py_RETURN_FALSE;
}

void written(const at::Tensor* t) {
  if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

// index(pages, index, table, lens, cu, T, stream) -> status, or None
PyObject* host_index(PyObject* const* a, Py_ssize_t n) {
  srw_kv_t c{};
  srw_kv_index_t x{};
  int device;
  int64_t T, stream;
  if (n != 7 || !pages_of(a[0], &c, &device) || !index_of(a[1], c, device, &x) || !i64(a[5], &T) || !i64(a[6], &stream))
    return none();
  if (T < 0 || !sequences(a[2], a[3], a[4], T, device, &c)) return none();
  const int status = srw_kv_index(&c, &x, reinterpret_cast<void*>(stream));
  written(tensor(PyTuple_GET_ITEM(a[1], 0)));
  written(tensor(PyTuple_GET_ITEM(a[1], 1)));
  return PyLong_FromLong(status);
}

// select(pages, index, q, table, lens, cu, n, first, last, stream) -> keep, or None
PyObject* host_select(PyObject* const* a, Py_ssize_t n) {
  srw_kv_select_t s{};
  int device;
  int64_t most, first, last, stream;
  if (n != 10 || !pages_of(a[0], &s.kv, &device) || !index_of(a[1], s.kv, device, &s.index) || !i64(a[6], &most) ||
      !i64(a[7], &first) || !i64(a[8], &last) || !i64(a[9], &stream))
    return none();
  const at::Tensor* q = tensor(a[2]);
  if (!plain(q, at::kBFloat16, 3, device) || wants_grad(q) || q->size(1) > kMost ||
      !rows(q, 4, s.kv.head_dim, &s.q_token_stride, &s.q_head_stride))
    return none();
  if (most < 1 || most > kMost || first < 0 || first > kMost || last < 0 || last > kMost) return none();
  const int64_t T = q->size(0);
  if (!sequences(a[3], a[4], a[5], T, device, &s.kv)) return none();
  s.q = q->data_ptr();
  s.n_heads = static_cast<int32_t>(q->size(1));
  s.n = static_cast<int32_t>(most);
  s.first = static_cast<int32_t>(first);
  s.last = static_cast<int32_t>(last);
  at::Tensor keep = at::empty({T, s.kv.n_kv_heads, most}, at::TensorOptions().device(at::kCUDA, device).dtype(at::kInt));
  s.keep = static_cast<int32_t*>(keep.data_ptr());
  if (srw_kv_select(&s, reinterpret_cast<void*>(stream)) != SRW_OK) return none();
  return THPVariable_Wrap(std::move(keep));
}

// attention_kept(pages, q, table, lens, cu, scale, keep, stream) -> out, or None
PyObject* host_attention_kept(PyObject* const* a, Py_ssize_t n) {
  srw_attention_t s{};
  int device;
  int64_t stream;
  if (n != 8 || !pages_of(a[0], &s.kv, &device) || !PyFloat_Check(a[5]) || !i64(a[7], &stream)) return none();
  const at::Tensor *q = tensor(a[1]), *keep = tensor(a[6]);
  if (!plain(q, at::kBFloat16, 3, device) || wants_grad(q) || q->size(1) > kMost ||
      !rows(q, 8, s.kv.head_dim, &s.q_token_stride, &s.q_head_stride))
    return none();
  const int64_t T = q->size(0);
  if (T == 0 || !plain(keep, at::kInt, 3, device) || !keep->is_contiguous() || keep->size(0) != T ||
      keep->size(1) != s.kv.n_kv_heads || !sequences(a[2], a[3], a[4], T, device, &s.kv))
    return none();
  s.q = q->data_ptr();
  s.n_heads = static_cast<int32_t>(q->size(1));
  s.scale = static_cast<float>(PyFloat_AS_DOUBLE(a[5]));
  const int32_t* lists = static_cast<const int32_t*>(keep->data_ptr());
  size_t need = 0;
  if (srw_attention_kept_workspace_size(&s, keep->size(2), &need) != SRW_OK) return none();
  const auto opt = at::TensorOptions().device(at::kCUDA, device);
  at::Tensor out = at::empty({T, q->size(1), s.kv.head_dim}, opt.dtype(at::kBFloat16)), ws;
  if (need) ws = at::empty({static_cast<int64_t>(need)}, opt.dtype(at::kByte));
  s.out = out.data_ptr();
  if (srw_attention_kept(&s, lists, keep->size(2), need ? ws.data_ptr() : nullptr, need,
                         reinterpret_cast<void*>(stream)) != SRW_OK)
    return none();
  return THPVariable_Wrap(std::move(out));
}

// The tensors of a copy: [layers, n_pages, ...], a layer's pages contiguous.
bool copied(PyObject* list, int device, srw_kv_copy_t* c) {
  if (!PyList_CheckExact(list) && !PyTuple_CheckExact(list)) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
  if (n < 1 || n > SRW_KV_COPY_TENSORS) return false;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t = tensor(PySequence_Fast_GET_ITEM(list, i));
    if (!t || t->dim() < 2 || !t->is_cuda() || t->get_device() != device || !t->is_contiguous() || wants_grad(t)) return false;
    int64_t bytes = static_cast<int64_t>(t->element_size());
    for (int64_t d = 2; d < t->dim(); ++d) bytes *= t->size(d);
    const int64_t pages = t->size(1), stride = pages * bytes;
    if (i == 0) {
      c->n_layers = t->size(0);
      c->n_src_pages = c->n_dst_pages = pages;
    }
    if (t->size(0) != c->n_layers || pages != c->n_src_pages) return false;
    c->src[i] = c->dst[i] = t->data_ptr();
    c->page_bytes[i] = bytes;
    c->src_layer_stride[i] = c->dst_layer_stride[i] = stride;
  }
  c->n_tensors = static_cast<int32_t>(n);
  return true;
}

// copy(tensors, src, dst, device, stream) -> status, or None: within contiguous tensors of the
// current device; src and dst arrays of C ints
PyObject* host_copy(PyObject* const* a, Py_ssize_t n) {
  srw_kv_copy_t c{};
  int64_t stream, device;
  if (n != 5 || !i64(a[3], &device) || !i64(a[4], &stream) || !copied(a[0], static_cast<int>(device), &c)) return none();
  Py_buffer src, dst;
  if (PyObject_GetBuffer(a[1], &src, PyBUF_SIMPLE)) return none();
  if (PyObject_GetBuffer(a[2], &dst, PyBUF_SIMPLE)) {
    PyBuffer_Release(&src);
    return none();
  }
  int status = -1;
  if (src.len == dst.len) {
    c.src_page = static_cast<const int32_t*>(src.buf);
    c.dst_page = static_cast<const int32_t*>(dst.buf);
    c.n_pairs = static_cast<int64_t>(src.len / 4);
    status = srw_kv_copy(&c, reinterpret_cast<void*>(stream));
  }
  PyBuffer_Release(&src);
  PyBuffer_Release(&dst);
  if (status != SRW_OK) return none();  // (the general path says what is wrong)
  if (c.n_pairs)
    for (Py_ssize_t i = 0; i < c.n_tensors; ++i) written(tensor(PySequence_Fast_GET_ITEM(a[0], i)));
  return PyLong_FromLong(status);
}

// A parameter of sampling: a tensor [B] of this type, or a number that its check takes.
bool parameter(PyObject* o, at::ScalarType type, int64_t B, int device, const void** array, double* number) {
  if (const at::Tensor* t = tensor(o)) {
    if (!plain(t, type, 1, device) || t->size(0) != B || !t->is_contiguous() || wants_grad(t)) return false;
    *array = t->data_ptr();
    return true;
  }
  if (type == at::kInt) {
    int64_t v;
    if (!i64(o, &v) || v < 0 || v > kMost) return false;
    *number = static_cast<double>(v);
    return true;
  }
  if (!PyFloat_Check(o) && !PyLong_CheckExact(o)) return false;
  *number = PyFloat_AsDouble(o);
  return *number >= 0 && (*number <= FLT_MAX || *number == HUGE_VAL);  // (an error gives -1; inf is a temperature)
}

// sample(logits, u, temperature, top_k, top_p, min_p, device, stream) -> (tokens, logprobs), or None
PyObject* host_sample(PyObject* const* a, Py_ssize_t n) {
  int64_t device, stream;
  if (n != 8 || !i64(a[6], &device) || !i64(a[7], &stream)) return none();
  const at::Tensor *logits = tensor(a[0]), *u = tensor(a[1]);
  if (!logits || (logits->scalar_type() != at::kFloat && logits->scalar_type() != at::kBFloat16)) return none();
  if (!plain(logits, logits->scalar_type(), 2, static_cast<int>(device)) || wants_grad(logits)) return none();
  const int64_t B = logits->size(0), V = logits->size(1);
  if (V < 1 || (V > 1 && logits->stride(1) != 1)) return none();
  if (!plain(u, at::kFloat, 1, static_cast<int>(device)) || u->size(0) != B || !u->is_contiguous() || wants_grad(u)) return none();
  const void *t = nullptr, *k = nullptr, *p = nullptr, *m = nullptr;
  double number[4] = {0, 0, 0, 0};
  if (!parameter(a[2], at::kFloat, B, static_cast<int>(device), &t, &number[0]) ||
      !parameter(a[3], at::kInt, B, static_cast<int>(device), &k, &number[1]) ||
      !parameter(a[4], at::kFloat, B, static_cast<int>(device), &p, &number[2]) ||
      !parameter(a[5], at::kFloat, B, static_cast<int>(device), &m, &number[3]))
    return none();
  const auto opt = at::TensorOptions().device(at::kCUDA, static_cast<c10::DeviceIndex>(device));
  at::Tensor token = at::empty({B}, opt.dtype(at::kLong)), logprob = at::empty({B}, opt.dtype(at::kFloat)), ws;
  srw_sample_t d{};
  d.logits = logits->data_ptr();
  d.row_stride = logits->stride(0);
  d.B = B;
  d.V = V;
  d.u = static_cast<const float*>(u->data_ptr());
  d.temperature = static_cast<const float*>(t);
  d.top_k = static_cast<const int32_t*>(k);
  d.top_p = static_cast<const float*>(p);
  d.min_p = static_cast<const float*>(m);
  d.temperature_all = static_cast<float>(number[0]);
  d.top_k_all = static_cast<int32_t>(number[1]);
  d.top_p_all = static_cast<float>(number[2]);
  d.min_p_all = static_cast<float>(number[3]);
  d.token = static_cast<int64_t*>(token.data_ptr());
  d.logprob = static_cast<float*>(logprob.data_ptr());
  d.dtype = logits->scalar_type() == at::kFloat ? SRW_F32 : SRW_BF16;
  size_t need = 0;
  if (srw_sample_workspace_size(&d, &need) != SRW_OK) return none();
  if (need) ws = at::empty({static_cast<int64_t>(need)}, opt.dtype(at::kByte));
  if (srw_sample(&d, need ? ws.data_ptr() : nullptr, need, reinterpret_cast<void*>(stream)) != SRW_OK) return none();
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(token)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(logprob)));
  return out;
}

// Nothing thrown leaves through Python's C frames: a tensor without memory of its
// own, no memory for an output -- the general path meets it again and says so.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* caught(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(a, n);
  } catch (...) {
    return none();
  }
}

PyMethodDef methods[] = {
    {"pages", reinterpret_cast<PyCFunction>(caught<host_pages>), METH_FASTCALL, nullptr},
    {"write", reinterpret_cast<PyCFunction>(caught<host_write>), METH_FASTCALL, nullptr},
    {"read", reinterpret_cast<PyCFunction>(caught<host_read>), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(caught<host_attention>), METH_FASTCALL, nullptr},
    {"index_pair", reinterpret_cast<PyCFunction>(caught<host_index_pair>), METH_FASTCALL, nullptr},
    {"index", reinterpret_cast<PyCFunction>(caught<host_index>), METH_FASTCALL, nullptr},
    {"select", reinterpret_cast<PyCFunction>(caught<host_select>), METH_FASTCALL, nullptr},
    {"attention_kept", reinterpret_cast<PyCFunction>(caught<host_attention_kept>), METH_FASTCALL, nullptr},
    {"copy", reinterpret_cast<PyCFunction>(caught<host_copy>), METH_FASTCALL, nullptr},
    {"sample", reinterpret_cast<PyCFunction>(caught<host_sample>), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_srw_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__srw_host(void) { return PyModule_Create(&module); }
