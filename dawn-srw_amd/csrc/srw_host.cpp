// srw_host.cpp -- the Python side of the paged cache's calls in native code.
//
// For single tokens the kernels take a few microseconds, and checking a call's
// tensors and describing it from Python takes more than that.  Here a call whose
// tensors are as the C entry points take them is described and made in about a
// microsecond beside its launch.  Anything else -- another type, shape, stride or
// alignment, whether an error or a case that kv.py prepares first -- gives None
// (False), and kv.py goes through its own checks, which say what is wrong.
//
// Tensors are looked at, nothing is kept of them; the current stream is the
// caller's last argument.

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

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
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_srw_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__srw_host(void) { return PyModule_Create(&module); }
