// The tensors of append_kv, paged_attention, key_bounds, select_pages and
// selected_attention (attention.py) to the structs and arguments of include/hypno_hip.h.
// What the Python functions check one attribute at a time (5 to 7 us a call, more than a
// token's kernel takes) is read from the tensors here, 1 to 2 us.  Only calls that are
// right are made: for any other the answer is NotImplemented, and the Python functions
// say what is wrong with it.
#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/hypno_hip.h"

namespace {

decltype(&hypno_hip_append_kv_dev) g_append = nullptr;
decltype(&hypno_hip_paged_attention_dev) g_attend = nullptr;
decltype(&hypno_hip_key_bounds_dev) g_bounds = nullptr;
decltype(&hypno_hip_select_pages_dev) g_select = nullptr;
decltype(&hypno_hip_selected_attention_dev) g_selected = nullptr;
PyObject* g_device = nullptr;  // current device, and the raw stream of one
PyObject* g_stream = nullptr;

PyObject* other() { Py_RETURN_NOTIMPLEMENTED; }

const at::Tensor* tensor(PyObject* o, int dev, at::ScalarType type, int64_t dim) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || (dev >= 0 && t.get_device() != dev) || t.scalar_type() != type ||
      t.dim() != dim || t.layout() != at::kStrided)
    return nullptr;
  return &t;
}

struct Rows {
  const at::Tensor* t;
  int64_t n, h, d, stride;
};

// [tokens, heads, head_dim] fp32 whose heads are contiguous (none empty).
bool rows(PyObject* o, int dev, Rows& r) {
  r.t = tensor(o, dev, at::kFloat, 3);
  if (!r.t) return false;
  const auto s = r.t->sizes(), st = r.t->strides();
  r.n = s[0], r.h = s[1], r.d = s[2], r.stride = st[0];
  if (r.n <= 0 || r.h <= 0 || r.d <= 0 || (r.d > 1 && st[2] != 1) || (r.h > 1 && st[1] != r.d))
    return false;
  if (r.n == 1) r.stride = r.h * r.d;
  return r.stride >= r.h * r.d;
}

// Elements from one page to the next (0: no gap), or -1.
int64_t page_stride(const at::Tensor& t) {
  if (t.is_contiguous()) return 0;
  int64_t inner = 1;
  for (int64_t i = t.dim() - 1; i > 0; i--) {
    if (t.size(i) > 1 && t.stride(i) != inner) return -1;
    inner *= t.size(i);
  }
  if (t.size(0) <= 1 || t.stride(0) == inner) return 0;
  return t.stride(0) > inner ? t.stride(0) : -1;
}

bool cache(PyObject* k, PyObject* v, PyObject* ks, PyObject* vs, int dev, hypno_hip_kv_cache& c) {
  if (!THPVariable_Check(k)) return false;
  const auto type = THPVariable_Unpack(k).scalar_type();
  const bool fp4 = type == at::kByte;
  if (type != at::kHalf && type != at::kChar && !fp4) return false;
  const at::Tensor *kt = tensor(k, dev, type, 4), *vt = tensor(v, dev, type, 4);
  if (!kt || !vt || kt->sizes() != vt->sizes()) return false;
  const int64_t kp = page_stride(*kt), vp = page_stride(*vt);
  if (kp < 0 || vp < 0) return false;
  const auto s = kt->sizes();
  const int64_t dim = fp4 ? 2 * s[3] : s[3];
  c = hypno_hip_kv_cache{fp4                 ? HYPNO_HIP_KV_FP4
                         : type == at::kChar ? HYPNO_HIP_KV_INT8
                                             : HYPNO_HIP_KV_FP16,
                         kt->data_ptr(), vt->data_ptr(), nullptr, nullptr, (size_t)s[0],
                         (size_t)s[1], (size_t)s[2], (size_t)dim, (size_t)kp, (size_t)vp, 0, 0};
  if (type == at::kHalf) return ks == Py_None && vs == Py_None;
  const at::ScalarType scales = fp4 ? at::kHalf : at::kFloat;
  const at::Tensor *kst = tensor(ks, dev, scales, fp4 ? 4 : 3),
                   *vst = tensor(vs, dev, scales, fp4 ? 4 : 3);
  const int64_t groups[] = {s[0], s[1], dim / 32, s[2]};
  const at::IntArrayRef want = fp4 ? at::IntArrayRef(groups, 4) : s.slice(0, 3);
  if (!kst || !vst || kst->sizes() != want || vst->sizes() != want) return false;
  const int64_t ksp = page_stride(*kst), vsp = page_stride(*vst);
  if (ksp < 0 || vsp < 0) return false;
  c.k_scale = (float*)kst->data_ptr(), c.v_scale = (float*)vst->data_ptr();
  c.k_scale_page_stride = (size_t)ksp, c.v_scale_page_stride = (size_t)vsp;
  return true;
}

bool batch(PyObject* table, PyObject* lens, PyObject* cu, int64_t tokens, int dev,
           hypno_hip_kv_batch& b) {
  const at::Tensor *t = tensor(table, dev, at::kInt, 2), *l = tensor(lens, dev, at::kInt, 1),
                   *c = tensor(cu, dev, at::kInt, 1);
  if (!t || !l || !c || !t->is_contiguous() || !l->is_contiguous() || !c->is_contiguous())
    return false;
  const int64_t n = t->size(0);
  if (l->size(0) != n || c->size(0) != n + 1) return false;
  b = hypno_hip_kv_batch{(const int32_t*)c->data_ptr(), (const int32_t*)l->data_ptr(),
                         (const int32_t*)t->data_ptr(), (size_t)n, (size_t)t->size(1),
                         (size_t)tokens};
  return true;
}

// (page_size and the cache's other sizes: the bounds' own)
bool key_bounds_of(PyObject* codes, PyObject* scale, int64_t page_size, int dev,
                   hypno_hip_key_bounds& o) {
  const at::Tensor *c = tensor(codes, dev, at::kChar, 4), *s = tensor(scale, dev, at::kFloat, 2);
  if (!c || !s || c->size(2) != 2 || s->sizes() != c->sizes().slice(0, 2)) return false;
  const int64_t cp = page_stride(*c), sp = page_stride(*s);
  if (cp < 0 || sp < 0) return false;
  o = hypno_hip_key_bounds{(int8_t*)c->data_ptr(), (float*)s->data_ptr(), (size_t)c->size(0),
                           (size_t)c->size(1), (size_t)page_size, (size_t)c->size(3), (size_t)cp,
                           (size_t)sp};
  return true;
}

// A Python int (or `none` for None) of `least` or more.
bool whole(PyObject* x, long long least, long long& v, long long none = -1) {
  if (x == Py_None && none >= 0) {
    v = none;
    return true;
  }
  if (!PyLong_Check(x)) return false;
  v = PyLong_AsLongLong(x);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return v >= least;
}

// The stream that torch queues on, if `dev` is the current device.
bool stream_of(int dev, void** s) {
  PyObject* cur = PyObject_CallNoArgs(g_device);
  const bool here = cur && PyLong_AsLong(cur) == dev;
  Py_XDECREF(cur);
  PyObject* raw = nullptr;
  if (here) {
    PyObject* d = PyLong_FromLong(dev);
    raw = d ? PyObject_CallOneArg(g_stream, d) : nullptr;
    Py_XDECREF(d);
  }
  if (raw) *s = PyLong_AsVoidPtr(raw);
  Py_XDECREF(raw);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return raw != nullptr;
}

// `out` as it was given, or the new tensor; a status that is not 0 as a number.
PyObject* result(int status, PyObject* given, at::Tensor& made) {
  if (status) return PyLong_FromLong(status);
  if (made.defined()) return THPVariable_Wrap(std::move(made));
  Py_INCREF(given);
  return given;
}

// (q, k, v, k_cache, v_cache, page_table, kv_lens, cu_q, inv_freq, style, k_scale,
// v_scale, out); style: HYPNO_HIP_ROPE_*
PyObject* append_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 13 || !g_append) return other();
  try {
    Rows q = {}, k, v, o = {};
    if (!rows(a[1], -1, k)) return other();
    const int dev = (int)k.t->get_device();
    if (!rows(a[2], dev, v) || v.n != k.n || v.h != k.h || v.d != k.d) return other();
    const long style = PyLong_Check(a[9]) ? PyLong_AsLong(a[9]) : -1;
    hypno_hip_kv_cache c;
    hypno_hip_kv_batch b;
    if (style < 0 || !cache(a[3], a[4], a[10], a[11], dev, c) ||
        !batch(a[5], a[6], a[7], k.n, dev, b) || (int64_t)c.kv_heads != k.h ||
        (int64_t)c.head_dim != k.d)
      return other();
    const float* freq = nullptr;
    size_t rot = 0;
    if (a[8] != Py_None) {
      const at::Tensor* f = tensor(a[8], dev, at::kFloat, 1);
      if (!f || !f->is_contiguous() || 2 * f->size(0) > k.d) return other();
      freq = (const float*)f->data_ptr(), rot = 2 * (size_t)f->size(0);
    }
    at::Tensor made;
    const float* qp = nullptr;
    float* op = nullptr;
    if (a[0] != Py_None) {
      if (!rows(a[0], dev, q) || q.n != k.n || q.d != k.d) return other();
      qp = (const float*)q.t->data_ptr();
      if (a[12] == Py_None) {
        made = at::empty(q.t->sizes(), q.t->options());
        o.stride = q.h * q.d, op = (float*)made.data_ptr();
      } else {
        if (!rows(a[12], dev, o) || o.n != q.n || o.h != q.h || o.d != q.d) return other();
        op = (float*)o.t->data_ptr();
      }
    } else if (a[12] != Py_None) {
      return other();
    }
    void* s = nullptr;
    if (!stream_of(dev, &s)) return other();
    const float *kp = (const float*)k.t->data_ptr(), *vp = (const float*)v.t->data_ptr();
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = g_append(&c, &b, op, (size_t)o.stride, qp, (size_t)q.stride, (size_t)q.h, kp,
                      (size_t)k.stride, vp, (size_t)v.stride, freq, rot, (uint32_t)style, s);
    Py_END_ALLOW_THREADS
    return result(status, a[12], made);
  } catch (...) {
    return other();
  }
}

// (q, k_cache, v_cache, page_table, kv_lens, cu_q, scale, window, k_scale, v_scale,
// max_kv_len, out)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 12 || !g_attend) return other();
  try {
    Rows q;
    if (!rows(a[0], -1, q)) return other();
    const int dev = (int)q.t->get_device();
    hypno_hip_kv_cache c;
    hypno_hip_kv_batch b;
    if (!cache(a[1], a[2], a[8], a[9], dev, c) || !batch(a[3], a[4], a[5], q.n, dev, b) ||
        (int64_t)c.head_dim != q.d || c.kv_heads == 0 || q.h % (int64_t)c.kv_heads)
      return other();
    if ((a[6] != Py_None && !PyFloat_Check(a[6])) || !PyLong_Check(a[7]) ||
        (a[10] != Py_None && !PyLong_Check(a[10])))
      return other();
    const double scale = a[6] == Py_None ? 1.0 / std::sqrt((double)q.d) : PyFloat_AsDouble(a[6]);
    const long long window = PyLong_AsLongLong(a[7]);
    const long long most = a[10] == Py_None ? 0 : PyLong_AsLongLong(a[10]);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      return other();
    }
    if (window < 0 || most < 0) return other();
    at::Tensor made;
    float* op = nullptr;
    if (a[11] == Py_None) {
      made = at::empty(q.t->sizes(), q.t->options());
      op = (float*)made.data_ptr();
    } else {
      const at::Tensor* o = tensor(a[11], dev, at::kFloat, 3);
      if (!o || o->sizes() != q.t->sizes() || !o->is_contiguous()) return other();
      op = (float*)o->data_ptr();
    }
    void* s = nullptr;
    if (!stream_of(dev, &s)) return other();
    const float* qp = (const float*)q.t->data_ptr();
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = g_attend(op, qp, (size_t)q.stride, (size_t)q.h, &c, &b, (float)scale,
                      (size_t)window, (size_t)most, s);
    Py_END_ALLOW_THREADS
    return result(status, a[11], made);
  } catch (...) {
    return other();
  }
}

// (k_cache, bounds, bounds_scale, page_table, kv_lens, cu_q, k_scale)
PyObject* key_bounds(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7 || !g_bounds) return other();
  try {
    if (!THPVariable_Check(a[0]) || !THPVariable_Unpack(a[0]).is_cuda()) return other();
    const int dev = (int)THPVariable_Unpack(a[0]).get_device();
    hypno_hip_kv_cache c;
    hypno_hip_kv_batch b;
    hypno_hip_key_bounds o;
    if (!cache(a[0], a[0], a[6], a[6], dev, c) ||
        !key_bounds_of(a[1], a[2], (int64_t)c.page_size, dev, o) || o.pages != c.pages ||
        o.kv_heads != c.kv_heads || o.head_dim != c.head_dim ||
        !batch(a[3], a[4], a[5], 0x7FFFFFFF, dev, b))
      return other();
    void* s = nullptr;
    if (!stream_of(dev, &s)) return other();
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = g_bounds(&o, &c, &b, s);
    Py_END_ALLOW_THREADS
    if (status) return PyLong_FromLong(status);
    Py_RETURN_NONE;
  } catch (...) {
    return other();
  }
}

// (q, bounds, bounds_scale, page_size, page_table, kv_lens, cu_q, count, first, last,
// max_kv_len, out)
PyObject* select_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 12 || !g_select) return other();
  try {
    Rows q;
    if (!rows(a[0], -1, q)) return other();
    const int dev = (int)q.t->get_device();
    long long size, count, first, last, most;
    hypno_hip_kv_batch b;
    hypno_hip_key_bounds o;
    if (!whole(a[3], 1, size) || !whole(a[7], 1, count) || !whole(a[8], 0, first) ||
        !whole(a[9], 1, last) || !whole(a[10], 0, most, 0) || count > 1024 || first > count ||
        last > count - first || !key_bounds_of(a[1], a[2], size, dev, o) ||
        !batch(a[4], a[5], a[6], q.n, dev, b) || (int64_t)o.head_dim != q.d || o.kv_heads == 0 ||
        q.h % (int64_t)o.kv_heads)
      return other();
    const int64_t shape[] = {q.n, (int64_t)o.kv_heads, count};
    at::Tensor made;
    int32_t* op = nullptr;
    if (a[11] == Py_None) {
      made = at::empty(shape, q.t->options().dtype(at::kInt));
      op = (int32_t*)made.data_ptr();
    } else {
      const at::Tensor* t = tensor(a[11], dev, at::kInt, 3);
      if (!t || t->sizes() != at::IntArrayRef(shape, 3) || !t->is_contiguous()) return other();
      op = (int32_t*)t->data_ptr();
    }
    void* s = nullptr;
    if (!stream_of(dev, &s)) return other();
    const float* qp = (const float*)q.t->data_ptr();
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = g_select(op, (size_t)count, (size_t)first, (size_t)last, qp, (size_t)q.stride,
                      (size_t)q.h, &o, &b, (size_t)most, s);
    Py_END_ALLOW_THREADS
    return result(status, a[11], made);
  } catch (...) {
    return other();
  }
}

// (q, k_cache, v_cache, selected, page_table, kv_lens, cu_q, scale, k_scale, v_scale, out)
PyObject* selected_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11 || !g_selected) return other();
  try {
    Rows q;
    if (!rows(a[0], -1, q)) return other();
    const int dev = (int)q.t->get_device();
    hypno_hip_kv_cache c;
    hypno_hip_kv_batch b;
    if (!cache(a[1], a[2], a[8], a[9], dev, c) || !batch(a[4], a[5], a[6], q.n, dev, b) ||
        (int64_t)c.head_dim != q.d || c.kv_heads == 0 || q.h % (int64_t)c.kv_heads)
      return other();
    const at::Tensor* sel = tensor(a[3], dev, at::kInt, 3);
    if (!sel || !sel->is_contiguous() || sel->size(0) != q.n ||
        sel->size(1) != (int64_t)c.kv_heads || sel->size(2) < 1 || sel->size(2) > 1024)
      return other();
    if (a[7] != Py_None && !PyFloat_Check(a[7])) return other();
    const double scale = a[7] == Py_None ? 1.0 / std::sqrt((double)q.d) : PyFloat_AsDouble(a[7]);
    at::Tensor made;
    float* op = nullptr;
    if (a[10] == Py_None) {
      made = at::empty(q.t->sizes(), q.t->options());
      op = (float*)made.data_ptr();
    } else {
      const at::Tensor* o = tensor(a[10], dev, at::kFloat, 3);
      if (!o || o->sizes() != q.t->sizes() || !o->is_contiguous()) return other();
      op = (float*)o->data_ptr();
    }
    void* s = nullptr;
    if (!stream_of(dev, &s)) return other();
    const float* qp = (const float*)q.t->data_ptr();
    const int32_t* sp = (const int32_t*)sel->data_ptr();
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = g_selected(op, qp, (size_t)q.stride, (size_t)q.h, &c, &b, (float)scale, sp,
                        (size_t)sel->size(2), s);
    Py_END_ALLOW_THREADS
    return result(status, a[10], made);
  } catch (...) {
    return other();
  }
}

// bind(addresses of hypno_hip_append_kv_dev, _paged_attention_dev, _key_bounds_dev,
// _select_pages_dev and _selected_attention_dev, function of the current device, function
// of a device's stream)
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long append = 0, attend = 0, bounds = 0, select = 0, selected = 0;
  PyObject *device = nullptr, *stream = nullptr;
  if (!PyArg_ParseTuple(args, "KKKKKOO", &append, &attend, &bounds, &select, &selected, &device,
                        &stream))
    return nullptr;
  Py_INCREF(device);
  Py_INCREF(stream);
  Py_XSETREF(g_device, device);
  Py_XSETREF(g_stream, stream);
  g_append = reinterpret_cast<decltype(g_append)>((uintptr_t)append);
  g_attend = reinterpret_cast<decltype(g_attend)>((uintptr_t)attend);
  g_bounds = reinterpret_cast<decltype(g_bounds)>((uintptr_t)bounds);
  g_select = reinterpret_cast<decltype(g_select)>((uintptr_t)select);
  g_selected = reinterpret_cast<decltype(g_selected)>((uintptr_t)selected);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"append_kv", (PyCFunction)(void (*)(void))append_kv, METH_FASTCALL, nullptr},
    {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
    {"key_bounds", (PyCFunction)(void (*)(void))key_bounds, METH_FASTCALL, nullptr},
    {"select_pages", (PyCFunction)(void (*)(void))select_pages, METH_FASTCALL, nullptr},
    {"selected_attention", (PyCFunction)(void (*)(void))selected_attention, METH_FASTCALL,
     nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attention_args", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__attention_args() { return PyModule_Create(&module); }
