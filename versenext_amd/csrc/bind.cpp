// Python binding of the 8-bit KV cache's entries: _vnx_bind.kv_write, kv_read
// and tree_attn_q8 take tensors, check them, allocate the results and call the
// C entries of vnx.h, in 1-2 us of host time a call beside the launch's
// 3.5, where the same checks in Python take 7-13 (a decode step's kernels take 3-9 us).
//
// Each function serves the call whose arguments the kernels read as they are.
// It returns None for every other one (a tensor elsewhere, another type, strides
// that need a copy, a bad shape): HipBackend then goes through its general
// checks, which convert, copy or raise.  A status of the C entry other than
// VNX_OK is returned as an int.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>

#include "../../include/vnx.h"

namespace {

decltype(&vnx_kv_write) g_write;
decltype(&vnx_kv_read) g_read;
decltype(&vnx_tree_attn_q8_workspace) g_attn_ws;
decltype(&vnx_tree_attn_q8) g_attn;

inline bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A tensor on GPU `dev` (nullptr else).
const at::Tensor* tensor(PyObject* o, int dev) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == dev && t.layout() == at::kStrided && !t.is_neg() ? &t : nullptr;
}

bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  return a.scalar_type() == b.scalar_type() && a.sizes() == b.sizes() && a.strides() == b.strides();
}

// Strides of the dims before the last are multiples of `bytes`, the last is 1,
// the data starts on 16 bytes.
bool rows_on(const at::Tensor& t, int64_t bytes) {
  const int n = (int)t.dim(), e = (int)t.element_size();
  if (t.stride(n - 1) != 1 || !aligned(t.data_ptr(), 16)) return false;
  for (int i = 0; i + 1 < n; ++i)
    if (t.stride(i) < 0 || t.stride(i) * e % bytes) return false;
  return true;
}

struct Cache {
  const at::Tensor *k, *v, *ks = nullptr, *vs = nullptr;
  int64_t B, Hkv, cap, d, s[2] = {0, 0};
  int code;
  bool get(PyObject* const* a, int dev) {
    k = tensor(a[0], dev);
    v = tensor(a[1], dev);
    if (!k || !v || k->dim() != 4 || !same_layout(*k, *v)) return false;
    B = k->size(0), Hkv = k->size(1), cap = k->size(2), d = k->size(3);
    if (B < 1 || Hkv < 1 || cap < 1 || d < 16 || Hkv > INT_MAX || d > INT_MAX || !rows_on(*k, 16) ||
        !aligned(v->data_ptr(), 16))
      return false;
    const auto t = k->scalar_type();
    if (t == at::kBFloat16) {
      code = VNX_BF16;
      return a[2] == Py_None && a[3] == Py_None;
    }
    if (t == at::kChar) code = VNX_I8;
    else if (t == at::kFloat8_e4m3fn) code = VNX_E4M3;
    else return false;
    ks = tensor(a[2], dev);
    vs = tensor(a[3], dev);
    if (!ks || !vs || ks->scalar_type() != at::kFloat || ks->dim() != 3 || !same_layout(*ks, *vs) ||
        ks->size(0) != B || ks->size(1) != Hkv || ks->size(2) != cap || ks->stride(2) != 1)
      return false;
    s[0] = ks->stride(0), s[1] = ks->stride(1);
    return true;
  }
  float* kscale() const { return ks ? static_cast<float*>(ks->data_ptr()) : nullptr; }
  float* vscale() const { return vs ? static_cast<float*>(vs->data_ptr()) : nullptr; }
};

// (B,) int32 contiguous; nullptr where it is not.
const int32_t* lens_of(PyObject* o, int64_t B, int dev) {
  const at::Tensor* t = tensor(o, dev);
  if (!t || t->scalar_type() != at::kInt || t->dim() != 1 || t->size(0) != B || (B > 1 && t->stride(0) != 1))
    return nullptr;
  return static_cast<const int32_t*>(t->data_ptr());
}

// A contiguous fp32 tensor on 16 bytes: (d,) or (rows, d).  None: *out = nullptr.
bool vec_of(PyObject* o, int dims, int64_t d, int dev, const float** out, int64_t* rows) {
  *out = nullptr;
  if (o == Py_None) return true;
  const at::Tensor* t = tensor(o, dev);
  if (!t || t->scalar_type() != at::kFloat || t->dim() != dims || t->size(dims - 1) != d || !t->is_contiguous() ||
      !aligned(t->data_ptr(), 16))
    return false;
  *out = static_cast<const float*>(t->data_ptr());
  if (rows) *rows = t->size(0);
  return true;
}

int code_of(at::ScalarType t) {
  return t == at::kFloat ? VNX_F32 : t == at::kBFloat16 ? VNX_BF16 : t == at::kHalf ? VNX_F16 : -1;
}

// An int argument in [lo, hi]; false for anything else.
bool int_of(PyObject* o, int64_t lo, int64_t hi, int64_t* out) {
  if (!PyLong_Check(o)) return false;
  int over = 0;
  *out = PyLong_AsLongLongAndOverflow(o, &over);
  return !over && *out >= lo && *out <= hi;
}

bool float_of(PyObject* o, double* out) {
  if (!PyFloat_Check(o)) return false;
  *out = PyFloat_AS_DOUBLE(o);
  return true;
}

bool stream_of(PyObject* dev_o, PyObject* st_o, int64_t* dev, void** st) {
  int64_t s;
  if (!int_of(dev_o, 0, INT_MAX, dev) || !PyLong_Check(st_o)) return false;
  s = (int64_t)PyLong_AsUnsignedLongLongMask(st_o);
  *st = reinterpret_cast<void*>(s);
  return true;
}

PyObject* status(int rc) { return PyLong_FromLong(rc); }

// kv_write(device, stream, k_cache, v_cache, k_scale, v_scale, qkv, lens, cos, sin, q_norm, k_norm, eps)
PyObject* kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t dev;
  void* st;
  Cache c;
  vnx_kv_write_args p{};
  double eps;
  if (n != 13 || !stream_of(a[0], a[1], &dev, &st) || !c.get(a + 2, (int)dev)) Py_RETURN_NONE;
  const at::Tensor* x = tensor(a[6], (int)dev);
  if (!x || x->dim() != 3 || x->size(0) != c.B || x->size(2) % c.d || !float_of(a[12], &eps)) Py_RETURN_NONE;
  const int64_t rows = x->size(1), H = x->size(2) / c.d - 2 * c.Hkv, ld = x->stride(1);
  p.dtype = code_of(x->scalar_type());
  if (rows < 1 || rows > INT_MAX || H < 1 || H > INT_MAX || p.dtype < 0 || ld < x->size(2) || !rows_on(*x, 16) ||
      (c.B > 1 && x->stride(0) != rows * ld))
    Py_RETURN_NONE;
  p.lens = lens_of(a[7], c.B, (int)dev);
  int64_t srows = 0;
  if (!p.lens || !vec_of(a[8], 2, c.d, (int)dev, &p.cos_table, &p.table_rows) ||
      !vec_of(a[9], 2, c.d, (int)dev, &p.sin_table, &srows) || p.table_rows != srows ||
      !p.cos_table != !p.sin_table || !vec_of(a[10], 1, c.d, (int)dev, &p.q_norm, nullptr) ||
      !vec_of(a[11], 1, c.d, (int)dev, &p.k_norm, nullptr))
    Py_RETURN_NONE;
  const c10::DeviceGuard guard(x->device());  // (the null stream is the current device's)
  at::Tensor q = at::empty({c.B, H, rows, c.d}, x->options().dtype(at::kBFloat16));
  p.qkv = x->data_ptr(), p.ldq = ld, p.q_out = q.data_ptr();
  p.k_cache = c.k->data_ptr(), p.v_cache = c.v->data_ptr();
  p.k_scale = c.kscale(), p.v_scale = c.vscale();
  for (int i = 0; i < 3; ++i) p.cache_strides[i] = c.k->stride(i);
  p.scale_strides[0] = c.s[0], p.scale_strides[1] = c.s[1];
  p.B = c.B, p.cap = c.cap, p.n = (int)rows, p.H = (int)H, p.Hkv = (int)c.Hkv, p.d = (int)c.d;
  p.cache_dtype = c.code, p.eps = (float)eps;
  const int rc = g_write(&p, st);
  return rc == VNX_OK ? THPVariable_Wrap(std::move(q)) : status(rc);
  END_HANDLE_TH_ERRORS
}

// kv_read(device, stream, k_cache, v_cache, k_scale, v_scale, start, rows, out_dtype)
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t dev, rows;
  void* st;
  Cache c;
  vnx_kv_read_args p{};
  if (n != 9 || !stream_of(a[0], a[1], &dev, &st) || !c.get(a + 2, (int)dev) || !THPDtype_Check(a[8])) Py_RETURN_NONE;
  if (a[6] != Py_None && !(p.start = lens_of(a[6], c.B, (int)dev))) Py_RETURN_NONE;
  if (a[7] == Py_None) rows = c.cap;
  else if (!int_of(a[7], 0, INT_MAX, &rows)) Py_RETURN_NONE;
  const auto t = reinterpret_cast<THPDtype*>(a[8])->scalar_type;
  p.out_dtype = code_of(t);
  if (rows > INT_MAX || p.out_dtype < 0) Py_RETURN_NONE;
  const c10::DeviceGuard guard(c.k->device());
  at::Tensor k = at::empty({c.B, c.Hkv, rows, c.d}, c.k->options().dtype(t)), v = at::empty_like(k);
  p.k_cache = c.k->data_ptr(), p.v_cache = c.v->data_ptr(), p.k_scale = c.kscale(), p.v_scale = c.vscale();
  p.k_out = k.data_ptr(), p.v_out = v.data_ptr();
  for (int i = 0; i < 3; ++i) p.cache_strides[i] = c.k->stride(i);
  p.scale_strides[0] = c.s[0], p.scale_strides[1] = c.s[1];
  p.out_strides[0] = c.Hkv * rows * c.d, p.out_strides[1] = rows * c.d, p.out_strides[2] = c.d;
  p.B = c.B, p.cap = c.cap, p.rows = (int)rows, p.Hkv = (int)c.Hkv, p.d = (int)c.d, p.cache_dtype = c.code;
  const int rc = g_read(&p, st);
  if (rc != VNX_OK) return status(rc);
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(v)));
  return r;
  END_HANDLE_TH_ERRORS
}

// Rows (B or `other`, heads, rows, d) of bf16 as the kernels read them.
const at::Tensor* heads(PyObject* o, int dev, int64_t d) {
  const at::Tensor* t = tensor(o, dev);
  return t && t->scalar_type() == at::kBFloat16 && t->dim() == 4 && t->size(3) == d && rows_on(*t, 16) ? t : nullptr;
}

struct Words {  // N ancestor words in host memory (a contiguous uint64 buffer)
  Py_buffer b{};
  bool held = false;
  ~Words() {
    if (held) PyBuffer_Release(&b);
  }
  bool get(PyObject* o, int64_t N) {
    if (PyObject_GetBuffer(o, &b, PyBUF_C_CONTIGUOUS | PyBUF_FORMAT)) {
      PyErr_Clear();
      return false;
    }
    held = true;
    return b.ndim == 1 && b.itemsize == 8 && b.len == 8 * N && b.format && (b.format[0] == 'L' || b.format[0] == 'Q') &&
           !b.format[1];
  }
};

// tree_attn_q8(device, stream, k_cache, v_cache, k_scale, v_scale, q, lens, anc, scale, seg2, gates, window, max_len,
//              out_dtype, out)
PyObject* tree_attn_q8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t dev, max_len, window;
  void* st;
  Cache c;
  vnx_attn_q8_args p{};
  Words words;
  if (n != 16 || !stream_of(a[0], a[1], &dev, &st) || !c.get(a + 2, (int)dev) || c.code == VNX_BF16) Py_RETURN_NONE;
  const at::Tensor* q = heads(a[6], (int)dev, c.d);
  if (!q || q->size(0) != c.B || q->size(1) < 1 || q->size(1) % c.Hkv || q->size(1) > INT_MAX || c.B > INT_MAX)
    Py_RETURN_NONE;
  const int64_t H = q->size(1), N = q->size(2);
  p.lens = lens_of(a[7], c.B, (int)dev);
  if (!p.lens || N < 1 || N > c.cap || c.cap > INT_MAX) Py_RETURN_NONE;
  if (a[13] == Py_None) max_len = c.cap - N;
  else if (!int_of(a[13], 0, c.cap - N, &max_len)) Py_RETURN_NONE;
  if (a[8] != Py_None) {
    if (!words.get(a[8], N)) Py_RETURN_NONE;
    p.anc_host = static_cast<const uint64_t*>(words.b.buf);
  }
  double scale = 1.0 / std::sqrt((double)c.d);
  if (a[9] != Py_None && !float_of(a[9], &scale)) Py_RETURN_NONE;
  if (!int_of(a[12], 0, INT_MAX, &window)) Py_RETURN_NONE;
  const int64_t ngates = a[10] != Py_None ? 2 : 1;
  if (a[11] != Py_None) {
    const at::Tensor* g = tensor(a[11], (int)dev);
    if (!g || g->scalar_type() != at::kFloat || g->dim() != 1 || g->size(0) < ngates || g->stride(0) != 1)
      Py_RETURN_NONE;
    p.gates = static_cast<const float*>(g->data_ptr());
  }
  if (a[10] != Py_None) {
    if (!PyTuple_Check(a[10]) || PyTuple_GET_SIZE(a[10]) != 2) Py_RETURN_NONE;
    const at::Tensor *k2 = heads(PyTuple_GET_ITEM(a[10], 0), (int)dev, c.d),
                     *v2 = heads(PyTuple_GET_ITEM(a[10], 1), (int)dev, c.d);
    if (!k2 || !v2 || !same_layout(*k2, *v2) || (k2->size(0) != 1 && k2->size(0) != c.B) || k2->size(1) != c.Hkv ||
        k2->size(2) < 1 || k2->size(2) > INT_MAX || !p.gates)
      Py_RETURN_NONE;
    p.k_seg2 = k2->data_ptr(), p.v_seg2 = v2->data_ptr();
    p.seg2_strides[0] = k2->size(0) == 1 ? 0 : k2->stride(0);
    p.seg2_strides[1] = k2->stride(1), p.seg2_strides[2] = k2->stride(2);
    p.T2 = (int)k2->size(2);
  }
  const c10::DeviceGuard guard(q->device());
  at::Tensor fresh;
  const at::Tensor* out;
  if (a[15] == Py_None) {
    if (!THPDtype_Check(a[14])) Py_RETURN_NONE;
    const auto t = reinterpret_cast<THPDtype*>(a[14])->scalar_type;
    if (t != at::kBFloat16 && t != at::kHalf) Py_RETURN_NONE;
    fresh = at::empty({c.B, H, N, c.d}, q->options().dtype(t));
    out = &fresh;
  } else {
    out = tensor(a[15], (int)dev);
    if (!out || (out->scalar_type() != at::kBFloat16 && out->scalar_type() != at::kHalf) || out->dim() != 4 ||
        out->size(0) != c.B || out->size(1) != H || out->size(2) != N || out->size(3) != c.d || !rows_on(*out, 16))
      Py_RETURN_NONE;
  }
  p.q = q->data_ptr(), p.out = out->data_ptr(), p.out_dtype = code_of(out->scalar_type());
  p.k_cache = c.k->data_ptr(), p.v_cache = c.v->data_ptr(), p.k_scale = c.kscale(), p.v_scale = c.vscale();
  for (int i = 0; i < 3; ++i) {
    p.q_strides[i] = q->stride(i);
    p.cache_strides[i] = c.k->stride(i);
    p.out_strides[i] = out->stride(i);
  }
  p.scale_strides[0] = c.s[0], p.scale_strides[1] = c.s[1];
  p.cap = c.cap, p.B = (int)c.B, p.H = (int)H, p.Hkv = (int)c.Hkv, p.Tp = (int)max_len, p.N = (int)N, p.d = (int)c.d;
  p.window = (int)window, p.kv_dtype = c.code, p.scale = (float)scale;
  // a workspace of this call's own: a captured graph keeps it in its pool
  const size_t need = g_attn_ws(&p);
  at::Tensor ws;
  if (need > 256) ws = at::empty({(int64_t)need}, q->options().dtype(at::kByte));
  const int rc = g_attn(&p, need > 256 ? ws.data_ptr() : nullptr, need > 256 ? need : 0, st);
  if (rc != VNX_OK) return status(rc);
  if (a[15] != Py_None) {
    Py_INCREF(a[15]);
    return a[15];
  }
  return THPVariable_Wrap(std::move(fresh));
  END_HANDLE_TH_ERRORS
}

// init(address of vnx_kv_write, vnx_kv_read, vnx_tree_attn_q8_workspace, vnx_tree_attn_q8)
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* f[4];
  if (n != 4) return PyErr_Format(PyExc_TypeError, "init takes four addresses");
  for (int i = 0; i < 4; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (!f[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "a null address");
  }
  g_write = reinterpret_cast<decltype(g_write)>(f[0]);
  g_read = reinterpret_cast<decltype(g_read)>(f[1]);
  g_attn_ws = reinterpret_cast<decltype(g_attn_ws)>(f[2]);
  g_attn = reinterpret_cast<decltype(g_attn)>(f[3]);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F));
}

PyMethodDef kMethods[] = {{"init", fast<init>(), METH_FASTCALL, nullptr},
                          {"kv_write", fast<kv_write>(), METH_FASTCALL, nullptr},
                          {"kv_read", fast<kv_read>(), METH_FASTCALL, nullptr},
                          {"tree_attn_q8", fast<tree_attn_q8>(), METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_vnx_bind", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// .torch: the PyTorch it was compiled against; .sizes: of the argument blocks
// that it fills.  Another PyTorch, or another library, must not get them.
PyMODINIT_FUNC PyInit__vnx_bind() {
  PyObject* m = PyModule_Create(&kModule);
  if (!m) return nullptr;
  PyObject* sizes =
      Py_BuildValue("(nnn)", (Py_ssize_t)sizeof(vnx_kv_write_args), (Py_ssize_t)sizeof(vnx_kv_read_args),
                    (Py_ssize_t)sizeof(vnx_attn_q8_args));
  if (!sizes || PyModule_AddObject(m, "sizes", sizes) < 0) {  // (takes sizes when it succeeds)
    Py_XDECREF(sizes);
    Py_DECREF(m);
    return nullptr;
  }
  if (PyModule_AddStringConstant(m, "torch", VNX_BIND_TORCH) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
