// The short way from torch tensors into libmpsa.so: checks, output allocation and the C call of the entry points that programs
// call most, in one step.  Up to the C call that took 8 - 11 us of the host's time through ctypes and struct, here 3: back to back, a pair
// of quantizers over 4500 tokens 16.5 -> 11.0 us, causal attention over 128 tokens 17.0 -> 11.0.  Outputs and workspaces come from torch's allocator through its dispatcher, as
// torch.empty does, and like there the interpreter's lock is released from the first of them to the end of the C call: an allocation may
// wait for the device, and a launch for room in its queue.  Operands that the one-launch paths do not take make a function return
// None, and the caller goes the long way; an error code of the C entry is returned as an int.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <exception>
#include <optional>

#include "../../include/mpsa.h"

namespace {

decltype(&mpsa_attention_workspace) workspace_fn;
decltype(&mpsa_attention) attention_fn;
decltype(&mpsa_quant_pair) quant_pair_fn;
decltype(&mpsa_gemm_block_scaled) gemm_fn;
decltype(&mpsa_norm_rope) norm_rope_fn;
decltype(&mpsa_kv_append) kv_append_fn;
decltype(&mpsa_kv_read) kv_read_fn;
decltype(&mpsa_kv_attention_workspace) kv_workspace_fn;
decltype(&mpsa_kv_attention) kv_attention_fn;
PyObject* out_of_memory = PyExc_MemoryError;              // torch.OutOfMemoryError

const at::ScalarType kOut[] = {at::kFloat, at::kHalf, at::kBFloat16, at::kFloat8_e5m2};

// Plain tensors only: a subclass may stand for something without memory of its own.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.has_storage() && t.layout() == at::kStrided ? &t : nullptr;
}

// 4-D, 16 bits, rows of the last dimension dense, everything 16-byte aligned
bool aligned16(const at::Tensor& t) {
  if (t.dim() != 4) return false;
  const auto s = t.strides();
  return s[3] == 1 && !((s[0] | s[1] | s[2]) & 7) && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15);
}

int in_dtype(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 0 : t.scalar_type() == at::kHalf ? 1 : -1; }

at::Tensor dense(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) { return at::empty(sizes, like.options().dtype(type).requires_grad(false)); }

// Other Python threads run while this lives.  (The caller's argument array keeps the tensors.)
struct Unlocked {
  PyThreadState* const state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// The operands' device for the time of a call: the usual case costs one look.
struct OnDevice {
  std::optional<c10::cuda::CUDAGuard> guard;
  explicit OnDevice(c10::DeviceIndex i) { if (c10::cuda::current_device() != i) guard.emplace(i); }
};

long long as_ll(PyObject* o) { return PyLong_AsLongLong(o); }

template <typename F>
PyObject* guarded(F f) {
  try {
    PyObject* r = f();
    if (r && PyErr_Occurred()) { Py_DECREF(r); return nullptr; }
    return r;
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(out_of_memory, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "mpsa: unknown error");
  }
  return nullptr;
}

bool counted(Py_ssize_t n, Py_ssize_t want, const char* name) {
  if (n != want) PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, want);
  return n == want;
}

PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 5, "init")) return nullptr;
  workspace_fn = reinterpret_cast<decltype(workspace_fn)>(PyLong_AsVoidPtr(a[0]));
  attention_fn = reinterpret_cast<decltype(attention_fn)>(PyLong_AsVoidPtr(a[1]));
  quant_pair_fn = reinterpret_cast<decltype(quant_pair_fn)>(PyLong_AsVoidPtr(a[2]));
  gemm_fn = reinterpret_cast<decltype(gemm_fn)>(PyLong_AsVoidPtr(a[3]));
  if (PyErr_Occurred()) return nullptr;
  Py_INCREF(a[4]);
  out_of_memory = a[4];
  Py_RETURN_NONE;
}

// attention(q, k, v, prepared, range_flag, status, out_dtype, causal, band, uniform, route, pv_mode, fp8_fmt, smooth_k, fp4_kind, q_scale, tau)
// k and v may be None: then prepared = (Hkv, Skv, Skv_pad, k8, k8_sf, k4, k4_sf, vt, vt8, v8_sf, vt4, v4_sf).
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 17, "attention")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* q = plain(a[0]);
    if (!q || !aligned16(*q)) Py_RETURN_NONE;
    mpsa_attention_args c = {};
    c.in_dtype = in_dtype(*q);
    if (c.in_dtype < 0) Py_RETURN_NONE;
    const auto size = q->sizes(), qs = q->strides();
    c.q = q->data_ptr();
    c.q_sb = qs[0]; c.q_sh = qs[1]; c.q_sl = qs[2];
    long long hkv, skv;
    if (a[1] == Py_None) {
      if (!PyTuple_CheckExact(a[3]) || PyTuple_GET_SIZE(a[3]) != 12) { PyErr_SetString(PyExc_TypeError, "attention: prepared operands missing"); return nullptr; }
      long long w[12];
      for (int i = 0; i < 12; ++i) w[i] = as_ll(PyTuple_GET_ITEM(a[3], i));
      hkv = w[0]; skv = w[1]; c.Skv_pad = (int)w[2];
      const void** p[] = {&c.k8, &c.k8_sf, &c.k4, &c.k4_sf, &c.vt, &c.vt8, &c.v8_sf, &c.vt4, &c.v4_sf};
      for (int i = 0; i < 9; ++i) *p[i] = reinterpret_cast<const void*>(w[3 + i]);
    } else {
      const at::Tensor *k = plain(a[1]), *v = plain(a[2]);
      if (!k || !v || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || !aligned16(*k) || !aligned16(*v) ||
          k->sizes() != v->sizes() || k->size(0) != size[0] || k->size(3) != size[3] || k->get_device() != q->get_device() ||
          v->get_device() != q->get_device())
        Py_RETURN_NONE;
      const auto ks = k->strides(), vs = v->strides();
      c.k = k->data_ptr(); c.v = v->data_ptr();
      c.k_sb = ks[0]; c.k_sh = ks[1]; c.k_sl = ks[2];
      c.v_sb = vs[0]; c.v_sh = vs[1]; c.v_sl = vs[2];
      hkv = k->size(1); skv = k->size(2);
    }
    if (PyErr_Occurred()) return nullptr;
    const long long most = 0x7fffffff;
    for (const long long x : {(long long)size[0], (long long)size[1], (long long)size[2], (long long)size[3], hkv, skv})
      if (x > most) Py_RETURN_NONE;
    c.B = (int)size[0]; c.Hq = (int)size[1]; c.S = (int)size[2]; c.D = (int)size[3]; c.Hkv = (int)hkv; c.Skv = (int)skv;
    c.causal = (int)as_ll(a[7]);
    if ((c.Hkv > 0 && c.Hq % c.Hkv) || (c.causal && c.Skv < c.S)) Py_RETURN_NONE;
    c.status = static_cast<int*>(PyLong_AsVoidPtr(a[5]));
    c.out_dtype = (int)as_ll(a[6]);
    c.band = (int)as_ll(a[8]); c.uniform = (int)as_ll(a[9]); c.route = (int)as_ll(a[10]); c.pv_mode = (int)as_ll(a[11]);
    c.fp8_fmt = (int)as_ll(a[12]); c.smooth_k = (int)as_ll(a[13]); c.fp4_kind = (int)as_ll(a[14]);
    c.q_scale = (float)PyFloat_AsDouble(a[15]); c.tau = (float)PyFloat_AsDouble(a[16]);
    if (PyErr_Occurred()) return nullptr;
    if (c.out_dtype < 0 || c.out_dtype > 2) Py_RETURN_NONE;
    if (a[4] != Py_None) {
      if (!THPVariable_Check(a[4])) { PyErr_SetString(PyExc_TypeError, "attention: range_flag must be a tensor"); return nullptr; }
      c.range_flag = static_cast<int*>(THPVariable_Unpack(a[4]).data_ptr());
    }
    at::Tensor out;
    long long rc;
    {
      const Unlocked unlocked;
      const OnDevice device(q->device().index());
      rc = workspace_fn(&c);                            // (refuses empty operands)
      if (rc >= 0) {
        const at::Tensor ws = dense({(int64_t)rc}, at::kByte, *q);
        out = dense(size, kOut[c.out_dtype], *q);
        c.out = out.data_ptr(); c.workspace = ws.data_ptr(); c.workspace_bytes = rc;
        rc = attention_fn(&c, c10::cuda::getCurrentCUDAStream(q->device().index()).stream());
      }
    }
    return rc ? PyLong_FromLongLong(rc) : THPVariable_Wrap(std::move(out));
  });
}

// quant_pair(q, k, q_scale, k_scale, fmt, hnd) -> (q codes, q scales, k codes, k scales)
PyObject* quant_pair(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 6, "quant_pair")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* x[2] = {plain(a[0]), plain(a[1])};
    if (!x[0] || !x[1] || !aligned16(*x[0]) || !aligned16(*x[1]) || x[0]->scalar_type() != x[1]->scalar_type() || x[0]->size(0) != x[1]->size(0) ||
        x[0]->size(3) != x[1]->size(3) || x[0]->get_device() != x[1]->get_device())
      Py_RETURN_NONE;
    mpsa_quant_pair_args c = {};
    c.in_dtype = in_dtype(*x[0]);
    const int64_t B = x[0]->size(0), D = x[0]->size(3);
    c.s[0] = (float)PyFloat_AsDouble(a[2]); c.s[1] = (float)PyFloat_AsDouble(a[3]);
    c.fp8_fmt = (int)as_ll(a[4]);
    const int hnd = PyObject_IsTrue(a[5]);
    if (PyErr_Occurred()) return nullptr;
    if (c.in_dtype < 0 || !(D == 64 || (D > 0 && D % 128 == 0)) || D > 0x7fffffff || B > 0x7fffffff || !(c.s[0] > 0.0f) || !(c.s[1] > 0.0f) ||
        c.fp8_fmt < 0 || c.fp8_fmt > 2)
      Py_RETURN_NONE;
    c.B = (int)B; c.D = (int)D;
    for (const at::Tensor* t : x)
      if (t->size(1) > 0x7fffffff || t->size(2) > 0x7fffffff) Py_RETURN_NONE;
    at::Tensor codes[2], scales[2];
    int rc;
    {
      const Unlocked unlocked;
      const OnDevice device(x[0]->device().index());
      const at::ScalarType type = c.fp8_fmt == 0 ? at::kByte : c.fp8_fmt == 1 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn;
      for (int i = 0; i < 2; ++i) {
        const auto z = x[i]->sizes(), st = x[i]->strides();
        const int h = hnd ? 1 : 2, l = hnd ? 2 : 1;       // where heads and length are
        codes[i] = dense(z, type, *x[i]);
        scales[i] = dense({B, z[h], z[l], D / 32}, at::kByte, *x[i]);
        const auto cs = codes[i].strides();
        c.x[i] = x[i]->data_ptr(); c.codes[i] = codes[i].data_ptr(); c.scales[i] = scales[i].data_ptr();
        c.H[i] = (int)z[h]; c.L[i] = (int)z[l];
        c.x_sb[i] = st[0]; c.x_sh[i] = st[h]; c.x_sl[i] = st[l];
        c.c_sb[i] = cs[0]; c.c_sh[i] = cs[h]; c.c_sl[i] = cs[l];
      }
      rc = quant_pair_fn(&c, c10::cuda::getCurrentCUDAStream(x[0]->device().index()).stream());
    }
    if (rc) return PyLong_FromLong(rc);
    PyObject* r = PyTuple_New(4);
    if (!r) return nullptr;
    for (int i = 0; i < 2; ++i) {
      PyTuple_SET_ITEM(r, 2 * i, THPVariable_Wrap(std::move(codes[i])));
      PyTuple_SET_ITEM(r, 2 * i + 1, THPVariable_Wrap(std::move(scales[i])));
    }
    return r;
  });
}

// gemm(a, a_scale, b, b_scale, M, N, K, mode, a_fmt, b_fmt, out_dtype, alpha, status)
PyObject* gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 13, "gemm")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *x = plain(a[0]), *xs = plain(a[1]), *y = plain(a[2]), *ys = plain(a[3]);
    if (!x || !xs || !y || !ys || x->dim() < 2 || y->dim() < 2 || x->stride(-1) != 1 || y->stride(-1) != 1 || !xs->is_contiguous() || !ys->is_contiguous())
      Py_RETURN_NONE;
    long long w[7];
    for (int i = 0; i < 7; ++i) w[i] = as_ll(a[4 + i]);
    const double alpha = PyFloat_AsDouble(a[11]);
    int* const status = static_cast<int*>(PyLong_AsVoidPtr(a[12]));
    if (PyErr_Occurred()) return nullptr;
    for (int i = 0; i < 3; ++i)
      if (w[i] <= 0 || w[i] > 0x7fffffff) Py_RETURN_NONE;
    if (w[6] < 0 || w[6] > 3) Py_RETURN_NONE;
    at::Tensor c;
    int rc;
    {
      const Unlocked unlocked;
      const OnDevice device(x->device().index());
      c = dense({(int64_t)w[0], (int64_t)w[1]}, kOut[w[6]], *x);
      rc = gemm_fn(x->data_ptr(), xs->data_ptr(), y->data_ptr(), ys->data_ptr(), c.data_ptr(), (int)w[0], (int)w[1], (int)w[2],
                   x->stride(0) * x->element_size(), y->stride(0) * y->element_size(), w[1], (int)w[3], (int)w[4], (int)w[5], (int)w[6],
                   (float)alpha, status, c10::cuda::getCurrentCUDAStream(x->device().index()).stream());
    }
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(std::move(c));
  });
}

// ---- serving token by token (mpsa/serving.py says what each takes; None: it checks, copies or refuses itself) ----

PyObject* init_serving(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 5, "init_serving")) return nullptr;
  norm_rope_fn = reinterpret_cast<decltype(norm_rope_fn)>(PyLong_AsVoidPtr(a[0]));
  kv_append_fn = reinterpret_cast<decltype(kv_append_fn)>(PyLong_AsVoidPtr(a[1]));
  kv_read_fn = reinterpret_cast<decltype(kv_read_fn)>(PyLong_AsVoidPtr(a[2]));
  kv_workspace_fn = reinterpret_cast<decltype(kv_workspace_fn)>(PyLong_AsVoidPtr(a[3]));
  kv_attention_fn = reinterpret_cast<decltype(kv_attention_fn)>(PyLong_AsVoidPtr(a[4]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// An optional plain tensor: false where the object is something else.
bool optional_plain(PyObject* o, const at::Tensor*& t) {
  t = o == Py_None ? nullptr : plain(o);
  return t || o == Py_None;
}

int any_dtype(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 2 : in_dtype(t); }
bool fits_int(int64_t n) { return n > 0 && n <= 0x7fffffff; }

// 4-D with dense rows, base and strides in multiples of `elements`
bool rows_aligned(const at::Tensor& t, int elements) {
  if (t.dim() != 4 || t.stride(3) != 1) return false;
  const auto s = t.strides();
  const uintptr_t bytes = elements * t.element_size() < 16 ? elements * t.element_size() : 16;
  return !((s[0] | s[1] | s[2]) & (elements - 1)) && !(reinterpret_cast<uintptr_t>(t.data_ptr()) & (bytes - 1)) && fits_int(t.size(0)) && fits_int(t.size(1)) &&
         fits_int(t.size(2)) && fits_int(t.size(3));
}

// A gradient, or a tangent of forward mode (no_grad leaves those on)
bool asks_gradient(const at::Tensor& t) { return (t.requires_grad() && at::GradMode::is_enabled()) || t._fw_grad(0).defined(); }

// int32 [B], dense, on `device`
bool indices(const at::Tensor& t, int64_t B, int device) {
  return t.dim() == 1 && t.size(0) == B && t.scalar_type() == at::kInt && t.is_contiguous() && t.get_device() == device;
}
bool page_table(const at::Tensor& t, int64_t B, int device) {
  return t.dim() == 2 && t.size(0) == B && fits_int(t.size(1)) && t.scalar_type() == at::kInt && t.stride(1) == 1 && t.get_device() == device;
}

// The argument block of a cache (block, k, k_scale, v, v_scale) if it is that of its buffers as they are now; own: the first of them.
const mpsa_kv_cache* cache_of(PyObject* o, const at::Tensor*& own) {
  if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 5 || !PyBytes_CheckExact(PyTuple_GET_ITEM(o, 0)) ||
      PyBytes_GET_SIZE(PyTuple_GET_ITEM(o, 0)) != sizeof(mpsa_kv_cache) || !(own = plain(PyTuple_GET_ITEM(o, 1))))
    return nullptr;
  const mpsa_kv_cache* const c = reinterpret_cast<const mpsa_kv_cache*>(PyBytes_AS_STRING(PyTuple_GET_ITEM(o, 0)));
  const void* const at[4] = {c->k, c->k_scale, c->v, c->v_scale};
  const int64_t row[2] = {c->elem == 2 ? c->D / 2 : c->D, c->D / 32};
  for (int i = 0; i < 4; ++i) {
    PyObject* const x = PyTuple_GET_ITEM(o, 1 + i);
    if (!THPVariable_CheckExact(x)) return nullptr;
    const c10::TensorImpl* const t = THPVariable_Unpack(x).unsafeGetTensorImpl();
    if (!t->has_storage() || t->data() != at[i] || t->dim() != 4 || !t->is_contiguous()) return nullptr;     // (the address is the device's, too)
    const auto z = t->sizes();
    if (z[0] != c->num_pages || z[1] != c->Hkv || z[2] != c->page_size || z[3] != row[i & 1]) return nullptr;
  }
  return c;
}

// kv_cache(k, k_scale, v, v_scale, elem) -> the cache's argument block as bytes
PyObject* kv_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 5, "kv_cache")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* t[4];
    for (int i = 0; i < 4; ++i)
      if (!(t[i] = plain(a[i])) || t[i]->dim() != 4 || t[i]->scalar_type() != at::kByte || !t[i]->is_contiguous() || t[i]->get_device() != t[0]->get_device()) Py_RETURN_NONE;
    const long long elem = as_ll(a[4]);
    if (PyErr_Occurred()) return nullptr;
    const auto z = t[0]->sizes();
    const int64_t D = elem == 2 ? 2 * z[3] : z[3];
    for (int i = 0; i < 4; ++i)
      if (!fits_int(z[i]) || (i < 3 && (t[1]->size(i) != z[i] || t[2]->size(i) != z[i] || t[3]->size(i) != z[i]))) Py_RETURN_NONE;
    if (t[2]->size(3) != z[3] || t[1]->size(3) != D / 32 || t[3]->size(3) != D / 32) Py_RETURN_NONE;
    mpsa_kv_cache c = {};
    c.k = t[0]->data_ptr(); c.k_scale = t[1]->data_ptr(); c.v = t[2]->data_ptr(); c.v_scale = t[3]->data_ptr();
    c.num_pages = (int)z[0]; c.Hkv = (int)z[1]; c.page_size = (int)z[2]; c.D = (int)D; c.elem = (int)elem;
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&c), sizeof c);
  });
}

// norm_rope(q, k, q_weight, k_weight, norm, eps, cos, sin, positions, sections, interleaved, hnd) -> (q, k) or q
PyObject* norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 12, "norm_rope")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor *x[2], *w[2], *cos, *sin, *pos;
    if (!(x[0] = plain(a[0])) || !optional_plain(a[1], x[1]) || !optional_plain(a[2], w[0]) || !optional_plain(a[3], w[1]) || !optional_plain(a[6], cos) ||
        !optional_plain(a[7], sin) || !optional_plain(a[8], pos))
      Py_RETURN_NONE;
    mpsa_norm_rope_args c = {};
    c.in_dtype = any_dtype(*x[0]);
    c.norm = (int)as_ll(a[4]);
    c.eps = (float)PyFloat_AsDouble(a[5]);
    c.interleaved = PyObject_IsTrue(a[10]);
    const int hnd = PyObject_IsTrue(a[11]), h = hnd ? 1 : 2, l = hnd ? 2 : 1;
    if (PyErr_Occurred()) return nullptr;
    if (c.in_dtype < 0 || (!c.norm && (w[0] || w[1])) || (!x[1] && w[1])) Py_RETURN_NONE;
    const int device = x[0]->get_device();
    for (int i = 0; i < (x[1] ? 2 : 1); ++i) {
      if (!rows_aligned(*x[i], 4) || x[i]->scalar_type() != x[0]->scalar_type() || x[i]->get_device() != device || asks_gradient(*x[i])) Py_RETURN_NONE;
      const auto z = x[i]->sizes(), s = x[i]->strides();
      if (z[0] != x[0]->size(0) || z[l] != x[0]->size(l) || z[3] != x[0]->size(3)) Py_RETURN_NONE;
      c.x[i] = x[i]->data_ptr();
      c.x_sb[i] = s[0]; c.x_sh[i] = s[h]; c.x_sl[i] = s[l];
      c.H[i] = (int)z[h];
      if (!w[i]) continue;
      const int64_t D = z[3], most = c.norm == 2 ? z[h] * D : D;
      const bool shaped = w[i]->dim() == 1 ? w[i]->size(0) == most : w[i]->dim() == 2 && c.norm == 2 && w[i]->size(0) == z[h] && w[i]->size(1) == D;
      c.w_dtype[i] = any_dtype(*w[i]);
      if (!shaped || (c.w_dtype[i] != 2 && c.w_dtype[i] != c.in_dtype) || (i && w[0] && c.w_dtype[0] != c.w_dtype[1]) || reinterpret_cast<uintptr_t>(w[i]->data_ptr()) % 16 || !w[i]->is_contiguous() || w[i]->get_device() != device || asks_gradient(*w[i])) Py_RETURN_NONE;
      c.weight[i] = w[i]->data_ptr();
    }
    c.B = (int)x[0]->size(0); c.L = (int)x[0]->size(l); c.D = (int)x[0]->size(3);
    c.axes = 1;
    if ((cos != nullptr) != (sin != nullptr) || (!cos && (pos || a[9] != Py_None))) Py_RETURN_NONE;
    if (cos) {
      for (const at::Tensor* t : {cos, sin})
        if (t->dim() != 2 || t->scalar_type() != at::kFloat || t->sizes() != cos->sizes() || !t->is_contiguous() || t->get_device() != device || reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 || asks_gradient(*t)) Py_RETURN_NONE;
      if (!fits_int(cos->size(0)) || !fits_int(cos->size(1)) || 2 * cos->size(1) > c.D) Py_RETURN_NONE;
      c.cos = cos->data_ptr(); c.sin = sin->data_ptr();
      c.table_rows = cos->size(0); c.rot = (int)(2 * cos->size(1));
      const bool several = a[9] != Py_None;
      if (several) {
        if (!pos || !PyTuple_CheckExact(a[9]) || PyTuple_GET_SIZE(a[9]) < 1 || PyTuple_GET_SIZE(a[9]) > 4) Py_RETURN_NONE;
        c.axes = (int)PyTuple_GET_SIZE(a[9]);
        long long end = 0;
        for (int i = 0; i < c.axes; ++i) {
          const long long k = as_ll(PyTuple_GET_ITEM(a[9], i));
          if (PyErr_Occurred()) return nullptr;
          if (k < 0 || k > c.rot) Py_RETURN_NONE;
          c.section_end[i] = (int)(end += k);
        }
        if (end != c.rot / 2) Py_RETURN_NONE;
      }
      if (pos) {
        const int64_t inner = several ? 2 : 1, d = pos->dim();
        if ((pos->scalar_type() != at::kInt && pos->scalar_type() != at::kLong) || !pos->is_contiguous() || pos->get_device() != device ||
            (d != inner && d != inner + 1) || (several && pos->size(-1) != c.axes) || pos->size(d - inner) != c.L || (d > inner && pos->size(0) != c.B))
          Py_RETURN_NONE;
        c.positions = pos->data_ptr();
        c.pos64 = pos->scalar_type() == at::kLong;
        c.pos_sb = d > inner ? (long long)c.L * c.axes : 0;
      } else if (c.L > c.table_rows) {
        Py_RETURN_NONE;
      }
    }
    at::Tensor y[2];
    int rc;
    {
      const Unlocked unlocked;
      const OnDevice guard(x[0]->device().index());
      for (int i = 0; i < (x[1] ? 2 : 1); ++i) {
        y[i] = dense(x[i]->sizes(), x[i]->scalar_type(), *x[i]);
        const auto s = y[i].strides();
        c.y[i] = y[i].data_ptr();
        c.y_sb[i] = s[0]; c.y_sh[i] = s[h]; c.y_sl[i] = s[l];
      }
      rc = norm_rope_fn(&c, c10::cuda::getCurrentCUDAStream(x[0]->device().index()).stream());
    }
    if (rc) return PyLong_FromLong(rc);
    if (!x[1]) return THPVariable_Wrap(std::move(y[0]));
    PyObject* r = PyTuple_New(2);
    for (int i = 0; r && i < 2; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(y[i])));
    return r;
  });
}

// kv_append(cache, k, v, page_table, start, counts, hnd) -> error code
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 7, "kv_append")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* own;
    const mpsa_kv_cache* cache = cache_of(a[0], own);
    const at::Tensor *k = plain(a[1]), *v = plain(a[2]), *table = plain(a[3]), *start = plain(a[4]), *counts;
    if (!cache || !k || !v || !table || !start || !optional_plain(a[5], counts)) Py_RETURN_NONE;
    const int hnd = PyObject_IsTrue(a[6]), h = hnd ? 1 : 2, l = hnd ? 2 : 1, device = own->get_device();
    if (!rows_aligned(*k, 8) || !rows_aligned(*v, 8) || asks_gradient(*k) || asks_gradient(*v) || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type() || any_dtype(*k) < 0 ||
        k->get_device() != device || v->get_device() != device || k->size(h) != cache->Hkv || k->size(3) != cache->D)
      Py_RETURN_NONE;
    const int64_t B = k->size(0);
    if (!page_table(*table, B, device) || !indices(*start, B, device) || (counts && !indices(*counts, B, device))) Py_RETURN_NONE;
    mpsa_kv_append_args c = {};
    c.cache = *cache;
    c.k = k->data_ptr(); c.v = v->data_ptr();
    const auto ks = k->strides(), vs = v->strides();
    c.k_sb = ks[0]; c.k_sh = ks[h]; c.k_sl = ks[l];
    c.v_sb = vs[0]; c.v_sh = vs[h]; c.v_sl = vs[l];
    c.table_sb = table->stride(0);
    c.page_table = static_cast<const int*>(table->data_ptr()); c.start = static_cast<const int*>(start->data_ptr());
    c.counts = counts ? static_cast<const int*>(counts->data_ptr()) : nullptr;
    c.in_dtype = any_dtype(*k); c.B = (int)B; c.T = (int)k->size(l); c.max_pages = (int)table->size(1);
    int rc;
    {
      const Unlocked unlocked;
      const OnDevice guard(own->device().index());
      rc = kv_append_fn(&c, c10::cuda::getCurrentCUDAStream(own->device().index()).stream());
    }
    return PyLong_FromLong(rc);
  });
}

// kv_read(cache, page_table, lengths, max_len, out_dtype) -> (k, v)
PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 5, "kv_read")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* own;
    const mpsa_kv_cache* cache = cache_of(a[0], own);
    const at::Tensor *table = plain(a[1]), *lengths = plain(a[2]);
    const long long len = as_ll(a[3]), type = as_ll(a[4]);
    if (PyErr_Occurred()) return nullptr;
    if (!cache || !table || !lengths || !fits_int(len) || type < 0 || type > 2 || table->dim() != 2) Py_RETURN_NONE;
    const int64_t B = table->size(0);
    if (!fits_int(B) || !page_table(*table, B, own->get_device()) || !indices(*lengths, B, own->get_device())) Py_RETURN_NONE;
    mpsa_kv_read_args c = {};
    c.cache = *cache;
    c.table_sb = table->stride(0);
    c.page_table = static_cast<const int*>(table->data_ptr()); c.lengths = static_cast<const int*>(lengths->data_ptr());
    c.out_dtype = (int)type; c.B = (int)B; c.max_len = (int)len; c.max_pages = (int)table->size(1);
    at::Tensor y[2];
    int rc;
    {
      const Unlocked unlocked;
      const OnDevice guard(own->device().index());
      for (at::Tensor& t : y) t = dense({B, cache->Hkv, len, cache->D}, kOut[type], *own);
      c.k_out = y[0].data_ptr(); c.v_out = y[1].data_ptr();
      rc = kv_read_fn(&c, c10::cuda::getCurrentCUDAStream(own->device().index()).stream());
    }
    if (rc) return PyLong_FromLong(rc);
    PyObject* r = PyTuple_New(2);
    for (int i = 0; r && i < 2; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(std::move(y[i])));
    return r;
  });
}

// kv_attention(cache, q, page_table, lengths, q_lens, mask, status, sm_scale, want_lse, hnd) -> out or (out, lse)
PyObject* kv_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counted(n, 10, "kv_attention")) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* own;
    const mpsa_kv_cache* cache = cache_of(a[0], own);
    const at::Tensor *q = plain(a[1]), *table = plain(a[2]), *lengths = plain(a[3]), *qlens, *mask;
    if (!cache || !q || !table || !lengths || !optional_plain(a[4], qlens) || !optional_plain(a[5], mask)) Py_RETURN_NONE;
    mpsa_kv_attention_args c = {};
    c.status = static_cast<int*>(PyLong_AsVoidPtr(a[6]));
    c.sm_scale = (float)PyFloat_AsDouble(a[7]);
    const int lse = PyObject_IsTrue(a[8]), hnd = PyObject_IsTrue(a[9]), h = hnd ? 1 : 2, l = hnd ? 2 : 1, device = own->get_device();
    if (PyErr_Occurred()) return nullptr;
    c.dtype = in_dtype(*q);
    if (c.dtype < 0 || !rows_aligned(*q, 8) || asks_gradient(*q) || q->get_device() != device || q->size(3) != cache->D || q->size(h) % cache->Hkv || q->size(l) > 1024) Py_RETURN_NONE;
    const int64_t B = q->size(0), T = q->size(l), Hq = q->size(h);
    if (!page_table(*table, B, device) || !indices(*lengths, B, device) || (qlens && !indices(*qlens, B, device))) Py_RETURN_NONE;
    if (mask) {
      const int64_t d = mask->dim();
      if ((d != 2 && d != 3) || mask->scalar_type() != at::kBool || mask->size(-1) != T || mask->size(-2) != T || (d == 3 && mask->size(0) != B) ||
          mask->get_device() != device || !mask->is_contiguous())
        Py_RETURN_NONE;
      c.mask = static_cast<const unsigned char*>(mask->data_ptr());
      c.mask_sb = d == 3 ? T * T : 0;
    }
    c.cache = *cache;
    c.q = q->data_ptr();
    const auto s = q->strides();
    c.q_sb = s[0]; c.q_sh = s[h]; c.q_sl = s[l];
    c.table_sb = table->stride(0);
    c.page_table = static_cast<const int*>(table->data_ptr()); c.lengths = static_cast<const int*>(lengths->data_ptr());
    c.q_lens = qlens ? static_cast<const int*>(qlens->data_ptr()) : nullptr;
    c.B = (int)B; c.T = (int)T; c.Hq = (int)Hq; c.max_pages = (int)table->size(1);
    at::Tensor out, sums;
    long long rc;
    {
      const Unlocked unlocked;
      const OnDevice guard(own->device().index());
      rc = kv_workspace_fn(&c);
      if (rc >= 0) {
        const at::Tensor ws = dense({(int64_t)rc}, at::kByte, *q);
        out = dense(q->sizes(), q->scalar_type(), *q);
        if (lse) sums = dense({B, Hq, T}, at::kFloat, *q);
        const auto os = out.strides();
        c.out = out.data_ptr(); c.lse = lse ? sums.data_ptr() : nullptr;
        c.o_sb = os[0]; c.o_sh = os[h]; c.o_sl = os[l];
        c.workspace = ws.data_ptr(); c.workspace_bytes = rc;
        rc = kv_attention_fn(&c, c10::cuda::getCurrentCUDAStream(own->device().index()).stream());
      }
    }
    if (rc) return PyLong_FromLongLong(rc);
    if (!lse) return THPVariable_Wrap(std::move(out));
    PyObject* r = PyTuple_New(2);
    if (!r) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(out)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(sums)));
    return r;
  });
}

PyMethodDef methods[] = {
    {"init", (PyCFunction)(void*)init, METH_FASTCALL, "addresses of mpsa_attention_workspace, mpsa_attention, mpsa_quant_pair, mpsa_gemm_block_scaled; torch.OutOfMemoryError"},
    {"attention", (PyCFunction)(void*)attention, METH_FASTCALL, "one attention call: output tensor, None (operands not taken) or an error code"},
    {"quant_pair", (PyCFunction)(void*)quant_pair, METH_FASTCALL, "two operands quantised: four tensors, None or an error code"},
    {"gemm", (PyCFunction)(void*)gemm, METH_FASTCALL, "block-scaled product: output tensor, None or an error code"},
    {"init_serving", (PyCFunction)(void*)init_serving, METH_FASTCALL, "addresses of mpsa_norm_rope, mpsa_kv_append, mpsa_kv_read, mpsa_kv_attention_workspace, mpsa_kv_attention"},
    {"kv_cache", (PyCFunction)(void*)kv_cache, METH_FASTCALL, "a cache's argument block as bytes, or None"},
    {"norm_rope", (PyCFunction)(void*)norm_rope, METH_FASTCALL, "norm and rotation: tensors, None or an error code"},
    {"kv_append", (PyCFunction)(void*)kv_append, METH_FASTCALL, "tokens into a cache: an error code or None"},
    {"kv_read", (PyCFunction)(void*)kv_read, METH_FASTCALL, "sequences from a cache: two tensors, None or an error code"},
    {"kv_attention", (PyCFunction)(void*)kv_attention, METH_FASTCALL, "attention over a cache: tensors, None or an error code"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", "torch tensors into libmpsa.so", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&module); }
