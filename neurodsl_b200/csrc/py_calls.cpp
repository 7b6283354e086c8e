// py_calls.cpp — the serving operators' calls from Python without the
// interpreter's share: a CPython extension that reads the tensors directly.
//
// A serving step makes these calls once a layer with kernels of a few
// microseconds, and the front end's argument checks and the foreign-function
// call cost more than that: back to back, a decode that takes the device 7.4 us
// took 12.5 a call and 7.4 here, a short store 9.8 and 3.5.  Each function
// here takes the arguments of its namesake in ops.py, checks that they are what
// nearly every call passes (tensors of the right types on the current device,
// outputs given, the current stream), and calls the C entry point, which
// validates sizes, alignment and the rest.  Returns its status; or None for
// anything else, which ops.py then checks, refuses or carries out itself.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>

#include "neurodsl_b200.h"

namespace {

constexpr auto kBF16 = at::kBFloat16;
constexpr auto kF32 = at::kFloat;
constexpr auto kI32 = at::kInt;

// The C entry points, by the addresses that the loader of the library gives
// (the extension does not link against it, so there is one copy of it).
decltype(&nd_window_attn_fwd) f_window = nullptr;
decltype(&nd_paged_decode_attn) f_decode = nullptr;
decltype(&nd_paged_kv_store) f_store = nullptr;
decltype(&nd_paged_kv_evict) f_evict = nullptr;
decltype(&nd_logits_penalty) f_logits = nullptr;

// What a call's arguments turned out to be; `ok` falls at the first that is
// for ops.py.
struct Args {
  PyObject* const* a;
  bool ok = true;
  int dev = -1;

  const at::Tensor* tensor(int i, at::ScalarType type, int dims, bool contiguous = true) {
    if (!ok) return nullptr;
    if (!THPVariable_Check(a[i])) return fail();
    const at::Tensor& t = THPVariable_Unpack(a[i]);
    if (!t.is_cuda() || t.layout() != at::kStrided || t.is_conj() || t.is_neg()) return fail();
    if (dev < 0) {
      dev = t.get_device();
      if (c10::cuda::current_device() != dev) return fail();
    }
    if (t.get_device() != dev || t.scalar_type() != type || (dims >= 0 && t.dim() != dims) ||
        (contiguous && !t.is_contiguous()))
      return fail();
    return &t;
  }
  const at::Tensor* optional(int i, at::ScalarType type, int dims, bool contiguous = true) {
    return a[i] == Py_None ? nullptr : tensor(i, type, dims, contiguous);
  }
  // float32 or bfloat16
  const at::Tensor* real(int i, int dims, bool contiguous = true) {
    if (!ok || !THPVariable_Check(a[i])) return fail();
    const auto type = THPVariable_Unpack(a[i]).scalar_type();
    return tensor(i, type == kBF16 ? kBF16 : kF32, dims, contiguous);
  }
  // A [rows][cols] int32 matrix with contiguous rows; its row stride.
  const at::Tensor* matrix(int i, int64_t rows, int64_t& ld) {
    const at::Tensor* t = tensor(i, kI32, 2, false);
    if (t != nullptr && !rows_of(*t, rows, ld)) return fail();
    return t;
  }
  bool rows_of(const at::Tensor& t, int64_t rows, int64_t& ld) {
    const int64_t cols = t.size(1);
    if (t.size(0) != rows || (cols > 1 && t.stride(1) != 1)) return false;
    ld = rows > 1 ? t.stride(0) : cols;
    return ld >= cols;
  }
  int integer(int i) {
    if (!ok || !PyLong_CheckExact(a[i])) return fail(), 0;
    int over = 0;
    const long long v = PyLong_AsLongLongAndOverflow(a[i], &over);
    if (over != 0 || v > INT_MAX || v < INT_MIN) return fail(), 0;
    return static_cast<int>(v);
  }
  // None: 1 / sqrt(d)
  float scale(int i, int64_t d) {
    if (!ok) return 0.f;
    if (a[i] == Py_None) return static_cast<float>(1.0 / std::sqrt(static_cast<double>(d)));
    if (!PyFloat_CheckExact(a[i])) return fail(), 0.f;
    return static_cast<float>(PyFloat_AS_DOUBLE(a[i]));
  }
  void need(bool x) { ok = ok && x; }
  std::nullptr_t fail() {
    ok = false;
    return nullptr;
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }
};

template <typename T = void>
T* ptr(const at::Tensor* t) {
  return t == nullptr ? nullptr : static_cast<T*>(t->data_ptr());
}
int dtype(const at::Tensor& t) { return t.scalar_type() == kBF16 ? ND_BF16 : ND_F32; }
int narrow(int64_t v, Args& a) {
  a.need(v <= INT_MAX);
  return static_cast<int>(v);
}

// The interpreter's lock let go for a scope (an exception takes it back too).
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// The status of `call` made without the interpreter's lock, or None.
template <typename F>
PyObject* status(const Args& a, F&& call) {
  if (!a.ok) Py_RETURN_NONE;
  int rc;
  {
    void* stream = a.stream();
    const Unlocked unlocked;
    rc = call(stream);
  }
  return PyLong_FromLong(rc);
}

// An exception of the tensor library becomes "for ops.py".
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// (Q, K, V, window, sinks, scale, out, lse, row_max)
PyObject* window_attn_fwd(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 9 || f_window == nullptr) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const at::Tensor *q = a.tensor(0, kBF16, 4, false), *k = a.tensor(1, kBF16, 4, false),
                     *x = a.tensor(2, kBF16, 4, false), *o = a.real(6, 4, false);
    const at::Tensor *lse = a.tensor(7, kF32, -1), *m = a.tensor(8, kF32, -1);
    const int window = a.integer(3), sinks = a.integer(4);
    if (!a.ok) Py_RETURN_NONE;
    const int64_t B = q->size(0), H = q->size(1), Sq = q->size(2), D = q->size(3);
    const int64_t Hkv = k->size(1), Sk = k->size(2);
    const float scale = a.scale(5, D);
    a.need(k->size(0) == B && k->size(3) == D && x->sizes() == k->sizes() && o->sizes() == q->sizes() &&
           lse->numel() == B * H * Sq && m->numel() == B * H * Sq);
    int64_t st[4][3];
    const at::Tensor* all[4] = {q, k, x, o};
    for (int i = 0; i < 4; ++i) {
      a.need(all[i]->stride(3) == 1);
      st[i][0] = all[i]->stride(2);
      st[i][1] = all[i]->stride(1);
      st[i][2] = all[i]->stride(0);
    }
    const int b = narrow(B, a), h = narrow(H, a), hk = narrow(Hkv, a), sq = narrow(Sq, a), sk = narrow(Sk, a);
    const int d = narrow(D, a);
    return status(a, [&](void* s) {
      return f_window(s, ptr(q), st[0], ptr(k), st[1], ptr(x), st[2], ptr(o), st[3], dtype(*o), ptr<float>(lse),
                      ptr<float>(m), b, h, hk, sq, sk, d, scale, window, sinks);
    });
  });
}

// (q, k_pages, v_pages, table, lens, k_new, v_new, window, sinks, scale, out, lse, weights, workspace)
PyObject* paged_decode_attn(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 14 || f_decode == nullptr) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const at::Tensor *q = a.tensor(0, kBF16, 3), *k = a.tensor(1, kBF16, 4), *x = a.tensor(2, kBF16, 4);
    if (!a.ok) Py_RETURN_NONE;
    const int64_t B = q->size(0), H = q->size(1), D = q->size(2), Hkv = k->size(1);
    int64_t ld = 0;
    const at::Tensor *table = a.matrix(3, B, ld), *lens = a.tensor(4, kI32, 1);
    const at::Tensor *kn = a.optional(5, kBF16, 3), *vn = a.optional(6, kBF16, 3);
    const int window = a.integer(7), sinks = a.integer(8);
    const float scale = a.scale(9, D);
    const at::Tensor *out = a.real(10, 3), *lse = a.optional(11, kF32, -1), *w = a.optional(12, kF32, 3);
    if (!a.ok || !THPVariable_Check(v[13])) Py_RETURN_NONE;
    const at::Tensor* ws = a.tensor(13, THPVariable_Unpack(v[13]).scalar_type(), -1);
    if (!a.ok) Py_RETURN_NONE;
    a.need(x->sizes() == k->sizes() && k->size(3) == D && lens->numel() == B && out->sizes() == q->sizes() &&
           (kn == nullptr) == (vn == nullptr));
    for (const at::Tensor* t : {kn, vn})
      if (t != nullptr) a.need(t->size(0) == B && t->size(1) == Hkv && t->size(2) == D);
    if (lse != nullptr) a.need(lse->numel() == B * H);
    if (w != nullptr) a.need(w->size(0) == B && w->size(1) == Hkv);
    const int np = narrow(k->size(0), a), ps = narrow(k->size(2), a), mp = narrow(table->size(1), a);
    const int b = narrow(B, a), h = narrow(H, a), hk = narrow(Hkv, a), d = narrow(D, a);
    return status(a, [&](void* s) {
      return f_decode(s, ptr(q), ptr(kn), ptr(vn), ptr(k), ptr(x), np, ps, ptr<int32_t>(table), ld, mp,
                      ptr<int32_t>(lens), ptr(out), dtype(*out), ptr<float>(lse), ptr<float>(w),
                      w == nullptr ? 0 : w->size(2), b, h, hk, d, window, sinks, scale, ptr(ws),
                      ws->nbytes());
    });
  });
}

// (src, k_col, v_col, k_pages, v_pages, table, B, S, pos0 tensor or int, lens)
PyObject* paged_kv_store(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 10 || f_store == nullptr) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const at::Tensor *src = a.tensor(0, kBF16, 2, false), *k = a.tensor(3, kBF16, 4), *x = a.tensor(4, kBF16, 4);
    const int k_col = a.integer(1), v_col = a.integer(2), B = a.integer(6), S = a.integer(7);
    int64_t ld = 0, t_ld = 0;
    if (!a.ok || B < 0 || S < 0 || !a.rows_of(*src, static_cast<int64_t>(B) * S, ld)) Py_RETURN_NONE;
    const at::Tensor* table = a.matrix(5, B, t_ld);
    const at::Tensor *pos = nullptr, *lens = a.optional(9, kI32, 1);
    int pos0 = 0;
    if (THPVariable_Check(v[8]))
      pos = a.tensor(8, kI32, 1);
    else
      pos0 = a.integer(8);
    if (!a.ok) Py_RETURN_NONE;
    const int64_t Hkv = k->size(1), D = k->size(3);
    a.need(x->sizes() == k->sizes() && (pos == nullptr || pos->numel() == B) &&
           (lens == nullptr || lens->numel() == B) && (k_col > v_col ? k_col : v_col) + Hkv * D <= src->size(1));
    const int np = narrow(k->size(0), a), ps = narrow(k->size(2), a), mp = narrow(table->size(1), a);
    const int hk = narrow(Hkv, a), d = narrow(D, a);
    return status(a, [&](void* s) {
      return f_store(s, ptr(src), ld, k_col, v_col, ptr(k), ptr(x), np, ps, ptr<int32_t>(table), t_ld, mp, B, S, hk,
                     pos0, ptr<int32_t>(pos), ptr<int32_t>(lens), d);
    });
  });
}

// (k_pages, v_pages, table, lens, weights, out_table, budget, sinks, recent, weights_out, kept, new_lens)
PyObject* paged_kv_evict(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 12 || f_evict == nullptr) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const at::Tensor *k = a.tensor(0, kBF16, 4), *x = a.tensor(1, kBF16, 4), *lens = a.tensor(3, kI32, 1);
    if (!a.ok) Py_RETURN_NONE;
    const int64_t B = lens->numel(), Hkv = k->size(1), D = k->size(3);
    int64_t ld = 0, out_ld = 0;
    const at::Tensor *table = a.matrix(2, B, ld), *out_table = a.matrix(5, B, out_ld);
    const at::Tensor *w = a.tensor(4, kF32, 3), *wo = a.tensor(9, kF32, 3);
    const at::Tensor *kept = a.tensor(10, kI32, -1), *nl = a.tensor(11, kI32, -1);
    const int budget = a.integer(6), sinks = a.integer(7), recent = a.integer(8);
    if (!a.ok) Py_RETURN_NONE;
    a.need(x->sizes() == k->sizes() && w->size(0) == B && w->size(1) == Hkv && wo->size(0) == B &&
           wo->size(1) == Hkv && budget >= 0 && kept->numel() == B * Hkv * budget && nl->numel() == B);
    const int np = narrow(k->size(0), a), ps = narrow(k->size(2), a), mp = narrow(table->size(1), a);
    const int mo = narrow(out_table->size(1), a), b = narrow(B, a), hk = narrow(Hkv, a);
    const int d = narrow(D, a);
    return status(a, [&](void* s) {
      return f_evict(s, ptr(k), ptr(x), np, ps, ptr<int32_t>(table), ld, mp, ptr<int32_t>(lens), ptr<float>(w),
                     w->size(2), ptr<int32_t>(out_table), out_ld, mo, ptr<float>(wo), wo->size(2), ptr<int32_t>(kept),
                     ptr<int32_t>(nl), b, hk, d, budget, sinks, recent);
    });
  });
}

// (logits, history, history_lens, repetition, presence, frequency, bias_ids, bias, mask, out, idx)
PyObject* logits_penalty(PyObject*, PyObject* const* v, Py_ssize_t n) {
  if (n != 11 || f_logits == nullptr) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Args a{v};
    const at::Tensor *x = a.real(0, 2, false), *out = a.real(9, 2, false);
    if (!a.ok) Py_RETURN_NONE;
    const int64_t rows = x->size(0), V = x->size(1);
    int64_t ld = 0, out_ld = 0, h_ld = 0, m_ld = 0;
    a.need(out->size(1) == V && a.rows_of(*x, rows, ld) && a.rows_of(*out, rows, out_ld));
    const at::Tensor* hist = v[1] == Py_None ? nullptr : a.matrix(1, rows, h_ld);
    const at::Tensor* hl = a.optional(2, kI32, 1);
    const at::Tensor *rep = a.optional(3, kF32, 1), *pres = a.optional(4, kF32, 1), *freq = a.optional(5, kF32, 1);
    const at::Tensor *ids = a.optional(6, kI32, 2), *bias = a.optional(7, kF32, 2);
    const at::Tensor *mask = a.optional(8, kI32, -1, false), *idx = a.optional(10, kI32, 1);
    if (!a.ok) Py_RETURN_NONE;
    for (const at::Tensor* t : {hl, rep, pres, freq, idx})
      if (t != nullptr) a.need(t->numel() == rows);
    a.need((ids == nullptr) == (bias == nullptr));
    if (bias != nullptr && ids != nullptr) a.need(ids->sizes() == bias->sizes() && bias->size(0) == rows);
    if (mask != nullptr) {
      const int64_t dims = mask->dim();
      a.need(dims == 1 || (dims == 2 && mask->size(0) == rows));
      if (!a.ok) Py_RETURN_NONE;
      const int64_t words = mask->size(dims - 1);
      a.need(words >= (V + 31) / 32 && (words <= 1 || mask->stride(dims - 1) == 1));
      if (dims == 2) m_ld = rows > 1 ? mask->stride(0) : words;
    }
    const int r = narrow(rows, a), nv = narrow(V, a), nh = hist == nullptr ? 0 : narrow(hist->size(1), a);
    const int nb = bias == nullptr ? 0 : narrow(bias->size(1), a);
    // a history without entries has no memory; it is still a history, and not read
    const void* h = hist != nullptr && nh == 0 ? ptr(x) : ptr(hist);
    return status(a, [&](void* s) {
      return f_logits(s, ptr(x), dtype(*x), ld, r, nv, static_cast<const int32_t*>(h), h_ld, nh, ptr<int32_t>(hl), ptr<float>(rep),
                      ptr<float>(pres), ptr<float>(freq), ptr<int32_t>(ids), ptr<float>(bias), nb, ptr<uint32_t>(mask),
                      m_ld, ptr(out), dtype(*out), out_ld, ptr<int32_t>(idx));
    });
  });
}

// bind(window, decode, store, evict, logits): the entry points' addresses
PyObject* bind(PyObject*, PyObject* const* v, Py_ssize_t n) {
  void* p[5];
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes five addresses");
    return nullptr;
  }
  for (int i = 0; i < 5; ++i) {
    p[i] = PyLong_AsVoidPtr(v[i]);
    if (p[i] == nullptr && PyErr_Occurred()) return nullptr;
  }
  f_window = reinterpret_cast<decltype(f_window)>(p[0]);
  f_decode = reinterpret_cast<decltype(f_decode)>(p[1]);
  f_store = reinterpret_cast<decltype(f_store)>(p[2]);
  f_evict = reinterpret_cast<decltype(f_evict)>(p[3]);
  f_logits = reinterpret_cast<decltype(f_logits)>(p[4]);
  Py_RETURN_NONE;
}

#define ND_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ND_METHOD(window_attn_fwd), ND_METHOD(paged_decode_attn), ND_METHOD(paged_kv_store),
                         ND_METHOD(paged_kv_evict),  ND_METHOD(logits_penalty),    ND_METHOD(bind),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
