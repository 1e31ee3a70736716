// pycall.cpp -- the Python calls of the chunk and eviction operators, for
// arguments that are as they should be: a tensor's type, device, sizes and
// strides are read here in nanoseconds, where a dozen tensors through the
// interpreter and ctypes take 15 to 25 us, more than the kernels of a decode
// step.  A call whose arguments are not as they should be returns None, and
// the caller's own checks say what is wrong.  The library's entry points come
// in by address (bind), so there is one library, whoever loaded it.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <limits>
#include <vector>

#include "kyro_spec.h"

namespace {

struct {
  decltype(&kyro_ctx_set_stream) set_stream;
  decltype(&kyro_qk_norm_rope_kv_write) rope;
  decltype(&kyro_chunk_attention) attention;
  decltype(&kyro_chunk_attention_workspace_size) attention_workspace;
  decltype(&kyro_kv_scores_add) scores;
  decltype(&kyro_kv_scores_add_workspace_size) scores_workspace;
  decltype(&kyro_kv_evict) evict;
  decltype(&kyro_kv_evict_workspace_size) evict_workspace;
} lib;

// The arguments of one call, until one of them is not as it should be.
struct Args {
  PyObject* const* a;
  bool ok = true;
  kyro_ctx* ctx = nullptr;
  int device = -1;

  explicit Args(PyObject* const* args) : a(args) {
    ctx = (kyro_ctx*)PyLong_AsVoidPtr(a[0]);
    device = (int)PyLong_AsLong(a[1]);
    ok = !PyErr_Occurred() && ctx && lib.rope;
  }
  bool need(bool x) { return ok = ok && x; }
  bool none(int i) const { return a[i] == Py_None; }

  const at::Tensor* any(PyObject* o, at::ScalarType type, int dim) {
    if (!need(THPVariable_CheckExact(o))) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    need(t.layout() == at::kStrided && t.scalar_type() == type && t.dim() == dim && t.is_cuda() &&
         t.get_device() == device);
    return ok ? &t : nullptr;
  }
  // a dense tensor; nullptr if it is not one, or by then `ok` is false
  const at::Tensor* dense(PyObject* o, at::ScalarType type, int dim) {
    const at::Tensor* t = any(o, type, dim);
    return t && need(t->is_contiguous()) ? t : nullptr;
  }
  const at::Tensor* dense(int i, at::ScalarType type, int dim) { return dense(a[i], type, dim); }
  int32_t size(int64_t n) {
    need(n >= 0 && n <= std::numeric_limits<int32_t>::max());
    return (int32_t)n;
  }
  int32_t integer(int i) {
    const long v = PyLong_AsLong(a[i]);
    need(!PyErr_Occurred() && v >= std::numeric_limits<int32_t>::min() &&
         v <= std::numeric_limits<int32_t>::max());
    return (int32_t)v;
  }
  float real(int i) {
    const double v = PyFloat_AsDouble(a[i]);
    need(!PyErr_Occurred());
    return (float)v;
  }

  // [T, heads, D] with dense heads; T rows may lie apart
  struct Rows {
    void* ptr = nullptr;
    int32_t T = 0, h = 0, d = 0;
    int64_t stride = 0;
    const at::Tensor* t = nullptr;
  };
  Rows rows(PyObject* o) {
    Rows r;
    r.t = any(o, at::kBFloat16, 3);
    if (!r.t) return r;
    const auto n = r.t->sizes(), s = r.t->strides();
    r.T = size(n[0]);
    r.h = size(n[1]);
    r.d = size(n[2]);
    const int64_t row = n[1] * n[2];
    r.stride = r.T <= 1 ? row : s[0];
    need((n[2] <= 1 || s[2] == 1) && (n[1] <= 1 || s[1] == n[2]) && r.stride >= row &&
         (r.T <= 1 || r.stride % 8 == 0));
    r.ptr = r.t->data_ptr();
    return r;
  }
  Rows rows(int i, int32_t T, int32_t h, int32_t d) {
    const Rows r = rows(a[i]);
    need(r.T == T && r.h == h && r.d == d);
    return r;
  }
};

// the sequences of a packed batch
struct Batch {
  const at::Tensor *starts, *table, *lens;
  int32_t B = 0, width = 0;

  Batch(Args& c, int i)
      : starts(c.dense(i, at::kInt, 1)), table(c.dense(i + 1, at::kLong, 2)),
        lens(c.dense(i + 2, at::kLong, 1)) {
    if (!c.ok) return;
    B = c.size(table->size(0));
    width = c.size(table->size(1));
    c.need(starts->size(0) == (int64_t)B + 1 && lens->size(0) == B);
  }
  const int32_t* s() const { return (const int32_t*)starts->data_ptr(); }
  int64_t* t() const { return (int64_t*)table->data_ptr(); }
  int64_t* l() const { return (int64_t*)lens->data_ptr(); }
};

PyObject* unsure() {
  PyErr_Clear();
  Py_RETURN_NONE;
}

// Runs `call` without the interpreter's lock; the result, or the status.
template <class Call>
PyObject* run(PyObject* result, Call&& call) {
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = call();
  Py_END_ALLOW_THREADS;
  if (status == KYRO_OK) return result;
  Py_DECREF(result);
  return PyLong_FromLong(status);
}

void* workspace(Args& c, int i, size_t need, size_t* bytes) {
  if (!c.ok) return nullptr;
  const at::Tensor* w = c.none(i) ? nullptr : c.dense(i, at::kByte, 1);
  *bytes = w ? (size_t)w->numel() : 0;
  return c.need(w && need && *bytes >= need) ? w->data_ptr() : nullptr;
}

// (ctx, device, q, k_new, v_new, starts, table, lens, k_cache, v_cache,
//  block_size, q_norm, k_norm, eps, theta, positions, q_out)
PyObject* rope_impl(PyObject* const* a) {
  Args c(a);
  const at::Tensor* kc = c.dense(8, at::kBFloat16, 4);
  const at::Tensor* vc = c.dense(9, at::kBFloat16, 4);
  const Batch b(c, 5);
  const Args::Rows q = c.rows(a[2]);
  if (!c.ok || kc->sizes() != vc->sizes()) return unsure();
  const int32_t nb = c.size(kc->size(0)), hkv = c.size(kc->size(1)), bs = c.size(kc->size(2));
  c.need(bs == c.integer(10) && kc->size(3) == q.d);
  const Args::Rows k = c.rows(3, q.T, hkv, q.d), v = c.rows(4, q.T, hkv, q.d);
  const void* norm[2] = {nullptr, nullptr};
  for (int i = 0; i < 2; ++i)
    if (!c.none(11 + i)) {
      const at::Tensor* w = c.dense(11 + i, at::kBFloat16, 1);
      if (w && c.need(w->numel() == q.d)) norm[i] = w->data_ptr();
    }
  const float eps = c.real(13), theta = c.real(14);
  const int64_t* pos = nullptr;
  if (!c.none(15)) {
    const at::Tensor* w = c.dense(15, at::kLong, 1);
    if (w && c.need(w->numel() == q.T)) pos = (const int64_t*)w->data_ptr();
  }
  Args::Rows o;
  if (!c.none(16)) o = c.rows(16, q.T, q.h, q.d);
  if (!c.ok) return unsure();
  PyObject* result = a[16];
  if (c.none(16)) {
    at::Tensor out = at::empty({q.T, q.h, q.d}, q.t->options());
    o.ptr = out.data_ptr();
    result = THPVariable_Wrap(std::move(out));
  } else {
    Py_INCREF(result);
  }
  const kyro_chunk_params p = {b.B,     q.T, q.h, hkv, q.d, bs, b.width, nb, 0.0f, q.stride,
                               k.stride, v.stride, o.stride};
  return run(result, [&] {
    return lib.rope(c.ctx, &p, theta, eps, norm[0], norm[1], pos, q.ptr, k.ptr, v.ptr, b.s(),
                    b.t(), b.l(), o.ptr, kc->data_ptr(), vc->data_ptr());
  });
}

// (ctx, device, q, k_cache, v_cache, starts, table, lens, scale, out, lse, workspace)
PyObject* attention_impl(PyObject* const* a) {
  Args c(a);
  const at::Tensor* kc = c.dense(3, at::kBFloat16, 4);
  const at::Tensor* vc = c.dense(4, at::kBFloat16, 4);
  const Batch b(c, 5);
  const Args::Rows q = c.rows(a[2]);
  if (!c.ok || kc->sizes() != vc->sizes() || kc->size(3) != q.d) return unsure();
  const float scale = c.none(8) ? 0.0f : c.real(8);
  Args::Rows o;
  if (!c.none(9)) o = c.rows(9, q.T, q.h, q.d);
  float* lse = nullptr;
  if (!c.none(10)) {
    const at::Tensor* w = c.dense(10, at::kFloat, 2);
    if (w && c.need(w->size(0) == q.T && w->size(1) == q.h)) lse = (float*)w->data_ptr();
  }
  const kyro_chunk_params p = {b.B, q.T, q.h, c.size(kc->size(1)), q.d, c.size(kc->size(2)),
                               b.width, c.size(kc->size(0)), scale, q.stride, 0, 0, o.stride};
  size_t bytes;
  void* ws = workspace(c, 11, c.ok ? lib.attention_workspace(&p) : 0, &bytes);
  if (!c.ok) return unsure();
  PyObject* result = a[9];
  if (c.none(9)) {
    at::Tensor out = at::empty({q.T, q.h, q.d}, q.t->options());
    o.ptr = out.data_ptr();
    result = THPVariable_Wrap(std::move(out));
  } else {
    Py_INCREF(result);
  }
  return run(result, [&] {
    return lib.attention(c.ctx, &p, q.ptr, kc->data_ptr(), vc->data_ptr(), b.s(), b.t(), b.l(),
                         o.ptr, lse, ws, bytes);
  });
}

// (ctx, device, q, k_cache, lse, starts, table, lens, scores, scale, out, workspace)
PyObject* scores_impl(PyObject* const* a) {
  Args c(a);
  const at::Tensor* kc = c.dense(3, at::kBFloat16, 4);
  const at::Tensor* lse = c.dense(4, at::kFloat, 2);
  const Batch b(c, 5);
  const Args::Rows q = c.rows(a[2]);
  const at::Tensor* s = c.dense(8, at::kFloat, 3);
  const at::Tensor* o = c.none(10) ? s : c.dense(10, at::kFloat, 3);
  if (!c.ok) return unsure();
  c.need(kc->size(3) == q.d && lse->size(0) == q.T && lse->size(1) == q.h &&
         s->size(0) == b.B && s->size(1) == kc->size(1) && s->sizes() == o->sizes());
  const float scale = c.none(9) ? 0.0f : c.real(9);
  const kyro_chunk_params p = {b.B, q.T, q.h, c.size(kc->size(1)), q.d, c.size(kc->size(2)),
                               b.width, c.size(kc->size(0)), scale, q.stride, 0, 0, 0};
  size_t bytes;
  void* ws = workspace(c, 11, c.ok ? lib.scores_workspace(&p) : 0, &bytes);
  if (!c.ok) return unsure();
  PyObject* result = c.none(10) ? a[8] : a[10];
  Py_INCREF(result);
  return run(result, [&] {
    return lib.scores(c.ctx, &p, q.ptr, kc->data_ptr(), (const float*)lse->data_ptr(), b.s(),
                      b.t(), b.l(), s->size(2), (const float*)s->data_ptr(),
                      (float*)o->data_ptr(), ws, bytes);
  });
}

// (ctx, device, budget, num_sink, num_recent, scores, k_caches, v_caches,
//  table, lens, free_stack, free_top, ref_counts, block_size, num_reserved,
//  kept, evicted, workspace)
PyObject* evict_impl(PyObject* const* a) {
  Args c(a);
  const at::Tensor* table = c.dense(8, at::kLong, 2);
  const at::Tensor* lens = c.dense(9, at::kLong, 1);
  const at::Tensor* stack = c.dense(10, at::kInt, 1);
  const at::Tensor* refs = c.dense(12, at::kInt, 1);
  if (!c.ok || !THPVariable_CheckExact(a[11])) return unsure();
  const at::Tensor* top = c.dense(11, at::kInt, (int)THPVariable_Unpack(a[11]).dim());
  std::vector<void*> ptr[3];
  const at::Tensor* first[3] = {nullptr, nullptr, nullptr};
  Py_ssize_t nl = 0;
  for (int i = 0; i < 3 && c.ok; ++i) {
    PyObject* l = a[5 + i];
    if (!c.need(PyList_CheckExact(l) || PyTuple_CheckExact(l))) break;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(l);
    if (i == 0) nl = n;
    if (!c.need(n == nl && n >= 1 && n < (1 << 20))) break;
    ptr[i].resize(n);
    for (Py_ssize_t j = 0; j < n; ++j) {
      const at::Tensor* t = c.dense(PySequence_Fast_GET_ITEM(l, j), i ? at::kBFloat16 : at::kFloat,
                                    i ? 4 : 3);
      if (!t) break;
      if (j == 0) first[i] = t;
      c.need(t->sizes() == first[i]->sizes());
      ptr[i][j] = t->data_ptr();
    }
  }
  if (!c.ok || first[1]->sizes() != first[2]->sizes()) return unsure();
  const auto cache = first[1]->sizes(), score = first[0]->sizes();
  const int32_t B = c.size(table->size(0)), budget = c.integer(2);
  c.need(budget >= 1 && stack->numel() == refs->numel() && lens->size(0) == B &&
         cache[0] == refs->numel() && cache[2] == c.integer(13) && score[0] == B &&
         score[1] == cache[1]);
  const kyro_evict_params p = {B, c.integer(13), c.size(table->size(1)), c.size(cache[0]),
                               c.size(nl), c.size(cache[1]), c.size(cache[3]), budget,
                               c.integer(3), c.integer(4), c.integer(14), score[2]};
  const at::Tensor* kept = c.none(15) ? nullptr : c.dense(15, at::kInt, 4);
  if (kept)
    c.need(kept->size(0) == nl && kept->size(1) == B && kept->size(2) == cache[1] &&
           kept->size(3) == budget);
  const at::Tensor* evicted = c.none(16) ? nullptr : c.dense(16, at::kInt, 1);
  if (evicted) c.need(evicted->numel() == B);
  size_t bytes;
  void* ws = workspace(c, 17, c.ok ? lib.evict_workspace(&p) : 0, &bytes);
  if (!c.ok) return unsure();
  at::Tensor own_kept, own_evicted;
  if (!kept) own_kept = at::empty({nl, B, cache[1], budget}, refs->options());
  int32_t* kp = (int32_t*)(kept ? kept->data_ptr() : own_kept.data_ptr());
  PyObject* result = a[16];
  int32_t* ep;
  if (evicted) {
    Py_INCREF(result);
    ep = (int32_t*)evicted->data_ptr();
  } else {
    own_evicted = at::empty({B}, refs->options());
    ep = (int32_t*)own_evicted.data_ptr();
    result = THPVariable_Wrap(own_evicted);
  }
  return run(result, [&] {
    return lib.evict(c.ctx, &p, (float* const*)ptr[0].data(), ptr[1].data(), ptr[2].data(),
                     (int64_t*)table->data_ptr(), (int64_t*)lens->data_ptr(),
                     (int32_t*)stack->data_ptr(), (int32_t*)top->data_ptr(),
                     (int32_t*)refs->data_ptr(), ep, kp, ws, bytes);
  });
}

template <PyObject* (*Impl)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return Impl(a);
  } catch (const std::exception&) {
    // (an allocation that fails, a tensor without storage: the caller's own
    // path meets it again and says so)
    return unsure();
  }
}

// (ctx, stream): the status of kyro_ctx_set_stream
PyObject* set_stream(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  kyro_ctx* ctx = (kyro_ctx*)PyLong_AsVoidPtr(a[0]);
  void* stream = PyErr_Occurred() ? nullptr : PyLong_AsVoidPtr(a[1]);
  if (PyErr_Occurred() || !lib.set_stream) return unsure();
  return PyLong_FromLong(lib.set_stream(ctx, stream));
}

// bind: the addresses of the library's entry points, in lib's order
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int kEntries = 8;
  if (n != kEntries) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  void* f[kEntries];
  for (int i = 0; i < kEntries; ++i) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  lib.set_stream = (decltype(lib.set_stream))f[0];
  lib.rope = (decltype(lib.rope))f[1];
  lib.attention = (decltype(lib.attention))f[2];
  lib.attention_workspace = (decltype(lib.attention_workspace))f[3];
  lib.scores = (decltype(lib.scores))f[4];
  lib.scores_workspace = (decltype(lib.scores_workspace))f[5];
  lib.evict = (decltype(lib.evict))f[6];
  lib.evict_workspace = (decltype(lib.evict_workspace))f[7];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
    {"set_stream", (PyCFunction)(void (*)(void))set_stream, METH_FASTCALL, nullptr},
    {"qk_norm_rope_kv_write", (PyCFunction)(void (*)(void))entry<rope_impl, 17>, METH_FASTCALL,
     nullptr},
    {"chunk_attention", (PyCFunction)(void (*)(void))entry<attention_impl, 12>, METH_FASTCALL,
     nullptr},
    {"kv_scores_add", (PyCFunction)(void (*)(void))entry<scores_impl, 12>, METH_FASTCALL, nullptr},
    {"kv_evict", (PyCFunction)(void (*)(void))entry<evict_impl, 18>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pycall", nullptr, -1, methods,
                      nullptr,               nullptr,   nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__pycall(void) { return PyModule_Create(&module); }
