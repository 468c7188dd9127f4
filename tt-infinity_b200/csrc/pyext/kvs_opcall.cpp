/* kvs_opcall.cpp -- CPython entry points of the operators on a paged cache (kvcache_manager.ops).
 *
 * A decode step calls these operators once per layer on work of a few microseconds; checking a dozen
 * tensors and filling the C structs in Python took 25-30 us per call, several times the kernels of a
 * small batch. This module reads the tensors through torch's C++ API, makes the same checks, allocates
 * the outputs and calls the functions of libkvs_b200.so through pointers that the package hands over
 * once (bind), so both bindings use the one loaded library.
 *
 * A call returns NotImplemented for whatever it does not take (a failed check, here or in the library, or
 * a tensor subclass); the caller then takes its ctypes path, which repeats the checks and raises the error
 * with its message. Any other error of the library comes back as its status, an int, for the caller to
 * raise: work may have been enqueued, and repeating it (rows turned in place, weights compacted in place)
 * would change what it reads. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>

#include "kvs.h"

namespace {

int (*g_fill)(const kvs_paged_cache *, const kvs_qkv_rows *, void *);
int (*g_workspace)(const kvs_paged_cache *, const kvs_decode_rows *, int32_t, uint64_t *);
int (*g_attend)(const kvs_paged_cache *, const kvs_decode_rows *, void *);
int (*g_evict)(const kvs_paged_cache *, const kvs_evict_rows *, void *);

// The arguments of one call: tensors on one GPU, of which none needs a gradient or carries a tangent.
struct Call {
  PyObject *const *args;
  c10::Device device{c10::kCPU};
  bool ok = true, grad = c10::GradMode::is_enabled();

  const at::Tensor *tensor(int i, int64_t dims, bool optional = false) {
    PyObject *o = args[i];
    if (o == Py_None && optional) return nullptr;
    if (!THPVariable_CheckExact(o)) return fail();
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.dim() != dims || t.layout() != c10::kStrided || (grad && t.requires_grad()) || t._fw_grad(0).defined())
      return fail();
    if (device.is_cpu()) device = t.device();
    if (t.device() != device) return fail();
    return &t;
  }
  // int32, contiguous
  const at::Tensor *ints(int i, int64_t dims, bool optional = false) {
    const at::Tensor *t = tensor(i, dims, optional);
    if (t && (t->scalar_type() != at::kInt || !t->is_contiguous())) return fail();
    return t;
  }
  // contiguous last dimension
  const at::Tensor *rows(int i, int64_t dims, bool optional = false) {
    const at::Tensor *t = tensor(i, dims, optional);
    if (t && t->size(dims - 1) > 1 && t->stride(dims - 1) != 1) return fail();
    return t;
  }
  double number(int i) {
    const double x = PyFloat_Check(args[i]) ? PyFloat_AS_DOUBLE(args[i]) : PyFloat_AsDouble(args[i]);
    if (x == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return x;
  }
  int64_t integer(int i, int64_t lo, int64_t hi) {
    if (!PyLong_Check(args[i])) {
      ok = false;
      return lo;
    }
    const long long x = PyLong_AsLongLong(args[i]);
    if ((x == -1 && PyErr_Occurred()) || x < lo || x > hi) {
      PyErr_Clear();
      ok = false;
      return lo;
    }
    return x;
  }
  const at::Tensor *fail() {
    ok = false;
    return nullptr;
  }
  void *stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
};

int code_of(at::ScalarType t) {
  return t == at::kBFloat16 ? KVS_DTYPE_BF16 : t == at::kHalf ? KVS_DTYPE_FP16 : t == at::kFloat8_e4m3fn ? KVS_DTYPE_E4M3 : -1;
}

// a dimension of one element has no stride
void strides(const at::Tensor &t, int n, int64_t unit, int64_t *out) {
  for (int i = 0; i < n; ++i) out[i] = t.size(i) > 1 ? t.stride(i) * unit : 0;
}

template <class T>
T *ptr(const at::Tensor *t) {
  return t ? static_cast<T *>(t->data_ptr()) : nullptr;
}

// arguments ik, ik + 1 (the caches) and ip (the page table)
bool cache_of(Call &c, int ik, int ip, int is, kvs_paged_cache *out) {
  const at::Tensor *k = c.rows(ik, 4), *v = c.rows(ik + 1, 4), *table = c.ints(ip, 2);
  if (!c.ok || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type()) return false;
  const int code = code_of(k->scalar_type());
  for (int i = 0; i < 4; ++i)
    if (k->size(i) > INT32_MAX) return false;
  if (code < 0 || table->size(0) > INT32_MAX || table->size(1) > INT32_MAX) return false;
  const int64_t unit = k->element_size();
  out->k = k->data_ptr();
  out->v = v->data_ptr();
  strides(*k, 3, unit, out->k_strides);
  strides(*v, 3, unit, out->v_strides);
  out->page_table = ptr<int32_t>(table);
  out->num_blocks = k->size(0);
  out->n_heads = k->size(1);
  out->block_size = k->size(2);
  out->head_dim = k->size(3);
  out->batch = table->size(0);
  out->max_blocks = table->size(1);
  out->dtype = code;
  out->k_scale = is < 0 ? 1.f : (float)c.number(is);
  out->v_scale = is < 0 ? 1.f : (float)c.number(is + 1);
  return c.ok;
}

// fp32 [batch, heads, at least `cover` tokens] with contiguous rows
bool sums_fit(const at::Tensor &t, int64_t batch, int64_t heads, int64_t cover) {
  return t.scalar_type() == at::kFloat && t.stride(2) == 1 && t.size(0) == batch && t.size(1) == heads && t.size(2) >= cover &&
         t.size(2) <= INT32_MAX;
}

// What a call has written counts as changed, so that autograd refuses a backward pass that saved it
// (tensors made in inference mode keep no count).
void changed(std::initializer_list<const at::Tensor *> written) {
  for (const at::Tensor *t : written)
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

PyObject *not_taken() { Py_RETURN_NOTIMPLEMENTED; }
// KVS_E_INVAL is a check's, before anything is enqueued
PyObject *failed(int rc) { return rc == KVS_E_INVAL ? not_taken() : PyLong_FromLong(rc); }

// A call whose C++ exceptions end here: before the library was called the ctypes path says what was wrong,
// after that nothing is repeated.
template <PyObject *(*call)(PyObject *const *, bool &)>
PyObject *guarded(PyObject *const *args) {
  bool called = false;
  try {
    return call(args, called);
  } catch (const std::exception &e) {
    if (PyErr_Occurred()) PyErr_Clear();
    if (!called) return not_taken();
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// fill(q, k, v, cos_sin, cu_seqlens, page_table, start_positions, cache_k, cache_v, q_weight, k_weight,
//      eps, positions, axes, interleaved, k_scale, v_scale, q_out, out_of_range) -> q_out
PyObject *take_fill(PyObject *const *args, bool &called) {
  Call c{args};
  kvs_paged_cache cache;
  if (!cache_of(c, 7, 5, 15, &cache)) return not_taken();
  const at::Tensor *q = c.rows(0, 3), *k = c.rows(1, 3), *v = c.rows(2, 3), *cs = c.tensor(3, 2), *cu = c.ints(4, 1),
                   *start = c.ints(6, 1), *wq = c.tensor(9, 1, true), *wk = c.tensor(10, 1, true), *axes = c.ints(13, 1, true),
                   *out = c.rows(17, 3, true);
  const at::Tensor *positions = nullptr, *count = nullptr;
  if (args[12] != Py_None) {
    if (!THPVariable_CheckExact(args[12])) return not_taken();
    positions = c.ints(12, THPVariable_Unpack(args[12]).dim() == 2 ? 2 : 1);
  }
  if (args[18] != Py_None) {
    if (!THPVariable_CheckExact(args[18])) return not_taken();
    count = c.tensor(18, THPVariable_Unpack(args[18]).dim());
  }
  if (!c.ok) return not_taken();
  const int64_t tokens = q->size(0), heads = q->size(1), dim = q->size(2);
  const at::ScalarType type = q->scalar_type();
  if (tokens > INT32_MAX / 2 || heads > 65535 || dim != cache.head_dim || k->sizes() != v->sizes() || k->size(0) != tokens ||
      k->size(1) != cache.n_heads || k->size(2) != dim || k->scalar_type() != type || v->scalar_type() != type)
    return not_taken();
  for (const at::Tensor *w : {wq, wk})
    if (w && (w->size(0) != dim || w->scalar_type() != type || !w->is_contiguous())) return not_taken();
  if (cs->scalar_type() != at::kFloat || !cs->is_contiguous() || cs->size(0) > INT32_MAX || cs->size(1) > INT32_MAX) return not_taken();
  if (start->size(0) != cache.batch || cu->size(0) != (int64_t)cache.batch + 1) return not_taken();
  const int64_t n_axes = !positions ? 0 : positions->dim() == 2 ? positions->size(0) : 1;
  if (positions && (positions->size(positions->dim() - 1) != tokens || n_axes < 1)) return not_taken();
  if (axes ? axes->size(0) * 2 != cs->size(1) : n_axes > 1) return not_taken();
  if (n_axes > 32 || (count && (count->scalar_type() != at::kInt || count->numel() < 1))) return not_taken();
  if (out && (out->sizes() != q->sizes() || out->scalar_type() != type)) return not_taken();
  if (!PyBool_Check(args[14])) return not_taken();
  at::Tensor fresh;
  if (!out) fresh = at::empty({tokens, heads, dim}, q->options());
  const at::Tensor &o = out ? *out : fresh;
  kvs_qkv_rows r{};
  r.q = q->data_ptr(), r.k = k->data_ptr(), r.v = v->data_ptr(), r.q_out = o.data_ptr();
  strides(*q, 2, 2, r.q_strides);
  strides(*k, 2, 2, r.k_strides);
  strides(*v, 2, 2, r.v_strides);
  strides(o, 2, 2, r.q_out_strides);
  r.cos_sin = ptr<float>(cs), r.cu_seqlens = ptr<int32_t>(cu), r.start_positions = ptr<int32_t>(start);
  r.positions = ptr<int32_t>(positions), r.axes = ptr<int32_t>(axes), r.q_weight = ptr<void>(wq), r.k_weight = ptr<void>(wk);
  r.out_of_range = ptr<uint32_t>(count);
  r.n_tokens = tokens, r.q_heads = heads, r.rotary = cs->size(1), r.n_positions = cs->size(0), r.n_axes = n_axes;
  r.dtype = code_of(type), r.eps = (float)c.number(11), r.interleaved = args[14] == Py_True, r.zero_rest = !out;
  if (!c.ok) return not_taken();
  void *stream = c.stream();
  int rc;
  called = true;
  Py_BEGIN_ALLOW_THREADS
  rc = g_fill(&cache, &r, stream);
  Py_END_ALLOW_THREADS
  if (rc != KVS_OK) return failed(rc);
  changed({&THPVariable_Unpack(args[7]), &THPVariable_Unpack(args[8]), out, count});
  if (out) {
    Py_INCREF(args[17]);
    return args[17];
  }
  return THPVariable_Wrap(fresh);
}
PyObject *fill(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return n == 19 && g_fill ? guarded<take_fill>(args) : not_taken();
}

// attend(q, cache_k, cache_v, page_table, seq_lens, scale, window, k_scale, v_scale, out, return_lse, weights,
//        weights_out) -> out or (out, lse)
PyObject *take_attend(PyObject *const *args, bool &called) {
  Call c{args};
  kvs_paged_cache cache;
  if (!cache_of(c, 1, 3, 7, &cache)) return not_taken();
  const at::Tensor *q = c.rows(0, 3), *lens = c.ints(4, 1), *out = c.rows(9, 3, true), *w = c.tensor(11, 3, true),
                   *wo = c.tensor(12, 3, true);
  const int64_t window = args[6] == Py_None ? 0 : c.integer(6, 1, INT32_MAX);
  if (!c.ok || !PyBool_Check(args[10])) return not_taken();
  const int64_t batch = q->size(0), heads = q->size(1), dim = q->size(2);
  if (batch != cache.batch || dim != cache.head_dim || heads > INT32_MAX || lens->size(0) != batch || (wo && !w)) return not_taken();
  if (out && (out->sizes() != q->sizes() || out->scalar_type() != q->scalar_type())) return not_taken();
  if (w && !wo) wo = w;
  const int64_t cover = (int64_t)cache.max_blocks * cache.block_size;
  if (w && !(sums_fit(*w, batch, cache.n_heads, cover) && sums_fit(*wo, batch, cache.n_heads, cover))) return not_taken();
  kvs_decode_rows r{};
  at::Tensor fresh, lse;
  if (!out) fresh = at::empty({batch, heads, dim}, q->options());
  const at::Tensor &o = out ? *out : fresh;
  r.q = q->data_ptr(), r.out = o.data_ptr();
  strides(*q, 2, 2, r.q_strides);
  strides(o, 2, 2, r.out_strides);
  r.seq_lens = ptr<int32_t>(lens);
  if (args[10] == Py_True) {
    lse = at::empty({batch, heads}, q->options().dtype(at::kFloat));
    r.lse = static_cast<float *>(lse.data_ptr());
  }
  if (w) {
    r.weights = ptr<float>(w), r.weights_out = ptr<float>(wo);
    strides(*w, 2, 1, r.weights_strides);
    strides(*wo, 2, 1, r.weights_out_strides);
    r.w_len = std::min(w->size(2), wo->size(2));
  }
  r.q_heads = heads, r.window = window, r.dtype = code_of(q->scalar_type());
  r.scale = args[5] == Py_None ? (float)(1.0 / std::sqrt((double)dim)) : (float)c.number(5);
  if (!c.ok) return not_taken();
  if (const int bad = g_workspace(&cache, &r, c.device.index(), &r.workspace_bytes)) return failed(bad);
  const at::Tensor workspace = at::empty({(int64_t)r.workspace_bytes}, q->options().dtype(at::kByte));
  r.workspace = workspace.data_ptr();
  void *stream = c.stream();
  int rc;
  called = true;
  Py_BEGIN_ALLOW_THREADS
  rc = g_attend(&cache, &r, stream);
  Py_END_ALLOW_THREADS
  if (rc != KVS_OK) return failed(rc);
  changed({out, wo});
  PyObject *result;
  if (out) {
    Py_INCREF(args[9]);
    result = args[9];
  } else {
    result = THPVariable_Wrap(fresh);
  }
  if (!r.lse || !result) return result;
  PyObject *second = THPVariable_Wrap(lse);
  PyObject *both = second ? PyTuple_Pack(2, result, second) : nullptr;
  Py_DECREF(result);
  Py_XDECREF(second);
  return both;
}
PyObject *attend(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return n == 13 && g_attend ? guarded<take_attend>(args) : not_taken();
}

// evict(cache_k, cache_v, page_table, seq_lens, weights, keep, first, recent, dst_page_table, weights_out,
//       out_of_range) -> (kept, new_lens)
PyObject *take_evict(PyObject *const *args, bool &called) {
  Call c{args};
  kvs_paged_cache cache;
  if (!cache_of(c, 0, 2, -1, &cache)) return not_taken();
  const at::Tensor *lens = c.ints(3, 1), *w = c.tensor(4, 3), *dst = c.ints(8, 2, true), *wo = c.tensor(9, 3, true);
  const at::Tensor *count = nullptr;
  if (args[10] != Py_None) {
    if (!THPVariable_CheckExact(args[10])) return not_taken();
    count = c.tensor(10, THPVariable_Unpack(args[10]).dim());
  }
  const int64_t keep = c.integer(5, 1, INT32_MAX), first = c.integer(6, 0, INT32_MAX), recent = c.integer(7, 0, INT32_MAX);
  if (!c.ok || first + recent > keep) return not_taken();
  if (!wo) wo = w;
  const int64_t batch = cache.batch, heads = cache.n_heads, cover = (int64_t)cache.max_blocks * cache.block_size;
  if (lens->size(0) != batch || (dst && (dst->size(0) != batch || dst->size(1) < 1 || dst->size(1) > INT32_MAX)) || !sums_fit(*w, batch, heads, cover) ||
      !sums_fit(*wo, batch, heads, cover) || (count && (count->scalar_type() != at::kInt || count->numel() < 1)))
    return not_taken();
  const at::Tensor kept = at::empty({batch, heads, keep}, lens->options()), fresh = at::empty({batch}, lens->options());
  kvs_evict_rows r{};
  r.seq_lens = ptr<int32_t>(lens), r.dst_table = ptr<int32_t>(dst);
  r.weights = ptr<float>(w), r.weights_out = ptr<float>(wo);
  strides(*w, 2, 1, r.weights_strides);
  strides(*wo, 2, 1, r.weights_out_strides);
  r.kept = static_cast<int32_t *>(kept.data_ptr()), r.new_lens = static_cast<int32_t *>(fresh.data_ptr());
  r.out_of_range = ptr<uint32_t>(count);
  r.dst_blocks = dst ? dst->size(1) : 0, r.w_len = w->size(2), r.wo_len = wo->size(2);
  r.keep = keep, r.first = first, r.recent = recent;
  void *stream = c.stream();
  int rc;
  called = true;
  Py_BEGIN_ALLOW_THREADS
  rc = g_evict(&cache, &r, stream);
  Py_END_ALLOW_THREADS
  if (rc != KVS_OK) return failed(rc);
  changed({&THPVariable_Unpack(args[0]), &THPVariable_Unpack(args[1]), wo, count});
  PyObject *a = THPVariable_Wrap(kept), *b = a ? THPVariable_Wrap(fresh) : nullptr;
  PyObject *both = b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return both;
}
PyObject *evict(PyObject *, PyObject *const *args, Py_ssize_t n) {
  return n == 11 && g_evict ? guarded<take_evict>(args) : not_taken();
}

PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long f, w, a, e;
  if (!PyArg_ParseTuple(args, "KKKK", &f, &w, &a, &e)) return nullptr;
  g_fill = reinterpret_cast<decltype(g_fill)>((uintptr_t)f);
  g_workspace = reinterpret_cast<decltype(g_workspace)>((uintptr_t)w);
  g_attend = reinterpret_cast<decltype(g_attend)>((uintptr_t)a);
  g_evict = reinterpret_cast<decltype(g_evict)>((uintptr_t)e);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"bind", bind, METH_VARARGS, "Addresses of the library's entry points."},
    {"fill", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fill)), METH_FASTCALL, "qk_norm_rope_fill"},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, "paged_decode_attention"},
    {"evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(evict)), METH_FASTCALL, "evict_paged_kv"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_opcall", "Compiled entry of the operators on a paged cache.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__opcall(void) { return PyModule_Create(&kModule); }
