// pa_host.cpp — the usual calls of the extended operators, from Python objects to
// the C ABI in one step (a CPython extension over torch's C++ tensors).
//
// Reading some sixty tensor attributes and filling the argument structures through
// ctypes takes a call 20 to 25 us of host time, several times a small call's device
// time; here it takes 1 to 2.  A function below launches only when every argument is
// exactly what the kernels take; otherwise it returns None and the Python caller
// goes the long way, which converts, explains and raises.  So the checks' meaning
// and every message stand in one place, in Python.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <utility>

#include "../../include/paged_attention_b200.h"

namespace {

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool on(const at::Tensor& t, c10::Device dev) { return t.device() == dev; }

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PA_DTYPE_FLOAT32;
    case at::kHalf: return PA_DTYPE_FLOAT16;
    case at::kBFloat16: return PA_DTYPE_BFLOAT16;
    default: return -1;
  }
}

pa_cache_view view_of(const at::Tensor& t) {
  return {t.data_ptr(), t.size(0), t.stride(0), t.stride(1), t.stride(2)};
}

// The caches of one layer, as the Python checks want them.
bool caches_ok(const at::Tensor& k, const at::Tensor& v) {
  return k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() &&
         k.stride(3) == 1 && v.stride(3) == 1 && k.is_cuda() && v.device() == k.device();
}

bool scales_ok(const at::Tensor& s, const at::Tensor& cache) {
  return s.dim() == 2 && s.size(0) == cache.size(0) && s.size(1) == cache.size(1) && s.scalar_type() == at::kFloat &&
         s.device() == cache.device();
}

bool rows_ok(const at::Tensor& t, int64_t B, int64_t H, int64_t q, int64_t D, c10::Device dev) {
  return t.dim() == 4 && t.size(0) == B && t.size(1) == H && t.size(2) == q && t.size(3) == D && t.stride(3) == 1 &&
         on(t, dev) && dtype_code(t.scalar_type()) >= 0;
}

bool int32_vector(const at::Tensor& t, int64_t n, c10::Device dev) {
  return t.dim() == 1 && t.numel() == n && t.scalar_type() == at::kInt && on(t, dev) && t.is_contiguous();
}

bool tables_ok(const at::Tensor& t, int64_t B, c10::Device dev) {
  return t.dim() == 2 && t.size(0) == B && t.size(1) > 0 && t.stride(1) == 1 && t.scalar_type() == at::kInt &&
         on(t, dev);
}

bool is_current(c10::Device dev) { return c10::cuda::current_device() == dev.index(); }

bool capturing() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }

void* stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

PyObject* none() { Py_RETURN_NONE; }

pa_cache_scales scales_of(const at::Tensor& ks, const at::Tensor& vs) {
  return {static_cast<float*>(ks.data_ptr()), ks.stride(0), ks.stride(1),
          static_cast<float*>(vs.data_ptr()), vs.stride(0), vs.stride(1)};
}

void set_rows(pa_kv_append_args& a, const at::Tensor& key, const at::Tensor& value) {
  a.key = key.data_ptr();
  a.key_stride_b = key.stride(0), a.key_stride_h = key.stride(1), a.key_stride_t = key.stride(2);
  a.value = value.data_ptr();
  a.value_stride_b = value.stride(0), a.value_stride_h = value.stride(1), a.value_stride_t = value.stride(2);
}

// Fills and launches an append; false when an argument is not the kernels'.
bool append(const at::Tensor& key, const at::Tensor& value, const at::Tensor& kc, const at::Tensor& vc,
            const pa_cache_scales* sc, const at::Tensor* slots, const at::Tensor* tables, const at::Tensor* positions,
            int64_t position_offset, void* word, void* stream) {
  const auto dev = kc.device();
  const int64_t B = key.dim() == 4 ? key.size(0) : 0, q = key.dim() == 4 ? key.size(2) : 0;
  if (B <= 0 || q <= 0 || !rows_ok(key, B, kc.size(1), q, kc.size(3), dev) ||
      !rows_ok(value, B, kc.size(1), q, kc.size(3), dev) || key.scalar_type() != value.scalar_type() ||
      (sc == nullptr && key.scalar_type() != kc.scalar_type()))
    return false;
  pa_kv_append_args a = {};
  set_rows(a, key, value);
  a.key_cache = view_of(kc);
  a.value_cache = view_of(vc);
  if (slots != nullptr) {
    if (slots->scalar_type() != at::kLong || !on(*slots, dev) || slots->numel() != B * q || !slots->is_contiguous())
      return false;
    a.slot_mapping = static_cast<const int64_t*>(slots->data_ptr());
  } else {
    if (tables == nullptr || positions == nullptr || !tables_ok(*tables, B, dev)) return false;
    const auto pt = positions->scalar_type();
    if ((pt != at::kInt && pt != at::kLong) || !on(*positions, dev) || positions->numel() != B ||
        !positions->is_contiguous())
      return false;
    a.block_tables = static_cast<const int32_t*>(tables->data_ptr());
    a.block_table_stride = tables->stride(0);
    a.max_blocks = static_cast<int32_t>(tables->size(1));
    a.positions = positions->data_ptr();
    a.positions_is_int64 = pt == at::kLong;
    a.position_offset = static_cast<int32_t>(position_offset);
  }
  a.batch = B, a.q_len = q, a.num_kv_heads = kc.size(1), a.head_dim = kc.size(3), a.block_size = kc.size(2);
  a.dtype = dtype_code(key.scalar_type());
  a.error_flags = static_cast<uint32_t*>(word);
  return (sc != nullptr ? pa_kv_append_8bit(&a, sc, stream) : pa_kv_append(&a, stream)) == PA_OK;
}

bool long_arg(PyObject* o, int64_t* out) {
  *out = PyLong_AsLongLong(o);
  if (*out == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool word_is_set(void* word) { return *static_cast<volatile uint32_t*>(word) != 0; }

// append8(key, value, key_cache, value_cache, key_scales, value_scales, slots | None, tables | None,
//         positions | None, position_offset, word) -> True | None
PyObject* py_append8(PyObject*, PyObject* const* o, Py_ssize_t n) {
  if (n != 11) return none();
  const at::Tensor* t[6];
  for (int i = 0; i < 6; ++i)
    if ((t[i] = tensor(o[i])) == nullptr) return none();
  int64_t offset, word;
  if (!long_arg(o[9], &offset) || !long_arg(o[10], &word) || word_is_set(reinterpret_cast<void*>(word))) return none();
  const at::Tensor &kc = *t[2], &vc = *t[3];
  if (!caches_ok(kc, vc) || kc.scalar_type() != at::kFloat8_e4m3fn || !scales_ok(*t[4], kc) || !scales_ok(*t[5], vc) ||
      !is_current(kc.device()))
    return none();
  const pa_cache_scales sc = scales_of(*t[4], *t[5]);
  const at::Tensor* slots = o[6] == Py_None ? nullptr : tensor(o[6]);
  if (o[6] != Py_None && slots == nullptr) return none();
  if (!append(*t[0], *t[1], kc, vc, &sc, slots, tensor(o[7]), tensor(o[8]), offset, reinterpret_cast<void*>(word),
              stream_of(kc.device())))
    return none();
  Py_RETURN_TRUE;
}

// decode(query, key_cache, value_cache, tables, lens, scale, slots, key, value, out, include_new, key_scales,
//        value_scales, modifiers, workspace, word, weights, n_weights) -> out | None
// modifiers: None or (softcap, window, alibi_slopes, key_starts, prefix_lens).  A call that is being captured
// goes the long way, which notes that a graph holds the workspace.
PyObject* py_decode(PyObject*, PyObject* const* o, Py_ssize_t n) {
  if (n != 18) return none();
  const at::Tensor *pq = tensor(o[0]), *pk = tensor(o[1]), *pv = tensor(o[2]), *pt = tensor(o[3]), *pl = tensor(o[4]);
  const at::Tensor* ws = tensor(o[14]);
  if (!pq || !pk || !pv || !pt || !pl || !ws) return none();
  const at::Tensor &query = *pq, &kc = *pk, &vc = *pv, &tables = *pt, &lens = *pl;
  int64_t word, weights, n_weights;
  if (!long_arg(o[15], &word) || !long_arg(o[16], &weights) || !long_arg(o[17], &n_weights)) return none();
  void* flags = reinterpret_cast<void*>(word);
  if (word_is_set(flags) || !caches_ok(kc, vc) || query.dim() != 4) return none();
  const auto dev = kc.device();
  const int64_t B = query.size(0), Hq = query.size(1), q = query.size(2), D = query.size(3);
  const int64_t Hkv = kc.size(1);
  const int code = dtype_code(query.scalar_type());
  if (B <= 0 || q <= 0 || code < 0 || D != kc.size(3) || !on(query, dev) || query.stride(3) != 1 || Hkv <= 0 ||
      Hq % Hkv != 0 || !tables_ok(tables, B, dev) || !int32_vector(lens, B, dev) || !is_current(dev) || capturing())
    return none();
  const double scale = PyFloat_AsDouble(o[5]);
  if (scale == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  pa_cache_scales sc;
  const bool eight = kc.scalar_type() == at::kFloat8_e4m3fn;
  if (eight) {
    const at::Tensor *ks = tensor(o[11]), *vs = tensor(o[12]);
    if (!ks || !vs || code == PA_DTYPE_FLOAT32 || !scales_ok(*ks, kc) || !scales_ok(*vs, vc)) return none();
    sc = scales_of(*ks, *vs);
  } else if (o[11] != Py_None || o[12] != Py_None || query.scalar_type() != kc.scalar_type()) {
    return none();
  }
  pa_score_modifiers sm = {};
  const bool scored = o[13] != Py_None;
  if (scored) {
    if (!PyTuple_Check(o[13]) || PyTuple_GET_SIZE(o[13]) != 5) return none();
    PyObject* m[5];
    for (int i = 0; i < 5; ++i) m[i] = PyTuple_GET_ITEM(o[13], i);
    const double cap = PyFloat_AsDouble(m[0]);
    int64_t window;
    if ((cap == -1.0 && PyErr_Occurred()) || !(cap == 0.0 || (cap > 1e-30 && cap < 1e30))) {
      PyErr_Clear();
      return none();
    }
    if (!long_arg(m[1], &window) || window < 0 || window >= (int64_t(1) << 31)) return none();
    sm.softcap = static_cast<float>(cap);
    sm.window = static_cast<int32_t>(window);
    if (m[2] != Py_None) {
      const at::Tensor* s = tensor(m[2]);
      if (!s || s->dim() != 1 || s->size(0) != Hq || s->scalar_type() != at::kFloat || !on(*s, dev) ||
          !s->is_contiguous())
        return none();
      sm.alibi_slopes = static_cast<const float*>(s->data_ptr());
    }
    if (m[3] != Py_None) {
      const at::Tensor* s = tensor(m[3]);
      if (!s || s->scalar_type() != at::kInt || !on(*s, dev) || s->dim() < 1 || s->dim() > 2 || s->size(0) != B ||
          (s->dim() == 2 && s->size(1) != q))
        return none();
      sm.key_starts = static_cast<const int32_t*>(s->data_ptr());
      sm.key_starts_stride_b = s->stride(0);
      sm.key_starts_stride_t = s->dim() == 2 ? s->stride(1) : 0;
    }
    if (m[4] != Py_None) {
      const at::Tensor* s = tensor(m[4]);
      if (!s || !int32_vector(*s, B, dev)) return none();
      sm.prefix_lens = static_cast<const int32_t*>(s->data_ptr());
    }
  }
  if (!eight && !scored) return none();
  const int include_new = PyObject_IsTrue(o[10]);
  const size_t need = pa_decode_ext_workspace_bytes(B, Hq, Hkv, q, D, code, dev.index());
  if (need == 0 || static_cast<size_t>(ws->numel()) < need || !on(*ws, dev)) return none();
  const at::Tensor *key = tensor(o[7]), *value = tensor(o[8]), *slots = tensor(o[6]);
  if ((o[7] != Py_None && !key) || (o[8] != Py_None && !value) || (o[6] != Py_None && !slots) ||
      (key == nullptr) != (value == nullptr) || (slots != nullptr && key == nullptr))
    return none();
  at::Tensor out;
  const at::Tensor* given = nullptr;
  if (o[9] != Py_None) {
    given = tensor(o[9]);
    if (!given || given->dim() != 4 || given->sizes() != query.sizes() ||
        given->scalar_type() != query.scalar_type() || !on(*given, dev) || given->stride(3) != 1)
      return none();
    out = *given;
  } else {
    out = at::empty(query.sizes(), query.options().memory_format(at::MemoryFormat::Contiguous));
  }
  void* stream = stream_of(dev);
  if (key != nullptr && (key->dim() != 4 || key->size(0) != B || key->size(2) != q ||
                         !append(*key, *value, kc, vc, eight ? &sc : nullptr, slots, &tables, &lens,
                                 include_new ? -q : 0, flags, stream)))
    return none();
  pa_decode_args a = {};
  a.query = query.data_ptr();
  a.query_stride_b = query.stride(0), a.query_stride_h = query.stride(1), a.query_stride_t = query.stride(2);
  a.key_cache = view_of(kc);
  a.value_cache = view_of(vc);
  a.block_tables = static_cast<const int32_t*>(tables.data_ptr());
  a.block_table_stride = tables.stride(0);
  a.max_blocks = static_cast<int32_t>(tables.size(1));
  a.context_lens = static_cast<const int32_t*>(lens.data_ptr());
  a.len_offset = include_new ? 0 : static_cast<int32_t>(q);
  a.out = out.data_ptr();
  a.out_stride_b = out.stride(0), a.out_stride_h = out.stride(1), a.out_stride_t = out.stride(2);
  a.batch = B, a.q_len = q, a.num_q_heads = Hq, a.num_kv_heads = Hkv, a.head_dim = D, a.block_size = kc.size(2);
  a.dtype = code;
  a.scale = static_cast<float>(scale);
  a.workspace = ws->data_ptr();
  a.workspace_bytes = ws->numel();
  a.allow_overlap_with_previous = key != nullptr;
  a.sm_weights = n_weights > 0 ? reinterpret_cast<const float*>(weights) : nullptr;
  a.num_sm_weights = static_cast<int32_t>(n_weights);
  if (pa_decode_ext(&a, eight ? &sc : nullptr, scored ? &sm : nullptr, static_cast<uint32_t*>(flags), stream) != PA_OK)
    return none();
  if (given != nullptr) {
    Py_INCREF(o[9]);
    return o[9];
  }
  return THPVariable_Wrap(out);
}

// The pages t[i] of a cache as equal runs of bytes (device_pages._view).
bool page_view(const at::Tensor& t, pa_page_view* v) {
  const int64_t e = t.element_size();
  std::pair<int64_t, int64_t> dims[16];  // stride, size
  int nd = 0;
  if (t.dim() < 1 || t.dim() > 16) return false;
  for (int64_t i = 1; i < t.dim(); ++i) {
    if (t.size(i) == 1) continue;
    if (t.stride(i) == 0) return false;
    dims[nd++] = {t.stride(i), t.size(i)};
  }
  std::sort(dims, dims + nd);
  int64_t run = 1, segments = 1, stride = 0;
  bool strided = false;
  for (int i = 0; i < nd; ++i) {
    if (!strided && dims[i].first == run) {
      run *= dims[i].second;
    } else if (strided && dims[i].first == segments * stride) {
      segments *= dims[i].second;
    } else if (!strided) {
      strided = true;
      stride = dims[i].first;
      segments = dims[i].second;
    } else {
      return false;
    }
  }
  // pages one after the other, or interleaved with one another's runs: no byte twice
  std::pair<int64_t, int64_t> levels[2] = {{t.stride(0), t.size(0)}, {stride, segments}};
  std::sort(levels, levels + 2);
  int64_t extent = run;
  for (const auto& l : levels) {
    if (l.second <= 1) continue;
    if (l.first < extent) return false;
    extent += (l.second - 1) * l.first;
  }
  *v = {t.data_ptr(), t.stride(0) * e, segments, stride * e, run * e};
  return true;
}

// Caches of a call; -1 when one is not the kernels'.  num_blocks and dev are taken from the first when unset.
int page_views(PyObject* caches, pa_page_view* v, int64_t* num_blocks, c10::Device* dev, bool* known) {
  if (!PyList_Check(caches) && !PyTuple_Check(caches)) return -1;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(caches);
  if (n > PA_MAX_PAGE_VIEWS) return -1;
  PyObject** items = PySequence_Fast_ITEMS(caches);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t = tensor(items[i]);
    if (!t || t->dim() < 1 || !t->is_cuda() || t->numel() == 0) return -1;
    if (!*known) {
      *num_blocks = t->size(0);
      *dev = t->device();
      *known = true;
    }
    if (t->size(0) != *num_blocks || t->device() != *dev || !page_view(*t, &v[i])) return -1;
  }
  return static_cast<int>(n);
}

bool ids_ok(const at::Tensor* t, c10::Device dev) {
  return t != nullptr && t->dim() == 1 && t->scalar_type() == at::kInt && on(*t, dev) && t->is_contiguous();
}

// copy_pages(caches, src, dst, word) -> True | None
PyObject* py_copy_pages(PyObject*, PyObject* const* o, Py_ssize_t n) {
  if (n != 4) return none();
  int64_t word, num_blocks = 0;
  c10::Device dev(c10::kCUDA, 0);
  bool known = false;
  pa_page_view v[PA_MAX_PAGE_VIEWS];
  const int nv = page_views(o[0], v, &num_blocks, &dev, &known);
  const at::Tensor *src = tensor(o[1]), *dst = tensor(o[2]);
  if (nv <= 0 || !long_arg(o[3], &word) || word_is_set(reinterpret_cast<void*>(word)) || !is_current(dev) ||
      !ids_ok(src, dev) || !ids_ok(dst, dev) || src->numel() != dst->numel() || src->numel() >= (int64_t(1) << 31) ||
      num_blocks >= (int64_t(1) << 31))
    return none();
  if (pa_pages_copy(v, nv, num_blocks, static_cast<const int32_t*>(src->data_ptr()),
                    static_cast<const int32_t*>(dst->data_ptr()), src->numel(), reinterpret_cast<uint32_t*>(word),
                    stream_of(dev)) != PA_OK)
    return none();
  Py_RETURN_TRUE;
}

// pages(op, tables, lens, refs, block_size, scratch, word, a, b, caches) -> True (compact: live) | None
// op 0: free(a), 1: fork(a -> b, caches), 2: reserve(a, b tokens), 3: compact(caches).  The object's own tensors
// were checked when it was made.
PyObject* py_pages(PyObject*, PyObject* const* o, Py_ssize_t n) {
  if (n != 10) return none();
  int64_t op, bs, word;
  const at::Tensor *t = tensor(o[1]), *lens = tensor(o[2]), *refs = tensor(o[3]), *scratch = tensor(o[5]);
  if (!t || !lens || !refs || !scratch || !long_arg(o[0], &op) || !long_arg(o[4], &bs) || !long_arg(o[6], &word) ||
      word_is_set(reinterpret_cast<void*>(word)))
    return none();
  c10::Device dev = t->device();
  if (!is_current(dev)) return none();
  pa_page_tables a = {};
  a.block_tables = static_cast<int32_t*>(t->data_ptr());
  a.block_table_stride = std::max(t->stride(0), t->size(1));
  a.num_seqs = t->size(0), a.max_blocks = t->size(1);
  a.seq_lens = static_cast<int32_t*>(lens->data_ptr());
  a.ref_counts = static_cast<int32_t*>(refs->data_ptr());
  a.num_blocks = refs->numel(), a.block_size = bs;
  a.scratch = static_cast<int32_t*>(scratch->data_ptr());
  a.error_flags = reinterpret_cast<uint32_t*>(word);
  const at::Tensor *x = tensor(o[7]), *y = tensor(o[8]);
  if (op != 3 && (!ids_ok(x, dev) || x->numel() > a.num_seqs)) return none();
  if ((op == 1 || op == 2) && (!ids_ok(y, dev) || y->numel() != x->numel())) return none();
  pa_page_view v[PA_MAX_PAGE_VIEWS];
  int64_t num_blocks = a.num_blocks;
  bool known = true;
  int nv = 0;
  if ((op == 1 || op == 3) && (nv = page_views(o[9], v, &num_blocks, &dev, &known)) < 0) return none();
  void* stream = stream_of(dev);
  const int32_t* xi = x ? static_cast<const int32_t*>(x->data_ptr()) : nullptr;
  const int32_t* yi = y ? static_cast<const int32_t*>(y->data_ptr()) : nullptr;
  int rc = PA_ERR_INVALID_ARGUMENT;
  if (op == 0) rc = pa_pages_free(&a, xi, x->numel(), stream);
  if (op == 1) rc = pa_pages_fork(&a, xi, yi, x->numel(), v, nv, stream);
  if (op == 2) rc = pa_pages_reserve(&a, xi, yi, x->numel(), stream);
  if (op == 3) {
    at::Tensor live = at::empty({1}, refs->options());
    if (pa_pages_compact(&a, v, nv, static_cast<int32_t*>(live.data_ptr()), stream) != PA_OK) return none();
    return THPVariable_Wrap(live);
  }
  if (rc != PA_OK) return none();
  Py_RETURN_TRUE;
}

// C++ exceptions (an allocation that fails, say) become Python's.
template <PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* o, Py_ssize_t n) {
  try {
    return f(self, o, n);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

template <PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<f>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<py_append8>("append8"), method<py_decode>("decode"),
                         method<py_copy_pages>("copy_pages"), method<py_pages>("pages"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "pa_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_pa_host() { return PyModule_Create(&module); }
