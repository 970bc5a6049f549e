// CPython binding of the operators' common calls: reads the torch tensors'
// addresses, sizes and strides in C++ and calls libkvx. It takes only calls
// that are valid as they stand; for anything else (other argument types, a
// failed check, tensors without storage) a function returns None and queues
// nothing, and the Python operator then makes its checks one by one, raising
// or handling what it finds. Otherwise it returns libkvx's status.
//
// Why: an eager call from Python through ctypes is bound by the host. On the
// MI355X boxes store_kvcache took 7.1 us a call, 4.1 of them in the C call
// (of which ctypes took about 1.2) and 2.9 in Python's argument checks, while
// its kernel runs for 2.3 us at decode sizes.

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <type_traits>
#include <vector>

#include "kvx.h"

namespace {

// libkvx's entry points, set by bind() from the library Python has loaded and
// whose version it has checked.
decltype(&kvx_store_kvcache) store_fn = nullptr;
decltype(&kvx_save_blocks) save_fn = nullptr;
decltype(&kvx_restore_blocks) restore_fn = nullptr;
decltype(&kvx_entry_layout) entry_layout_fn = nullptr;
decltype(&kvx_rotary_embed) rotary_fn = nullptr;
decltype(&kvx_store_kvcache_fp8) store_fp8_fn = nullptr;
decltype(&kvx_attention_fp8_workspace) workspace_fn = nullptr;
decltype(&kvx_attention_fp8) attention_fn = nullptr;
decltype(&kvx_attention_weights_fp8) weights_fn = nullptr;
decltype(&kvx_select_tokens) select_fn = nullptr;
decltype(&kvx_compact_kvcache_fp8) compact_fn = nullptr;

const at::Tensor* tensor_of(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;  // subclasses may redefine what a tensor is
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.unsafeGetTensorImpl()->has_storage() ? &t
                                                                                                          : nullptr;
}

bool fits32(int64_t v) { return v >= 0 && v <= INT32_MAX; }

void* stream_of(const at::Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int scale_code(at::ScalarType t) {
  return t == at::kBFloat16 ? KVX_SCALE_BF16 : t == at::kFloat ? KVX_SCALE_FP32 : -1;
}

// Lets other Python threads run for the scope's lifetime, also if it is left by an exception.
class WithoutGil {
 public:
  WithoutGil() : state_(PyEval_SaveThread()) {}
  ~WithoutGil() { PyEval_RestoreThread(state_); }

 private:
  PyThreadState* state_;
};

// Runs `call` (a libkvx status) without the GIL: a launch may block on a full queue.
template <typename F>
PyObject* status(F call) {
  int rc;
  {
    WithoutGil released;
    rc = call();
  }
  return PyLong_FromLong(rc);
}

template <typename F>
PyObject* guarded(F body) {
  try {
    if (PyObject* r = body()) return r;
  } catch (const std::exception&) {
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

// store(key, value, k_cache, v_cache, slot_mapping)
PyObject* store(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 5 || !store_fn) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    const at::Tensor* t[5];
    for (int i = 0; i < 5; ++i)
      if (!(t[i] = tensor_of(args[i])) || t[i]->device() != t[0]->device()) return nullptr;
    const at::Tensor &key = *t[0], &value = *t[1], &kc = *t[2], &vc = *t[3], &slots = *t[4];
    if (key.dim() != 3 || kc.dim() < 2 || vc.dim() < 2 || key.sizes() != value.sizes()) return nullptr;
    const int64_t n = key.size(0), heads = key.size(1), hd = key.size(2), row = heads * hd;
    if (n <= 0 || row <= 0 || !fits32(heads) || !fits32(hd)) return nullptr;
    if (key.stride(2) != 1 || value.stride(2) != 1 || key.stride(1) != hd || value.stride(1) != hd) return nullptr;
    if (kc.stride(1) != row || vc.stride(1) != row || slots.numel() != n) return nullptr;
    if (key.scalar_type() != value.scalar_type() || key.scalar_type() != kc.scalar_type() ||
        key.scalar_type() != vc.scalar_type() || slots.scalar_type() != at::kInt)
      return nullptr;
    if (!kc.is_contiguous() || !vc.is_contiguous() || kc.numel() != vc.numel() || !slots.is_contiguous()) return nullptr;
    const void *k = key.mutable_data_ptr(), *v = value.mutable_data_ptr(), *s = slots.mutable_data_ptr();
    void *kd = kc.mutable_data_ptr(), *vd = vc.mutable_data_ptr();
    const int64_t ks = key.stride(0), vs = value.stride(0), cache_slots = kc.numel() / row;
    const int32_t es = (int32_t)key.element_size();
    void* stream = stream_of(key);
    return status([&] {
      return store_fn(k, ks, v, vs, kd, vd, (const int32_t*)s, n, (int32_t)heads, (int32_t)hd, es, cache_slots, stream);
    });
  });
}

// codec(save, values, payload, scale): values whose leading dims are one uniformly strided run of planes.
PyObject* codec(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4 || !save_fn || !restore_fn) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    const bool save = args[0] == Py_True;
    const at::Tensor* t[3];
    for (int i = 0; i < 3; ++i)
      if (!(t[i] = tensor_of(args[1 + i])) || t[i]->device() != t[0]->device()) return nullptr;
    const at::Tensor &x = *t[0], &payload = *t[1], &scale = *t[2];
    const int64_t dims = x.dim(), scales = scale_code(scale.scalar_type());
    if (dims < 1 || x.scalar_type() != at::kBFloat16 || payload.scalar_type() != at::kFloat8_e4m3fn || scales < 0)
      return nullptr;
    if (payload.sizes() != x.sizes() || !payload.is_contiguous() || !scale.is_contiguous() || scale.dim() != dims ||
        scale.size(dims - 1) != 1 || scale.sizes().slice(0, dims - 1) != x.sizes().slice(0, dims - 1))
      return nullptr;
    const int64_t hd = x.size(dims - 1);
    if (x.numel() == 0 || x.stride(dims - 1) != 1) return nullptr;
    // The longest run of trailing dims packed back to back are rows; the dims before them must be one strided run.
    int64_t i = dims - 2, rows = 1;
    for (; i >= 0 && (x.size(i) == 1 || x.stride(i) == rows * hd); --i) rows *= x.size(i);
    int64_t planes = 1, plane_stride = rows * hd;
    for (bool first = true; i >= 0; --i) {
      if (x.size(i) == 1) continue;
      if (first) plane_stride = x.stride(i);
      else if (x.stride(i) != plane_stride * planes) return nullptr;
      first = false;
      planes *= x.size(i);
    }
    if (!fits32(rows) || !fits32(planes) || !fits32(hd)) return nullptr;
    const kvx_block_layout layout{plane_stride, 0, (int32_t)planes, (int32_t)rows, (int32_t)hd, 1, 2, (int32_t)scales};
    void* values = x.mutable_data_ptr();
    const uint64_t entry = (uint64_t)(uintptr_t)payload.mutable_data_ptr();
    const int64_t offset = (int64_t)((uint64_t)(uintptr_t)scale.mutable_data_ptr() - entry);
    const int32_t id = 0;
    void* stream = stream_of(x);
    return status([&] {
      return save ? save_fn(values, &layout, KVX_FORMAT_FP8, &id, &entry, 1, offset, stream)
                  : restore_fn(values, &layout, KVX_FORMAT_FP8, &id, &entry, 1, offset, stream);
    });
  });
}

// The list, tuple or range `o` of exact ints within [0, most], appended to `out`.
template <typename T>
bool ints_of(PyObject* o, uint64_t most, std::vector<T>& out) {
  if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o) && !PyRange_Check(o)) return false;
  PyObject* seq = PySequence_Fast(o, "");
  if (!seq) return false;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  out.reserve((size_t)n);
  bool ok = true;
  for (Py_ssize_t i = 0; ok && i < n; ++i) {
    PyObject* item = PySequence_Fast_GET_ITEM(seq, i);
    uint64_t v = 0;
    ok = PyLong_CheckExact(item);
    if (ok) {
      v = PyLong_AsUnsignedLongLong(item);
      ok = !PyErr_Occurred() && v <= most;
    }
    if (ok) out.push_back((T)v);
  }
  Py_DECREF(seq);
  return ok;
}

// blocks(save, pool, block_ids, entries, format, scale dtype or None)
PyObject* blocks(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 6 || !save_fn || !restore_fn || !entry_layout_fn) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    const bool save = args[0] == Py_True;
    const at::Tensor* pool = tensor_of(args[1]);
    if (!pool || pool->dim() != 6 || pool->size(0) != 2 || !pool->is_contiguous() || !PyLong_CheckExact(args[4]))
      return nullptr;
    int scales = scale_code(pool->scalar_type());
    if (args[5] != Py_None) {
      if (!THPDtype_Check(args[5])) return nullptr;
      scales = scale_code(((THPDtype*)args[5])->scalar_type);
      if (scales < 0) return nullptr;
    }
    std::vector<int32_t> ids;
    std::vector<uint64_t> entries;
    if (!ints_of(args[2], INT32_MAX, ids) || !ints_of(args[3], UINT64_MAX, entries) || ids.size() != entries.size() ||
        !fits32((int64_t)ids.size()))
      return nullptr;
    const int64_t layers = pool->size(1), nb = pool->size(2), hd = pool->size(5);
    const int64_t rows = pool->size(3) * pool->size(4);
    if (!fits32(2 * layers) || !fits32(nb) || !fits32(rows) || !fits32(hd)) return nullptr;
    const long format = PyLong_AsLong(args[4]);
    if (format != KVX_FORMAT_RAW && format != KVX_FORMAT_FP8) return nullptr;
    // Without a scale dtype, pools of other dtypes only use RAW entries, which carry no scales.
    const kvx_block_layout layout{nb * rows * hd, rows * hd, (int32_t)(2 * layers), (int32_t)rows, (int32_t)hd,
                                  (int32_t)nb, (int32_t)pool->element_size(), scales < 0 ? KVX_SCALE_BF16 : scales};
    int64_t logical, offset, stride;
    if (entry_layout_fn(&layout, (int32_t)format, &logical, &offset, &stride) != KVX_OK) return nullptr;
    void* base = pool->mutable_data_ptr();
    void* stream = stream_of(*pool);
    return status([&] {
      return save ? save_fn(base, &layout, (int32_t)format, ids.data(), entries.data(), (int32_t)ids.size(), offset, stream)
                  : restore_fn(base, &layout, (int32_t)format, ids.data(), entries.data(), (int32_t)ids.size(), offset, stream);
    });
  });
}

// ---------------------------------------------------------------------------
// Operators around an e4m3 cache. Those that make their outputs return them,
// or libkvx's status where that is an error.

int dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? KVX_DTYPE_BF16 : t == at::kHalf ? KVX_DTYPE_FP16 : t == at::kFloat ? KVX_DTYPE_FP32 : -1;
}

// Reads a call's arguments: `ok` stays true while each is what its reader asks for.
struct Reader {
  explicit Reader(PyObject* const* a) : args(a) {}
  PyObject* const* args;
  bool ok = true;

  // A tensor on the device of those before it.
  const at::Tensor* tensor(int i) {
    const at::Tensor* t = tensor_of(args[i]);
    if (!t || (first_ && t->device() != first_->device())) {
      ok = false;
      return nullptr;
    }
    if (!first_) first_ = t;
    return t;
  }
  const at::Tensor* tensor_or_none(int i) { return args[i] == Py_None ? nullptr : tensor(i); }
  int64_t integer(int i, int64_t none = -1) {
    if (args[i] == Py_None) return none;
    if (!PyLong_CheckExact(args[i])) {
      ok = false;
      return none;
    }
    const long long v = PyLong_AsLongLong(args[i]);
    if (PyErr_Occurred() || !fits32(v)) ok = false;
    return v;
  }
  double number(int i) {
    if (!PyFloat_CheckExact(args[i])) {
      ok = false;
      return 0.0;
    }
    return PyFloat_AS_DOUBLE(args[i]);
  }
  bool flag(int i) {
    if (!PyBool_Check(args[i])) ok = false;
    return args[i] == Py_True;
  }

 private:
  const at::Tensor* first_ = nullptr;
};

// [tokens, heads, head_dim] with packed heads.
bool packed_heads(const at::Tensor& t) {
  return t.dim() == 3 && (t.numel() == 0 || (t.stride(2) == 1 && t.stride(1) == t.size(2)));
}

// A layer's codes and scales; v and vs may both be null (keys only).
bool cache_of(const at::Tensor& k, const at::Tensor& ks, const at::Tensor* v, const at::Tensor* vs, kvx_fp8_cache* out) {
  if (k.dim() != 4 || ks.dim() != 4 || k.scalar_type() != at::kFloat8_e4m3fn || ks.scalar_type() != at::kFloat ||
      !k.is_contiguous() || !ks.is_contiguous())
    return false;
  const int64_t nb = k.size(0), bs = k.size(1), heads = k.size(2), hd = k.size(3), groups = ks.size(1);
  if (groups <= 0 || bs % groups || ks.size(0) != nb || ks.size(2) != heads || ks.size(3) != 1) return false;
  if (v && (v->scalar_type() != at::kFloat8_e4m3fn || v->sizes() != k.sizes() || !v->is_contiguous() ||
            vs->scalar_type() != at::kFloat || vs->sizes() != ks.sizes() || !vs->is_contiguous()))
    return false;
  if (!fits32(nb) || !fits32(bs) || !fits32(heads) || !fits32(hd)) return false;
  *out = {k.mutable_data_ptr(), v ? v->mutable_data_ptr() : nullptr, (float*)ks.mutable_data_ptr(),
          v ? (float*)vs->mutable_data_ptr() : nullptr, (int32_t)nb, (int32_t)bs, (int32_t)(bs / groups), (int32_t)heads,
          (int32_t)hd};
  return true;
}

bool int32_vector(const at::Tensor& t, int64_t n) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous();
}

// cu may be null; max_seqlen -1: not given.
bool batch_of(const at::Tensor& tables, const at::Tensor& lens, const at::Tensor* cu, int64_t max_seqlen,
              int64_t num_tokens, kvx_paged_batch* out) {
  if (tables.scalar_type() != at::kInt || tables.dim() != 2 ||
      (tables.numel() && tables.size(1) > 1 && tables.stride(1) != 1))
    return false;
  const int64_t seqs = tables.size(0);
  if (!int32_vector(lens, seqs) || !fits32(num_tokens) || !fits32(seqs) || !fits32(tables.size(1))) return false;
  if (cu ? !int32_vector(*cu, seqs + 1) : max_seqlen != -1 && max_seqlen != 1) return false;
  if (max_seqlen < 0 || !cu) max_seqlen = cu ? num_tokens : 1;
  *out = {(const int32_t*)tables.mutable_data_ptr(), (const int32_t*)lens.mutable_data_ptr(),
          cu ? (const int32_t*)cu->mutable_data_ptr() : nullptr, tables.stride(0), (int32_t)tables.size(1),
          (int32_t)seqs, (int32_t)max_seqlen, (int32_t)num_tokens};
  return true;
}

// `rc`'s status where it is an error, else the outputs (a tensor, or a tuple of several).
PyObject* outputs(int rc, std::initializer_list<const at::Tensor*> tensors) {
  if (rc != KVX_OK) return PyLong_FromLong(rc);
  if (tensors.size() == 1) return THPVariable_Wrap(**tensors.begin());
  PyObject* tuple = PyTuple_New((Py_ssize_t)tensors.size());
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor* t : tensors) {
    PyObject* o = THPVariable_Wrap(*t);
    if (!o) {
      Py_DECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}

template <typename F>
int without_gil(F call) {
  WithoutGil released;
  return call();
}

// rotary(query, key, positions, frequencies, interleaved, magnitude, query_out or None, key_out or None)
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 8 || !rotary_fn) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Reader r(args);
    const at::Tensor *q = r.tensor(0), *k = r.tensor(1), *where = r.tensor(2), *f = r.tensor(3);
    const bool interleaved = r.flag(4);
    const double magnitude = r.number(5);
    const at::Tensor *qo = r.tensor_or_none(6), *ko = r.tensor_or_none(7);
    if (!r.ok || !packed_heads(*q) || !packed_heads(*k)) return nullptr;
    const int64_t n = q->size(0), hd = q->size(2);
    const int dtype = dtype_code(q->scalar_type());
    if (n <= 0 || dtype < 0 || k->size(0) != n || k->size(2) != hd || k->scalar_type() != q->scalar_type()) return nullptr;
    if (where->dim() != 1 || where->size(0) != n || !where->is_contiguous() ||
        (where->scalar_type() != at::kInt && where->scalar_type() != at::kLong))
      return nullptr;
    if (f->dim() != 1 || f->scalar_type() != at::kDouble || !f->is_contiguous()) return nullptr;
    if (!fits32(hd) || !fits32(q->size(1)) || !fits32(k->size(1)) || !fits32(2 * f->size(0))) return nullptr;
    for (const at::Tensor* o : {qo, ko}) {
      const at::Tensor* in = o == qo ? q : k;
      if (o && (!packed_heads(*o) || o->sizes() != in->sizes() || o->scalar_type() != in->scalar_type())) return nullptr;
    }
    const at::Tensor q_out = qo ? *qo : at::empty(q->sizes(), q->options());
    const at::Tensor k_out = ko ? *ko : at::empty(k->sizes(), k->options());
    void* stream = stream_of(*q);
    const int rc = without_gil([&] {
      return rotary_fn(q->mutable_data_ptr(), q->stride(0), k->mutable_data_ptr(), k->stride(0),
                       q_out.mutable_data_ptr(), q_out.stride(0), k_out.mutable_data_ptr(), k_out.stride(0),
                       where->mutable_data_ptr(), (int32_t)where->element_size(), (const double*)f->mutable_data_ptr(), n,
                       (int32_t)q->size(1), (int32_t)k->size(1), (int32_t)hd, (int32_t)(2 * f->size(0)), interleaved,
                       (float)magnitude, dtype, stream);
    });
    return outputs(rc, {&q_out, &k_out});
  });
}

// store_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
PyObject* store_fp8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 7 || !store_fp8_fn) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Reader r(args);
    const at::Tensor* t[7];
    for (int i = 0; i < 7; ++i) t[i] = r.tensor(i);
    if (!r.ok) return nullptr;
    const at::Tensor &key = *t[0], &value = *t[1], &slots = *t[6];
    kvx_fp8_cache cache;
    const int dtype = dtype_code(key.scalar_type());
    if (dtype < 0 || !packed_heads(key) || !packed_heads(value) || key.sizes() != value.sizes() ||
        key.scalar_type() != value.scalar_type() || !cache_of(*t[2], *t[4], t[3], t[5], &cache) ||
        key.size(1) != cache.num_heads || key.size(2) != cache.head_dim || !int32_vector(slots, key.size(0)))
      return nullptr;
    const void *k = key.mutable_data_ptr(), *v = value.mutable_data_ptr(), *s = slots.mutable_data_ptr();
    void* stream = stream_of(key);
    return status([&] {
      return store_fp8_fn(&cache, k, key.stride(0), v, value.stride(0), dtype, (const int32_t*)s, key.size(0), stream);
    });
  });
}

// attention(query, k_cache, v_cache, k_scale, v_scale, block_tables, context_lens, softmax_scale, cu_seqlens or None,
//           max_seqlen or None, out or None, return_lse)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 12 || !attention_fn || !workspace_fn) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Reader r(args);
    const at::Tensor* t[7];
    for (int i = 0; i < 7; ++i) t[i] = r.tensor(i);
    const double scale = args[7] == Py_None ? 0.0 : r.number(7);
    const at::Tensor* cu = r.tensor_or_none(8);
    const int64_t max_seqlen = r.integer(9);
    const at::Tensor* given = r.tensor_or_none(10);
    const bool with_lse = r.flag(11);
    if (!r.ok) return nullptr;
    const at::Tensor& q = *t[0];
    kvx_fp8_cache cache;
    kvx_paged_batch batch;
    const int dtype = dtype_code(q.scalar_type());
    if (dtype < 0 || dtype == KVX_DTYPE_FP32 || !packed_heads(q) || !cache_of(*t[1], *t[3], t[2], t[4], &cache) ||
        q.size(2) != cache.head_dim || !fits32(q.size(1)) || !batch_of(*t[5], *t[6], cu, max_seqlen, q.size(0), &batch))
      return nullptr;
    if (given && (given->sizes() != q.sizes() || given->scalar_type() != q.scalar_type() || !given->is_contiguous()))
      return nullptr;
    const int32_t heads = (int32_t)q.size(1);
    int64_t need = 0;
    if (workspace_fn(&cache, &batch, heads, &need) != KVX_OK) return nullptr;
    const at::Tensor out = given ? *given : at::empty(q.sizes(), q.options());
    at::Tensor lse, workspace;
    if (with_lse) lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
    if (need > 0) workspace = at::empty({need}, q.options().dtype(at::kByte));
    const float softmax_scale = args[7] == Py_None ? (float)(1.0 / std::sqrt((double)cache.head_dim)) : (float)scale;
    void* stream = stream_of(q);
    const int rc = without_gil([&] {
      return attention_fn(&cache, &batch, q.mutable_data_ptr(), q.stride(0), heads, dtype, softmax_scale,
                          out.mutable_data_ptr(), with_lse ? (float*)lse.mutable_data_ptr() : nullptr,
                          need > 0 ? workspace.mutable_data_ptr() : nullptr, need, stream);
    });
    return with_lse ? outputs(rc, {&out, &lse}) : outputs(rc, {&out});
  });
}

// attention_weights(query, lse, k_cache, k_scale, block_tables, context_lens, softmax_scale, cu_seqlens or None,
//                   max_seqlen or None, weights or None, out)
PyObject* attention_weights(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 11 || !weights_fn) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Reader r(args);
    const at::Tensor* t[6];
    for (int i = 0; i < 6; ++i) t[i] = r.tensor(i);
    const double scale = args[6] == Py_None ? 0.0 : r.number(6);
    const at::Tensor* cu = r.tensor_or_none(7);
    const int64_t max_seqlen = r.integer(8);
    const at::Tensor *weights = r.tensor_or_none(9), *out = r.tensor(10);
    if (!r.ok) return nullptr;
    const at::Tensor &q = *t[0], &lse = *t[1];
    kvx_fp8_cache cache;
    kvx_paged_batch batch;
    const int dtype = dtype_code(q.scalar_type());
    if (dtype < 0 || dtype == KVX_DTYPE_FP32 || !packed_heads(q) || !cache_of(*t[2], *t[3], nullptr, nullptr, &cache) ||
        q.size(2) != cache.head_dim || !fits32(q.size(1)) || !batch_of(*t[4], *t[5], cu, max_seqlen, q.size(0), &batch))
      return nullptr;
    if (lse.scalar_type() != at::kFloat || lse.dim() != 2 || lse.size(0) != q.size(0) || lse.size(1) != q.size(1) ||
        !lse.is_contiguous())
      return nullptr;
    for (const at::Tensor* w : {weights, out})
      if (w && (w->scalar_type() != at::kFloat || w->dim() != 3 || w->size(0) != batch.num_seqs ||
                w->size(1) != cache.num_heads || w->size(2) != out->size(2) || !w->is_contiguous()))
        return nullptr;
    const float softmax_scale = args[6] == Py_None ? (float)(1.0 / std::sqrt((double)cache.head_dim)) : (float)scale;
    void* stream = stream_of(q);
    return status([&] {
      return weights_fn(&cache, &batch, q.mutable_data_ptr(), q.stride(0), (int32_t)q.size(1), dtype, softmax_scale,
                        (const float*)lse.mutable_data_ptr(), weights ? (const float*)weights->mutable_data_ptr() : nullptr,
                        (float*)out->mutable_data_ptr(), out->size(2), stream);
    });
  });
}

// select(weights, context_lens, keep, recent)
PyObject* select(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 4 || !select_fn) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Reader r(args);
    const at::Tensor *w = r.tensor(0), *lens = r.tensor(1);
    const int64_t keep = r.integer(2), recent = r.integer(3);
    if (!r.ok || keep < 0 || recent < 0 || w->scalar_type() != at::kFloat || w->dim() != 3 || !w->is_contiguous() ||
        w->size(1) <= 0 || !fits32(w->size(0)) || !fits32(w->size(1)) || !int32_vector(*lens, w->size(0)))
      return nullptr;
    const at::Tensor indices = at::empty({w->size(0), w->size(1), keep}, lens->options());
    const at::Tensor counts = at::empty({w->size(0)}, lens->options());
    const at::Tensor kept = at::empty({w->size(0), w->size(1), keep}, w->options());
    void* stream = stream_of(*w);
    const int rc = without_gil([&] {
      return select_fn((const float*)w->mutable_data_ptr(), (const int32_t*)lens->mutable_data_ptr(), (int32_t)w->size(0),
                       (int32_t)w->size(1), w->size(2), (int32_t)keep, (int32_t)recent,
                       (int32_t*)indices.mutable_data_ptr(), (int32_t*)counts.mutable_data_ptr(),
                       (float*)kept.mutable_data_ptr(), stream);
    });
    return outputs(rc, {&indices, &counts, &kept});
  });
}

// compact(k_cache, v_cache, k_scale, v_scale, block_tables, indices, counts, new_block_tables, context_lens or None)
PyObject* compact(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 9 || !compact_fn) Py_RETURN_NONE;
  return guarded([&]() -> PyObject* {
    Reader r(args);
    const at::Tensor* t[8];
    for (int i = 0; i < 8; ++i) t[i] = r.tensor(i);
    const at::Tensor* lens = r.tensor_or_none(8);
    if (!r.ok) return nullptr;
    const at::Tensor &indices = *t[5], &counts = *t[6];
    kvx_fp8_cache cache;
    kvx_paged_batch from, to;
    if (!cache_of(*t[0], *t[2], t[1], t[3], &cache) || !batch_of(*t[4], lens ? *lens : counts, nullptr, -1, 0, &from) ||
        !batch_of(*t[7], counts, nullptr, -1, 0, &to) || to.num_seqs != from.num_seqs)
      return nullptr;
    if (!lens) from.context_lens = nullptr;
    if (indices.scalar_type() != at::kInt || indices.dim() != 3 || indices.size(0) != from.num_seqs ||
        indices.size(1) != cache.num_heads || !fits32(indices.size(2)) || !indices.is_contiguous())
      return nullptr;
    const void *i = indices.mutable_data_ptr(), *c = counts.mutable_data_ptr();
    void* stream = stream_of(indices);
    return status([&] {
      return compact_fn(&cache, &from, (const int32_t*)i, (const int32_t*)c, (int32_t)indices.size(2), to.block_tables,
                        to.table_stride, to.table_width, stream);
    });
  });
}

// bind(address, ...): of libkvx's functions, in this order.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long a[11];
  if (!PyArg_ParseTuple(args, "KKKKKKKKKKK", a, a + 1, a + 2, a + 3, a + 4, a + 5, a + 6, a + 7, a + 8, a + 9, a + 10))
    return nullptr;
  auto set = [](auto& fn, unsigned long long address) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>((uintptr_t)address); };
  set(store_fn, a[0]);
  set(save_fn, a[1]);
  set(restore_fn, a[2]);
  set(entry_layout_fn, a[3]);
  set(rotary_fn, a[4]);
  set(store_fp8_fn, a[5]);
  set(workspace_fn, a[6]);
  set(attention_fn, a[7]);
  set(weights_fn, a[8]);
  set(select_fn, a[9]);
  set(compact_fn, a[10]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"store", (PyCFunction)(void (*)(void))store, METH_FASTCALL, nullptr},
    {"codec", (PyCFunction)(void (*)(void))codec, METH_FASTCALL, nullptr},
    {"blocks", (PyCFunction)(void (*)(void))blocks, METH_FASTCALL, nullptr},
    {"rotary", (PyCFunction)(void (*)(void))rotary, METH_FASTCALL, nullptr},
    {"store_fp8", (PyCFunction)(void (*)(void))store_fp8, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)(void))attention, METH_FASTCALL, nullptr},
    {"attention_weights", (PyCFunction)(void (*)(void))attention_weights, METH_FASTCALL, nullptr},
    {"select", (PyCFunction)(void (*)(void))select, METH_FASTCALL, nullptr},
    {"compact", (PyCFunction)(void (*)(void))compact, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods};

}  // namespace

// ABI_VERSION: of the kvx.h it was compiled against; TORCH_VERSION: the torch whose tensors it reads.
PyMODINIT_FUNC PyInit__bind() {
  PyObject* m = PyModule_Create(&module);
  if (m && (PyModule_AddIntConstant(m, "ABI_VERSION", KVX_ABI_VERSION) ||
            PyModule_AddStringConstant(m, "TORCH_VERSION", KVX_TORCH_VERSION))) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
