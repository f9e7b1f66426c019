// Descriptor building for kvx_amd/paged.py: write(), gather() and the
// operators' functions fill the kvx_abi.h and kvx_ext.h structs of a call from torch tensors and call the library's entry
// point.  Filling them field by field through ctypes bound every small call:
// on the MI355X host a gather of eight short sequences took 19.3 us, 4.8 us
// through this module (of which the launch is about 3).
//
// All return the kvx_status_t, or None for anything that the ctypes helpers
// must decide (an argument that is not a plain tensor, a dtype outside the
// ABI's, more than five axes, sizes past 32 bits): the caller then takes
// those helpers, which raise what they always raised.  The entry points are
// passed as addresses, so that the module calls whichever libkvx_amd.so the
// process has loaded.  A plain CPython module rather than a torch operator:
// the calls stay outside torch's dispatcher, as ctypes calls are.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/hip/HIPFunctions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <vector>

#include "kvx_ext.h"
#include "kvx_paged_kv.h"

namespace {

kvx_dtype_t dtype_of(at::ScalarType t) {
  switch (t) {
    case at::ScalarType::Half: return KVX_DTYPE_F16;
    case at::ScalarType::BFloat16: return KVX_DTYPE_BF16;
    case at::ScalarType::Float: return KVX_DTYPE_F32;
    case at::ScalarType::Float8_e4m3fn: return KVX_DTYPE_F8_E4M3;
    case at::ScalarType::Float8_e5m2: return KVX_DTYPE_F8_E5M2;
    case at::ScalarType::Int: return KVX_DTYPE_S32;
    case at::ScalarType::Long: return KVX_DTYPE_S64;
    default: return KVX_DTYPE_INVALID;
  }
}

// The argument's tensor, or null: exactly torch.Tensor (or Parameter), with
// storage of its own, so that no subclass override is passed by.
const at::Tensor *plain(PyObject *o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  if (!t.defined() || t.layout() != at::kStrided || !t.has_storage() || t.is_neg() || t.is_conj())
    return nullptr;
  return &t;
}

bool fits32(int64_t v) { return v >= 0 && v <= 0xFFFFFFFFll; }

// paged.tensor_desc
bool describe(kvx_tensor_desc_t *d, const at::Tensor &t, int layout) {
  const kvx_dtype_t dt = dtype_of(t.scalar_type());
  if (dt == KVX_DTYPE_INVALID || t.dim() > KVX_MAX_TENSOR_DIMS) return false;
  d->size = sizeof(kvx_tensor_desc_t);
  d->dtype = dt;
  d->layout = static_cast<kvx_layout_t>(layout);
  d->memory = t.is_cuda() ? KVX_MEMORY_DEVICE : KVX_MEMORY_HOST;
  d->ndim = static_cast<uint32_t>(t.dim());
  const auto sizes = t.sizes();
  const auto strides = t.strides();
  for (size_t i = 0; i < sizes.size(); ++i) {
    d->shape[i] = sizes[i];
    d->stride[i] = strides[i];
  }
  d->data = t.data_ptr();
  return true;
}

// paged.scale_desc_of: granularity -1 for a tensor that is a per-tensor scale.
bool describe_scale(kvx_scale_desc_t *d, const at::Tensor &t, int granularity) {
  d->size = sizeof(kvx_scale_desc_t);
  d->dtype = KVX_DTYPE_F32;
  d->granularity = granularity < 0 ? KVX_SCALE_PER_TENSOR
                                   : static_cast<kvx_scale_granularity_t>(granularity);
  d->ndim = 1;
  d->shape[0] = 1;
  d->stride[0] = 1;
  if (granularity >= 0 && t.dim() > 0) {
    if (t.dim() > KVX_MAX_TENSOR_DIMS) return false;
    d->ndim = static_cast<uint32_t>(t.dim());
    for (int64_t i = 0; i < t.dim(); ++i) {
      d->shape[i] = t.size(i);
      d->stride[i] = t.stride(i);
    }
  }
  d->data = t.data_ptr();
  return true;
}

// Arguments in order, each a plain tensor or number; `ok` turns false at the
// first that is not.
struct Args {
  PyObject *const *v;
  Py_ssize_t n;
  Py_ssize_t at = 0;
  bool ok = true;

  PyObject *next() {
    if (at >= n) {
      ok = false;
      return Py_None;
    }
    return v[at++];
  }
  const at::Tensor *tensor() {
    const at::Tensor *t = plain(next());
    if (t == nullptr) ok = false;
    return t;
  }
  const at::Tensor *tensor_or_none() {
    PyObject *o = next();
    if (o == Py_None) return nullptr;
    const at::Tensor *t = plain(o);
    if (t == nullptr) ok = false;
    return t;
  }
  int64_t number() {
    PyObject *o = next();
    if (!ok || !PyLong_Check(o)) {
      ok = false;
      return 0;
    }
    const int64_t x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return x;
  }
  uint32_t number32() {
    const int64_t x = number();
    if (!fits32(x)) ok = false;
    return static_cast<uint32_t>(x);
  }
  double real() {
    PyObject *o = next();
    if (!ok || !(PyFloat_Check(o) || PyLong_Check(o))) {
      ok = false;
      return 0.0;
    }
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return x;
  }
  template <class F>
  F function() {
    PyObject *o = next();
    void *p = ok && PyLong_Check(o) ? PyLong_AsVoidPtr(o) : nullptr;
    if (p == nullptr) {
      PyErr_Clear();
      ok = false;
    }
    return reinterpret_cast<F>(p);
  }
};

// (key_cache, value_cache, k_layout, v_layout, num_blocks, block_size, heads,
// head_dim) of a PagedCache.
bool cache_of(Args &a, kvx_cache_desc_t *c) {
  const at::Tensor *k = a.tensor();
  const at::Tensor *v = a.tensor();
  const int64_t kl = a.number();
  const int64_t vl = a.number();
  c->size = sizeof(kvx_cache_desc_t);
  c->num_blocks = a.number32();
  c->block_size = a.number32();
  c->num_kv_heads = a.number32();
  c->head_dim = a.number32();
  return a.ok && describe(&c->k, *k, static_cast<int>(kl)) &&
         describe(&c->v, *v, static_cast<int>(vl));
}

// The stream argument: a handle, or None for torch's current stream.
void *stream_of(Args &a) {
  PyObject *o = a.next();
  if (o == Py_None)
    return reinterpret_cast<void *>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream());
  void *p = PyLong_Check(o) ? PyLong_AsVoidPtr(o) : nullptr;
  if (p == nullptr && PyErr_Occurred()) {
    PyErr_Clear();
    a.ok = false;
  }
  if (!PyLong_Check(o)) a.ok = false;
  return p;
}

template <class F>
PyObject *status_of(F &&call) {
  kvx_status_t st;
  Py_BEGIN_ALLOW_THREADS
  st = call();
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(static_cast<long>(st));
}

typedef kvx_status_t (*WriteFn)(const kvx_cache_desc_t *, const kvx_write_desc_t *, void *);
typedef kvx_status_t (*PrefillFn)(const kvx_cache_desc_t *, const kvx_write_desc_t *, int32_t,
                                  void *);
typedef kvx_status_t (*GatherFn)(const kvx_cache_desc_t *, const kvx_gather_desc_t *, void *);
typedef kvx_status_t (*DequantFn)(const kvx_cache_desc_t *, const kvx_gather_desc_t *,
                                  const kvx_scale_desc_t *, const kvx_scale_desc_t *, void *);

// write(fn, tokens_per_seq (None: fn takes none), stream, cache..., key, value,
//       slots, k_scale, k_granularity, v_scale, v_granularity)
PyObject *host_write(Args a) {
  void *fn = a.function<void *>();
  const bool prefill = a.at < a.n && a.v[a.at] != Py_None;
  int64_t per_seq = 0;
  if (prefill) per_seq = a.number();
  else a.next();
  void *stream = stream_of(a);
  kvx_cache_desc_t c{};
  if (!a.ok || !cache_of(a, &c)) Py_RETURN_NONE;
  kvx_write_desc_t w{};
  const at::Tensor *key = a.tensor();
  const at::Tensor *value = a.tensor();
  const at::Tensor *slots = a.tensor();
  const at::Tensor *ks = a.tensor_or_none();
  const int64_t kg = a.number();
  const at::Tensor *vs = a.tensor_or_none();
  const int64_t vg = a.number();
  if (!a.ok || a.at != a.n || key->dim() != 3 || !fits32(key->size(0)) ||
      !fits32(key->size(1)) || !fits32(key->size(2)) || !fits32(slots->numel()) ||
      per_seq > 0x7FFFFFFF || per_seq < -0x80000000ll)
    Py_RETURN_NONE;
  w.size = sizeof(kvx_write_desc_t);
  w.io.size = sizeof(kvx_kv_io_desc_t);
  const kvx_dtype_t sdt = dtype_of(slots->scalar_type());
  if (!describe(&w.io.key, *key, KVX_LAYOUT_BLOCK_CUSTOM) ||
      !describe(&w.io.value, *value, KVX_LAYOUT_BLOCK_CUSTOM) || sdt == KVX_DTYPE_INVALID)
    Py_RETURN_NONE;
  w.io.num_tokens = static_cast<uint32_t>(key->size(0));
  w.io.num_kv_heads = static_cast<uint32_t>(key->size(1));
  w.io.head_dim = static_cast<uint32_t>(key->size(2));
  w.slots.size = sizeof(kvx_slot_mapping_t);
  w.slots.dtype = sdt;
  w.slots.token_count = static_cast<uint32_t>(slots->numel());
  w.slots.invalid_slot = -1;
  w.slots.slots = slots->data_ptr();
  if (ks && !describe_scale(&w.k_scale_desc, *ks, static_cast<int>(kg))) Py_RETURN_NONE;
  if (vs && !describe_scale(&w.v_scale_desc, *vs, static_cast<int>(vg))) Py_RETURN_NONE;
  if (prefill)
    return status_of([&] {
      return reinterpret_cast<PrefillFn>(fn)(&c, &w, static_cast<int32_t>(per_seq), stream);
    });
  return status_of([&] { return reinterpret_cast<WriteFn>(fn)(&c, &w, stream); });
}

// paged._table_desc, and the pool fields of paged.gather_cache_desc.
bool table_of(const at::Tensor &table, const at::Tensor *indptr, const at::Tensor *primary,
              const at::Tensor *secondary, uint32_t bytes_per_block, kvx_block_table_t *out,
              kvx_cache_desc_t *c) {
  kvx_block_table_t &t = *out;
  const kvx_dtype_t tdt = dtype_of(table.scalar_type());
  if (tdt == KVX_DTYPE_INVALID) return false;
  t.size = sizeof(kvx_block_table_t);
  t.index_dtype = tdt;
  t.beam_width = 1;
  t.indices = table.data_ptr();
  if (indptr != nullptr) {
    const kvx_dtype_t pdt = dtype_of(indptr->scalar_type());
    if (pdt == KVX_DTYPE_INVALID || indptr->numel() < 1 || !fits32(indptr->numel()) ||
        !fits32(table.numel()))
      return false;
    t.format = KVX_BLOCK_TABLE_RAGGED;
    t.indptr_dtype = pdt;
    t.seq_count = static_cast<uint32_t>(indptr->numel() - 1);
    t.max_blocks_per_seq = 1;
    t.indptr = indptr->data_ptr();
    t.indices_count = static_cast<uint32_t>(table.numel());
    t.indptr_count = static_cast<uint32_t>(indptr->numel());
  } else if (primary != nullptr) {
    if (table.dim() != 4 || table.size(2) != 2 || tdt != KVX_DTYPE_S32 ||
        !fits32(table.size(0)) || !fits32(table.size(1)) || !fits32(table.size(3)) ||
        !fits32(table.numel()))
      return false;
    t.format = KVX_BLOCK_TABLE_KV_OFFSETS;
    t.seq_count = static_cast<uint32_t>(table.size(0));
    t.beam_width = static_cast<uint32_t>(table.size(1));
    t.max_blocks_per_seq = static_cast<uint32_t>(table.size(3));
    t.indices_count = static_cast<uint32_t>(table.numel());
    t.flags = KVX_BLOCK_TABLE_FLAG_KVCACHEINDEX;
    c->pool.size = sizeof(kvx_pool_desc_t);
    c->pool.memory = primary->is_cuda() ? KVX_MEMORY_DEVICE : KVX_MEMORY_HOST;
    c->pool.bytes_per_block = bytes_per_block;
    c->pool.primary = primary->data_ptr();
    c->pool.secondary = secondary ? secondary->data_ptr() : nullptr;
  } else {
    if (table.dim() != 2 || !fits32(table.size(0)) || !fits32(table.size(1)) ||
        !fits32(table.numel()))
      return false;
    t.format = KVX_BLOCK_TABLE_PACKED;
    t.seq_count = static_cast<uint32_t>(table.size(0));
    t.max_blocks_per_seq = static_cast<uint32_t>(table.size(1));
    t.indices_count = static_cast<uint32_t>(table.numel());
  }
  return true;
}

// gather(fn, stream, cache..., key_out, value_out, table, indptr, primary,
//        secondary, bytes_per_block, lens, max_seq_len, k_scale,
//        k_granularity, v_scale, v_granularity): indptr set for a RAGGED
//        table (`table` its indices), primary for a KV_OFFSETS one (`table`
//        its offsets); with scales fn is the dequantizing gather.
PyObject *host_gather(Args a) {
  void *fn = a.function<void *>();
  void *stream = stream_of(a);
  kvx_cache_desc_t c{};
  if (!a.ok || !cache_of(a, &c)) Py_RETURN_NONE;
  const at::Tensor *ko = a.tensor();
  const at::Tensor *vo = a.tensor();
  const at::Tensor *table = a.tensor();
  const at::Tensor *indptr = a.tensor_or_none();
  const at::Tensor *primary = a.tensor_or_none();
  const at::Tensor *secondary = a.tensor_or_none();
  const uint32_t bytes_per_block = a.number32();
  const at::Tensor *lens = a.tensor();
  const uint32_t width = a.number32();
  const at::Tensor *ks = a.tensor_or_none();
  const int64_t kg = a.number();
  const at::Tensor *vs = a.tensor_or_none();
  const int64_t vg = a.number();
  if (!a.ok || a.at != a.n || (ks == nullptr) != (vs == nullptr) || ko->dim() != 4 ||
      !fits32(ko->size(2)) || !fits32(ko->size(3)) || !fits32(lens->numel()))
    Py_RETURN_NONE;
  kvx_gather_desc_t g{};
  g.size = sizeof(kvx_gather_desc_t);
  g.io.size = sizeof(kvx_kv_io_desc_t);
  const kvx_dtype_t ldt = dtype_of(lens->scalar_type());
  if (!describe(&g.io.key, *ko, KVX_LAYOUT_BLOCK_CUSTOM) ||
      !describe(&g.io.value, *vo, KVX_LAYOUT_BLOCK_CUSTOM) || ldt == KVX_DTYPE_INVALID)
    Py_RETURN_NONE;
  kvx_block_table_t &t = g.block_table;
  if (!table_of(*table, indptr, primary, secondary, bytes_per_block, &t, &c)) Py_RETURN_NONE;
  if ((uint64_t)t.seq_count * width > 0xFFFFFFFFull) Py_RETURN_NONE;
  g.io.num_tokens = t.seq_count * width;
  g.io.num_kv_heads = static_cast<uint32_t>(ko->size(2));
  g.io.head_dim = static_cast<uint32_t>(ko->size(3));
  g.seq_lens.size = sizeof(kvx_seq_lens_t);
  g.seq_lens.dtype = ldt;
  g.seq_lens.seq_count = static_cast<uint32_t>(lens->numel());
  g.seq_lens.lengths = lens->data_ptr();
  g.max_seq_len = width;
  if (ks == nullptr)
    return status_of([&] { return reinterpret_cast<GatherFn>(fn)(&c, &g, stream); });
  kvx_scale_desc_t ksd{}, vsd{};
  if (!describe_scale(&ksd, *ks, static_cast<int>(kg)) ||
      !describe_scale(&vsd, *vs, static_cast<int>(vg)))
    Py_RETURN_NONE;
  return status_of([&] { return reinterpret_cast<DequantFn>(fn)(&c, &g, &ksd, &vsd, stream); });
}

// Whether all tensors (null: none) are on the current device, so that neither
// a device guard nor an error message is needed.
bool here(std::initializer_list<const at::Tensor *> tensors) {
  const auto now = c10::hip::current_device();
  for (const at::Tensor *t : tensors)
    if (t != nullptr && (!t->is_cuda() || t->get_device() != now)) return false;
  return true;
}

bool is_index(const at::Tensor &t) {
  return (t.scalar_type() == at::ScalarType::Int || t.scalar_type() == at::ScalarType::Long) &&
         t.is_contiguous();
}

// Scales (null: none) that kernels can read.
bool are_scales(std::initializer_list<const at::Tensor *> scales) {
  for (const at::Tensor *t : scales)
    if (t != nullptr && t->scalar_type() != at::ScalarType::Float) return false;
  return here(scales);
}

bool is_line(const at::Tensor &t, int64_t n) { return is_index(t) && t.dim() == 1 && t.size(0) == n; }

// The cache's tensors, which come next among the arguments.
bool cache_here(const Args &a) {
  if (a.at + 2 > a.n) return false;
  const at::Tensor *k = plain(a.v[a.at]), *v = plain(a.v[a.at + 1]);
  return k != nullptr && v != nullptr && here({k, v});
}

// rope_write(fn, stream, cache..., query, query_out (None: no queries), key,
//            value, positions, inv_freq, interleaved, magnitude, slots,
//            k_scale, k_granularity, v_scale, v_granularity): None for what
//            paged.rope_write_kv refuses, too.
PyObject *host_rope_write(Args a) {
  typedef kvx_status_t (*Fn)(const kvx_cache_desc_t *, const kvx_write_desc_t *,
                             const kvx_rope_desc_t *, void *);
  const Fn fn = a.function<Fn>();
  void *stream = stream_of(a);
  kvx_cache_desc_t c{};
  if (!a.ok || !cache_here(a) || !cache_of(a, &c)) Py_RETURN_NONE;
  const at::Tensor *q = a.tensor_or_none();
  const at::Tensor *o = a.tensor_or_none();
  const at::Tensor *key = a.tensor();
  const at::Tensor *value = a.tensor();
  const at::Tensor *pos = a.tensor();
  const at::Tensor *inv = a.tensor();
  const int64_t interleaved = a.number();
  const double magnitude = a.real();
  const at::Tensor *slots = a.tensor();
  const at::Tensor *ks = a.tensor_or_none();
  const int64_t kg = a.number();
  const at::Tensor *vs = a.tensor_or_none();
  const int64_t vg = a.number();
  if (!a.ok || a.at != a.n || (q == nullptr) != (o == nullptr) ||
      !here({q, o, key, value, pos, inv, slots}) || !are_scales({ks, vs}) || key->dim() != 3 || value->dim() != 3 ||
      (q != nullptr && (q->dim() != 3 || o->dim() != 3)) || !is_line(*pos, key->size(0)) ||
      !is_line(*slots, key->size(0)) || inv->scalar_type() != at::ScalarType::Float ||
      !inv->is_contiguous() || !fits32(key->size(0)) || !fits32(key->size(1)) ||
      !fits32(key->size(2)) || !fits32(2 * inv->numel()))
    Py_RETURN_NONE;
  kvx_write_desc_t w{};
  kvx_rope_desc_t r{};
  if (!describe(&w.io.key, *key, KVX_LAYOUT_BLOCK_CUSTOM) ||
      !describe(&w.io.value, *value, KVX_LAYOUT_BLOCK_CUSTOM) ||
      (q != nullptr && (!describe(&r.query, *q, KVX_LAYOUT_BLOCK_CUSTOM) ||
                        !describe(&r.query_out, *o, KVX_LAYOUT_BLOCK_CUSTOM))))
    Py_RETURN_NONE;
  w.size = sizeof(kvx_write_desc_t);
  w.io.size = sizeof(kvx_kv_io_desc_t);
  w.io.num_tokens = static_cast<uint32_t>(key->size(0));
  w.io.num_kv_heads = static_cast<uint32_t>(key->size(1));
  w.io.head_dim = static_cast<uint32_t>(key->size(2));
  w.slots.size = sizeof(kvx_slot_mapping_t);
  w.slots.dtype = dtype_of(slots->scalar_type());
  w.slots.token_count = static_cast<uint32_t>(slots->numel());
  w.slots.invalid_slot = -1;
  w.slots.slots = slots->data_ptr();
  if (ks && !describe_scale(&w.k_scale_desc, *ks, static_cast<int>(kg))) Py_RETURN_NONE;
  if (vs && !describe_scale(&w.v_scale_desc, *vs, static_cast<int>(vg))) Py_RETURN_NONE;
  r.size = sizeof(kvx_rope_desc_t);
  r.style = interleaved ? KVX_ROPE_INTERLEAVED : KVX_ROPE_HALF;
  r.rot_dim = static_cast<uint32_t>(2 * inv->numel());
  r.magnitude = static_cast<float>(magnitude);
  r.position_dtype = dtype_of(pos->scalar_type());
  r.positions = pos->data_ptr();
  r.inv_freq = inv->data_ptr<float>();
  return status_of([&] { return fn(&c, &w, &r, stream); });
}

// attention(fn, workspace_size fn, stream, cache..., query, out, table, indptr,
//           primary, secondary, bytes_per_block, lens, query_indptr, causal,
//           scale, window, softcap, lse, max_seq_len, max_query_len, k_scale,
//           k_granularity, v_scale, v_granularity, workspace): the table as
//           gather's; None for what paged.attention refuses, and for a
//           workspace that another stream than the current one uses, too.
PyObject *host_attention(Args a) {
  typedef kvx_status_t (*SizeFn)(const kvx_cache_desc_t *, const kvx_attention_desc_t *,
                                 uint64_t *);
  typedef kvx_status_t (*Fn)(const kvx_cache_desc_t *, const kvx_attention_desc_t *, void *);
  const Fn fn = a.function<Fn>();
  const SizeFn size_fn = a.function<SizeFn>();
  const bool current = a.at < a.n && a.v[a.at] == Py_None;
  void *stream = stream_of(a);
  kvx_cache_desc_t c{};
  if (!a.ok || !cache_here(a) || !cache_of(a, &c)) Py_RETURN_NONE;
  const at::Tensor *q = a.tensor();
  const at::Tensor *o = a.tensor();
  const at::Tensor *table = a.tensor();
  const at::Tensor *indptr = a.tensor_or_none();
  const at::Tensor *primary = a.tensor_or_none();
  const at::Tensor *secondary = a.tensor_or_none();
  const uint32_t bytes_per_block = a.number32();
  const at::Tensor *lens = a.tensor();
  const at::Tensor *rows = a.tensor_or_none();
  const int64_t causal = a.number();
  const double scale = a.real();
  const uint32_t window = a.number32();
  const double softcap = a.real();
  const at::Tensor *lse = a.tensor_or_none();
  const uint32_t max_seq = a.number32();
  const uint32_t max_query = a.number32();
  const at::Tensor *ks = a.tensor_or_none();
  const int64_t kg = a.number();
  const at::Tensor *vs = a.tensor_or_none();
  const int64_t vg = a.number();
  const at::Tensor *workspace = a.tensor_or_none();
  if (!a.ok || a.at != a.n ||
      !here({q, o, table, indptr, primary, secondary, lens, rows, lse, workspace}) ||
      !are_scales({ks, vs}) ||
      q->dim() != 3 || o->dim() != 3 || !is_index(*table) || !is_index(*lens) ||
      (indptr != nullptr && !is_index(*indptr)))
    Py_RETURN_NONE;
  kvx_attention_desc_t d{};
  kvx_block_table_t &t = d.block_table;
  if (!table_of(*table, indptr, primary, secondary, bytes_per_block, &t, &c) ||
      !is_line(*lens, t.seq_count) || (rows != nullptr && !is_line(*rows, (int64_t)t.seq_count + 1)) ||
      (lse != nullptr && (lse->scalar_type() != at::ScalarType::Float || !lse->is_contiguous() ||
                          lse->dim() != 2 || lse->size(0) != q->size(0) ||
                          lse->size(1) != q->size(1))) ||
      (workspace != nullptr && !workspace->is_contiguous()))
    Py_RETURN_NONE;
  d.size = sizeof(kvx_attention_desc_t);
  d.flags = causal ? KVX_ATTENTION_CAUSAL : 0;
  if (!describe(&d.query, *q, KVX_LAYOUT_BLOCK_CUSTOM) ||
      !describe(&d.out, *o, KVX_LAYOUT_BLOCK_CUSTOM))
    Py_RETURN_NONE;
  d.lse = lse != nullptr ? lse->data_ptr<float>() : nullptr;
  if (rows != nullptr) {
    d.query_indptr = rows->data_ptr();
    d.query_indptr_dtype = dtype_of(rows->scalar_type());
  }
  d.window = window;
  d.scale = static_cast<float>(scale);
  d.softcap = static_cast<float>(softcap);
  d.max_seq_len = max_seq;
  d.max_query_len = max_query;
  d.seq_lens.size = sizeof(kvx_seq_lens_t);
  d.seq_lens.dtype = dtype_of(lens->scalar_type());
  d.seq_lens.seq_count = static_cast<uint32_t>(lens->numel());
  d.seq_lens.lengths = lens->data_ptr();
  if (ks && !describe_scale(&d.k_scale, *ks, static_cast<int>(kg))) Py_RETURN_NONE;
  if (vs && !describe_scale(&d.v_scale, *vs, static_cast<int>(vg))) Py_RETURN_NONE;
  uint64_t need = 0;
  const kvx_status_t st = size_fn(&c, &d, &need);
  if (st != KVX_STATUS_OK) return PyLong_FromLong(static_cast<long>(st));
  at::Tensor own;
  if (workspace == nullptr && need > 0) {
    if (!current || need > 0x7FFFFFFFFFFFFFFFull) Py_RETURN_NONE;
    // from the current stream's memory, which the caching allocator hands out
    // again in that stream's order
    own = at::empty({static_cast<int64_t>(need)}, q->options().dtype(at::kByte));
    workspace = &own;
  }
  if (workspace != nullptr) {
    d.workspace = workspace->data_ptr();
    d.workspace_size = workspace->nbytes();
  }
  return status_of([&] { return fn(&c, &d, stream); });
}

// copy_blocks(fn, stream, PagedCache type, list of caches, pairs): caches of
//             exactly that type.
PyObject *host_copy_blocks(Args a) {
  typedef kvx_status_t (*Fn)(const kvx_cache_desc_t *const *, uint32_t, const void *, kvx_dtype_t,
                             uint32_t, void *);
  static PyObject *const names[8] = {
      PyUnicode_InternFromString("key_cache"),  PyUnicode_InternFromString("value_cache"),
      PyUnicode_InternFromString("k_layout"),   PyUnicode_InternFromString("v_layout"),
      PyUnicode_InternFromString("num_blocks"), PyUnicode_InternFromString("block_size"),
      PyUnicode_InternFromString("heads"),      PyUnicode_InternFromString("head_dim")};
  const Fn fn = a.function<Fn>();
  void *stream = stream_of(a);
  PyObject *type = a.next();
  PyObject *list = a.next();
  const at::Tensor *pairs = a.tensor();
  if (!a.ok || a.at != a.n || !PyList_Check(list) || !here({pairs}) || !is_index(*pairs) ||
      pairs->dim() != 2 || pairs->size(1) != 2 || !fits32(pairs->size(0)))
    Py_RETURN_NONE;
  const Py_ssize_t count = PyList_GET_SIZE(list);
  if (!fits32(count)) Py_RETURN_NONE;
  std::vector<kvx_cache_desc_t> caches(static_cast<size_t>(count));
  std::vector<const kvx_cache_desc_t *> pointers(caches.size());
  for (Py_ssize_t i = 0; i < count; ++i) {
    PyObject *o = PyList_GET_ITEM(list, i);
    if (reinterpret_cast<PyObject *>(Py_TYPE(o)) != type) Py_RETURN_NONE;
    PyObject *v[8] = {};
    bool ok = true;
    for (int k = 0; k < 8 && ok; ++k) ok = (v[k] = PyObject_GetAttr(o, names[k])) != nullptr;
    if (ok) {
      Args c{v, 8};
      ok = cache_here(c) && cache_of(c, &caches[i]);
    }
    for (PyObject *x : v) Py_XDECREF(x);  // the cache object keeps them
    if (!ok) {
      PyErr_Clear();
      Py_RETURN_NONE;
    }
    pointers[i] = &caches[i];
  }
  const void *ids = pairs->data_ptr();
  const kvx_dtype_t dt = dtype_of(pairs->scalar_type());
  const uint32_t n = static_cast<uint32_t>(pairs->size(0));
  return status_of([&] {
    return fn(pointers.data(), static_cast<uint32_t>(pointers.size()), ids, dt, n, stream);
  });
}

template <PyObject *(*F)(Args)>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  try {
    return F(Args{args, n});
  } catch (...) {
    // torch refuses a tensor (no data to point at, say): the ctypes helpers
    // raise for it
    Py_RETURN_NONE;
  }
}

PyMethodDef kMethods[] = {
    {"write", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<host_write>)),
     METH_FASTCALL, nullptr},
    {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<host_gather>)),
     METH_FASTCALL, nullptr},
    {"rope_write",
     reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<host_rope_write>)),
     METH_FASTCALL, nullptr},
    {"attention",
     reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<host_attention>)),
     METH_FASTCALL, nullptr},
    {"copy_blocks",
     reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<host_copy_blocks>)),
     METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_paged_host", nullptr, -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_host(void) { return PyModule_Create(&kModule); }
