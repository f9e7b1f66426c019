// Entry points of kvx_ext.h's operators: the rotary write, the attention over
// a paged cache and the block copy.  Every check runs on the host before any
// HIP call; what a kernel reads of device data (ids, lengths, row numbers) it
// checks itself.
#include <hip/hip_runtime.h>

#include <cmath>
#include <vector>

#include "kvx_ext.h"
#include "operators_internal.h"

namespace kvx {
namespace {

constexpr int64_t kMost32 = 0x7FFFFFFF;

bool on_device(const kvx_tensor_desc_t &t) {
  return t.memory == KVX_MEMORY_DEVICE || t.memory == KVX_MEMORY_UNIFIED;
}

// An axis of n elements spans less than 2^56 of them: no offset on the host or the
// device overflows.
bool spans(int64_t n, int64_t stride) {
  const int64_t most = ((int64_t)1 << 56) / (n > 1 ? n : 1);
  return stride >= -most && stride <= most;
}

// fill_geom, with strides of axes of one element as 0 (they are never used) and
// the others' spans checked.
kvx_status_t cache_geom(const kvx_cache_desc_t *c, const kvx_tensor_desc_t *t, Geom *g) {
  const kvx_status_t st = fill_geom(c, t, g);
  if (st != KVX_STATUS_OK) return st;
  const int64_t pack = g->pack > 0 ? g->pack : 1;
  struct {
    int64_t n, *stride;
  } const axes[5] = {{(int64_t)c->num_blocks, &g->s_block}, {(int64_t)c->block_size, &g->s_off},
                     {(int64_t)c->num_kv_heads, &g->s_head},
                     {(int64_t)c->head_dim / pack, &g->s_piece}, {pack, &g->s_inner}};
  for (const auto &x : axes) {
    if (x.n <= 1) *x.stride = 0;
    else if (!spans(x.n, *x.stride)) return KVX_STATUS_INVALID_ARGUMENT;
  }
  return KVX_STATUS_OK;
}

bool is_index(kvx_dtype_t dt) { return dt == KVX_DTYPE_S32 || dt == KVX_DTYPE_S64; }

// A [tokens, heads, head_dim] tensor of rows with adjacent head elements and
// any other strides.  A stride of a size-1 axis is never used.
kvx_status_t check_rows(const kvx_tensor_desc_t &t, int64_t tokens, int64_t heads,
                        int64_t head_dim, int64_t *tok, int64_t *head) {
  if (t.size < sizeof(kvx_tensor_desc_t) || t.ndim != 3) return KVX_STATUS_INVALID_ARGUMENT;
  if (t.shape[0] != tokens || t.shape[1] != heads || t.shape[2] != head_dim)
    return KVX_STATUS_INVALID_ARGUMENT;
  if (!on_device(t)) return KVX_STATUS_INVALID_ARGUMENT;
  if (t.stride[2] != 1 && head_dim > 1) return KVX_STATUS_UNSUPPORTED;
  *tok = tokens > 1 ? t.stride[0] : 0;
  *head = heads > 1 ? t.stride[1] : 0;
  return spans(tokens, *tok) && spans(heads, *head) ? KVX_STATUS_OK : KVX_STATUS_INVALID_ARGUMENT;
}

// A written tensor: no two of its elements may share an address.
bool rows_overlap(int64_t tokens, int64_t heads, int64_t head_dim, int64_t tok, int64_t head) {
  if (tokens == 0 || heads == 0 || head_dim == 0) return false;
  const int64_t t = tok < 0 ? -tok : tok, h = head < 0 ? -head : head;
  if (heads > 1 && h < head_dim) return true;
  if (tokens <= 1) return false;
  if (heads <= 1) return t < head_dim;
  // tokens outside heads, or heads outside tokens
  return !(t >= (heads - 1) * h + head_dim || (t >= head_dim && h >= (tokens - 1) * t + head_dim));
}

kvx_status_t check_cache(const kvx_cache_desc_t *cache) {
  if (cache == nullptr || cache->size < sizeof(kvx_cache_desc_t))
    return KVX_STATUS_INVALID_ARGUMENT;
  if (cache->k.dtype != cache->v.dtype) return KVX_STATUS_INVALID_ARGUMENT;
  if (!is_io_float(cache->k.dtype) && !is_fp8(cache->k.dtype)) return KVX_STATUS_UNSUPPORTED;
  if (cache->num_blocks > kMost32 || cache->block_size > kMost32 ||
      cache->num_kv_heads > kMost32 || cache->head_dim > kMost32)
    return KVX_STATUS_INVALID_ARGUMENT;
  if (!on_device(cache->k) || !on_device(cache->v)) return KVX_STATUS_INVALID_ARGUMENT;
  return KVX_STATUS_OK;
}

}  // namespace

static kvx_status_t plan_rope(const kvx_cache_desc_t *cache, const kvx_write_desc_t *write,
                              const kvx_rope_desc_t *rope, RopePlan *p, bool *empty) {
  if (write == nullptr || rope == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
  kvx_status_t st = check_cache(cache);
  if (st != KVX_STATUS_OK) return st;
  if (write->size < sizeof(kvx_write_desc_t) || write->io.size < sizeof(kvx_kv_io_desc_t) ||
      write->slots.size < sizeof(kvx_slot_mapping_t) || rope->size < sizeof(kvx_rope_desc_t))
    return KVX_STATUS_INVALID_ARGUMENT;
  const kvx_dtype_t cdt = cache->k.dtype, io = write->io.key.dtype;
  if (write->io.value.dtype != io || !is_io_float(io) || (!is_fp8(cdt) && io != cdt))
    return KVX_STATUS_UNSUPPORTED;
  const int64_t T = write->io.num_tokens, H = cache->num_kv_heads, D = cache->head_dim;
  if (T > kMost32 || write->io.num_kv_heads != H || write->io.head_dim != D)
    return KVX_STATUS_INVALID_ARGUMENT;
  *p = RopePlan{};
  st = check_rows(write->io.key, T, H, D, &p->k_tok, &p->k_head);
  if (st != KVX_STATUS_OK) return st;
  st = check_rows(write->io.value, T, H, D, &p->v_tok, &p->v_head);
  if (st != KVX_STATUS_OK) return st;
  if (write->slots.token_count != write->io.num_tokens) return KVX_STATUS_INVALID_ARGUMENT;
  if (rope->style != KVX_ROPE_HALF && rope->style != KVX_ROPE_INTERLEAVED)
    return KVX_STATUS_INVALID_ARGUMENT;
  if (rope->rot_dim % 2 != 0 || rope->rot_dim > D) return KVX_STATUS_INVALID_ARGUMENT;
  if (rope->rot_dim > 8192) return KVX_STATUS_UNSUPPORTED;
  const bool query = rope->query.ndim != 0;
  int64_t Hq = 0;
  if (query) {
    Hq = rope->query.shape[1];
    if (Hq < 0 || Hq > kMost32 || rope->query.dtype != io || rope->query_out.dtype != io)
      return Hq < 0 || Hq > kMost32 ? KVX_STATUS_INVALID_ARGUMENT : KVX_STATUS_UNSUPPORTED;
    st = check_rows(rope->query, T, Hq, D, &p->q_tok, &p->q_head);
    if (st != KVX_STATUS_OK) return st;
    st = check_rows(rope->query_out, T, Hq, D, &p->o_tok, &p->o_head);
    if (st != KVX_STATUS_OK) return st;
    if (rows_overlap(T, Hq, D, p->o_tok, p->o_head)) return KVX_STATUS_UNSUPPORTED;
  }
  WritePlan &w = p->w;
  st = cache_geom(cache, &cache->k, &w.gk);
  if (st != KVX_STATUS_OK) return st;
  st = cache_geom(cache, &cache->v, &w.gv);
  if (st != KVX_STATUS_OK) return st;
  if (is_fp8(cdt)) {
    st = resolve_write_scale(&write->k_scale_desc, write->k_scale, cache, &w.k_scale);
    if (st != KVX_STATUS_OK) return st;
    st = resolve_write_scale(&write->v_scale_desc, write->v_scale, cache, &w.v_scale);
    if (st != KVX_STATUS_OK) return st;
  }
  *empty = T == 0 || D == 0 || (H == 0 && Hq == 0);
  if (*empty) return KVX_STATUS_OK;
  if (!is_index(write->slots.dtype) || !is_index(rope->position_dtype))
    return KVX_STATUS_INVALID_ARGUMENT;
  if (cache->block_size == 0 || rope->positions == nullptr ||
      (rope->rot_dim > 0 && rope->inv_freq == nullptr) || write->slots.slots == nullptr ||
      (H > 0 && (write->io.key.data == nullptr || write->io.value.data == nullptr ||
                 cache->k.data == nullptr || cache->v.data == nullptr)) ||
      (Hq > 0 && (rope->query.data == nullptr || rope->query_out.data == nullptr)))
    return KVX_STATUS_INVALID_ARGUMENT;
  w.src_k = write->io.key.data;
  w.src_v = write->io.value.data;
  w.dst_k = cache->k.data;
  w.dst_v = cache->v.data;
  w.slots = write->slots.slots;
  w.num_tokens = T;
  w.slot_is64 = write->slots.dtype == KVX_DTYPE_S64;
  w.heads = (int32_t)H;
  w.head_dim = (int32_t)D;
  w.block_size = (int32_t)cache->block_size;
  w.num_blocks = (int32_t)cache->num_blocks;
  w.conv = is_fp8(cdt) ? kConvQuant : kConvCopy;
  w.io_dtype = io;
  w.cache_dtype = cdt;
  p->query = rope->query.data;
  p->query_out = rope->query_out.data;
  p->positions = rope->positions;
  p->inv_freq = rope->inv_freq;
  p->magnitude = rope->magnitude;
  p->position_is64 = rope->position_dtype == KVX_DTYPE_S64;
  p->query_heads = (int32_t)Hq;
  p->rot_dim = (int32_t)rope->rot_dim;
  p->interleaved = rope->style == KVX_ROPE_INTERLEAVED;
  return KVX_STATUS_OK;
}

// `pointers` false: the descriptors' data pointers are not looked at.
static kvx_status_t plan_attention(const kvx_cache_desc_t *cache, const kvx_attention_desc_t *a,
                                   bool pointers, AttentionPlan *p, bool *empty) {
  if (a == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
  kvx_status_t st = check_cache(cache);
  if (st != KVX_STATUS_OK) return st;
  if (a->size < sizeof(kvx_attention_desc_t) || a->block_table.size < sizeof(kvx_block_table_t) ||
      a->seq_lens.size < sizeof(kvx_seq_lens_t))
    return KVX_STATUS_INVALID_ARGUMENT;
  const kvx_dtype_t cdt = cache->k.dtype, io = a->query.dtype;
  if (a->out.dtype != io || !is_io_float(io) || (!is_fp8(cdt) && io != cdt))
    return KVX_STATUS_UNSUPPORTED;
  const kvx_block_table_t &tb = a->block_table;
  const kvx_block_table_format_t fmt = tb.format;
  if (fmt != KVX_BLOCK_TABLE_PACKED && fmt != KVX_BLOCK_TABLE_RAGGED &&
      fmt != KVX_BLOCK_TABLE_KV_OFFSETS)
    return KVX_STATUS_UNSUPPORTED;
  const int64_t T = a->query.ndim == 3 ? a->query.shape[0] : -1;
  const int64_t Hq = a->query.ndim == 3 ? a->query.shape[1] : -1;
  const int64_t H = cache->num_kv_heads, D = cache->head_dim, S = tb.seq_count;
  if (T < 0 || T > kMost32 || Hq < 0 || Hq > kMost32 || S > kMost32)
    return KVX_STATUS_INVALID_ARGUMENT;
  *p = AttentionPlan{};
  st = check_rows(a->query, T, Hq, D, &p->q_tok, &p->q_head);
  if (st != KVX_STATUS_OK) return st;
  st = check_rows(a->out, T, Hq, D, &p->o_tok, &p->o_head);
  if (st != KVX_STATUS_OK) return st;
  if (rows_overlap(T, Hq, D, p->o_tok, p->o_head)) return KVX_STATUS_UNSUPPORTED;
  if (H > 0 ? Hq % H != 0 : Hq != 0) return KVX_STATUS_INVALID_ARGUMENT;
  if (a->seq_lens.seq_count != tb.seq_count) return KVX_STATUS_INVALID_ARGUMENT;
  if (a->flags & ~(uint32_t)KVX_ATTENTION_CAUSAL) return KVX_STATUS_INVALID_ARGUMENT;
  const bool causal = (a->flags & KVX_ATTENTION_CAUSAL) != 0;
  if (a->window > kMost32 || (a->window > 0 && !causal)) return KVX_STATUS_INVALID_ARGUMENT;
  if (!(a->softcap >= 0.0f) || std::isinf(a->softcap) || a->max_seq_len > kMost32 || a->max_query_len > kMost32)
    return KVX_STATUS_INVALID_ARGUMENT;
  if (D > 512) return KVX_STATUS_UNSUPPORTED;
  GatherPlan &g = p->g;
  st = cache_geom(cache, &cache->k, &g.gk);
  if (st != KVX_STATUS_OK) return st;
  st = cache_geom(cache, &cache->v, &g.gv);
  if (st != KVX_STATUS_OK) return st;
  if (is_fp8(cdt)) {
    // Without pointers a descriptor's data may be NULL: anything stands for it.
    static const float kSome = 1.0f;
    kvx_scale_desc_t ks = a->k_scale, vs = a->v_scale;
    if (!pointers) ks.data = vs.data = &kSome;
    const bool block_ok = fmt != KVX_BLOCK_TABLE_KV_OFFSETS;
    st = resolve_scale_desc(&ks, cache, block_ok, &g.k_scale);
    if (st != KVX_STATUS_OK) return st;
    st = resolve_scale_desc(&vs, cache, block_ok, &g.v_scale);
    if (st != KVX_STATUS_OK) return st;
  }
  *empty = T == 0 || Hq == 0 || D == 0 || S == 0;
  if (*empty) return KVX_STATUS_OK;
  if (!is_index(tb.index_dtype) || !is_index(a->seq_lens.dtype))
    return KVX_STATUS_INVALID_ARGUMENT;
  const kvx_pool_blocks_t *pools = a->pool_blocks;
  if (pools != nullptr && (pools->size < sizeof(kvx_pool_blocks_t) || pools->primary < 0 ||
                           pools->secondary < 0))
    return KVX_STATUS_INVALID_ARGUMENT;
  if (cache->block_size == 0) return KVX_STATUS_INVALID_ARGUMENT;
  const int64_t bs = cache->block_size;
  if (fmt == KVX_BLOCK_TABLE_KV_OFFSETS) {
    if (tb.index_dtype != KVX_DTYPE_S32 || (tb.flags & KVX_BLOCK_TABLE_FLAG_KVCACHEINDEX) == 0 ||
        tb.beam_width == 0)
      return KVX_STATUS_INVALID_ARGUMENT;
    if (tb.beam_width != 1) return KVX_STATUS_UNSUPPORTED;
    if ((bs & (bs - 1)) != 0 || cache->pool.bytes_per_block == 0 ||
        (pointers && cache->pool.primary == nullptr) ||
        (uint64_t)tb.indices_count != (uint64_t)tb.seq_count * 2u * tb.max_blocks_per_seq)
      return KVX_STATUS_INVALID_ARGUMENT;
    const int esize = dtype_size(cdt);
    if (!block_fits(g.gk, bs, H, D, esize, cache->pool.bytes_per_block) ||
        !block_fits(g.gv, bs, H, D, esize, cache->pool.bytes_per_block))
      return KVX_STATUS_INVALID_ARGUMENT;
  } else if (tb.index_dtype != a->seq_lens.dtype) {
    return KVX_STATUS_INVALID_ARGUMENT;
  }
  if (fmt == KVX_BLOCK_TABLE_RAGGED) {
    if (!is_index(tb.indptr_dtype) || (pointers && tb.indptr == nullptr) ||
        (int64_t)tb.indptr_count != S + 1)
      return KVX_STATUS_INVALID_ARGUMENT;
  } else if (tb.max_blocks_per_seq > kMost32 || tb.max_blocks_per_seq * bs > kMost32 - 65536) {
    return KVX_STATUS_UNSUPPORTED;  // token numbers are 32-bit
  }
  if (a->query_indptr != nullptr ? !is_index(a->query_indptr_dtype) : T != S)
    return KVX_STATUS_INVALID_ARGUMENT;
  if (a->query_indptr != nullptr && T + S > kMost32)
    return KVX_STATUS_UNSUPPORTED;  // tile numbers are 32-bit
  if (pointers &&
      (a->query.data == nullptr || a->out.data == nullptr || a->seq_lens.lengths == nullptr ||
       (fmt != KVX_BLOCK_TABLE_KV_OFFSETS &&
        (cache->k.data == nullptr || cache->v.data == nullptr)) ||
       (tb.indices == nullptr &&
        (fmt == KVX_BLOCK_TABLE_PACKED ? tb.max_blocks_per_seq > 0 : tb.indices_count > 0))))
    return KVX_STATUS_INVALID_ARGUMENT;

  g.src_k = cache->k.data;
  g.src_v = cache->v.data;
  g.block_table = tb.indices;
  g.seq_lens = a->seq_lens.lengths;
  g.indptr = tb.indptr;
  g.table_count = tb.indices_count;
  g.pool[0] = static_cast<const char *>(cache->pool.primary);
  g.pool[1] = static_cast<const char *>(cache->pool.secondary);
  g.bytes_per_block = cache->pool.bytes_per_block;
  const int64_t nb = cache->num_blocks;
  const int64_t counts[2] = {pools ? pools->primary : 0, pools ? pools->secondary : 0};
  for (int i = 0; i < 2; ++i)
    g.pool_blocks[i] = (int32_t)(counts[i] > 0 && counts[i] < nb ? counts[i] : nb);
  g.format = fmt;
  g.index_is64 = tb.index_dtype == KVX_DTYPE_S64;
  g.indptr_is64 = tb.indptr_dtype == KVX_DTYPE_S64;
  g.lens_is64 = a->seq_lens.dtype == KVX_DTYPE_S64;
  g.seq_count = (int32_t)S;
  g.max_blocks_per_seq = (int32_t)tb.max_blocks_per_seq;
  g.heads = (int32_t)H;
  g.head_dim = (int32_t)D;
  g.block_size = (int32_t)bs;
  g.num_blocks = (int32_t)nb;
  g.io_dtype = io;
  g.cache_dtype = cdt;
  p->query = a->query.data;
  p->out = a->out.data;
  p->lse = a->lse;
  p->query_indptr = a->query_indptr;
  p->workspace = a->workspace;
  p->scale = a->scale;
  p->softcap = a->softcap;
  p->indptr_is64 = a->query_indptr_dtype == KVX_DTYPE_S64;
  p->tokens = (int32_t)T;
  p->query_heads = (int32_t)Hq;
  p->causal = causal;
  p->window = (int32_t)a->window;
  p->max_seq_len = (int32_t)a->max_seq_len;
  p->max_query_len = (int32_t)(a->query_indptr == nullptr ? 1 : a->max_query_len);
  return KVX_STATUS_OK;
}

}  // namespace kvx

// kvx_ext.h's structs on LP64.
static_assert(sizeof(kvx_rope_desc_t) == 264, "abi");
static_assert(offsetof(kvx_rope_desc_t, positions) == 24, "abi");
static_assert(offsetof(kvx_rope_desc_t, query) == 40, "abi");
static_assert(sizeof(kvx_attention_desc_t) == 592, "abi");
static_assert(offsetof(kvx_attention_desc_t, lse) == 232, "abi");
static_assert(offsetof(kvx_attention_desc_t, block_table) == 272, "abi");
static_assert(offsetof(kvx_attention_desc_t, k_scale) == 360, "abi");
static_assert(offsetof(kvx_attention_desc_t, workspace) == 576, "abi");

extern "C" {

KVX_API kvx_status_t kvx_launch_rope_write_kv(const kvx_cache_desc_t *cache,
                                              const kvx_write_desc_t *write,
                                              const kvx_rope_desc_t *rope, void *stream) {
  kvx::RopePlan p;
  bool empty = false;
  const kvx_status_t st = kvx::plan_rope(cache, write, rope, &p, &empty);
  if (st != KVX_STATUS_OK || empty) return st;
  return kvx::enqueue_rope_write(p, stream);
}

KVX_API kvx_status_t kvx_attention_workspace_size(const kvx_cache_desc_t *cache,
                                                  const kvx_attention_desc_t *attention,
                                                  uint64_t *out_bytes) {
  if (out_bytes == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
  kvx::AttentionPlan p;
  bool empty = false;
  const kvx_status_t st = kvx::plan_attention(cache, attention, false, &p, &empty);
  if (st != KVX_STATUS_OK) return st;
  *out_bytes = empty ? 0 : kvx::attention_workspace_bound(p);
  return KVX_STATUS_OK;
}

KVX_API kvx_status_t kvx_launch_attention(const kvx_cache_desc_t *cache,
                                          const kvx_attention_desc_t *attention, void *stream) {
  kvx::AttentionPlan p;
  bool empty = false;
  const kvx_status_t st = kvx::plan_attention(cache, attention, true, &p, &empty);
  if (st != KVX_STATUS_OK || empty) return st;
  const uint64_t need = kvx::attention_workspace(p);
  if (need > 0 && (p.workspace == nullptr || attention->workspace_size < need ||
                   (uintptr_t)p.workspace % 16 != 0))
    return KVX_STATUS_INVALID_ARGUMENT;
  return kvx::enqueue_attention(p, stream);
}

KVX_API kvx_status_t kvx_launch_copy_blocks(const kvx_cache_desc_t *const *caches,
                                            uint32_t cache_count, const void *pairs,
                                            kvx_dtype_t index_dtype, uint32_t pair_count,
                                            void *stream) {
  if (caches == nullptr && cache_count > 0) return KVX_STATUS_INVALID_ARGUMENT;
  if (!kvx::is_index(index_dtype)) return KVX_STATUS_INVALID_ARGUMENT;
  if (pair_count > kvx::kMost32) return KVX_STATUS_INVALID_ARGUMENT;
  try {
    std::vector<kvx::CopyTensor> tensors;
    tensors.reserve(2 * (size_t)cache_count);
    for (uint32_t i = 0; i < cache_count; ++i) {
      const kvx_cache_desc_t *c = caches[i];
      kvx_status_t st = kvx::check_cache(c);
      if (st != KVX_STATUS_OK) return st;
      for (const kvx_tensor_desc_t *t : {&c->k, &c->v}) {
        kvx::CopyTensor x{};
        st = kvx::cache_geom(c, t, &x.g);
        if (st != KVX_STATUS_OK) return st;
        if (c->block_size == 0) return KVX_STATUS_INVALID_ARGUMENT;
        if (c->num_blocks == 0 || c->num_kv_heads == 0 || c->head_dim == 0) continue;
        if (t->data == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
        if (t == &c->v && c->v.data == c->k.data) continue;  // one pool for both
        x.data = static_cast<char *>(t->data);
        x.num_blocks = c->num_blocks;
        x.block_size = (int32_t)c->block_size;
        x.heads = (int32_t)c->num_kv_heads;
        x.head_dim = (int32_t)c->head_dim;
        x.esize = kvx::dtype_size(t->dtype);
        tensors.push_back(x);
      }
    }
    if (tensors.empty() || pair_count == 0) return KVX_STATUS_OK;
    if (pairs == nullptr) return KVX_STATUS_INVALID_ARGUMENT;
    return kvx::enqueue_copy_blocks(tensors.data(), (int64_t)tensors.size(), pairs,
                                    index_dtype == KVX_DTYPE_S64, pair_count, stream);
  } catch (...) {  // no memory for the list
    return KVX_STATUS_INTERNAL_ERROR;
  }
}

}  // extern "C"
