// Internal interface of the operators (kvx_ext.h's attention, rotary write and
// block copy): between operators.cpp and their kernels, and what operators.cpp
// shares with launch.cpp.  Apart from kvx_internal.h, so that the write's and
// gather's sources do not change with the operators'.  Nothing here is exported.
#pragma once

#include "kvx_internal.h"

namespace kvx {

// Everything the rotary write needs, already validated on the host.  `w`
// describes keys, values and their cache rows; strides are in elements.
struct RopePlan {
  WritePlan w;
  const void *query;
  void *query_out;
  const void *positions;
  const float *inv_freq;
  int64_t k_tok, k_head, v_tok, v_head;
  int64_t q_tok, q_head, o_tok, o_head;
  float magnitude;
  int32_t position_is64;
  int32_t query_heads;  // 0: no queries
  int32_t rot_dim;
  int32_t interleaved;
};

// Everything the attention needs, already validated on the host.  The cache
// and its table are described as a gather's (`g`: its dst, max_seq_len and conv
// are not used); strides are in elements.
struct AttentionPlan {
  GatherPlan g;
  const void *query;
  void *out;
  float *lse;
  const void *query_indptr;
  void *workspace;
  int64_t q_tok, q_head, o_tok, o_head;
  float scale;
  float softcap;
  int32_t indptr_is64;
  int32_t tokens;
  int32_t query_heads;
  int32_t causal;
  int32_t window;         // 0: none
  int32_t max_seq_len;    // hints, 0: not known
  int32_t max_query_len;
};

// One K or V tensor of a block copy.
struct CopyTensor {
  char *data;
  int64_t num_blocks;
  Geom g;
  int32_t block_size;
  int32_t heads;
  int32_t head_dim;
  int32_t esize;
};

// Enqueue the kernels on `stream`, as enqueue_write and enqueue_gather do.
kvx_status_t enqueue_rope_write(const RopePlan &plan, void *stream);
kvx_status_t enqueue_attention(const AttentionPlan &plan, void *stream);
kvx_status_t enqueue_copy_blocks(const CopyTensor *tensors, int64_t count, const void *pairs,
                                 bool index_is64, int64_t pair_count, void *stream);

// Bytes of workspace that enqueue_attention uses for the plan, whose pointers'
// alignment takes part in the choice of the kernel, and the most that it uses
// whatever that alignment is.  Neither reads through a pointer.
uint64_t attention_workspace(const AttentionPlan &plan);
uint64_t attention_workspace_bound(const AttentionPlan &plan);

// Checks and conversions that the entry points share (launch.cpp).
bool is_io_float(kvx_dtype_t dt);
bool is_fp8(kvx_dtype_t dt);
kvx_status_t fill_geom(const kvx_cache_desc_t *cache, const kvx_tensor_desc_t *t, Geom *g);
bool block_fits(const Geom &g, int64_t bs, int64_t heads, int64_t head_dim, int esize,
                int64_t pitch);
kvx_status_t resolve_scale_desc(const kvx_scale_desc_t *d, const kvx_cache_desc_t *cache,
                                bool block_ok, ScaleRef *out);
kvx_status_t resolve_write_scale(const kvx_scale_desc_t *desc, const void *raw,
                                 const kvx_cache_desc_t *cache, ScaleRef *out);

}  // namespace kvx
