/*
 * Extensions to the KVX v1 ABI that kvx_abi.h cannot carry unchanged.
 *
 * FP8 KV cache (OCP E4M3 "e4m3fn", KVX_DTYPE_F8_E4M3, or OCP E5M2,
 * KVX_DTYPE_F8_E5M2) with F32 scales:
 *
 *   write:  kvx_launch_write_kv / kvx_launch_write_kv_prefill with an FP8
 *           cache and io of dtype F16, BF16 or F32.  The scale is read from
 *           write->k_scale_desc / v_scale_desc when their `data` is non-NULL,
 *           otherwise from write->k_scale / v_scale as one F32 each
 *           (KVX_SPEC.md:258-259).  Scale pointers are device pointers, read
 *           by the kernel.
 *             q = fp8_rne(saturate(f32(x) / scale))
 *           saturating to +-448 (E4M3) / +-57344 (E5M2), infinities included;
 *           NaN -> 0x7F (E4M3) / 0x7E (E5M2).  With io of the cache's own
 *           FP8 dtype the bytes are copied unscaled.
 *
 *   gather: kvx_launch_gather_kv_dequant below, because kvx_gather_desc_t
 *           (reference kvx_abi.h:182-188) has no scale fields.
 *             y = round_to_io_dtype(f32(q) * scale)   (RNE; NaN -> quiet NaN)
 *           kvx_launch_gather_kv with an FP8 cache and the same FP8 io copies
 *           bytes.
 *
 * Scale descriptors (kvx_scale_desc_t, dtype F32; strides in elements; the
 * field names are the spec's, KVX_SPEC.md:190-197, the shapes this build's):
 *   PER_TENSOR      data[0]
 *   PER_HEAD        ndim 1, shape [num_kv_heads]
 *   PER_BLOCK       ndim 1, shape [num_blocks], indexed by physical block id
 *   PER_BLOCK_HEAD  ndim 2, shape [num_blocks, num_kv_heads]
 * A wrong shape is KVX_STATUS_INVALID_ARGUMENT; other granularities and
 * dtypes, and block-indexed scales on KV_OFFSETS gathers, are
 * KVX_STATUS_UNSUPPORTED.
 *
 * The reference has no FP8 kernels (KVX_CONFORMANCE.md:24, :35); this is new
 * functionality.
 *
 * Block-table formats beyond PACKED (KVX_SPEC.md:99-122), gathered by
 * kvx_launch_gather_kv, kvx_launch_gather_kv_dequant and kvx_gather_kv (the
 * reference returns UNSUPPORTED for them, kernels/kvx_paged_kv.cu:788-790):
 *   RAGGED      row t of sequence s is token indptr[s] + t, valid for
 *               t < indptr[s+1] - indptr[s]; its block id is indices[token]
 *               (skipped when < 0 or >= num_blocks), its offset t % block_size.
 *   KV_OFFSETS  int32 KVCacheIndex entries [seq_count, 1, 2, max_blocks_per_seq]
 *               (K then V): bit 31 selects the secondary pool, bits 0-30 the
 *               block; the block's address is pool + index * bytes_per_block.
 *               An entry is skipped when its index is >= num_blocks or its
 *               pool is NULL.  kvx_pool_desc_t carries no pool sizes, so
 *               through kvx_launch_gather_kv, kvx_launch_gather_kv_dequant and
 *               kvx_gather_kv BOTH pools must hold at least num_blocks blocks
 *               of bytes_per_block bytes: a smaller secondary pool (an offload
 *               pool, say) is read out of bounds by indices between its size
 *               and num_blocks.  kvx_launch_gather_kv_pools below takes each
 *               pool's block count and skips the entries past it.
 */
#ifndef KVX_EXT_H
#define KVX_EXT_H

#include "kvx_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Dequantizing gather from an F8_E4M3 or F8_E5M2 paged cache into an
 * F16/BF16/F32 [seq_count, max_seq_len, H, D] buffer, over any block-table
 * format.  Same validation order, codes and untouched-row semantics as
 * kvx_launch_gather_kv; k_scale / v_scale must be non-NULL F32 scale
 * descriptors (granularities above) whose data is a device pointer.
 * No reference counterpart (the reference gather returns UNSUPPORTED for FP8,
 * kernels/kvx_paged_kv.cu:900-909). */
KVX_API kvx_status_t kvx_launch_gather_kv_dequant(
    const kvx_cache_desc_t *cache, const kvx_gather_desc_t *gather,
    const kvx_scale_desc_t *k_scale, const kvx_scale_desc_t *v_scale,
    void *stream);

/* Block counts of the two pools of a KV_OFFSETS table (kvx_pool_desc_t,
 * reference kvx_abi.h:84-90, has none).  A count of 0, or one of
 * num_blocks or more, means num_blocks. */
typedef struct kvx_pool_blocks_t {
  uint32_t size; /* sizeof(kvx_pool_blocks_t) */
  uint32_t reserved;
  int64_t primary;   /* blocks in cache->pool.primary */
  int64_t secondary; /* blocks in cache->pool.secondary */
} kvx_pool_blocks_t;

/* kvx_launch_gather_kv (k_scale and v_scale NULL) or
 * kvx_launch_gather_kv_dequant (both non-NULL), with a KV_OFFSETS entry also
 * skipped when its index is at or past its pool's count in pool_blocks, so
 * that a secondary pool smaller than num_blocks is never read past its end.
 * pool_blocks may be NULL (no narrowing); it is not read for PACKED and
 * RAGGED tables.  KVX_STATUS_INVALID_ARGUMENT for a pool_blocks->size below
 * sizeof(kvx_pool_blocks_t), a negative count, or one scale descriptor
 * without the other; otherwise the same validation order and codes as the
 * gather it stands for.  No reference counterpart: an extension for callers
 * whose KV_OFFSETS pools differ in size (an offload pool beside the
 * primary one). */
KVX_API kvx_status_t kvx_launch_gather_kv_pools(
    const kvx_cache_desc_t *cache, const kvx_gather_desc_t *gather,
    const kvx_pool_blocks_t *pool_blocks, const kvx_scale_desc_t *k_scale,
    const kvx_scale_desc_t *v_scale, void *stream);

/* ---------------------------------------------------------------------------
 * Operators of a serving step beside the write and the gather.  No reference
 * counterparts.  Their tensors are device memory: a KVX_MEMORY_HOST tensor
 * descriptor is KVX_STATUS_INVALID_ARGUMENT.  Asynchronous on `stream`, which
 * belongs to the current device; capturable into a HIP graph.
 */

/* Which elements of a head rotate together. */
typedef enum kvx_rope_style KVX_ENUM_BASE {
  KVX_ROPE_HALF = 0,       /* i and i + rot_dim / 2 */
  KVX_ROPE_INTERLEAVED = 1 /* 2 i and 2 i + 1 */
} kvx_rope_style_t;

/* Rotary positions.  Pair i of a row at position p turns by the angle
 * p * inv_freq[i], which is reduced by whole turns in 64 bits:
 *   (x0, x1) -> magnitude * (x0 cos - x1 sin, x1 cos + x0 sin);
 * elements from rot_dim on stay as they are.  inv_freq carries any scaling
 * for long contexts. */
typedef struct kvx_rope_desc {
  uint32_t size; /* sizeof(kvx_rope_desc_t) */
  kvx_rope_style_t style;
  uint32_t rot_dim; /* even, at most head_dim and 8192 */
  float magnitude;
  kvx_dtype_t position_dtype; /* S32 or S64 */
  uint32_t reserved;
  const void *positions;   /* [num_tokens] */
  const float *inv_freq;   /* F32 [rot_dim / 2] */
  kvx_tensor_desc_t query; /* [num_tokens, query_heads, head_dim]; ndim 0: none */
  kvx_tensor_desc_t query_out; /* same shape; the query itself or apart from it */
} kvx_rope_desc_t;

/* Rotates query rows into query_out and key rows into the paged cache, and
 * writes the value rows beside them: kvx_launch_write_kv of the rotated keys
 * without a round trip through memory, each value rounded once from 32 bits.
 * `write` is that call's descriptor, except that key, value, query and
 * query_out may have any token and head strides (elements of a head are
 * adjacent), as views of one projection's output have.  Rows whose slot is
 * skipped by the write are skipped in the cache; their queries are rotated.
 * The query has the dtype of key and value. */
KVX_API kvx_status_t kvx_launch_rope_write_kv(const kvx_cache_desc_t *cache,
                                              const kvx_write_desc_t *write,
                                              const kvx_rope_desc_t *rope, void *stream);

typedef enum kvx_attention_flags KVX_ENUM_BASE {
  KVX_ATTENTION_CAUSAL = 1 << 0
} kvx_attention_flags_t;

/* Attention of new tokens over a paged cache that holds them already.
 * Sequence s has the query rows query_indptr[s] .. query_indptr[s + 1] - 1
 * (NULL: the one row s) and seq_lens[s] cached tokens, its query rows' own
 * among them: its row i of n is at position p = seq_lens[s] - n + i.  It
 * attends to the cached tokens t < seq_lens[s], with KVX_ATTENTION_CAUSAL to
 * t <= p, with a window also t > p - window:
 *   x_t = scale * q . k_t, softcap > 0: softcap * tanh(x_t / softcap),
 *   out = sum_t softmax(x)_t v_t,   lse = ln sum_t exp(x_t).
 * Query head h reads kv head h / (query heads / num_kv_heads).  Tokens that a
 * gather would skip (a block id out of range, no table entry, past the RAGGED
 * count) are not attended to.  A row that attends to nothing is 0 with lse
 * -infinity.  Rows behind the last sequence are left as they were.  Scales of
 * blocks that a row attends to nothing of may be anything, as their tokens may.
 * Sums and softmax statistics are F32, and so are logits: past 9e7 (F16 queries;
 * else 1e9) in size their rounding alone leaves the weights' range, and a row may
 * turn NaN. */
typedef struct kvx_attention_desc {
  uint32_t size;  /* sizeof(kvx_attention_desc_t) */
  uint32_t flags; /* kvx_attention_flags_t */
  kvx_tensor_desc_t query; /* [num_tokens, query_heads, head_dim], F16/BF16/F32, the
                              cache's dtype unless that is FP8; elements of a head
                              adjacent, any other strides */
  kvx_tensor_desc_t out;   /* same shape and dtype; the query itself or apart from it */
  float *lse;              /* F32 [num_tokens, query_heads], or NULL */
  const void *query_indptr; /* [seq_count + 1] row numbers, or NULL */
  kvx_dtype_t query_indptr_dtype; /* S32 or S64 */
  uint32_t window;         /* tokens seen, its own included; 0: all.  Causal only */
  float scale;
  float softcap;           /* 0: none; any finite one.  Past 64 (F16; BF16: 512) chunks take
                              longer */
  uint32_t max_seq_len;    /* largest sequence and most query rows of one, as far as */
  uint32_t max_query_len;  /* known (0: not): they steer the split, not the result */
  kvx_block_table_t block_table; /* PACKED, RAGGED or KV_OFFSETS, as a gather's */
  kvx_seq_lens_t seq_lens;
  kvx_scale_desc_t k_scale; /* of an FP8 cache, as the dequantizing gather's */
  kvx_scale_desc_t v_scale;
  const kvx_pool_blocks_t *pool_blocks; /* KV_OFFSETS, or NULL */
  void *workspace;         /* device memory, 16-byte aligned, for this call alone */
  uint64_t workspace_size; /* at least kvx_attention_workspace_size's */
} kvx_attention_desc_t;

/* Bytes of workspace that kvx_launch_attention needs for these descriptors;
 * of the data pointers only whether query_indptr is NULL matters, and the
 * workspace fields themselves are not read. */
KVX_API kvx_status_t kvx_attention_workspace_size(const kvx_cache_desc_t *cache,
                                                  const kvx_attention_desc_t *attention,
                                                  uint64_t *out_bytes);

/* Runs the attention.  Head dims to 512 elements.  KVX_STATUS_INVALID_ARGUMENT
 * for a workspace that is too small; otherwise checks and codes as the gather. */
KVX_API kvx_status_t kvx_launch_attention(const kvx_cache_desc_t *cache,
                                          const kvx_attention_desc_t *attention, void *stream);

/* Copies blocks inside caches (the layers of a model): for every pair
 * (src, dst) = pairs[2 i], pairs[2 i + 1] of block ids, block src of K and of
 * V to block dst, in each of cache_count caches.  Pairs with an id outside
 * [0, num_blocks) are skipped.  No dst may be another pair's src or dst.
 * Block-indexed scales are not copied.  Caches may differ in everything. */
KVX_API kvx_status_t kvx_launch_copy_blocks(const kvx_cache_desc_t *const *caches,
                                            uint32_t cache_count, const void *pairs,
                                            kvx_dtype_t index_dtype, uint32_t pair_count,
                                            void *stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* KVX_EXT_H */
