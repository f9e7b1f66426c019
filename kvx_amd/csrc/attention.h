// What the kernels of the attention over a paged cache share: their
// arguments, the map from workgroups to query rows, and the map from token
// numbers to cache rows.
//
// Rows.  A kv head's query rows are its `group` query heads at each new token.
// A workgroup takes a tile of them: `tile_tokens` tokens by `tile_heads` heads
// (the group, or a part of one wider than the tile), all of which read the
// same keys and values.  The host knows only how many tiles there can be; each
// workgroup counts those of the sequences before its own (of the sequences that
// its kernel takes), so that the ones that are left over lie together.
// Scattered among the others they would cost far more than their own time:
// workgroups go round the machine in order, and a part of it would get all of
// them and run empty (64 sequences of 4 drafts at 2048 tokens: 155 us instead of
// 99).  Counting many sequences takes time as well: where they are said to have
// one tile each, or are more than 256 and have few rows, the first tile of each
// has the sequence's number and only further ones are counted (1024 sequences
// of one token at 200: 226 us instead of 291, without the hint 252 instead of
// 307).
//
// Splits.  Where the tiles alone do not fill the machine, a tile's tokens are
// divided among `splits` workgroups.  Each writes its unnormalised sum, its
// maximum and its sum of weights to the workspace, and
// attention_join_kernel adds them up.
//
// Logits are kept in units of log2, so that a weight is one exp2.
#pragma once

#include <hip/hip_runtime.h>

#include "kernels.h"
#include "operators_internal.h"

namespace kvx {
namespace dev {

constexpr int kRowTile = 16;       // rows of a tile of the kernels for few rows
constexpr int kManyRowTile = 128;  // and of the one for many
constexpr float near_cap(int io) { return io == KVX_DTYPE_BF16 ? 512.0f : 64.0f; }  // see cap_logits
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

constexpr int kDies = 8;  // that take workgroups in turn

struct AttentionArgs {
  // cache and table
  const char *k, *v;
  const char *pool[2];
  int64_t bytes_per_block;
  int64_t table_count;
  const void *table, *indptr, *lens;
  GeomBytes gk, gv;
  ScaleRef ks, vs;
  int32_t pool_blocks[2];
  int32_t format, index64, indptr64, lens64;
  int32_t max_blocks, block_size, block_log2, num_blocks;  // block_log2 < 0: not a power of two
  int32_t entry_log2;    // bytes of a table entry
  int64_t entry_second;  // from an entry's low word (or K's entry) to its high (V's)
  // queries; strides in bytes
  const char *q;
  char *out;
  float *lse;
  const void *qptr;
  int64_t q_tok, q_head, o_tok, o_head;
  int32_t qptr64;
  int32_t seqs, tokens, heads, group, head_dim;
  int32_t causal, window;
  float scale, softcap;  // as given; softcap 0: none
  float scale_log2;  // scale * log2 e
  float cap, cap_in; // softcap / 4 * log2 e (finite for any softcap), scale / softcap
  float scale_rest, cap_rest;  // what rounding left of scale_log2 and cap
  // tiles
  int32_t tile_heads, head_tiles, tile_tokens, tiles;
  int32_t least_rows, most_rows;  // new tokens of the sequences this kernel takes
  int32_t splits;
  int32_t split_steps;  // least steps of 64 tokens in a split
  int32_t first_tiles; // each sequence's first tile has its number, others follow
  int32_t heads_near;  // the heads of a tile's part run on one die (few rows)
  int32_t part_rows;  // partial row of (s, i): s * part_rows + i; 0: the row number
  float *part_o;      // [partial row, query head, split, head_dim]
  float *part_ml;     // the same without head_dim: (maximum, sum of weights)
  int32_t chunk_k;    // keys' elements load four at a time (rows kernel)
};

struct QueryTile {
  int32_t seq;
  int32_t first;   // first row of the tile in its sequence
  int32_t count;   // tokens of the tile
  int64_t begin;   // row number of the sequence's first row
  int32_t rows;    // the sequence's new tokens
  int64_t length;  // its cached tokens, as given
  int32_t usable;  // of those, the ones the table can hold
  const char *entries;  // its table entries: one per block (RAGGED: per token)
};

__device__ __forceinline__ int64_t index_at(const void *p, bool is64, int64_t i) {
  return is64 ? static_cast<const int64_t *>(p)[i] : (int64_t)static_cast<const int32_t *>(p)[i];
}

__device__ __forceinline__ int64_t query_begin(const AttentionArgs &a, int64_t s) {
  const int64_t b = index_at(a.qptr, a.qptr64, s);
  return b < 0 ? 0 : b > a.tokens ? a.tokens : b;
}

// The last s in [0, seqs) for which `before(s)`, a property that holds up to
// some s, is true (0 where it never is): 64 pivots at a time.  Uniform over
// the wave, all of whose lanes call.
template <typename F>
__device__ __forceinline__ int last_sequence(int seqs, const F &before) {
  const int lane = (int)(threadIdx.x % kWave);
  int lo = 0, span = seqs;
  while (span > 1) {
    const int step = (span + kWave - 1) / kWave;
    const int hits = __popcll(__ballot(lane * step < span && before(lo + lane * step)));
    const int at = hits > 0 ? hits - 1 : 0;
    lo += at * step;
    span = min(step, span - at * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// The sequence and rows of a tile, or false behind the last one.  A lane counts
// the tiles of four sequences, without the first `skip` of each, and the wave
// scans the sums.
__device__ __forceinline__ bool find_rows(const AttentionArgs &a, int tile, int skip,
                                          QueryTile *t) {
  constexpr int kEach = 4;
  const int lane = (int)(threadIdx.x % kWave);
  int left = tile;  // behind the tiles counted so far
  for (int s0 = 0; s0 < a.seqs; s0 += kEach * kWave) {
    const int s = s0 + kEach * lane;
    int64_t begin[kEach + 1];
    int count[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i <= kEach; ++i) begin[i] = query_begin(a, min(s + i, a.seqs));
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int64_t n = begin[i + 1] - begin[i];
      const bool mine = n > 0 && n >= a.least_rows && n <= a.most_rows;
      count[i] =
          mine ? (int)((uint32_t)(n + a.tile_tokens - 1) / (uint32_t)a.tile_tokens) - skip : 0;
      sum += count[i];
    }
    int upto = sum;
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const int x = __shfl_up(upto, d);
      upto += lane >= d ? x : 0;
    }
    const int from = __builtin_amdgcn_readfirstlane(__popcll(__ballot(upto <= left)));
    if (from < kWave) {
      left -= __builtin_amdgcn_readlane(upto - sum, from);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int c = __builtin_amdgcn_readlane(count[i], from);
        if (left < c) {
          const int b = __builtin_amdgcn_readlane((int)begin[i], from);
          t->seq = s0 + kEach * from + i;
          t->begin = b;
          t->rows = __builtin_amdgcn_readlane((int)begin[i + 1], from) - b;
          t->first = (left + skip) * a.tile_tokens;
          t->count = min(a.tile_tokens, t->rows - t->first);
          return true;
        }
        left -= c;
      }
    }
    left -= __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return false;
}

// The tile with number `tile`, or false where it has no rows or another
// kernel takes its sequence.  Uniform over the wave, all of whose lanes call.
__device__ __forceinline__ bool find_tile(const AttentionArgs &a, int tile, QueryTile *t) {
  if (a.qptr == nullptr) {
    t->seq = tile;
    t->first = 0;
    t->count = 1;
    t->begin = tile;
    t->rows = 1;
  } else if (a.first_tiles && tile < a.seqs) {
    const int64_t b = query_begin(a, tile), n = query_begin(a, tile + 1) - b;
    if (n <= 0 || n < a.least_rows || n > a.most_rows) return false;
    t->seq = tile;
    t->first = 0;
    t->count = (int32_t)min(n, (int64_t)a.tile_tokens);
    t->begin = b;
    t->rows = (int32_t)n;
  } else {
    const int skip = a.first_tiles ? 1 : 0;
    if (!find_rows(a, tile - skip * a.seqs, skip, t)) return false;
  }
  t->length = index_at(a.lens, a.lens64, t->seq);
  int64_t hold, first;
  if (a.format == KVX_BLOCK_TABLE_RAGGED) {
    first = index_at(a.indptr, a.indptr64, t->seq);
    hold = index_at(a.indptr, a.indptr64, t->seq + 1);
    hold = first < 0 ? 0 : min(hold, a.table_count) - first;
    if (hold > 0x7FFF0000) hold = 0x7FFF0000;
  } else {
    first = (int64_t)t->seq * a.max_blocks * (a.format == KVX_BLOCK_TABLE_KV_OFFSETS ? 2 : 1);
    hold = (int64_t)a.max_blocks * a.block_size;
  }
  hold = min(hold, t->length);
  t->usable = hold < 0 ? 0 : (int32_t)hold;
  t->entries = static_cast<const char *>(a.table) + first * (a.index64 ? 8 : 4);
  return true;
}

// Tokens [lo, hi) that row i of the sequence attends to.
__device__ __forceinline__ void row_range(const AttentionArgs &a, const QueryTile &t, int i,
                                          int *lo, int *hi) {
  *lo = 0;
  *hi = t.usable;
  if (!a.causal) return;
  const int64_t pos = t.length - t.rows + i;
  if (pos + 1 < t.usable) *hi = pos < 0 ? 0 : (int)(pos + 1);
  if (a.window > 0 && pos - a.window + 1 > 0)
    *lo = (int)min(pos - a.window + 1, (int64_t)t.usable);
}

// Tokens of split z of a tile that sees [lo, hi): split_steps steps of 64 each, or
// more where the sequence is longer than the host knew; from a multiple of 64 on.
__device__ __forceinline__ void split_range(const AttentionArgs &a, int lo, int hi, int z,
                                            int *from, int *to) {
  const int start = lo & ~63;
  if (hi <= lo) {
    *from = *to = start;
    return;
  }
  const int steps = (hi - start + 63) >> 6;
  const int per = max((steps + a.splits - 1) / a.splits, a.split_steps);
  *from = (int)min((int64_t)start + (int64_t)z * per * 64, (int64_t)hi);
  *to = (int)min((int64_t)start + (int64_t)(z + 1) * per * 64, (int64_t)hi);
}

// Table entry of token `at` of a sequence, as loaded: nothing looks at it, so
// that the load stays in flight until token_rows does.  `at` < the sequence's
// usable tokens.
struct TokenEntry {
  uint32_t lo, hi;  // an id's words (hi = lo for 32 bits); KV_OFFSETS: of K and of V
};

__device__ __forceinline__ TokenEntry token_entry(const AttentionArgs &a, const QueryTile &t,
                                                  int at) {
  uint32_t i = (uint32_t)at;
  if (a.format != KVX_BLOCK_TABLE_RAGGED)
    i = a.block_log2 >= 0 ? i >> a.block_log2 : i / (uint32_t)a.block_size;
  const char *p = t.entries + ((int64_t)i << a.entry_log2);
  return {*reinterpret_cast<const uint32_t *>(p),
          *reinterpret_cast<const uint32_t *>(p + a.entry_second)};
}

// Where the token with that entry lies: the addresses of its K and V rows (head
// 0), or false for a token that is not there.  `block` is the physical block
// for block-indexed scales.
struct TokenRows {
  const char *k, *v;
  int32_t block;
};

__device__ __forceinline__ bool token_rows(const AttentionArgs &a, const TokenEntry &e, int at,
                                           TokenRows *r) {
  const int off = (int)(a.block_log2 >= 0 ? (uint32_t)at & (uint32_t)(a.block_size - 1)
                                          : (uint32_t)at % (uint32_t)a.block_size);
  const char *kb, *vb;
  if (a.format == KVX_BLOCK_TABLE_KV_OFFSETS) {
    const uint32_t ek = e.lo, ev = e.hi;
    // selected, not indexed: arguments stay in scalar registers
    const char *pk = ek >> 31 ? a.pool[1] : a.pool[0], *pv = ev >> 31 ? a.pool[1] : a.pool[0];
    const int32_t nk = ek >> 31 ? a.pool_blocks[1] : a.pool_blocks[0];
    const int32_t nv = ev >> 31 ? a.pool_blocks[1] : a.pool_blocks[0];
    const int32_t ik = (int32_t)(ek & 0x7FFFFFFFu), iv = (int32_t)(ev & 0x7FFFFFFFu);
    if (pk == nullptr || pv == nullptr || ik >= nk || iv >= nv) return false;
    kb = pk + ik * a.bytes_per_block;
    vb = pv + iv * a.bytes_per_block;
    r->block = 0;
  } else {
    const int64_t b = a.index64 ? (int64_t)(((uint64_t)e.hi << 32) | e.lo) : (int64_t)(int32_t)e.lo;
    if (b < 0 || b >= a.num_blocks) return false;
    kb = a.k + b * a.gk.s_block;
    vb = a.v + b * a.gv.s_block;
    r->block = (int32_t)b;
  }
  r->k = kb + off * a.gk.s_off;
  r->v = vb + off * a.gv.s_off;
  return true;
}

__device__ __forceinline__ float scale_of(const ScaleRef &s, int32_t block, int32_t head) {
  return s.p[s.indexed ? block * s.s_block + head * s.s_head : 0];
}

// Four times tanh of a raw product's logit over the softcap, to be multiplied by
// a.cap: good to a few units of F32 for every softcap.  A quotient, as scale /
// softcap may be subnormal or infinite.
__device__ __forceinline__ float capped_part(const AttentionArgs &a, float dot) {
  return 4.0f * tanhf(dot * a.scale / a.softcap);
}

// x = scale * q.k (in log2 units) of a raw product.
__device__ __forceinline__ float logit(const AttentionArgs &a, float dot) {
  if (a.softcap != 0.0f) return a.cap * capped_part(a, dot);
  return dot * a.scale_log2;
}

// One element of a cache or query tensor as f32.
template <int C>
__device__ __forceinline__ float value_at(const char *p) {
  if constexpr (C == KVX_DTYPE_F32) return *reinterpret_cast<const float *>(p);
  else if constexpr (C == KVX_DTYPE_BF16)
    return bf16_to_f32(*reinterpret_cast<const uint16_t *>(p));
  else if constexpr (C == KVX_DTYPE_F16) return (float)*reinterpret_cast<const _Float16 *>(p);
  else return decode_pair<C == KVX_DTYPE_F8_E5M2>((int)*reinterpret_cast<const uint8_t *>(p), false)[0];
}

template <int C>
constexpr int bytes_of_type() {
  return C == KVX_DTYPE_F32 ? 4 : C == KVX_DTYPE_BF16 || C == KVX_DTYPE_F16 ? 2 : 1;
}

template <int IO>
__device__ __forceinline__ void store_out(char *p, float x) {
  if constexpr (IO == KVX_DTYPE_F32) *reinterpret_cast<float *>(p) = x;
  else *reinterpret_cast<uint16_t *>(p) = (uint16_t)(pack_pair<IO>(f32x2{x, x}) & 0xFFFFu);
}

// Number of (row, head) among the partial results.
__device__ __forceinline__ int64_t part_index(const AttentionArgs &a, const QueryTile &t, int i,
                                              int head) {
  const int64_t row = a.part_rows > 0 ? (int64_t)t.seq * a.part_rows + i : t.begin + i;
  return row * (a.heads * a.group) + head;
}

// Other lanes of the wave see what this one wrote to LDS.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A launch of one of the kernels.
struct AttentionPart {
  AttentionArgs a;
  uint32_t grid;  // workgroups
  bool stream;    // few rows: no two tiles read the same keys and values
};

void run_attention_rows(const AttentionPart &p, int io, int cache, hipStream_t s);
// vt: values with the token axis innermost; grouped: blocks hold whole groups of
// the tokens that a wave loads together, whose rows follow from the first's
void run_attention_few_f32(const AttentionPart &p, bool vt, bool grouped, hipStream_t s);
void run_attention_few_f32_e4m3(const AttentionPart &p, bool vt, bool grouped, hipStream_t s);
void run_attention_few_f32_e5m2(const AttentionPart &p, bool vt, bool grouped, hipStream_t s);
void run_attention_few_bf16(const AttentionPart &p, bool vt, bool grouped, hipStream_t s);
void run_attention_few_bf16_e4m3(const AttentionPart &p, bool vt, bool grouped, hipStream_t s);
void run_attention_few_bf16_e5m2(const AttentionPart &p, bool vt, bool grouped, hipStream_t s);
void run_attention_few_f16(const AttentionPart &p, bool vt, bool grouped, hipStream_t s);
void run_attention_few_f16_e4m3(const AttentionPart &p, bool vt, bool grouped, hipStream_t s);
void run_attention_few_f16_e5m2(const AttentionPart &p, bool vt, bool grouped, hipStream_t s);
// few: sequences of few new tokens in the same launch, or null
void run_attention_many_bf16(const AttentionPart &p, const AttentionPart *few, bool vt,
                             bool grouped, hipStream_t s);
void run_attention_many_bf16_e4m3(const AttentionPart &p, const AttentionPart *few, bool vt,
                                  bool grouped, hipStream_t s);
void run_attention_many_bf16_e5m2(const AttentionPart &p, const AttentionPart *few, bool vt,
                                  bool grouped, hipStream_t s);
void run_attention_many_f16(const AttentionPart &p, const AttentionPart *few, bool vt,
                            bool grouped, hipStream_t s);
void run_attention_many_f16_e4m3(const AttentionPart &p, const AttentionPart *few, bool vt,
                                 bool grouped, hipStream_t s);
void run_attention_many_f16_e5m2(const AttentionPart &p, const AttentionPart *few, bool vt,
                                 bool grouped, hipStream_t s);

}  // namespace dev
}  // namespace kvx
