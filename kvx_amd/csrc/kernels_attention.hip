// Host planning of the attention over a paged cache, and the kernel that
// joins the splits of a tile.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>

#include "attention.h"
#include "operators_internal.h"

namespace kvx {
namespace dev {
namespace {

constexpr int kMostSplits = 256;
constexpr double kLog2eWide = 1.44269504088896340736;

// Rows that have partial sums.
__host__ __device__ __forceinline__ int64_t join_rows(const AttentionArgs &a) {
  return a.part_rows > 0 ? (int64_t)a.seqs * a.part_rows : a.tokens;
}

// Adds up the splits of one row and head: with M the largest maximum,
//   out = sum_z 2^(m_z - M) o_z / sum_z 2^(m_z - M) l_z.
// A workgroup has a row and head.  Its threads weigh one split each, then take
// VEC elements of every G-th split, G as many as fit beside each other, and add
// the G sums up through LDS: loads of many splits are in flight at once.
template <int IO, int VEC, int kJoinThreads>
__device__ __forceinline__ void join_splits(const AttentionArgs &a, uint32_t unit) {
  __shared__ float weights[kJoinThreads];  // of the splits; < 0: nothing was written for it
  __shared__ float waves[2][kJoinThreads / kWave];
  __shared__ float sums[kJoinThreads * VEC];
  const int tid = (int)threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int hq = a.heads * a.group;
  const int64_t part = unit / (uint32_t)hq;
  const int head = (int)(unit % (uint32_t)hq);
  int64_t row = part;
  if (a.qptr != nullptr) {
    const int s = a.part_rows > 0 ? (int)(part / a.part_rows)
                                  : last_sequence(a.seqs, [&](int q) {
                                      return query_begin(a, q) <= part;
                                    });
    const int64_t b = query_begin(a, s), n = query_begin(a, s + 1) - b;
    if (a.part_rows > 0) row = b + part - (int64_t)s * a.part_rows;
    if (row < b || row >= b + n || n < a.least_rows || n > a.most_rows) return;
  }
  const int64_t at = (part * hq + head) * a.splits;
  const bool split = tid < a.splits;
  const float m = split ? a.part_ml[2 * (at + tid)] : -INFINITY;
  const float l = split ? a.part_ml[2 * (at + tid) + 1] : 0.0f;
  float top = m;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) waves[0][wave] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoinThreads / kWave; ++i) top = fmaxf(top, waves[0][i]);
  const float w = l == 0.0f ? -1.0f : exp2f(m - (top == -INFINITY ? 0.0f : top));
  weights[tid] = w;
  float total = l == 0.0f ? 0.0f : w * l;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) total += __shfl_xor(total, d);
  if (lane == 0) waves[1][wave] = total;
  __syncthreads();
  total = 0.0f;
#pragma unroll
  for (int i = 0; i < kJoinThreads / kWave; ++i) total += waves[1][i];
  const bool none = top == -INFINITY && total == 0.0f;

  const int columns = a.head_dim / VEC;
  int across = 1;  // threads of a split
  while (across < columns && across < kJoinThreads) across *= 2;
  const int g = tid / across, groups = kJoinThreads / across;
  for (int c0 = 0; c0 < columns; c0 += across) {
    const int c = c0 + tid % across;
    float sum[VEC] = {};
    if (c < columns) {
#pragma unroll 4
      for (int z = g; z < a.splits; z += groups) {
        const float by = weights[z];
        const Raw<4 * VEC> x =
            ld<4 * VEC>(reinterpret_cast<const char *>(a.part_o + (at + z) * a.head_dim + c * VEC));
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[j] = by < 0.0f ? sum[j] : fmaf(by, __uint_as_float(x.w[j]), sum[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) sums[tid * VEC + j] = sum[j];
    __syncthreads();
    for (int d = tid; d < across * VEC && c0 * VEC + d < a.head_dim; d += kJoinThreads) {
      float x = 0.0f;
      for (int i = 0; i < groups; ++i) x += sums[i * across * VEC + d];
      store_out<IO>(a.out + row * a.o_tok + head * a.o_head +
                        (int64_t)(c0 * VEC + d) * bytes_of_type<IO>(),
                    none ? 0.0f : x / total);
    }
    __syncthreads();
  }
  if (tid == 0 && a.lse != nullptr)
    a.lse[row * hq + head] = none ? -INFINITY : (top + log2f(total)) * kLn2;
}

// Up to two parts' sums: of the sequences of many new tokens and of few.
struct JoinArgs {
  AttentionArgs part[2];
  uint32_t units;  // rows and heads of the first
};

template <int IO, int VEC, int kJoinThreads>
__global__ void __launch_bounds__(kJoinThreads) attention_join_kernel(JoinArgs j) {
  if (blockIdx.x < j.units) join_splits<IO, VEC, kJoinThreads>(j.part[0], blockIdx.x);
  else join_splits<IO, VEC, kJoinThreads>(j.part[1], blockIdx.x - j.units);
}

GeomBytes bytes_of(const Geom &g, int esize) {
  return {g.s_block * esize, g.s_off * esize, g.s_head * esize, g.s_piece * esize,
          g.s_inner * esize, g.pack, 0};
}

// `n` elements of a head that start at a multiple of n lie together and
// aligned.
bool chunks(const AttentionPlan &p, const Geom &g, const void *base, int n) {
  const int e = dtype_size((kvx_dtype_t)p.g.cache_dtype);
  if (g.s_inner != 1 || g.pack % n != 0 || p.g.head_dim % n != 0) return false;
  const int64_t b = (int64_t)n * e;
  uint64_t low = (uint64_t)((g.s_off | g.s_head | g.s_piece) * e);
  if (p.g.format == KVX_BLOCK_TABLE_KV_OFFSETS)
    low |= (uint64_t)(uintptr_t)p.g.pool[0] | (uint64_t)(uintptr_t)p.g.pool[1] |
           (uint64_t)p.g.bytes_per_block;
  else
    low |= (uint64_t)(uintptr_t)base | (uint64_t)(g.s_block * e);
  return low % (uint64_t)b == 0;
}

// Most tokens that one sequence can have, as far as the host knows.
int64_t longest(const AttentionPlan &p) {
  const int64_t hold = p.g.format == KVX_BLOCK_TABLE_RAGGED
                           ? p.g.table_count
                           : (int64_t)p.g.max_blocks_per_seq * p.g.block_size;
  return p.max_seq_len > 0 && p.max_seq_len < hold ? p.max_seq_len : hold;
}

// Rows of a kv head in tiles of at most `rows`.
void tile_rows(AttentionArgs *a, int rows) {
  a->tile_heads = a->group < rows ? a->group : rows;
  a->head_tiles = (a->group + a->tile_heads - 1) / a->tile_heads;
  a->tile_tokens = rows / a->tile_heads;
  a->tiles = a->qptr != nullptr ? a->tokens / a->tile_tokens + a->seqs : a->seqs;
}

enum Kind { kRows, kFew, kMany };

// Workgroups that share a tile's tokens.  The machine holds about 512 at once;
// with fewer tiles, each is divided until they fill it, into four parts or more
// of `least` tokens: starting a workgroup and joining its sums takes as long.
// With many rows the sums are large, and parts are short only where there are
// few tiles (8 kv heads, us, whole and in parts of 128: one chunk of 100 tokens
// at 1000 tokens 37 and 25, of 512 at 512 24 and 35).
// Sequences of different lengths even out over a few rounds of workgroups, so
// that parts of 2048 tokens at least are made for up to 3200 of them (5
// sequences of 16384 to 32768 tokens: 97 us at 512 workgroups, 86 at 640).
// `rows`: rows of partial sums per query head.
void split_tokens(const AttentionPlan &p, AttentionArgs *a, Kind kind, int64_t rows) {
  // about as many tiles as there are: of many rows, between full ones and a part
  // of one in each sequence
  int64_t tiles = a->qptr == nullptr ? a->seqs : a->tokens / a->tile_tokens;
  if (a->least_rows > 0) tiles = (tiles + a->tiles) / 2;
  else tiles = std::max<int64_t>(tiles, a->seqs);
  tiles = std::min<int64_t>(tiles, a->tiles);
  const int64_t units = std::max<int64_t>(tiles * a->heads * a->head_tiles, 1);
  int64_t tokens = longest(p);  // that a tile sees
  if (a->causal && a->window > 0)
    tokens = std::min(tokens, (int64_t)a->window + a->tile_tokens);
  const int64_t least =
      kind == kMany ? std::min<int64_t>(std::max<int64_t>(4 * units, 128), 512) : 256;
  int64_t n = tokens < 4 * least ? 1 : std::min(512 / units, tokens / least);
  if (kind != kMany) n = std::max(n, std::min(3200 / units, tokens / 2048));
  // partial sums of at most 1 GiB
  const int64_t each = rows * a->heads * a->group * (a->head_dim + 2) * 4;
  if (n * each > ((int64_t)1 << 30)) n = ((int64_t)1 << 30) / each;
  a->splits = (int)(n < 1 ? 1 : n > kMostSplits ? kMostSplits : n);
  a->split_steps = (int)((tokens + 64 * (int64_t)a->splits - 1) / (64 * (int64_t)a->splits));
}

int64_t workgroups(const AttentionArgs &a) {
  int64_t parts = (int64_t)a.tiles * a.splits;
  if (a.heads_near) parts = (parts + kDies - 1) / kDies * kDies;
  return parts * a.heads * a.head_tiles;
}

// Up to two parts: sequences of many new tokens, and of few beside them.
struct Plan {
  AttentionPart part[2];
  int parts;
  Kind kind;  // of the first; a second one is kFew
  bool many;  // there is a kernel for many rows
  bool vt;
  bool grouped;
  uint64_t workspace;
};

// `n` tokens of one element of a value lie together and aligned.
bool tokens_inner(const AttentionPlan &p, int n) {
  const Geom &g = p.g.gv;
  const int e = dtype_size((kvx_dtype_t)p.g.cache_dtype);
  if (g.s_off != 1 || p.g.block_size % n != 0) return false;
  uint64_t low = (uint64_t)((g.s_inner | g.s_head | g.s_piece) * e);
  if (p.g.format == KVX_BLOCK_TABLE_KV_OFFSETS)
    low |= (uint64_t)(uintptr_t)p.g.pool[0] | (uint64_t)(uintptr_t)p.g.pool[1] |
           (uint64_t)p.g.bytes_per_block;
  else
    low |= (uint64_t)(uintptr_t)p.g.src_v | (uint64_t)(g.s_block * e);
  return low % (uint64_t)(n * e) == 0;
}

// Offsets inside a head fit 32 bits.
bool near(const AttentionPlan &p, const Geom &g) {
  const int64_t e = dtype_size((kvx_dtype_t)p.g.cache_dtype), most = (int64_t)1 << 30;
  const int64_t pieces = p.g.head_dim / g.pack;
  return g.s_piece >= 0 && g.s_inner >= 0 && g.s_piece < most && g.s_inner < most &&
         (pieces * g.s_piece + (int64_t)g.pack * g.s_inner) * e < most;
}

// The matrix-core kernels read queries and keys 16 bytes at a time and write 8
// elements of the output at a time.
bool matrix_cores(const AttentionPlan &p) {
  const int D = p.g.head_dim, e = dtype_size((kvx_dtype_t)p.g.cache_dtype);
  if (D % 8 != 0 || D > 256) return false;
  const int n = 16 / dtype_size((kvx_dtype_t)p.g.io_dtype);
  if (((p.q_tok | p.q_head | p.o_tok | p.o_head) % n) != 0 ||
      (uintptr_t)p.query % 16 != 0 || (uintptr_t)p.out % 16 != 0)
    return false;
  return near(p, p.g.gk) && near(p, p.g.gv) && chunks(p, p.g.gk, p.g.src_k, 16 / e);
}

// Values: DP / 16 elements at a time, or 16 bytes of more (few rows), or 16 bytes
// (many); with the token axis innermost 4 tokens or 8 (vt).
bool values_fit(const AttentionPlan &p, Kind kind, bool *vt) {
  const int D = p.g.head_dim, e = dtype_size((kvx_dtype_t)p.g.cache_dtype);
  const int n = kind == kMany || D > 128 || e == 4 ? 16 / e : D <= 64 ? 4 : 8;
  *vt = !chunks(p, p.g.gv, p.g.src_v, n);
  return !*vt || tokens_inner(p, kind == kMany ? 8 : 4);
}

// most: the kernel for the largest chunks that may be taken.
Plan make_plan(const AttentionPlan &p, Kind most) {
  const GatherPlan &g = p.g;
  const int cs = dtype_size((kvx_dtype_t)g.cache_dtype), is = dtype_size((kvx_dtype_t)g.io_dtype);
  AttentionArgs a{};
  a.k = static_cast<const char *>(g.src_k);
  a.v = static_cast<const char *>(g.src_v);
  a.pool[0] = g.pool[0];
  a.pool[1] = g.pool[1];
  a.bytes_per_block = g.bytes_per_block;
  a.table_count = g.table_count;
  a.table = g.block_table;
  a.indptr = g.indptr;
  a.lens = g.seq_lens;
  a.gk = bytes_of(g.gk, cs);
  a.gv = bytes_of(g.gv, cs);
  a.ks = g.k_scale;
  a.vs = g.v_scale;
  a.pool_blocks[0] = g.pool_blocks[0];
  a.pool_blocks[1] = g.pool_blocks[1];
  a.format = g.format;
  a.index64 = g.index_is64;
  a.indptr64 = g.indptr_is64;
  a.lens64 = g.lens_is64;
  a.max_blocks = g.max_blocks_per_seq;
  a.block_size = g.block_size;
  a.block_log2 = (g.block_size & (g.block_size - 1)) == 0 ? __builtin_ctz(g.block_size) : -1;
  a.num_blocks = g.num_blocks;
  a.entry_log2 = g.index_is64 ? 3 : 2;
  a.entry_second = g.format == KVX_BLOCK_TABLE_KV_OFFSETS ? (int64_t)g.max_blocks_per_seq * 4
                   : g.index_is64                         ? 4
                                                          : 0;
  a.q = static_cast<const char *>(p.query);
  a.out = static_cast<char *>(p.out);
  a.lse = p.lse;
  a.qptr = p.query_indptr;
  a.q_tok = p.q_tok * is;
  a.q_head = p.q_head * is;
  a.o_tok = p.o_tok * is;
  a.o_head = p.o_head * is;
  a.qptr64 = p.indptr_is64;
  a.seqs = g.seq_count;
  a.tokens = p.tokens;
  a.heads = g.heads;
  a.group = p.query_heads / g.heads;
  a.head_dim = g.head_dim;
  a.causal = p.causal;
  a.window = p.window;
  a.scale_log2 = p.scale * kLog2e;
  a.scale = p.scale;
  a.softcap = p.softcap;
  // a quarter, so that no softcap is infinite; positive for every one
  a.cap = p.softcap > 0.0f ? std::max(p.softcap * (0.25f * kLog2e), FLT_MIN) : 0.0f;
  a.scale_rest = (float)((double)p.scale * kLog2eWide - (double)a.scale_log2);
  a.cap_rest = a.cap > FLT_MIN ? (float)((double)p.softcap * (0.25 * kLog2eWide) - (double)a.cap) : 0.0f;
  // infinite for the smallest softcaps: 0 * infinity would be NaN
  a.cap_in = p.softcap > 0.0f ? std::clamp(p.scale / p.softcap, -FLT_MAX, FLT_MAX) : 0.0f;
  a.least_rows = 0;
  a.most_rows = 0x7FFFFFFF;
  Plan r{};
  auto add = [&](Kind kind, const AttentionArgs &x) -> AttentionArgs & {
    if (r.parts == 0) r.kind = kind;
    r.part[r.parts].a = x;
    return r.part[r.parts++].a;
  };
  const bool cores = matrix_cores(p);
  // Sequences of at most `few` new tokens go to the kernel for few rows: two of
  // its tiles (8 sequences of 7 tokens at 8192, groups of 4: 91 us, with the
  // other kernel 122; 64 of them at 2048: 133 and 145; with three tiles, 12
  // tokens, 236 and 139).  How many new tokens each has is known here where
  // there is one sequence, one token each, or a hint that bounds all; else one
  // launch has workgroups of both kinds and each kind takes its own.
  const int few = a.group >= 2 * kRowTile ? 1 : 2 * kRowTile / a.group;
  const bool all_few = a.qptr == nullptr || a.tokens <= few ||
                       (p.max_query_len > 0 && p.max_query_len <= few);
  const bool all_many = !all_few && a.seqs == 1;
  // Groups of 16 tokens at most share a load.  RAGGED tables name every token's
  // block.
  auto steps_fit = [&](const Geom &x) { return x.s_off >= 0 && x.s_off * cs < (1 << 24); };
  r.grouped = g.block_size % 16 == 0 && g.format != KVX_BLOCK_TABLE_RAGGED && steps_fit(g.gk) &&
              steps_fit(g.gv);
  const bool few_ok = most != kRows && cores && values_fit(p, kFew, &r.vt);
  bool vt_many = false;
  r.many = most == kMany && few_ok && g.io_dtype != KVX_DTYPE_F32 && p.softcap <= near_cap(g.io_dtype) &&
           values_fit(p, kMany, &vt_many) && vt_many == r.vt;
  if (!few_ok) {
    AttentionArgs &x = add(kRows, a);
    tile_rows(&x, kRowTile);
    x.chunk_k = chunks(p, g.gk, g.src_k, 4);
    split_tokens(p, &x, kRows, x.tokens);
  } else if (all_few || !r.many) {
    AttentionArgs &x = add(kFew, a);
    tile_rows(&x, kRowTile);
    split_tokens(p, &x, kFew, x.tokens);
    // Heads that share 128-byte lines run on one die, or each die would read
    // their lines (200 sequences of 1000 tokens, 8 FP8 heads of 64: 53 us, 74
    // spread over the dies).  Heads of one line are better off together too
    // where there are more workgroups than the machine holds (of 128: 89 and 99
    // us; 16 sequences of 4096 tokens: 38 and 37), wider ones are not (BF16 of
    // 128: 160 and 158).  Two tiles of a sequence would part instead (164 us
    // become 201), so that this is for sequences of one.
    const bool one = x.head_tiles == 1 && (x.qptr == nullptr || (p.max_query_len > 0 &&
                                                                 p.max_query_len <= x.tile_tokens));
    r.part[0].stream = one || !(r.many || g.io_dtype == KVX_DTYPE_F32);
    const auto near_lines = [&](const GeomBytes &g) {
      const int64_t s = g.s_head < 0 ? -g.s_head : g.s_head;
      return s < 256 && (s % 128 != 0 || workgroups(x) > 512);
    };
    x.first_tiles = one;
    x.heads_near = one && a.heads > 1 && near_lines(a.gk) && near_lines(a.gv);
  } else {
    AttentionArgs &x = add(kMany, a);
    tile_rows(&x, kManyRowTile);
    if (!all_many) {
      x.least_rows = few + 1;
      // no more sequences than that have so many tokens
      x.tiles = x.tokens / x.tile_tokens + std::min(x.seqs, x.tokens / x.least_rows);
    }
    split_tokens(p, &x, kMany, x.tokens);
    if (!all_many) {
      AttentionArgs &y = add(kFew, a);
      tile_rows(&y, kRowTile);
      y.most_rows = few;
      y.part_rows = few;
      const int64_t most = (int64_t)y.seqs * ((few + y.tile_tokens - 1) / y.tile_tokens);
      y.tiles = (int)std::min<int64_t>(y.tiles, most);
      y.first_tiles = y.seqs > 256;
      split_tokens(p, &y, kFew, (int64_t)y.seqs * few);
    }
  }
  for (int i = 0; i < r.parts; ++i) {
    AttentionArgs &x = r.part[i].a;
    if (x.splits == 1) continue;
    const int64_t sums = join_rows(x) * p.query_heads * x.splits;
    // as numbers: the workspace is null where only its size is asked for
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.workspace) + r.workspace;
    x.part_o = reinterpret_cast<float *>(at);
    x.part_ml = reinterpret_cast<float *>(at + (uint64_t)sums * x.head_dim * 4);
    r.workspace += ((uint64_t)sums * (x.head_dim + 2) * 4 + 15) & ~(uint64_t)15;
  }
  return r;
}

// Few splits are joined by one wave a row and head, many by four.
template <int IO>
void launch_join(const Plan &p, hipStream_t s) {
  JoinArgs j{};
  uint32_t units = 0;
  int splits = 1;
  for (int i = 0; i < p.parts; ++i) {
    const AttentionArgs &a = p.part[i].a;
    j.part[i] = a;
    splits = std::max(splits, a.splits);
    if (a.splits > 1) units += (uint32_t)(join_rows(a) * a.heads * a.group);
    if (i == 0) j.units = units;
  }
  if (units == 0) return;
  auto go = [&](auto vec) {
    constexpr int kVec = decltype(vec)::value;
    if (splits <= 16) attention_join_kernel<IO, kVec, 64><<<dim3(units), 64, 0, s>>>(j);
    else attention_join_kernel<IO, kVec, kMostSplits><<<dim3(units), kMostSplits, 0, s>>>(j);
  };
  if (p.part[0].a.head_dim % 4 == 0) go(std::integral_constant<int, 4>{});
  else go(std::integral_constant<int, 1>{});
}

bool launchable(const Plan &p) {
  int64_t grid = 0, units = 0;
  for (int i = 0; i < p.parts; ++i) {
    const AttentionArgs &a = p.part[i].a;
    if (a.splits > 1) units += join_rows(a) * a.heads * a.group;
    grid += workgroups(a);
    if (p.kind == kRows && (int64_t)a.heads * a.head_tiles > 65535) return false;
  }
  return units * kMostSplits <= 0xFFFFFF00ll && grid * 256 <= 0xFFFFFFFFll;
}

void run_parts(Plan &p, int io, int cache, hipStream_t s) {
  const bool e4 = cache == KVX_DTYPE_F8_E4M3, e5 = cache == KVX_DTYPE_F8_E5M2;
  for (int i = 0; i < p.parts; ++i) p.part[i].grid = (uint32_t)workgroups(p.part[i].a);
  AttentionPart a = p.part[0];
  const AttentionPart *few = p.parts > 1 ? &p.part[1] : nullptr;
  if (p.kind == kFew && !a.stream && io != KVX_DTYPE_F32) {  // the unstreamed kernel is there
    few = &p.part[0];
    a.grid = 0;
  }
  if (p.kind == kRows)
    run_attention_rows(a, io, cache, s);
  else if (p.kind == kFew && io == KVX_DTYPE_F32)
    (e4 ? run_attention_few_f32_e4m3 : e5 ? run_attention_few_f32_e5m2
                                          : run_attention_few_f32)(a, p.vt, p.grouped, s);
  else if (p.kind == kFew && p.part[0].stream && io == KVX_DTYPE_BF16)
    (e4 ? run_attention_few_bf16_e4m3 : e5 ? run_attention_few_bf16_e5m2
                                           : run_attention_few_bf16)(a, p.vt, p.grouped, s);
  else if (p.kind == kFew && p.part[0].stream)
    (e4 ? run_attention_few_f16_e4m3 : e5 ? run_attention_few_f16_e5m2
                                          : run_attention_few_f16)(a, p.vt, p.grouped, s);
  else if (io == KVX_DTYPE_BF16)
    (e4 ? run_attention_many_bf16_e4m3 : e5 ? run_attention_many_bf16_e5m2
                                            : run_attention_many_bf16)(a, few, p.vt, p.grouped, s);
  else
    (e4 ? run_attention_many_f16_e4m3 : e5 ? run_attention_many_f16_e5m2
                                           : run_attention_many_f16)(a, few, p.vt, p.grouped, s);
}

}  // namespace
}  // namespace dev

using namespace dev;

uint64_t attention_workspace(const AttentionPlan &p) { return make_plan(p, kMany).workspace; }

// Enough whatever kernels the alignment of the call's tensors allows.
uint64_t attention_workspace_bound(const AttentionPlan &p) {
  AttentionPlan x = p;  // as if everything were aligned: all pointers null
  x.query = nullptr;
  x.out = nullptr;
  x.g.src_k = x.g.src_v = nullptr;
  x.g.pool[0] = x.g.pool[1] = nullptr;
  uint64_t bytes = 0;
  for (const Kind most : {kRows, kFew, kMany}) bytes = std::max(bytes, make_plan(x, most).workspace);
  return bytes;
}

kvx_status_t enqueue_attention(const AttentionPlan &p, void *stream) {
  Plan plan = make_plan(p, kMany);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (!launchable(plan)) return KVX_STATUS_UNSUPPORTED;
  run_parts(plan, p.g.io_dtype, p.g.cache_dtype, s);
  if (p.g.io_dtype == KVX_DTYPE_F32) launch_join<KVX_DTYPE_F32>(plan, s);
  else if (p.g.io_dtype == KVX_DTYPE_F16) launch_join<KVX_DTYPE_F16>(plan, s);
  else launch_join<KVX_DTYPE_BF16>(plan, s);
  return hipGetLastError() == hipSuccess ? KVX_STATUS_OK : KVX_STATUS_INTERNAL_ERROR;
}

}  // namespace kvx
