// Rotary positions and the paged write in one pass (kvx_launch_rope_write_kv).
//
// A row at position p turns pair i by the angle p * f_i, f_i = inv_freq[i]:
//   (x0, x1) -> m (x0 cos - x1 sin, x1 cos + x0 sin).
// Every query element is read and written once, every key and value element
// read once and written to its cache row: T * D * (2 Hq io + 2 H (io + cache))
// bytes over the HBM rate is the floor; the few operations an element needs
// stay far below the vector rate as long as a row's sines and cosines are
// computed once and shared by its heads.  So a workgroup takes `tile` whole
// tokens (or a slice of one token's heads where there are few tokens),
// computes their rot / 2 angles into LDS, and then walks over units of 2 * VEC
// elements: VEC pairs of a query or key head, two chunks past the rotated part,
// or of a value head.
//
// Angles: p * f_i / 2 pi in f64 (exact to 2^-52 of the number of turns, so a
// position of a million still has its angle to 1e-9), whole turns dropped,
// the rest split into f32 and a correction that enters by the first term of
// the addition theorem: cosines and sines are right to about one unit of f32.
//
// Measured: 32768 tokens of 32 + 8 + 8 heads of 128, BF16, 163 us (4.9 TB/s);
// 4 tokens 5.2 us, 251 into an FP8 cache 7.2 us, where a launch's latency is
// nearly all; prefill into an FP8 cache 165 us (4.5 TB/s), in F32 313 (5.1).  With
// one query and one key head a token's angles cost more than its bytes (90000 tokens
// into FP8: 75 to 82 us, 1.4 to 1.6 TB/s).
#include <hip/hip_runtime.h>

#include "kernels.h"
#include "operators_internal.h"

namespace kvx {
namespace dev {
namespace {

constexpr int kRopeThreads = 128;
constexpr int kRopeUnits = 3;        // of a thread
constexpr uint32_t kDies = 8;        // that take workgroups in turn

struct RopeArgs {
  const char *q, *key, *value;
  char *qo, *dst_k, *dst_v;
  const void *slots, *positions;
  const float *inv_freq;
  ScaleRef k_scale, v_scale;
  GeomBytes gk, gv;                                               // cache, bytes
  int64_t q_tok, q_head, o_tok, o_head, k_tok, k_head, v_tok, v_head;  // bytes
  int64_t tokens;
  int32_t slot64, pos64;
  int32_t query_heads, heads, head_dim, half;  // half: rot_dim / 2
  int32_t block_size, num_blocks;
  int32_t interleaved;
  int32_t chunks_k, chunks_v;  // cache chunks of VEC elements are contiguous
  int32_t tile;                // tokens of a workgroup
  int32_t slices;              // workgroups that share them (grid.y)
  int32_t pair_units, rest_units, value_units;  // of one head
  uint32_t head_magic, value_magic;             // of pair_units + rest_units, value_units
  float magnitude;
};

template <int IO>
__device__ __forceinline__ float element(const char *p) {
  if constexpr (IO == KVX_DTYPE_F32) return *reinterpret_cast<const float *>(p);
  else if constexpr (IO == KVX_DTYPE_BF16)
    return bf16_to_f32(*reinterpret_cast<const uint16_t *>(p));
  else return (float)*reinterpret_cast<const _Float16 *>(p);
}

template <int IO, int VEC>
__device__ __forceinline__ void load(const char *p, float (&x)[VEC]) {
  const Raw<VEC * IoType<IO>::kBytes> r = ld<VEC * IoType<IO>::kBytes>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = io_to_f32<IO>(r, i);
}

// Rounds to nearest even, once.
template <int IO, int VEC>
__device__ __forceinline__ Raw<VEC * IoType<IO>::kBytes> narrow(const float (&x)[VEC]) {
  Raw<VEC * IoType<IO>::kBytes> r;
  if constexpr (IO == KVX_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.w[i] = f32_bits(x[i]);
  } else if constexpr (VEC == 1) {
    r.w[0] = pack_pair<IO>(f32x2{x[0], x[0]}) & 0xFFFFu;
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) r.w[i] = pack_pair<IO>(f32x2{x[2 * i], x[2 * i + 1]});
  }
  return r;
}

// VEC elements into a cache tensor: d = first element of the head.
template <int IO, int C, int VEC>
__device__ __forceinline__ void store_cache(char *row, const GeomBytes &g, int d, bool chunk,
                                            const float (&x)[VEC], const QuantScale &qs) {
  constexpr bool kQuant = C != IO;
  constexpr int E = kQuant ? 1 : IoType<IO>::kBytes;
  Raw<VEC * E> r;
  if constexpr (kQuant) {
    float q[VEC < 4 ? 4 : VEC] = {};
#pragma unroll
    for (int i = 0; i < VEC; ++i) q[i] = qs.fast ? quant_quotient(qs, x[i]) : x[i] / qs.s;
#pragma unroll
    for (int k = 0; k < Raw<VEC * E>::kWords; ++k)
      r.w[k] = encode4<C, (VEC >= 4)>(q[4 * k], q[4 * k + 1], q[4 * k + 2], q[4 * k + 3]);
  } else {
    r = narrow<IO, VEC>(x);
  }
  if (chunk) {
    st<VEC * E>(row + (d / g.pack) * g.s_piece + (d % g.pack) * g.s_inner, r);
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    Raw<E> e;
    if constexpr (E == 4) e.w[0] = r.w[i];
    else if constexpr (E == 2) e.w[0] = get16(r, i);
    else e.w[0] = get8(r, i);
    const int at = d + i;
    st<E>(row + (at / g.pack) * g.s_piece + (at % g.pack) * g.s_inner, e);
  }
}

template <int IO, int C, int VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_write_kernel(RopeArgs a) {
  extern __shared__ __align__(16) char lds[];
  constexpr int E = IoType<IO>::kBytes;
  // Workgroups go round the dies in order.  Tiles of neighbouring tokens go to
  // one die, whose L2 then puts their pieces of a packed cache's lines together.
  const uint32_t die = blockIdx.x % kDies, each = gridDim.x / kDies, more = gridDim.x % kDies;
  const uint32_t number = die * each + min(die, more) + blockIdx.x / kDies;
  const int64_t first = (int64_t)number * a.tile;
  const int n = (int)min((int64_t)a.tile, a.tokens - first);
  int64_t *slot_of = reinterpret_cast<int64_t *>(lds);
  float *cos_of = reinterpret_cast<float *>(lds + 8 * a.tile);
  float *sin_of = cos_of + a.tile * a.half;

  for (int t = (int)threadIdx.x; t < n; t += kRopeThreads)
    slot_of[t] = a.slot64 ? static_cast<const int64_t *>(a.slots)[first + t]
                          : (int64_t)static_cast<const int32_t *>(a.slots)[first + t];
  for (int i = (int)threadIdx.x; i < n * a.half; i += kRopeThreads) {
    const int t = i / a.half, pair = i - t * a.half;
    const double p = a.pos64 ? (double)static_cast<const int64_t *>(a.positions)[first + t]
                             : (double)static_cast<const int32_t *>(a.positions)[first + t];
    double turns = p * (double)a.inv_freq[pair] * 0.15915494309189533577;
    turns -= rint(turns);
    const float near = (float)turns;
    const float rest = (float)((turns - (double)near) * 6.28318530717958647693);
    float s, c;
    sincospif(2.0f * near, &s, &c);
    cos_of[i] = a.magnitude * fmaf(-s, rest, c);
    sin_of[i] = a.magnitude * fmaf(c, rest, s);
  }
  __syncthreads();

  const int per_head = a.pair_units + a.rest_units;
  const int row_units = a.query_heads * per_head;
  const int key_units = a.heads * per_head;
  const int units = row_units + key_units + a.heads * a.value_units;
  const int per_slice = (units + a.slices - 1) / a.slices;
  const int u0 = (int)blockIdx.y * per_slice;
  const int mine = min(per_slice, units - u0);
  if (mine <= 0) return;
  int t = 0, left = (int)threadIdx.x;
  while (true) {
    while (left >= mine) {  // the unit's token
      left -= mine;
      if (++t >= n) return;
    }
    int u = u0 + left;
    left += kRopeThreads;
    const int64_t tok = first + t;
    const bool is_query = u < row_units;
    const bool is_key = !is_query && u < row_units + key_units;
    char *row = nullptr;
    QuantScale qs{};
    if (!is_query) {
      u -= row_units;
      const int64_t slot = slot_of[t];
      if (slot < 0) continue;
      const int64_t block = slot / a.block_size;
      if (block >= a.num_blocks) continue;
      const int off = (int)(slot - block * a.block_size);
      if (!is_key) u -= key_units;
      const uint32_t magic = is_key ? a.head_magic : a.value_magic;
      const int head = magic == 0 ? u : (int)div_magic((uint32_t)u, magic);
      const GeomBytes &g = is_key ? a.gk : a.gv;
      row = (is_key ? a.dst_k : a.dst_v) + block * g.s_block + off * g.s_off + head * g.s_head;
      if constexpr (C != IO) {
        const ScaleRef &sc = is_key ? a.k_scale : a.v_scale;
        qs = quant_scale(sc.p[sc.indexed ? block * sc.s_block + head * sc.s_head : 0]);
      }
      if (!is_key) {
        const int d = (u - head * a.value_units) * 2 * VEC;
        const char *x = a.value + tok * a.v_tok + head * a.v_head + (int64_t)d * E;
        float v[VEC];
        load<IO, VEC>(x, v);
        if (d + VEC < a.head_dim) {
          float v1[VEC];
          load<IO, VEC>(x + VEC * E, v1);
          store_cache<IO, C, VEC>(row, g, d + VEC, a.chunks_v, v1, qs);
        }
        store_cache<IO, C, VEC>(row, g, d, a.chunks_v, v, qs);
        continue;
      }
    }
    const int head = a.head_magic == 0 ? u : (int)div_magic((uint32_t)u, a.head_magic);
    const int i = u - head * per_head;
    const char *x = is_query ? a.q + tok * a.q_tok + head * a.q_head
                             : a.key + tok * a.k_tok + head * a.k_head;
    int d0, d1;
    float x0[VEC], x1[VEC];
    bool two = true;
    if (i < a.pair_units) {
      d0 = a.interleaved ? 2 * VEC * i : VEC * i;
      d1 = a.interleaved ? d0 + VEC : d0 + a.half;
      load<IO, VEC>(x + (int64_t)d0 * E, x0);
      load<IO, VEC>(x + (int64_t)d1 * E, x1);
      const float *c = cos_of + t * a.half + VEC * i;
      const float *s = sin_of + t * a.half + VEC * i;
      if (a.interleaved) {
        // x0 and x1 are 2 VEC adjacent elements: pairs (2 j, 2 j + 1)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float &a0 = 2 * j < VEC ? x0[(2 * j) % VEC] : x1[(2 * j) % VEC];
          float &a1 = 2 * j + 1 < VEC ? x0[(2 * j + 1) % VEC] : x1[(2 * j + 1) % VEC];
          const float y = fmaf(a0, c[j], -(a1 * s[j]));
          a1 = fmaf(a1, c[j], a0 * s[j]);
          a0 = y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float y = fmaf(x0[j], c[j], -(x1[j] * s[j]));
          x1[j] = fmaf(x1[j], c[j], x0[j] * s[j]);
          x0[j] = y;
        }
      }
    } else {
      d0 = 2 * a.half + 2 * VEC * (i - a.pair_units);
      d1 = d0 + VEC;
      two = d1 < a.head_dim;
      load<IO, VEC>(x + (int64_t)d0 * E, x0);
      if (two) load<IO, VEC>(x + (int64_t)d1 * E, x1);
    }
    if (is_query) {
      char *o = a.qo + tok * a.o_tok + head * a.o_head;
      st<VEC * E>(o + (int64_t)d0 * E, narrow<IO, VEC>(x0));
      if (two) st<VEC * E>(o + (int64_t)d1 * E, narrow<IO, VEC>(x1));
    } else {
      store_cache<IO, C, VEC>(row, a.gk, d0, a.chunks_k, x0, qs);
      if (two) store_cache<IO, C, VEC>(row, a.gk, d1, a.chunks_k, x1, qs);
    }
  }
}

GeomBytes bytes_of(const Geom &g, int esize) {
  return {g.s_block * esize, g.s_off * esize, g.s_head * esize, g.s_piece * esize,
          g.s_inner * esize, g.pack, 0};
}

bool multiple(const void *p, int64_t b) { return (uintptr_t)p % (uintptr_t)b == 0; }

// Chunks of VEC elements that start at multiples of VEC lie in one piece of a
// cache row, aligned to their size.
bool cache_chunks(const Geom &g, const void *base, int esize, int vec) {
  const int64_t b = (int64_t)vec * esize;
  if (vec > 1 && (g.s_inner != 1 || g.pack % vec != 0)) return false;
  return multiple(base, b) && (g.s_block * esize) % b == 0 && (g.s_off * esize) % b == 0 &&
         (g.s_head * esize) % b == 0 && (g.s_piece * esize) % b == 0;
}

uint32_t magic_of(int d) { return d <= 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + d - 1) / d); }

template <int IO, int C>
void launch_rope(const RopeArgs &a, int vec, dim3 grid, size_t lds, hipStream_t s) {
  constexpr int kWide = 16 / IoType<IO>::kBytes;
  if (vec == kWide)
    rope_write_kernel<IO, C, kWide><<<grid, kRopeThreads, lds, s>>>(a);
  else
    rope_write_kernel<IO, C, 1><<<grid, kRopeThreads, lds, s>>>(a);
}

template <int IO>
void launch_rope_io(const RopeArgs &a, int cache, int vec, dim3 grid, size_t lds, hipStream_t s) {
  if (cache == KVX_DTYPE_F8_E4M3) launch_rope<IO, KVX_DTYPE_F8_E4M3>(a, vec, grid, lds, s);
  else if (cache == KVX_DTYPE_F8_E5M2) launch_rope<IO, KVX_DTYPE_F8_E5M2>(a, vec, grid, lds, s);
  else launch_rope<IO, IO>(a, vec, grid, lds, s);
}

}  // namespace
}  // namespace dev

using namespace dev;

kvx_status_t enqueue_rope_write(const RopePlan &p, void *stream) {
  const WritePlan &w = p.w;
  const int is = dtype_size((kvx_dtype_t)w.io_dtype), cs = dtype_size((kvx_dtype_t)w.cache_dtype);
  RopeArgs a{};
  a.q = static_cast<const char *>(p.query);
  a.qo = static_cast<char *>(p.query_out);
  a.key = static_cast<const char *>(w.src_k);
  a.value = static_cast<const char *>(w.src_v);
  a.dst_k = static_cast<char *>(w.dst_k);
  a.dst_v = static_cast<char *>(w.dst_v);
  a.slots = w.slots;
  a.positions = p.positions;
  a.inv_freq = p.inv_freq;
  a.k_scale = w.k_scale;
  a.v_scale = w.v_scale;
  a.gk = bytes_of(w.gk, cs);
  a.gv = bytes_of(w.gv, cs);
  a.q_tok = p.q_tok * is;
  a.q_head = p.q_head * is;
  a.o_tok = p.o_tok * is;
  a.o_head = p.o_head * is;
  a.k_tok = p.k_tok * is;
  a.k_head = p.k_head * is;
  a.v_tok = p.v_tok * is;
  a.v_head = p.v_head * is;
  a.tokens = w.num_tokens;
  a.slot64 = w.slot_is64;
  a.pos64 = p.position_is64;
  a.query_heads = p.query_heads;
  a.heads = w.heads;
  a.head_dim = w.head_dim;
  a.half = p.rot_dim / 2;
  a.block_size = w.block_size;
  a.num_blocks = w.num_blocks;
  a.interleaved = p.interleaved;
  a.magnitude = p.magnitude;

  // 16-byte chunks where rows, pairs and the part past them allow; else
  // single elements.
  int vec = 16 / is;
  const int64_t strides = p.q_tok | p.q_head | p.o_tok | p.o_head | p.k_tok | p.k_head | p.v_tok |
                          p.v_head;
  if (a.half % vec != 0 || w.head_dim % vec != 0 || (strides * is) % 16 != 0 ||
      !multiple(a.q, 16) || !multiple(a.qo, 16) || !multiple(a.key, 16) || !multiple(a.value, 16))
    vec = 1;
  a.chunks_k = cache_chunks(w.gk, w.dst_k, cs, vec);
  a.chunks_v = cache_chunks(w.gv, w.dst_v, cs, vec);
  const auto units_of = [&](int64_t n) { return (int32_t)((n + 2 * vec - 1) / (2 * vec)); };
  a.pair_units = a.half / vec;
  a.rest_units = units_of(w.head_dim - p.rot_dim);
  a.value_units = units_of(w.head_dim);
  a.head_magic = magic_of(a.pair_units + a.rest_units);
  a.value_magic = magic_of(a.value_units);
  const int64_t heads = (int64_t)p.query_heads + w.heads;
  const int64_t units =
      heads * (a.pair_units + a.rest_units) + (int64_t)w.heads * a.value_units;
  // div_magic is exact while unit * divisor stays within 2^32.
  if (units * (a.value_units + 1) > ((int64_t)1 << 32)) return KVX_STATUS_UNSUPPORTED;
  // Few tokens: slices of one token, so that the machine has work for a
  // decode batch; many: as many whole tokens as give each thread three units,
  // within 16 KiB of angles.  Small workgroups, whose angles and loads overlap
  // others': 32768 tokens of 32 + 8 + 8 heads of 128 take 167 us (4.8 TB/s, a
  // copy's rate) with 128 threads a token, 172 with 256 for two, 180 with 512
  // for four, 205 with 256 for four; 196 without the order by die.
  int64_t tile = kRopeUnits * kRopeThreads / units;
  const int64_t fit = a.half > 0 ? 16384 / (8 * a.half) : tile;
  if (tile > fit) tile = fit;
  if (tile < 1) tile = 1;
  while (tile > 1 && (w.num_tokens + tile - 1) / tile < 1024) --tile;
  a.tile = (int32_t)tile;
  const int64_t groups = (w.num_tokens + tile - 1) / tile;
  int64_t slices = 1;
  while (groups * slices < 512 && (units + slices - 1) / slices > kRopeThreads) ++slices;
  a.slices = (int32_t)slices;
  if (groups * kRopeThreads > 0xFFFFFFFFll) return KVX_STATUS_UNSUPPORTED;
  const size_t lds = (size_t)(8 * tile + 8 * tile * a.half);
  const dim3 grid((uint32_t)groups, (uint32_t)slices);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (w.io_dtype == KVX_DTYPE_F32) launch_rope_io<KVX_DTYPE_F32>(a, w.cache_dtype, vec, grid, lds, s);
  else if (w.io_dtype == KVX_DTYPE_F16)
    launch_rope_io<KVX_DTYPE_F16>(a, w.cache_dtype, vec, grid, lds, s);
  else launch_rope_io<KVX_DTYPE_BF16>(a, w.cache_dtype, vec, grid, lds, s);
  return hipGetLastError() == hipSuccess ? KVX_STATUS_OK : KVX_STATUS_INTERNAL_ERROR;
}

}  // namespace kvx
