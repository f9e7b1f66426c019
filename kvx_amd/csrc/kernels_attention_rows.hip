// Attention over a paged cache for everything the matrix-core kernels do not
// take: head dims that are not multiples of 8 (from an FP8 cache of 16) or past 256,
// strides without 16-byte chunks.
//
// A workgroup of four waves has 16 query rows of one kv head; each wave takes
// every fourth step of 64 tokens.  Products: lane = token, so that its key
// stays in the lane's registers four elements at a time while 16 rows of
// queries come from LDS as broadcasts.  Sums: lane = element of the head, 16
// weights a token from LDS, again broadcasts.  Each key or value element is
// used 16 times per load, in F32 throughout; LDS and the vector unit bound it
// (16 sequences of 4096 tokens, 8 kv heads of 100 F32: 335 us, 1.2 TB/s; where
// the matrix cores can be used, heads of 128 take 107; 64 of 2048, FP8 heads of 72:
// 534 us, 0.3 TB/s).
#include <hip/hip_runtime.h>

#include "attention.h"

namespace kvx {
namespace dev {
namespace {

constexpr int kRowsThreads = 256;
constexpr int kRowsWaves = kRowsThreads / kWave;

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) x += __shfl_xor(x, d);
  return x;
}

template <int IO, int C, int DJ>
__global__ void __launch_bounds__(kRowsThreads) attention_rows_kernel(AttentionArgs a) {
  constexpr int E = bytes_of_type<C>();
  constexpr int EQ = bytes_of_type<IO>();
  extern __shared__ __align__(16) float lds[];
  const int D = a.head_dim, D4 = (D + 3) & ~3;
  float *q_of = lds;                              // [16][D4], later the joined sums
  float *p_of = q_of + kRowTile * D4;             // [wave][64][16]
  float *state = p_of + kRowsWaves * kWave * kRowTile;  // [wave][16] maxima, then sums
  const char **v_of =
      reinterpret_cast<const char **>(state + 2 * kRowsWaves * kRowTile);  // [wave][64]

  QueryTile t;
  if (!find_tile(a, (int)blockIdx.x, &t)) return;
  const int lane = (int)(threadIdx.x % kWave);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const int kvh = (int)blockIdx.y / a.head_tiles;
  const int head0 = ((int)blockIdx.y - kvh * a.head_tiles) * a.tile_heads;
  const int nheads = min(a.tile_heads, a.group - head0);
  const int z = (int)blockIdx.z;
  const int rows = t.count * a.tile_heads;

  for (int i = (int)threadIdx.x; i < kRowTile * D4; i += kRowsThreads) {
    const int r = i / D4, d = i - r * D4;
    const int tok = r / a.tile_heads, h = r - tok * a.tile_heads;
    float x = 0.0f;
    if (r < rows && h < nheads && d < D)
      x = value_at<IO>(a.q + (t.begin + t.first + tok) * a.q_tok +
                       (int64_t)(kvh * a.group + head0 + h) * a.q_head + (int64_t)d * EQ);
    q_of[i] = x;
  }
  int lo, hi, x0, x1, from, to;
  row_range(a, t, t.first, &lo, &x0);
  row_range(a, t, t.first + t.count - 1, &x1, &hi);
  split_range(a, lo, hi, z, &from, &to);
  __syncthreads();

  float m[kRowTile], l[kRowTile], acc[kRowTile][DJ];
#pragma unroll
  for (int r = 0; r < kRowTile; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.0f;
#pragma unroll
    for (int j = 0; j < DJ; ++j) acc[r][j] = 0.0f;
  }
  float *pw = p_of + wave * kWave * kRowTile;
  const char **vw = v_of + wave * kWave;

  for (int base = from + wave * kWave; base < to; base += kRowsThreads) {
    const int at = base + lane;
    TokenRows tr{nullptr, nullptr, 0};
    const bool there = at < to && token_rows(a, token_entry(a, t, at), at, &tr);
    float s[kRowTile];
#pragma unroll
    for (int r = 0; r < kRowTile; ++r) s[r] = 0.0f;
    float ks = 1.0f, vs = 1.0f;
    if (there) {
      if constexpr (C != IO) {
        ks = scale_of(a.ks, tr.block, kvh);
        vs = scale_of(a.vs, tr.block, kvh);
      }
      const char *krow = tr.k + kvh * a.gk.s_head;
      for (int d = 0; d < D; d += 4) {
        float kx[4];
        if (a.chunk_k) {
          const Raw<4 * E> raw =
              ld<4 * E>(krow + (d / a.gk.pack) * a.gk.s_piece + (int64_t)(d % a.gk.pack) * E);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (E == 4) kx[i] = bits_f32(raw.w[i]);
            else if constexpr (E == 2) kx[i] = io_to_f32<C>(raw, i);
            else kx[i] = decode_pair<C == KVX_DTYPE_F8_E5M2>((int)raw.w[0], i >= 2)[i & 1];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = d + i;
            kx[i] = e < D ? value_at<C>(krow + (e / a.gk.pack) * a.gk.s_piece +
                                        (e % a.gk.pack) * a.gk.s_inner)
                          : 0.0f;
          }
        }
#pragma unroll
        for (int r = 0; r < kRowTile; ++r) {
          const float *qr = q_of + r * D4 + d;
#pragma unroll
          for (int i = 0; i < 4; ++i) s[r] = fmaf(kx[i], qr[i], s[r]);
        }
      }
    }
    vw[lane] = there ? tr.v + kvh * a.gv.s_head : nullptr;
#pragma unroll
    for (int r = 0; r < kRowTile; ++r) {
      int rlo, rhi;
      row_range(a, t, t.first + min(r / a.tile_heads, t.count - 1), &rlo, &rhi);
      const bool seen = there && r < rows && at >= rlo && at < rhi;
      const float x = seen ? logit(a, s[r] * ks) : -INFINITY;
      const float top = fmaxf(m[r], wave_max(x));  // NaN logits do not move it
      const float base_m = top == -INFINITY ? 0.0f : top;
      const float p = seen ? exp2f(x - base_m) : 0.0f;
      const float alpha = exp2f(m[r] - base_m);
      m[r] = top;
      l[r] = l[r] * alpha + wave_sum(p);
#pragma unroll
      for (int j = 0; j < DJ; ++j) acc[r][j] *= alpha;
      // 0: the row does not see the token, whose page may have any scale.  A weight
      // that vanished is the smallest number instead, so that a value that is not
      // finite still reaches the row.
      const float w = p * vs;
      pw[lane * kRowTile + r] = !seen ? 0.0f : w == 0.0f ? 0x1p-149f : w;
    }
    wave_sync();
    const int count = min(kWave, to - base);
    for (int k = 0; k < count; ++k) {
      const char *vrow = vw[k];
      if (vrow == nullptr) continue;
      float vx[DJ];
      bool odd = false;
#pragma unroll
      for (int j = 0; j < DJ; ++j) {
        const int d = lane + j * kWave;
        vx[j] = d < D ? value_at<C>(vrow + (d / a.gv.pack) * a.gv.s_piece +
                                    (d % a.gv.pack) * a.gv.s_inner)
                      : 0.0f;
        odd |= !isfinite(vx[j]);
      }
      const float *pk = pw + k * kRowTile;
      if (__any(odd)) {  // a row that does not see the token takes nothing of it
#pragma unroll
        for (int r = 0; r < kRowTile; ++r)
#pragma unroll
          for (int j = 0; j < DJ; ++j)
            acc[r][j] = pk[r] != 0.0f ? fmaf(pk[r], vx[j], acc[r][j]) : acc[r][j];
      } else {
#pragma unroll
        for (int r = 0; r < kRowTile; ++r)
#pragma unroll
          for (int j = 0; j < DJ; ++j) acc[r][j] = fmaf(pk[r], vx[j], acc[r][j]);
      }
    }
    wave_sync();
  }

  // Join the waves: common maxima, then each wave in turn adds its part.
  if (lane == 0) {
#pragma unroll
    for (int r = 0; r < kRowTile; ++r) {
      state[wave * kRowTile + r] = m[r];
      state[(kRowsWaves + wave) * kRowTile + r] = l[r];
    }
  }
  __syncthreads();
  float top[kRowTile], weight[kRowTile];
#pragma unroll
  for (int r = 0; r < kRowTile; ++r) {
    top[r] = -INFINITY;
    for (int w = 0; w < kRowsWaves; ++w) top[r] = fmaxf(top[r], state[w * kRowTile + r]);
    const float base_m = top[r] == -INFINITY ? 0.0f : top[r];
    weight[r] = exp2f(m[r] - base_m);
    l[r] = 0.0f;
    for (int w = 0; w < kRowsWaves; ++w)
      l[r] += state[(kRowsWaves + w) * kRowTile + r] * exp2f(state[w * kRowTile + r] - base_m);
  }
  for (int w = 0; w < kRowsWaves; ++w) {
    if (w == wave) {
#pragma unroll
      for (int r = 0; r < kRowTile; ++r)
#pragma unroll
        for (int j = 0; j < DJ; ++j) {
          const int d = lane + j * kWave;
          if (d < D) {
            const float part = acc[r][j] * weight[r];
            q_of[r * D4 + d] = w == 0 ? part : q_of[r * D4 + d] + part;
          }
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kRowTile; ++r) {
    const int tok = r / a.tile_heads, h = r - tok * a.tile_heads;
    if (r >= rows || h >= nheads || r % kRowsWaves != wave) continue;
    const int head = kvh * a.group + head0 + h;
    if (a.splits > 1) {
      const int64_t at = part_index(a, t, t.first + tok, head) * a.splits + z;
      for (int d = lane; d < D; d += kWave) a.part_o[at * D + d] = q_of[r * D4 + d];
      if (lane == 0) {
        a.part_ml[2 * at] = top[r];
        a.part_ml[2 * at + 1] = l[r];
      }
      continue;
    }
    const int64_t row = t.begin + t.first + tok;
    const bool none = top[r] == -INFINITY && l[r] == 0.0f;
    for (int d = lane; d < D; d += kWave)
      store_out<IO>(a.out + row * a.o_tok + head * a.o_head + (int64_t)d * EQ,
                    none ? 0.0f : q_of[r * D4 + d] / l[r]);
    if (lane == 0 && a.lse != nullptr)
      a.lse[row * (a.heads * a.group) + head] =
          none ? -INFINITY : (top[r] + log2f(l[r])) * kLn2;
  }
}

template <int IO, int C>
void launch_rows(const AttentionArgs &a, hipStream_t s) {
  const int D4 = (a.head_dim + 3) & ~3;
  const size_t lds = (size_t)(kRowTile * D4 + kRowsWaves * kWave * kRowTile +
                              2 * kRowsWaves * kRowTile) * 4 + kRowsWaves * kWave * 8;
  const dim3 grid((uint32_t)a.tiles, (uint32_t)(a.heads * a.head_tiles), (uint32_t)a.splits);
  if (a.head_dim <= 128)
    attention_rows_kernel<IO, C, 2><<<grid, kRowsThreads, lds, s>>>(a);
  else if (a.head_dim <= 256)
    attention_rows_kernel<IO, C, 4><<<grid, kRowsThreads, lds, s>>>(a);
  else
    attention_rows_kernel<IO, C, 8><<<grid, kRowsThreads, lds, s>>>(a);
}

template <int IO>
void launch_rows_io(const AttentionArgs &a, int cache, hipStream_t s) {
  if (cache == KVX_DTYPE_F8_E4M3) launch_rows<IO, KVX_DTYPE_F8_E4M3>(a, s);
  else if (cache == KVX_DTYPE_F8_E5M2) launch_rows<IO, KVX_DTYPE_F8_E5M2>(a, s);
  else launch_rows<IO, IO>(a, s);
}

}  // namespace

void run_attention_rows(const AttentionPart &p, int io, int cache, hipStream_t s) {
  const AttentionArgs &a = p.a;
  if (io == KVX_DTYPE_F32) launch_rows_io<KVX_DTYPE_F32>(a, cache, s);
  else if (io == KVX_DTYPE_F16) launch_rows_io<KVX_DTYPE_F16>(a, cache, s);
  else launch_rows_io<KVX_DTYPE_BF16>(a, cache, s);
}

}  // namespace dev
}  // namespace kvx
