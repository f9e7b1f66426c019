// What the matrix-core kernels of the attention share: operands and products,
// conversions, and exchanges between lanes.
#pragma once

#include "attention.h"

namespace kvx {
namespace dev {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Four dwords that hold eight 16-bit elements: an operand of the product.
struct Frag {
  uint32_t w[4];
};

// c + a b: v_mfma_f32_16x16x32 or v_mfma_f32_32x32x16 by c's type.
template <int IO, typename Acc>
__device__ __forceinline__ Acc mma(const Frag &a, const Frag &b, Acc c) {
  u32x4 x, y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = a.w[i];
    y[i] = b.w[i];
  }
  if constexpr (sizeof(Acc) == 16) {
    if constexpr (IO == KVX_DTYPE_BF16)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x),
                                                     __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x),
                                                    __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
  } else {
    if constexpr (IO == KVX_DTYPE_BF16)
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x),
                                                     __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x),
                                                    __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
  }
}

// c + a b: v_mfma_f32_16x16x4_f32.
__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// Weights are 2^(x - m), m the maximum of the logits x less this.  An F16 weight
// has 11 digits down to 2^-14 and none below 2^-25: with a maximum of 1 a long
// context would lose the many tokens of small weights (32768 tokens of e^-17.75
// beside one of 1: all of them).  `room`: how far the maximum may grow, in powers
// of two, before m follows it; the largest weight is 2^14 or 2^15.  Past 2^20 a
// maximum has few digits behind the point, which are all of its weight's (2^e, e the
// rounding of m): m is the maximum itself then, so that F16 weights hold out to
// logits of 2^27, as others to 2^31.
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > 0x1p20f; }
template <int IO>
__device__ __forceinline__ float reference_maximum(float top, int room) {
  if constexpr (IO != KVX_DTYPE_F16) return top;
  return is_far(top) ? top : top - (room > 0 ? 15.0f - (float)room : 14.0f);
}

// Block-indexed scales of values multiply the weights, which the products take in
// the queries' type.  BF16 and F32 have the range for that.  F16 has not: a row's
// weights are taken relative to a reference near the largest product of weight
// and scale so far (not of the scale alone: a page of a large one may have next
// to no weight), and its sums count in units of it.
//
// kLeastScale: the smallest reference; a sum of so small a scale is 0 in an F16
// output (2^-64 * 57344).
constexpr float kLeastScale = 0x1p-64f;

// The reference of a row, `was` until now, for a step whose largest weight is
// `most`: weights may grow to 2^14 before a new one is taken, 2^-7 of the largest.
__device__ __forceinline__ float reference_of(float was, float most) {
  return most > was * 0x1p14f || was < kLeastScale ? fmaxf(most * 0x1p-7f, kLeastScale) : was;
}

// Two f32 to two 16-bit elements, to nearest even.
template <int IO>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
  if constexpr (IO == KVX_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// Two FP8 codes (a halfword of w) as two 16-bit elements: exact, every code of
// both formats is a bf16 and an f16 value.
template <int IO, int C>
__device__ __forceinline__ uint32_t widen(uint32_t w, bool hi) {
  if constexpr (IO == KVX_DTYPE_BF16) {
    if constexpr (C == KVX_DTYPE_F8_E5M2)
      return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, false));
    else
      return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
  } else {
    if constexpr (C == KVX_DTYPE_F8_E5M2)
      return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, false));
    else
      return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
  }
}

// FP8 code number i of w.
template <int C>
__device__ __forceinline__ float code(uint32_t w, int i) {
  if constexpr (bytes_of_type<C>() == 1)
    return decode_pair<C == KVX_DTYPE_F8_E5M2>((int)w, i >= 2)[i & 1];
  else return 0.0f;
}

// An element of w that is NaN or infinite.
template <int C>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (C == KVX_DTYPE_F32) return ((w & 0x7F800000u) + 0x00800000u) & 0x80000000u;
  else if constexpr (C == KVX_DTYPE_BF16) return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
  else if constexpr (C == KVX_DTYPE_F16) return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
  else if constexpr (C == KVX_DTYPE_F8_E4M3)
    return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
  else return ((w & 0x7C7C7C7Cu) + 0x04040404u) & 0x80808080u;
}

// w with its NaN and infinite elements 0.
template <int C>
__device__ __forceinline__ uint32_t only_finite(uint32_t w) {
  const uint32_t top = not_finite<C>(w);  // the top bit of each such element
  constexpr int kBits = bytes_of_type<C>() * 8 - 1;
  return w & ~(top | (top - (top >> kBits)));
}

// 0 * infinity must not reach a row that does not see a token.  The kernels
// therefore take NaN and infinities out of the values of steps that not all
// rows of a tile see whole, note that there were some, and call this after the
// tile's outputs are written (and a barrier): it looks at those steps again and
// adds what they hold to the rows that see it.  A thread has elements of its
// own, so the additions need no order.  tile, z, y: the workgroup's tile, split,
// and kv head and part of its group; STEP: tokens of a step; HOLES: they were
// also taken out of steps some of whose tokens are not there.
//
// Not inlined, and with the address of its arguments instead of the caller's
// copy: what this rare path uses must not wait in scalar registers through the
// loops before it, which have too few of them.
template <int IO, int C, int STEP, bool HOLES>
__device__ __attribute__((noinline)) void add_infinities(uint64_t args, int tile, int z, int y) {
  args = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)args) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(args >> 32)) << 32;
  const AttentionArgs &a =
      *(const AttentionArgs *)(const __attribute__((address_space(4))) AttentionArgs *)args;
  QueryTile t;
  if (!find_tile(a, __builtin_amdgcn_readfirstlane(tile), &t)) return;
  z = __builtin_amdgcn_readfirstlane(z);
  y = __builtin_amdgcn_readfirstlane(y);
  const int kvh = y / a.head_tiles;
  const int head0 = (y - kvh * a.head_tiles) * a.tile_heads;
  const int nheads = min(a.tile_heads, a.group - head0);
  int lo, hi, all_lo, all_hi, from, to;  // all rows see [all_lo, all_hi)
  row_range(a, t, t.first, &lo, &all_hi);
  row_range(a, t, t.first + t.count - 1, &all_lo, &hi);
  split_range(a, lo, hi, z, &from, &to);
  for (int d = (int)threadIdx.x; d < a.head_dim; d += (int)blockDim.x) {
    const int64_t at_d = (d / a.gv.pack) * a.gv.s_piece + (d % a.gv.pack) * a.gv.s_inner;
    for (int at = from > lo ? from : lo; at < to; ++at) {
      const int base = from + (at - from) / STEP * STEP;
      TokenRows r;
      if (base >= all_lo && base + STEP <= all_hi) {
        bool whole = true;
        if constexpr (HOLES)
          for (int i = base; i < base + STEP; ++i)
            whole &= token_rows(a, token_entry(a, t, i), i, &r);
        if (whole) {
          at = base + STEP - 1;
          continue;
        }
      }
      if (!token_rows(a, token_entry(a, t, at), at, &r)) continue;
      float x = value_at<C>(r.v + kvh * a.gv.s_head + at_d);
      if (fabsf(x) < INFINITY) continue;
      if constexpr (C != IO) x *= scale_of(a.vs, r.block, kvh);
      for (int i = 0; i < t.count; ++i) {
        int rlo, rhi;
        row_range(a, t, t.first + i, &rlo, &rhi);
        if (at < rlo || at >= rhi) continue;
        for (int h = 0; h < nheads; ++h) {
          const int head = kvh * a.group + head0 + h;
          if (a.splits > 1) {
            float *p = a.part_o + (part_index(a, t, t.first + i, head) * a.splits + z) * a.head_dim;
            p[d] += x;
          } else {
            char *p = a.out + (t.begin + t.first + i) * a.o_tok + head * a.o_head + d * bytes_of_type<IO>();
            store_out<IO>(p, value_at<IO>(p) + x);
          }
        }
      }
    }
  }
}

// The address of a kernel's arguments, `offset` bytes into them.
__device__ __forceinline__ uint64_t args_address(size_t offset) {
  return reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr()) + offset;
}

// The capped logits in units of log2 of raw products x (by: the scale of an FP8
// key), for 16-bit products.  With y = scale x / softcap:
//
// - softcap to near_cap: softcap * (1 - 2 / (1 + e^2y)), off by up to 2^-21 of the
//   softcap and so a sixteenth of a weight's rounding, 2^-15 of F16, 2^-12 of BF16;
// - larger ones, for which that grows: right to about 2^-20 of the logit, by
//   scale x * tanh(y) / y for |y| < 1/2, a polynomial in y^2 (least maximum error
//   on [0, 1/4], 1.5e-8), so that a cap far away leaves logits as they are.
//
// FAR: the second form too.  Only the streaming kernel for few rows has it, and
// takes chunks of any length with such a cap: in the kernel for many rows it costs
// chunks with near caps 27 to 43 % where it is the only form, and registers that
// other calls miss beside the first (a mixed batch without a cap: 62 us for 54).
// Two chunks of 2048 tokens at 4096 to 8192, BF16 heads of 128: 400 us with a cap
// of 30, 1763 with one of 10^5.
template <int IO, bool FAR, typename V, int N>
__device__ __forceinline__ void cap_logits(const AttentionArgs &a, float by, V &x) {
  if (!FAR || a.softcap <= near_cap(IO)) {
    const float cap = 4.0f * a.cap;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = __builtin_amdgcn_exp2f(x[i] * by * a.cap_in * (2.0f * kLog2e));
      x[i] = fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + e), cap);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = x[i] * by * a.cap_in, u = y * y;
    const float e = __builtin_amdgcn_exp2f(y * (2.0f * kLog2e));
    const float far = a.cap * fmaf(__builtin_amdgcn_rcpf(1.0f + e), -8.0f, 4.0f);
    float r = fmaf(u, 0.01724149f, -0.05304549f);
    r = fmaf(u, r, 0.13325879f);
    r = fmaf(u, r, -0.33333144f);
    r = fmaf(u, r, 1.0f);
    x[i] = fabsf(y) < 0.5f ? x[i] * by * a.scale_log2 * r : far;
  }
}

// The factor from products to logits in units of log2 (1 where a softcap has
// its own), made positive by changing the queries: maxima are taken of products
// then, and a logit costs one multiply-add in its exp2.  A scale of 0 makes
// the queries 0.
template <int IO, int N>
__device__ __forceinline__ float positive_scale(const AttentionArgs &a, float ks, Frag (&q)[N]) {
  if (a.softcap != 0.0f) return 1.0f;
  const float scale = a.scale_log2 * ks;
  const uint32_t keep = scale == 0.0f ? 0u : ~0u, flip = scale >= 0.0f             ? 0u
                                                            : IO == KVX_DTYPE_F32 ? 0x80000000u
                                                                                  : 0x80008000u;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) q[i].w[j] = (q[i].w[j] & keep) ^ flip;
  return scale == 0.0f ? 1.0f : fabsf(scale);
}

// Another lane's value; `at` = 4 * lane, so that constants added to it become
// the instruction's offset.
__device__ __forceinline__ uint32_t from_lane(uint32_t x, int at) {
  return (uint32_t)__builtin_amdgcn_ds_bpermute(at, (int)x);
}
__device__ __forceinline__ float from_lane(float x, int at) {
  return bits_f32(from_lane(f32_bits(x), at));
}
__device__ __forceinline__ uint64_t from_lane(uint64_t x, int at) {
  return from_lane((uint32_t)x, at) | (uint64_t)from_lane((uint32_t)(x >> 32), at) << 32;
}

// A wave-uniform copy of lane `lane`'s address.
__device__ __forceinline__ uint64_t address_of_lane(uint64_t x, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, lane) |
         (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), lane) << 32;
}

// K and V rows of kv head `kvh` for the tokens that a wave's lanes look up, one
// each: every token of a step, or (blocks that hold whole groups of 16) the
// first of a group, whose other rows follow from it.  Tokens that are not there
// get another's rows, so that loads need no conditions.
struct LaneRows {
  uint64_t k, v;
  uint64_t held;  // bit per lane whose token is there; none: k and v cannot be read
  float ks, vs;   // block-indexed scales
  bool apart;     // a value load's tokens are not all of one block
};

// VN: values with the token axis innermost, VN tokens a load from the lane of the
// first.  Only a RAGGED table can name different blocks for them; v is the row
// of the load's first token in the lane's own block then.
template <bool INDEXED, int VN = 0>
__device__ __forceinline__ LaneRows lane_rows(const AttentionArgs &a, const TokenEntry &entry,
                                              int at, bool looks, int kvh) {
  LaneRows r{0, 0, 0, 1.0f, 1.0f, false};
  TokenRows x{nullptr, nullptr, 0};
  const bool held = looks && token_rows(a, entry, at, &x);
  if (held) {
    r.k = reinterpret_cast<uint64_t>(x.k + kvh * a.gk.s_head);
    r.v = reinterpret_cast<uint64_t>(x.v + kvh * a.gv.s_head);
    if constexpr (VN > 0) {
      if (a.format == KVX_BLOCK_TABLE_RAGGED) r.v -= (at % VN) * a.gv.s_off;
    }
    if constexpr (INDEXED) {
      r.ks = scale_of(a.ks, x.block, kvh);
      r.vs = scale_of(a.vs, x.block, kvh);
    }
  }
  r.held = __ballot(held);
  if (r.held != 0 && r.held != ~0ull) {
    const int first = 4 * __builtin_ctzll(r.held);
    const uint64_t k = from_lane(r.k, first), v = from_lane(r.v, first);
    if (!held) {
      r.k = k;
      r.v = v;
    }
  }
  if constexpr (VN > 0) {
    if (a.format == KVX_BLOCK_TABLE_RAGGED && r.held != 0) {
      const int first = (int)(threadIdx.x % kWave) / VN * VN;
      const bool same = from_lane(r.v, 4 * first) == r.v && ((r.held >> first) & 1);
      r.apart = __any(held && !same);
    }
  }
  return r;
}

// Bits [from - base, to - base) of a mask of tokens from `base` on, n <= 64 of them.
__device__ __forceinline__ uint64_t tokens_between(int from, int to, int base, int n) {
  const int lo = from > base ? from - base : 0, hi = to < base + n ? to - base : n;
  if (lo >= hi) return 0;
  const uint64_t below = hi >= 64 ? ~0ull : (1ull << hi) - 1;
  return below & ~((1ull << lo) - 1);
}

// A bit for each of 4 groups of 16 tokens, as a bit for each token.
__device__ __forceinline__ uint64_t group_tokens(uint32_t groups) {
  return ((groups & 1) | (uint64_t)(groups & 2) << 15 | (uint64_t)(groups & 4) << 30 |
          (uint64_t)(groups & 8) << 45) *
         0xFFFFull;
}

// Bits of token `at` of a load of tokens, in its dword w.
template <int E>
__device__ __forceinline__ uint32_t token_bits(int at, int w) {
  constexpr int kEach = 4 / E;  // tokens of a dword
  const uint32_t one = E == 4 ? ~0u : (1u << (8 * E % 32)) - 1;
  return at / kEach == w ? one << (8 * E * (at % kEach) % 32) : 0u;
}

// B bytes of global memory at an address that went through another lane, and so
// is not known to be global.  A uniform address and a 32-bit offset make the
// scalar form of the load, without a vector operation for the address.  NT:
// streamed.
template <int B, bool NT>
__device__ __forceinline__ Raw<B> global_load(uint64_t base, uint32_t offset) {
  const auto *p = reinterpret_cast<const __attribute__((address_space(1))) char *>(base) + offset;
  auto read = [](const auto *q) { return NT ? __builtin_nontemporal_load(q) : *q; };
  Raw<B> r;
  if constexpr (B == 4) {
    r.w[0] = read(reinterpret_cast<const __attribute__((address_space(1))) uint32_t *>(p));
  } else if constexpr (B == 8) {
    const u32x2 v = read(reinterpret_cast<const __attribute__((address_space(1))) u32x2 *>(p));
    r.w[0] = v[0];
    r.w[1] = v[1];
  } else {
    const u32x4 v = read(reinterpret_cast<const __attribute__((address_space(1))) u32x4 *>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = v[i];
  }
  return r;
}

}  // namespace dev
}  // namespace kvx
