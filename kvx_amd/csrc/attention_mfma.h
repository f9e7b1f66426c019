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

// An element of w that is NaN or infinite.
template <int C>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (C == KVX_DTYPE_BF16) return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
  else if constexpr (C == KVX_DTYPE_F16) return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
  else if constexpr (C == KVX_DTYPE_F8_E4M3)
    return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
  else return ((w & 0x7C7C7C7Cu) + 0x04040404u) & 0x80808080u;
}

template <int IO>
constexpr uint32_t kOne = IO == KVX_DTYPE_BF16 ? 0x3F80u : 0x3C00u;
template <int IO>
constexpr uint32_t kInf = IO == KVX_DTYPE_BF16 ? 0x7F80u : 0x7C00u;

// acc + v w where v holds NaN or infinities that must not reach, as 0 * v, a
// row whose weight is 0: the finite values as ever, and three products of
// zeros and ones that say which rows meet an infinity of either sign or NaN
// with a weight.
template <int IO, typename Acc>
__device__ __forceinline__ Acc guarded(const Frag &v, const Frag &w, Acc acc) {
  Frag one, fine;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    one.w[i] = (w.w[i] & 0x7FFFu ? kOne<IO> : 0u) | (w.w[i] & 0x7FFF0000u ? kOne<IO> << 16 : 0u);
    fine.w[i] = ((v.w[i] & 0x7FFFu) < kInf<IO> ? v.w[i] & 0xFFFFu : 0u) |
                ((v.w[i] & 0x7FFF0000u) < kInf<IO> << 16 ? v.w[i] & 0xFFFF0000u : 0u);
  }
  acc = mma<IO>(fine, w, acc);
#pragma unroll
  for (int k = 0; k < 3; ++k) {  // infinity, -infinity, NaN: one at a time, in few registers
    __builtin_amdgcn_sched_barrier(0);
    Frag met;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      met.w[i] = 0;
#pragma unroll
      for (int half = 0; half < 32; half += 16) {
        const uint32_t e = (v.w[i] >> half) & 0xFFFFu;
        const bool is = k == 0 ? e == kInf<IO> : k == 1 ? e == (kInf<IO> | 0x8000u)
                                                        : (e & 0x7FFFu) > kInf<IO>;
        if (is) met.w[i] |= kOne<IO> << half;
      }
    }
    const Acc n = mma<IO>(met, one, Acc{});
    const float what = k == 0 ? INFINITY : k == 1 ? -INFINITY : NAN;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Acc) / 4); ++i) acc[i] += n[i] > 0.0f ? what : 0.0f;
  }
  __builtin_amdgcn_sched_barrier(0);
  return acc;
}

// scale * q.k in units of log2, the scale of an FP8 key included in the
// arguments; tanh(y) = 1 - 2 / (1 + e^2y).
__device__ __forceinline__ float capped(const AttentionArgs &a, float x) {
  const float e = __builtin_amdgcn_exp2f(x * a.cap_in * (2.0f * kLog2e));
  return a.cap - 2.0f * a.cap * __builtin_amdgcn_rcpf(1.0f + e);
}

// The factor from products to logits in units of log2 (1 where a softcap has
// its own), made positive by changing the queries: maxima are taken of products
// then, and a logit costs one multiply-add in its exp2.  A scale of 0 makes
// the queries 0.
template <int IO, int N>
__device__ __forceinline__ float positive_scale(const AttentionArgs &a, float ks, Frag (&q)[N]) {
  if (a.cap != 0.0f) return 1.0f;
  const float scale = a.scale_log2 * ks;
  const uint32_t keep = scale == 0.0f ? 0u : ~0u, flip = scale < 0.0f ? 0x80008000u : 0u;
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

// Streaming load of B bytes of global memory (an address that went through
// another lane is not known to be global).
template <int B>
__device__ __forceinline__ Raw<B> stream_load(uint64_t at) {
  Raw<B> r;
  if constexpr (B == 4) {
    r.w[0] = __builtin_nontemporal_load(reinterpret_cast<
        const __attribute__((address_space(1))) uint32_t *>(at));
  } else if constexpr (B == 8) {
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<
        const __attribute__((address_space(1))) u32x2 *>(at));
    r.w[0] = v[0];
    r.w[1] = v[1];
  } else {
    const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<
        const __attribute__((address_space(1))) u32x4 *>(at));
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = v[i];
  }
  return r;
}

}  // namespace dev
}  // namespace kvx
