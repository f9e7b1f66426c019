// Attention of many rows per kv head (prefill chunks) on the matrix cores.
//
// 4 * D operations for every (row, token) pair; rows of a tile share its keys
// and values, so that 128 rows make it compute-bound: the matrix cores, and
// beside them the vector unit, which owes every pair a maximum, a
// multiply-add, an exp2, a sum and half a conversion.
//
// Four waves with 32 rows each share steps of 64 tokens through LDS, two
// buffers, loaded one step ahead: straight from memory, or through registers
// where FP8 codes become 16-bit elements or something has to be left out.
//
// v_mfma_f32_32x32x16: lane l = 32 h + c holds A[row c][8 h .. 8 h + 7],
// B[8 h ..][column c], D[rows 8 (i / 4) + 4 h + i % 4][column c], i < 16.
//
//   S^T = K Q^T   lane c has row c of its wave's queries (held in registers)
//                 and half of the step's tokens: maximum and sum are a chain in
//                 the lane and one exchange with lane c ^ 32.
//   O^T = V^T P^T a lane's weights are the B operand as they stand: the sum's
//                 tokens may come in any order, and A takes them in that one,
//                 through ds_read_b64_tr_b16, which transposes 4 tokens by 16
//                 elements (values with the token axis innermost are kept as
//                 they are and read plainly).
//   The sums of a row are a lane's own, so rescaling them is one multiplication
//   each; it is put off until a maximum has grown by more than 8 (weights then
//   are 2^8 times as large, which changes neither their relative rounding nor the
//   F32 sums).
//
// Measured, 8 kv heads of 128, groups of 4, BF16 (from card to card): a chunk of
// 8192 tokens 583 to 645 us (850 to 940 TFLOP/s), two chunks of 2048 at 4096 to 8192
// 323 to 340 us (765 to 805); those from FP8 320 to 332, with block scales 380 to 395
// (F16 405 to 418: its weights need a reference), heads of 256 760 to 775 (680).
// Matrix and vector instructions of a SIMD's two waves add up to nearly all of
// it: they overlap little.  The next step's products written between the weights
// of this one ran slower (402 us for 340), and the products' priority gives 2 %.
//
// LDS rows are not padded; the 16-byte chunks of a row are permuted by the
// token's number, so that the 8 lanes that read one element range of 8 keys
// (and the 16 that transpose 4 values) meet all banks.
#pragma once

#include "kernels_attention_few.h"

namespace kvx {
namespace dev {

constexpr int kManyWaves = 4;
constexpr int kManyThreads = kManyWaves * kWave;
static_assert(kManyRowTile == 32 * kManyWaves, "32 rows a wave");
constexpr int kManyStep = 64;
constexpr int kRoom = 8;  // see reference_maximum

// Operands are read from LDS this many products before they are used (about 128
// cycles of 32 each); scheduling barriers, which vector and scalar operations
// may cross, keep the compiler from moving the reads to their uses.
constexpr int kAhead = 4;
constexpr int kMayCross = 0x2 | 0x4;

template <int DP, bool INDEXED>
constexpr size_t many_lds() {
  return (size_t)2 * (2 * kManyStep * DP * 2 + (INDEXED ? 2 * kManyStep * 4 : 0)) + 16;
}

// What is XORed to the number of a 16-byte chunk of a token's key or value.  LDS
// has 64 banks of 4 bytes: 16 lanes that read the same chunk of 16 keys, and 32
// that transpose 4 chunks of 4 values, meet all of them (a row of 128 bytes
// takes half of the banks, by its token's parity).
template <int DP>
__device__ __forceinline__ int key_swap(int token) {
  // DP 256: a thread's loads step by 8 tokens, which the permutation must not see
  return DP == 64 ? (token >> 1) & 7 : DP == 128 ? token & 15 : token & 7;
}
template <int DP>
__device__ __forceinline__ int value_swap(int token) {
  return DP == 64 ? 4 * ((token >> 1) & 1) : 4 * (token & 3);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) char lds_char;

// 16 bytes a lane of global memory into LDS, lane after lane from `to` (uniform)
// on; there once vmcnt is 0.
__device__ __forceinline__ void copy_to_lds(uint64_t base, uint32_t offset, lds_char *to) {
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const __attribute__((address_space(1))) uint32_t *>(
          reinterpret_cast<const __attribute__((address_space(1))) char *>(base) + offset),
      reinterpret_cast<__attribute__((address_space(3))) uint32_t *>(to), 16, 0, 0);
}

template <typename V>
__device__ __forceinline__ V lds_read(const lds_char *at) {
  return *reinterpret_cast<const __attribute__((address_space(3))) V *>(at);
}
__device__ __forceinline__ u32x2 lds_transposed(const lds_char *at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4 *)(at)));
}

// Workgroup `id` of its grid, whose arguments start at args_at.
template <int IO, int C, int DP, bool VT, bool INDEXED, bool GROUPED>
__device__ __forceinline__ void attention_many(const AttentionArgs &a, size_t args_at, uint32_t id,
                                               char *lds) {
  constexpr bool kFp8 = C != IO;
  constexpr bool kRelative = INDEXED && IO == KVX_DTYPE_F16;  // see kLeastScale
  constexpr int E = kFp8 ? 1 : 2;
  constexpr int KC = DP / 16;                   // products of 32 tokens' logits
  constexpr int NJ = DP / 32;                   // blocks of elements of the sums
  constexpr int ROW = DP * 2;                   // bytes of a row in LDS
  constexpr int CPR = DP * E / 16;              // 16-byte chunks of a cached row
  constexpr int NL = kManyStep * CPR / kManyThreads;  // of them a thread loads
  constexpr int NB = 2;                         // buffers
  constexpr int NVL = VT ? DP / 32 : NL;        // value loads (VT: 8 tokens of an element)
  constexpr int VLB = VT ? 8 * E : 16;
  constexpr int TENSOR = kManyStep * ROW;
  constexpr int BUFFER = 2 * TENSOR;  // keys, then values
  float *const scales = reinterpret_cast<float *>(lds + NB * BUFFER);  // [buffer][k, v][64]
  int *const infinities =
      reinterpret_cast<int *>(lds + many_lds<DP, INDEXED>() - 16);  // see add_infinities

  // The last tiles of a causal chunk see most tokens: they start first.
  const int hh = a.heads * a.head_tiles;
  const int y = (int)(id % (uint32_t)hh);
  id /= (uint32_t)hh;
  const int z = (int)(id % (uint32_t)a.splits);
  const int tile = a.tiles - 1 - (int)(id / (uint32_t)a.splits);
  QueryTile t;
  if (!find_tile(a, tile, &t)) return;
  const int tid = (int)threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int c = lane % 32, h = lane / 32;
  const int kvh = y / a.head_tiles;
  const int head0 = (y - kvh * a.head_tiles) * a.tile_heads;
  const int nheads = min(a.tile_heads, a.group - head0);
  const int D = a.head_dim;

  // This lane's row.
  const int r = 32 * wave + c;
  const int tok = r / a.tile_heads, rh = r - tok * a.tile_heads;
  const bool row = tok < t.count && rh < nheads;
  const int qh = kvh * a.group + head0 + rh;
  int rlo = 0, rhi = 0;
  if (row) row_range(a, t, t.first + tok, &rlo, &rhi);
  int lo, hi, first_hi, last_lo, from, to;
  row_range(a, t, t.first, &lo, &first_hi);
  row_range(a, t, t.first + t.count - 1, &last_lo, &hi);
  split_range(a, lo, hi, z, &from, &to);
  // The wave's rows see all of [all_lo, all_hi) and nothing outside [any_lo, any_hi).
  const int tok0 = 32 * wave / a.tile_heads;
  const int tok1 = min((32 * wave + 31) / a.tile_heads, t.count - 1);
  int any_lo = 0, any_hi = 0, all_lo = 0, all_hi = 0;
  if (tok0 < t.count) {
    row_range(a, t, t.first + tok0, &any_lo, &all_hi);
    row_range(a, t, t.first + tok1, &all_lo, &any_hi);
  }

  Frag q[KC];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    const int d = 16 * i + 8 * h;
    Raw<16> x{};
    if (row && d < D)
      x = ld<16>(a.q + (t.begin + t.first + tok) * a.q_tok + (int64_t)qh * a.q_head + 2 * d);
#pragma unroll
    for (int j = 0; j < 4; ++j) q[i].w[j] = x.w[j];
  }

  // What this thread loads of a step: a chunk each of the keys and values of
  // tokens tid / CPR + l * (256 / CPR); VT: 8 tokens of elements tid / 8 + 32 l.
  // Sixteen-bit elements go to LDS as they are, lane after lane, so that the
  // permutation of a row's chunks is one of what the lanes read.
  const int chunk = tid % CPR;
  const int kd0 = (kFp8 ? chunk : chunk ^ key_swap<DP>(tid / CPR)) * 16 / E;
  const int vd0 = (kFp8 ? chunk : chunk ^ value_swap<DP>(tid / CPR)) * 16 / E;
  const bool kinside = kd0 < D;
  const int kd = kinside ? kd0 : 0, vd = vd0 < D ? vd0 : 0;
  const uint32_t koff = (kd / a.gk.pack) * (int32_t)a.gk.s_piece + (kd % a.gk.pack) * E;
  const int vgroup8 = (tid % 8) ^ ((tid / 16) & 7);  // VT: 8 tokens of the step
  uint32_t voff[VT ? NVL : 1];
  if constexpr (VT) {
#pragma unroll
    for (int l = 0; l < NVL; ++l) {
      const int e = tid / 8 + 32 * l, d = e < D ? e : 0;
      voff[l] = (d / a.gv.pack) * (int32_t)a.gv.s_piece + (d % a.gv.pack) * (int32_t)a.gv.s_inner;
    }
  } else {
    voff[0] = (vd / a.gv.pack) * (int32_t)a.gv.s_piece + (vd % a.gv.pack) * E;
  }
  float ks = 1.0f, vs = 1.0f;
  if constexpr (kFp8 && !INDEXED) {
    ks = scale_of(a.ks, 0, kvh);
    vs = scale_of(a.vs, 0, kvh);
  }
  const float scale = positive_scale<IO>(a, ks, q);

  // GROUPED: lane i looks up the first token of the i-th group of 16, so that one
  // look serves 16 steps; else lane i looks up token i of one step.
  constexpr int kSteps = GROUPED ? 16 : 1;
  auto token_of_lane = [&](int base) { return base + (GROUPED ? 16 * lane : lane); };
  // Table entries are loaded one look ahead of their use.
  auto entries = [&](int base) -> TokenEntry {
    TokenEntry e{0, 0};
    if (token_of_lane(base) < to) e = token_entry(a, t, token_of_lane(base));
    return e;
  };
  struct Step {
    LaneRows rows;
    int lane0;       // GROUPED: the lane of its first group
    uint64_t there;  // bit per token that some row may see
  };
  auto step_at = [&](const LaneRows &rows, int base, int lane0) -> Step {
    // slots in front of a window hold anything
    const uint64_t held = GROUPED ? group_tokens((uint32_t)(rows.held >> lane0) & 15u) : rows.held;
    return {rows, lane0, held & tokens_between(lo, to, base, kManyStep)};
  };
  auto look = [&](int base, const TokenEntry &entry) {
    const int at = token_of_lane(base);
    return lane_rows<INDEXED, VT && !GROUPED ? 8 : 0>(a, entry, at, at < to, kvh);
  };

  // GROUPED: a wave's load takes kGroup tokens of one block, from one scalar
  // address.
  constexpr int kGroup = kWave / CPR;
  const uint32_t kgroup = koff + (uint32_t)((lane / CPR) * (int)a.gk.s_off);
  const uint32_t vgroup = voff[0] + (uint32_t)((lane / CPR) * (int)a.gv.s_off);
  // f(l, address, offset) for this thread's key and value loads.
  auto each_row = [&](const Step &s, uint64_t rows, int64_t s_off, uint32_t in_group,
                      uint32_t alone, auto f) {
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      constexpr int kLoad = kManyThreads / CPR;  // tokens of the workgroup's load
      const int at = wave * kGroup + l * kLoad;  // the wave's first
      if constexpr (GROUPED)
        f(l, address_of_lane(rows, s.lane0 + at / 16) + (at % 16) * s_off, in_group);
      else
        f(l, from_lane(rows, 4 * (at + lane / CPR)), alone);
    }
  };
  auto each_key = [&](const Step &s, auto f) {
    each_row(s, s.rows.k, a.gk.s_off, kgroup, koff, f);
  };
  auto each_value = [&](const Step &s, auto f) {
    if constexpr (VT) {
      uint64_t p;
      if constexpr (GROUPED)
        p = from_lane(s.rows.v, 4 * (s.lane0 + vgroup8 / 2)) + (vgroup8 % 2) * (8 * E);
      else
        p = from_lane(s.rows.v, 32 * vgroup8);
#pragma unroll
      for (int l = 0; l < NVL; ++l) f(l, p, voff[l]);
    } else {
      each_row(s, s.rows.v, a.gv.s_off, vgroup, voff[0], f);
    }
  };
  struct Staged {
    Raw<16> k[NL];
    Raw<VLB> v[NVL];
  };
  auto load = [&](const Step &s) -> Staged {
    Staged x{};
    if (s.rows.held == 0) return x;
    each_key(s, [&](int l, uint64_t p, uint32_t o) { x.k[l] = global_load<16, false>(p, o); });
    if constexpr (VT && !GROUPED) {
      if (s.rows.apart) {  // each token's block in turn
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          const uint64_t p = from_lane(s.rows.v, 32 * vgroup8 + 4 * e);
#pragma unroll
          for (int l = 0; l < NVL; ++l) {
            const Raw<VLB> r = global_load<VLB, false>(p, voff[l]);
#pragma unroll
            for (int w = 0; w < VLB / 4; ++w) {
              const uint32_t mine = token_bits<E>(e, w);
              x.v[l].w[w] = (x.v[l].w[w] & ~mine) | (r.w[w] & mine);
            }
          }
        }
        return x;
      }
    }
    each_value(s, [&](int l, uint64_t p, uint32_t o) { x.v[l] = global_load<VLB, false>(p, o); });
    return x;
  };
  // Straight into LDS, where nothing has to be changed on the way.
  auto load_lds = [&](const Step &s, lds_char *to) {
    to += wave * 1024;
    each_key(s, [&](int l, uint64_t p, uint32_t o) { copy_to_lds(p, o, to + l * 4096); });
    each_value(s, [&](int l, uint64_t p, uint32_t o) { copy_to_lds(p, o, to + TENSOR + l * 4096); });
  };
  // Whether all rows see all tokens of the step.
  auto plain = [&](const Step &s, int base) {
    return s.there == ~0ull && base >= last_lo && base + kManyStep <= first_hi;
  };
  // From registers: FP8 codes become elements, values of tokens that are not
  // there, NaN and infinities of steps that are not plain, and what is past a
  // key's end become 0.
  auto put = [&](char *line, int swap, const Raw<16> &x) {
    if constexpr (kFp8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        u32x4 o;
#pragma unroll
        for (int w = 0; w < 4; ++w) o[w] = widen<IO, C>(x.w[2 * i + w / 2], w % 2);
        *reinterpret_cast<u32x4 *>(line + 16 * ((2 * chunk + i) ^ swap)) = o;
      }
    } else {
      *reinterpret_cast<u32x4 *>(line + 16 * chunk) = u32x4{x.w[0], x.w[1], x.w[2], x.w[3]};
    }
  };
  auto store = [&](const Step &s, Staged &staged, int base, int buffer) {
    char *kb = lds + buffer * BUFFER, *vb = kb + TENSOR;
    if (!plain(s, base)) {
      uint32_t odd = 0;
#pragma unroll
      for (int l = 0; l < NVL; ++l) {
        const uint32_t have =
            VT ? (uint32_t)(s.there >> (8 * vgroup8)) & 0xFFu
               : (uint32_t)(s.there >> (tid / CPR + l * (kManyThreads / CPR))) & 1u ? 0xFFu : 0u;
#pragma unroll
        for (int w = 0; w < VLB / 4; ++w) {
          uint32_t keep;
          if constexpr (!VT) keep = have ? ~0u : 0u;
          else if constexpr (E == 2)
            keep = ((have >> (2 * w)) & 1 ? 0xFFFFu : 0u) |
                   ((have >> (2 * w + 1)) & 1 ? 0xFFFF0000u : 0u);
          else
            keep = ((have >> (4 * w)) & 1 ? 0xFFu : 0u) | ((have >> (4 * w)) & 2 ? 0xFF00u : 0u) |
                   ((have >> (4 * w)) & 4 ? 0xFF0000u : 0u) |
                   ((have >> (4 * w)) & 8 ? 0xFF000000u : 0u);
          const uint32_t x = staged.v[l].w[w] & keep;
          odd |= not_finite<C>(x);
          staged.v[l].w[w] = only_finite<C>(x);
        }
      }
      if (odd != 0) *infinities = 1;
    }
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      const int at = tid / CPR + l * (kManyThreads / CPR);
      put(kb + at * ROW, key_swap<DP>(at), D != DP && !kinside ? Raw<16>{} : staged.k[l]);
    }
    if constexpr (VT) {
#pragma unroll
      for (int l = 0; l < NVL; ++l) {
        u32x4 o;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if constexpr (kFp8) o[w] = widen<IO, C>(staged.v[l].w[w / 2], w % 2);
          else o[w] = staged.v[l].w[w];
        }
        *reinterpret_cast<u32x4 *>(vb + 16 * (tid + l * kManyThreads)) = o;
      }
    } else {
#pragma unroll
      for (int l = 0; l < NL; ++l) {
        const int at = tid / CPR + l * (kManyThreads / CPR);
        put(vb + at * ROW, value_swap<DP>(at), staged.v[l]);
      }
    }
    if constexpr (INDEXED && !GROUPED) {
      if (wave == 0) {
        scales[(2 * buffer) * kManyStep + lane] = s.rows.ks;
        scales[(2 * buffer + 1) * kManyStep + lane] = s.rows.vs;
      }
    }
  };

  float m = -INFINITY, l = 0.0f, unit = kLeastScale;
  f32x16 acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = f32x16{};

  // The scales of tokens 32 b + 8 i + 4 h .. + 3 of a step.
  auto token_scales = [&](const Step &s, float x, int buffer, int which, int b, int i) -> f32x4 {
    if constexpr (GROUPED) {
      const float y = bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(x),
                                                                  s.lane0 + 2 * b + i / 2));
      return f32x4{y, y, y, y};
    } else {
      return *reinterpret_cast<const f32x4 *>(scales + (2 * buffer + which) * kManyStep + 32 * b +
                                              8 * i + 4 * h);
    }
  };
  auto step = [&](const Step &now, int base, int buffer, const lds_char *cur) {
    if (base >= any_hi || base + kManyStep <= any_lo || now.there == 0) return;
    // Rows start at multiples of their length, so that the permutation is an
    // exclusive or of the address.
    const int kb = c * ROW + 16 * (h ^ key_swap<DP>(c));
    f32x16 s[2] = {};
    {
      // The two halves in turn: their sums do not wait for each other.
      auto key = [&](int i) -> Frag {
        const u32x4 x = lds_read<u32x4>(cur + (kb ^ (32 * (i / 2))) + (i % 2) * 32 * ROW);
        return {{x[0], x[1], x[2], x[3]}};
      };
      Frag k[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) k[i] = key(i);
      __builtin_amdgcn_s_setprio(1);  // products go before the other wave's weights
#pragma unroll
      for (int i = 0; i < 2 * KC; ++i) {
        __builtin_amdgcn_sched_barrier(kMayCross);
        s[i % 2] = mma<IO>(k[i % kAhead], q[i / 2], s[i % 2]);
        if (i + kAhead < 2 * KC) k[i % kAhead] = key(i + kAhead);
      }
      __builtin_amdgcn_sched_barrier(kMayCross);
      __builtin_amdgcn_s_setprio(0);
    }
    const bool whole = now.there == ~0ull && base >= all_lo && base + kManyStep <= all_hi;
    float top = -INFINITY;
    uint32_t hidden = 0;  // bit 16 b + i: this lane's row does not see its token i of half b
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if constexpr (INDEXED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = token_scales(now, now.rows.ks, buffer, 0, b, i);
#pragma unroll
          for (int w = 0; w < 4; ++w) s[b][4 * i + w] *= x[w];
        }
      }
      if (a.softcap != 0.0f) cap_logits<IO, false, f32x16, 16>(a, ks, s[b]);
      if (!whole) {
        const uint32_t there = (uint32_t)(now.there >> (32 * b)) >> (4 * h);
        const int start = base + 32 * b + 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = 8 * (i / 4) + i % 4;
          const bool seen = ((there >> at) & 1) & (start + at >= rlo) & (start + at < rhi);
          s[b][i] = seen ? s[b][i] : -INFINITY;
          hidden |= seen ? 0u : 1u << (16 * b + i);
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);  // NaN does not move it
    }
    top = reference_maximum<IO>(fmaxf(top, __shfl_xor(top, 32)) * scale, kRoom);
    if (__any(top > m + (IO == KVX_DTYPE_F16 && is_far(top) ? 0.0f : (float)kRoom))) {
      const float now_m = fmaxf(top, m);
      const float alpha = __builtin_amdgcn_exp2f(m - (now_m == -INFINITY ? 0.0f : now_m));
      m = now_m;
      l *= alpha;
      if constexpr (kRelative) {
        unit *= alpha;
      } else {
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] *= alpha;
      }
    }
    const float shift = m == -INFINITY ? 0.0f : m;
    Frag w[4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float part = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], scale, -shift));
        part += s[b][i];
      }
      l += part;
      asm volatile("" : "+v"(l));  // summed here, not after the products: fewer live registers
      if constexpr (INDEXED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // by selection: see the few-row kernel
          const f32x4 x = token_scales(now, now.rows.vs, buffer, 1, b, i);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            s[b][4 * i + k] *= (hidden >> (16 * b + 4 * i + k)) & 1 ? 0.0f : x[k];
        }
      }
    }
    if constexpr (kRelative) {
      float most = 0.0f;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(s[b][i]));
      most = fmaxf(most, __shfl_xor(most, 32));
      const float fresh = reference_of(unit, most);
      if (__any(fresh != unit)) {
        const float ratio = unit / fresh;
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[j] *= ratio;
        unit = fresh;
      }
      const float inv = __builtin_amdgcn_rcpf(unit);
#pragma unroll
      for (int b = 0; b < 2; ++b) s[b] *= inv;
    }
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[2 * b + i / 4].w[i % 4] = pair_of<IO>(s[b][2 * i], s[b][2 * i + 1]);
    // Values of 16 tokens (in the weights' order) of element 32 j + c.
    const int li = lane % 16;
    const lds_char *values_at = cur + TENSOR;
    const int vb = VT ? c * (kManyStep * 2) + 8 * h + 16 * ((c / 2) % 8)
                      : (4 * h + li / 4) * ROW + 8 * (li % 2) +
                            16 * ((2 * ((lane / 16) % 2) + (li % 4) / 2) ^ value_swap<DP>(li / 4));
    auto values = [&](int kk, int j) -> Frag {
      Frag f;
      u32x2 x, y;
      if constexpr (VT) {  // chunks of 8 tokens, permuted by the element
        x = lds_read<u32x2>(values_at + (vb ^ (32 * kk)) + 32 * j * (kManyStep * 2));
        y = lds_read<u32x2>(values_at + (vb ^ (32 * kk + 16)) + 32 * j * (kManyStep * 2));
      } else {
        x = lds_transposed(values_at + (vb ^ (64 * j)) + 16 * kk * ROW);
        y = lds_transposed(values_at + (vb ^ (64 * j)) + (16 * kk + 8) * ROW);
      }
      f.w[0] = x[0];
      f.w[1] = x[1];
      f.w[2] = y[0];
      f.w[3] = y[1];
      return f;
    };
    Frag v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = values(i / NJ, i % NJ);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < 4 * NJ; ++i) {
      __builtin_amdgcn_sched_barrier(kMayCross);
      acc[i % NJ] = mma<IO>(v[i % kAhead], w[i / NJ], acc[i % NJ]);
      if (i + kAhead < 4 * NJ) v[i % kAhead] = values((i + kAhead) / NJ, (i + kAhead) % NJ);
    }
    __builtin_amdgcn_sched_barrier(kMayCross);
    __builtin_amdgcn_s_setprio(0);
  };

  // The two buffers are told apart by the parameters' __restrict__: a transposing
  // read would else wait for the loads into the other buffer.
  auto turn = [&](const lds_char *__restrict__ cur, lds_char *__restrict__ other, const Step &now,
                  const Step &next, int base, int buffer, bool direct) {
    if (direct) load_lds(next, other);
    step(now, base, buffer, cur);
  };

  if (tid == 0) *infinities = 0;
  __syncthreads();
  if (from < to) {
    // The step after this one, from rows that serve kSteps steps; past `to`
    // nothing is there.
    LaneRows rows = look(from, entries(from));
    Step now = step_at(rows, from, 0);
    Staged staged = load(now);
    TokenEntry ahead = entries(from + kSteps * kManyStep);
    int count = 0;
    auto advance = [&](int at) -> Step {
      count = (count + 1) % kSteps;
      if (count == 0) {
        rows = look(at, ahead);
        ahead = entries(at + kSteps * kManyStep);
      }
      return step_at(rows, at, 4 * count);
    };
    store(now, staged, from, 0);
    Step next = advance(from + kManyStep);
    __syncthreads();
    int buffer = 0;
    for (int base = from;; base += kManyStep) {
      const bool more = base + kManyStep < to;
      const bool direct =
          !kFp8 && D == DP && plain(next, base + kManyStep) && !(VT && next.rows.apart);
      if (more) {
        if constexpr (kFp8) staged = load(next);
      }
      turn((lds_char *)lds + buffer * BUFFER, (lds_char *)lds + (buffer ^ 1) * BUFFER, now, next,
           base, buffer, direct && more);
      if (!more) break;
      buffer ^= 1;
      if (!direct) {
        if constexpr (!kFp8) staged = load(next);
        store(next, staged, base + kManyStep, buffer);
      }
      now = next;
      next = advance(base + 2 * kManyStep);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what went straight into LDS
      __syncthreads();
    }
  }
  l += __shfl_xor(l, 32);
  if constexpr (kRelative) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] *= unit;
  }
  const bool none = m == -INFINITY && l == 0.0f;
  const int64_t line = t.begin + t.first + tok;
  if (row && a.splits > 1) {
    const int64_t at = part_index(a, t, t.first + tok, qh) * a.splits + z;
    if (h == 0) {
      a.part_ml[2 * at] = m;
      a.part_ml[2 * at + 1] = l;
    }
    if (!none) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = 32 * j + 8 * i + 4 * h;
          if (d < D)
            *reinterpret_cast<f32x4 *>(a.part_o + at * D + d) =
                f32x4{acc[j][4 * i], acc[j][4 * i + 1], acc[j][4 * i + 2], acc[j][4 * i + 3]} * vs;
        }
    }
  } else if (row) {
    if (h == 0 && a.lse != nullptr)
      a.lse[line * (a.heads * a.group) + qh] = none ? -INFINITY : (m + log2f(l)) * kLn2;
    const float norm = vs / l;
    char *out = a.out + line * a.o_tok + (int64_t)qh * a.o_head;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = 32 * j + 8 * i + 4 * h;
        if (d >= D) continue;
        Raw<8> o;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float x0 = none ? 0.0f : acc[j][4 * i + 2 * k] * norm;
          const float x1 = none ? 0.0f : acc[j][4 * i + 2 * k + 1] * norm;
          o.w[k] = pack_pair<IO>(f32x2{x0, x1});
        }
        st<8>(out + 2 * d, o);
      }
  }
  __syncthreads();
  if (*infinities != 0)
    add_infinities<IO, C, kManyStep, true>(args_address(args_at), tile, z, y);
}

// A batch's sequences of few new tokens, beside the ones of many: their
// workgroups start first, and wait for memory while the others compute (12
// sequences, 4 of them chunks of 100 to 500 new tokens, with a window of 1024, 4 kv
// heads of 64: 53 us with the join, 9 more as two launches; a chunk that is alone
// takes 1 to 4 % longer for the code that it does not run).
//
// Heads of 64: three waves a SIMD, for which the FP8 forms move 3 to 25 registers
// through scratch memory (with block scales 15 to 45, those of 128 and 256 up to 20)
// and the BF16 ones with the token axis innermost 3 to 7.  Short chunks gain by the
// third wave, long ones lose: 10 chunks of 256 tokens at 2048, FP8, three and two
// waves: 91 and 109 us, with block scales 119 and 128; 2 of 2048 at 4096 to 8192: 233
// and 227, with block scales 329 and 295, token axis innermost 257 and 234; BF16 240
// and 238, token axis innermost 240 and 231.
struct MixedArgs {
  AttentionArgs many, few;
  uint32_t few_grid;
};

template <int IO, int C, int DP, bool VT, bool INDEXED, bool GROUPED>
__global__ void __launch_bounds__(kManyThreads, DP == 256 ? 1 : DP == 128 ? 2 : 3)
    attention_many_kernel(MixedArgs x) {
  extern __shared__ __align__(1024) char lds[];
  static_assert(sizeof(FewShared<DP>) <= many_lds<DP, INDEXED>() && kFewThreads == kManyThreads);
  if (blockIdx.x < x.few_grid)
    attention_few<IO, C, DP, VT, INDEXED, GROUPED, false>(
        x.few, offsetof(MixedArgs, few), blockIdx.x,
        *reinterpret_cast<FewShared<DP> *>(lds));
  else
    attention_many<IO, C, DP, VT, INDEXED, GROUPED>(x.many, offsetof(MixedArgs, many),
                                                     blockIdx.x - x.few_grid, lds);
}

// few: null where no sequence can have few new tokens; p.grid: 0 where none can
// have many.
template <int IO, int C>
void launch_many(const AttentionPart &p, const AttentionPart *few, bool vt, bool grouped,
                 hipStream_t s) {
  with_variant<IO, C>(p.a, vt, grouped, [&](auto dp, auto vt_, auto indexed_, auto grouped_) {
    constexpr int kDim = decltype(dp)::value;
    constexpr bool kIndexed = decltype(indexed_)::value;
    constexpr size_t kLds = many_lds<kDim, kIndexed>();
    const auto kernel =
        attention_many_kernel<IO, C, kDim, decltype(vt_)::value, kIndexed, decltype(grouped_)::value>;
    if (kLds > 65536)  // more than a kernel has unasked
      (void)hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds);
    const MixedArgs x{p.a, few ? few->a : p.a, few ? few->grid : 0};
    kernel<<<dim3(p.grid + x.few_grid), kManyThreads, kLds, s>>>(x);
  });
}

}  // namespace dev
}  // namespace kvx
