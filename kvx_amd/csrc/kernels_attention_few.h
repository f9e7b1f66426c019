// Attention of few rows per kv head (decode steps, drafts, short chunks) on
// the matrix cores.
//
// Every cached key and value is read once per tile of 16 rows and takes part
// in 16 products of each kind (4 * 16 operations for 2 elements), far below
// the matrix rate: HBM bounds it, and all that matters is loads in flight.  So
// the waves do not share anything while they run: a wave takes every fourth
// step of 32 tokens of its workgroup's range, loads its keys and values
// straight from HBM into the registers that the matrix instructions read, and
// the four waves join their sums through LDS at the end.
//
// v_mfma_f32_16x16x32: lane l = 16 g + c holds A[row c][8 g .. 8 g + 7],
// B[8 g .. 8 g + 7][column c] and D[rows 4 g .. 4 g + 3][column c].
//
//   S^T = K Q^T   A: 16 tokens, so that lane c reads 16 bytes of token c's key
//                 where they lie.  D: lane c has row c of the queries, tokens
//                 4 g + i of each half of the step.
//   O^T = V^T P^T B: row c's weights of tokens 4 g + i and 16 + 4 g + i, which
//                 are the lane's own logits; no exchange.  The order of the
//                 sum's 32 tokens is free, so A takes them in the same order.
//                 A: values by element, tokens across.  From rows, a lane
//                 loads NV = DP / 16 elements of eight tokens and transposes
//                 them with v_perm (half an operation an element); from a
//                 cache whose token axis is innermost it loads four tokens of
//                 one element, as they are.
//
// F32: v_mfma_f32_16x16x4, lane l has A[row c][g] and B[g][column c].  Element
// 16 i + 4 g + w of a key is the w-th of the lane's i-th load, and takes part in
// the product 4 i + w with the query's element of that place; values need no
// transposition, a product takes tokens 4 g + i of the four groups.  Wide F32
// rows take steps of 16 tokens for two waves a SIMD, which at heads of 128 still
// move 8 to 20 registers through scratch memory (16 sequences of 4096 tokens: 107 us,
// 111 with 32 tokens and one wave; heads of 256: 242, and 584 with 32 tokens).
//
// Measured, 64 sequences of 2048 tokens, 8 kv heads of 128, groups of 4: BF16 97 us
// (5.5 TB/s), FP8 62 us (4.3 TB/s; with block scales 63), F32 195 us (5.5 TB/s);
// heads of 256, BF16 193 us (5.6 TB/s), FP8 104 (5.2); 200 of 4000 tokens, FP8: 320 us
// (5.1 TB/s).  More waves a SIMD in fewer registers spill: BF16 at three 142 us.
//
// Keys and values that one tile reads are streamed past the caches (5 sequences
// of 16384 to 32768 tokens: 85 us, 94 without), unless a sequence may have two
// tiles, whose second reads come from L2 then (64 sequences of 2048 with 8 new
// tokens each: 133 us, 165 streamed).
//
// Maximum and sum are one register each, as a lane has one row; the maximum
// is shared over the four lane groups, the sum only at the end.  Weights are
// rounded to the queries' type for the product (half a step of 2^-8 or 2^-11
// relative, as the output is rounded), their sum is not.
#pragma once

#include "attention_mfma.h"

namespace kvx {
namespace dev {

constexpr int kFewWaves = 4;
constexpr int kFewThreads = kFewWaves * kWave;

// Token e of a lane's eight in a step, from its group's first.
__device__ __forceinline__ constexpr int place_of(int e) { return e < 4 ? e : 12 + e; }

template <int DP>
struct FewShared {
  float sums[2][kRowTile][DP + 4];
  float states[kFewWaves][2][kRowTile];
  int infinities;  // see add_infinities
};

// Workgroup `id` of its grid, whose arguments start at args_at.  IO: type of
// queries and of the products; C: the cache's type; DP: head_dim rounded up to 64,
// 128 or 256; VT: values with the token axis innermost; INDEXED: scales by block;
// GROUPED: blocks hold whole groups of 16 tokens; STREAM: keys and values are read
// past the caches (and 16-bit queries may have a softcap past near_cap).
template <int IO, int C, int DP, bool VT, bool INDEXED, bool GROUPED, bool STREAM>
__device__ __forceinline__ void attention_few(const AttentionArgs &a, size_t args_at, uint32_t id,
                                              FewShared<DP> &shared) {
  constexpr bool kFp8 = C != IO, kF32 = IO == KVX_DTYPE_F32;
  constexpr int E = bytes_of_type<C>();
  constexpr bool kRelative = INDEXED && IO == KVX_DTYPE_F16;  // see kLeastScale
  constexpr int KC = kF32 ? DP / 16 : DP / 32;  // operands of a half step's logits
  constexpr int KL = DP * E / 64;      // 16-byte key loads of a token and lane group
  constexpr int NV = DP / 16;          // products of a step's sums; elements a lane loads
  constexpr int VB = NV * E;           // bytes of them
  // groups of 16 tokens in a step
  constexpr int HALVES = kF32 && DP * E >= 512 ? 1 : 2;
  constexpr int kFewStep = 16 * HALVES;  // tokens
  constexpr uint32_t kAll = 0xFFFFFFFFu >> (32 - kFewStep);
  constexpr int VW = VB / 4;           // dwords (VT: of four tokens)
  auto &sums = shared.sums;
  auto &states = shared.states;
  int &infinities = shared.infinities;

  // Heads in turn, or (heads_near) eight tiles' parts in turn: one for each die.
  const uint32_t hh = (uint32_t)(a.heads * a.head_tiles);
  int y;
  if (a.heads_near) {
    y = (int)(id / kDies % hh);
    id = id / (kDies * hh) * kDies + id % kDies;
  } else {
    y = (int)(id % hh);
    id /= hh;
  }
  const int z = (int)(id % (uint32_t)a.splits);
  const int tile = (int)(id / (uint32_t)a.splits);
  QueryTile t;
  if (tile >= a.tiles || !find_tile(a, tile, &t)) return;
  const int lane = (int)(threadIdx.x % kWave);
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x / kWave));
  const int c = lane % 16, g = lane / 16;
  const int kvh = y / a.head_tiles;
  const int head0 = (y - kvh * a.head_tiles) * a.tile_heads;
  const int nheads = min(a.tile_heads, a.group - head0);
  const int D = a.head_dim;

  // This lane's row.
  const int tok = c / a.tile_heads, h = c - tok * a.tile_heads;
  const bool row = tok < t.count && h < nheads;
  const int qh = kvh * a.group + head0 + h;
  int rlo = 0, rhi = 0;
  if (row) row_range(a, t, t.first + tok, &rlo, &rhi);
  int lo, hi, first_hi, last_lo, from, to;
  row_range(a, t, t.first, &lo, &first_hi);
  row_range(a, t, t.first + t.count - 1, &last_lo, &hi);
  split_range(a, lo, hi, z, &from, &to);
  if (a.splits > 1 && from >= to) {  // nothing for this split: say so
    if (wave == 0 && g == 0 && row) {
      const int64_t at = part_index(a, t, t.first + tok, qh) * a.splits + z;
      a.part_ml[2 * at] = -INFINITY;
      a.part_ml[2 * at + 1] = 0.0f;
    }
    return;
  }

  if (threadIdx.x == 0) infinities = 0;
  __syncthreads();
  Frag q[KC];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    // FP8: two (F32: four) operands share a 16-byte load of 16 elements
    constexpr int N = kF32 ? 4 : 8, kShare = kFp8 ? 16 / N : 1;
    const int d = N * (4 * kShare * (i / kShare) + kShare * g + i % kShare);
    Raw<16> r{};
    if (row && d < D)
      r = ld<16>(a.q + (t.begin + t.first + tok) * a.q_tok + (int64_t)qh * a.q_head +
                 d * bytes_of_type<IO>());
#pragma unroll
    for (int j = 0; j < 4; ++j) q[i].w[j] = r.w[j];
  }

  // Offsets of the lane's pieces from a token's row; a piece past the head's
  // end is its first one (a key's counts as zero below, a value's sum is not
  // stored).
  uint32_t koff[KL];
#pragma unroll
  for (int i = 0; i < KL; ++i) {
    const int d0 = (i * 64 + g * 16) / E, d = d0 < D ? d0 : 0;
    koff[i] = (d / a.gk.pack) * (int32_t)a.gk.s_piece + (d % a.gk.pack) * E;
  }
  constexpr int VL = VT ? NV : (VB + 15) / 16;  // value loads a token (VT: four tokens)
  constexpr int VLB = VT ? 4 * E : VB / VL;      // bytes of one
  uint32_t voff[VL];
#pragma unroll
  for (int i = 0; i < VL; ++i) {
    const int d0 = VT ? 16 * i + c : c * NV + i * (VLB / E), d = d0 < D ? d0 : 0;
    voff[i] = (d / a.gv.pack) * (int32_t)a.gv.s_piece + (d % a.gv.pack) * (int32_t)a.gv.s_inner;
  }
  float ks = 1.0f, vs = 1.0f;
  if constexpr (kFp8 && !INDEXED) {
    ks = scale_of(a.ks, 0, kvh);
    vs = scale_of(a.vs, 0, kvh);
  }

  // F32: the factor's rest too, or all logits would be off by its rounding.
  float scale = positive_scale<IO>(a, ks, q), scale_rest = 0.0f;
  if constexpr (kF32) {
    const float hi = a.softcap != 0.0f ? a.cap : a.scale_log2, by = a.softcap != 0.0f ? 1.0f : ks;
    const float product = hi * by;
    if (product != 0.0f) {
      scale = fabsf(product);
      scale_rest = fmaf(hi, by, -product) + (a.softcap != 0.0f ? a.cap_rest : a.scale_rest) * by;
      scale_rest = product < 0.0f ? -scale_rest : scale_rest;
    }
  }
  float m = -INFINITY, l = 0.0f, unit = kLeastScale;
  f32x4 acc[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // GROUPED: blocks hold whole half steps, whose rows follow from the first, a
  // scalar address.
  const uint32_t krow = (uint32_t)(c * (int)a.gk.s_off);
  const uint32_t vrow = (uint32_t)(4 * g * (int)a.gv.s_off);

  constexpr int kStride = kFewWaves * kFewStep;
  // GROUPED: lane HALVES i + b looks up the first token of half b of the wave's
  // i-th step, so that one look serves 32 steps; else lane i looks up token i of
  // one.
  constexpr int kSteps = GROUPED ? kWave / HALVES : 1;
  auto token_of_lane = [&](int base) {
    return GROUPED ? base + (lane / HALVES) * kStride + 16 * (lane % HALVES) : base + lane;
  };
  auto looks = [&](int base) {
    return token_of_lane(base) < to && (GROUPED || lane < kFewStep);
  };
  // Table entries are loaded one look ahead of their use.
  auto entries = [&](int base) -> TokenEntry {
    TokenEntry e{0, 0};
    if (looks(base)) e = token_entry(a, t, token_of_lane(base));
    return e;
  };
  struct Step {
    LaneRows rows;
    int lane0;       // GROUPED: the lane of its first half
    uint32_t there;  // bit per token that some row may see
  };
  auto step_at = [&](const LaneRows &rows, int base, int lane0) -> Step {
    // Tokens in front of a window are of the block, but nobody's: they may hold
    // anything.
    const uint32_t in = (uint32_t)tokens_between(lo, to, base, kFewStep);
    const uint32_t held =
        GROUPED ? (uint32_t)group_tokens((uint32_t)(rows.held >> lane0) & (2u * HALVES - 1))
                : (uint32_t)rows.held;
    return {rows, lane0, held & in};
  };
  auto look = [&](int base, const TokenEntry &entry) {
    return lane_rows<INDEXED, VT && !GROUPED ? 4 : 0>(a, entry, token_of_lane(base), looks(base),
                                                      kvh);
  };
  // A token's scale, of the eight that the lane has.
  auto token_scale = [&](const Step &s, float x, int e) {
    return GROUPED ? from_lane(x, 4 * (s.lane0 + e / 4)) : from_lane(x, 16 * g + 4 * place_of(e));
  };
  uint32_t kw[HALVES][KL][4];
  auto load_keys = [&](const Step &s) {
    if (s.rows.held == 0) return;
    auto one = [&](int b, uint64_t p, uint32_t row) {
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const Raw<16> r = global_load<16, STREAM>(p, row + koff[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) kw[b][i][j] = r.w[j];
      }
    };
#pragma unroll
    for (int b = 0; b < HALVES; ++b) {
      if constexpr (GROUPED) one(b, address_of_lane(s.rows.k, s.lane0 + b), krow);
      else one(b, from_lane(s.rows.k, 4 * c + 64 * b), 0);
    }
  };
  // Rows: [token e][dword]; VT: [half b][element j][dword].
  uint32_t vw[VT ? HALVES * NV : 4 * HALVES][VT ? E : VW];
  auto load_values = [&](const Step &s) {
    if (s.rows.held == 0) return;
    if constexpr (VT && !GROUPED) {
      if (s.rows.apart) {  // each token's block in turn
#pragma unroll 1
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int b = 0; b < HALVES; ++b) {
            const uint64_t p = from_lane(s.rows.v, 16 * g + 64 * b + 4 * e);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
              const Raw<VLB> r = global_load<VLB, STREAM>(p, voff[j]);
#pragma unroll
              for (int w = 0; w < E; ++w) {
                const uint32_t mine = token_bits<E>(e, w);
                vw[b * NV + j][w] = (vw[b * NV + j][w] & ~mine) | (r.w[w] & mine);
              }
            }
          }
        return;
      }
    }
    if constexpr (VT) {
#pragma unroll
      for (int b = 0; b < HALVES; ++b) {
        uint64_t p;
        if constexpr (GROUPED) p = address_of_lane(s.rows.v, s.lane0 + b);
        else p = from_lane(s.rows.v, 16 * g + 64 * b);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const Raw<VLB> r = global_load<VLB, STREAM>(p, (GROUPED ? 4 * g * E : 0) + voff[j]);
#pragma unroll
          for (int w = 0; w < E; ++w) vw[b * NV + j][w] = r.w[w];
        }
      }
    } else {
      auto one = [&](int e, uint64_t p, uint32_t row) {
#pragma unroll
        for (int i = 0; i < VL; ++i) {
          const Raw<VLB> r = global_load<VLB, STREAM>(p, row + voff[i]);
#pragma unroll
          for (int w = 0; w < VLB / 4; ++w) vw[e][i * (VLB / 4) + w] = r.w[w];
        }
      };
#pragma unroll
      for (int e = 0; e < 4 * HALVES; ++e) {
        if constexpr (GROUPED)
          one(e, address_of_lane(s.rows.v, s.lane0 + e / 4) + (e % 4) * a.gv.s_off, vrow);
        else one(e, from_lane(s.rows.v, 16 * g + 4 * place_of(e)), 0);
      }
    }
  };
  // Values of tokens that are not there become 0: their slots hold anything.
  auto clear_values = [&](uint32_t there) {
    if constexpr (VT) {
#pragma unroll
      for (int b = 0; b < HALVES; ++b) {
        const uint32_t have = (there >> (4 * g)) >> (16 * b);
#pragma unroll
        for (int w = 0; w < E; ++w) {
          const uint32_t keep =
              E == 4   ? (have >> w) & 1 ? ~0u : 0u
              : E == 2 ? ((have >> (2 * w)) & 1 ? 0xFFFFu : 0u) |
                           ((have >> (2 * w + 1)) & 1 ? 0xFFFF0000u : 0u)
                     : (have & 1 ? 0xFFu : 0u) | (have & 2 ? 0xFF00u : 0u) |
                           (have & 4 ? 0xFF0000u : 0u) | (have & 8 ? 0xFF000000u : 0u);
#pragma unroll
          for (int j = 0; j < NV; ++j) vw[b * NV + j][w] &= keep;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4 * HALVES; ++e) {
        const uint32_t keep = ((there >> (4 * g)) >> place_of(e)) & 1 ? ~0u : 0u;
#pragma unroll
        for (int w = 0; w < VW; ++w) vw[e][w] &= keep;
      }
    }
  };

  int base = from + wave * kFewStep;
  if (base < to) {
    // The step after this one, from rows that serve kSteps steps; past `to`
    // nothing is there.
    LaneRows rows = look(base, entries(base));
    Step now = step_at(rows, base, 0);
    load_keys(now);
    load_values(now);
    TokenEntry ahead = entries(base + kSteps * kStride);
    int count = 0;
    auto advance = [&](int at) -> Step {
      count = (count + 1) % kSteps;
      if (count == 0) {
        rows = look(at, ahead);
        ahead = entries(at + kSteps * kStride);
      }
      return step_at(rows, at, HALVES * count);
    };
    Step next = advance(base + kStride);
    for (;;) {
      if (D != DP) {  // pieces past the head's end
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const uint32_t keep = (i * 64 + g * 16) / E < D ? ~0u : 0u;
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int b = 0; b < HALVES; ++b) kw[b][i][j] &= keep;
        }
      }
      // Logits: lane c has its row's tokens base + 16 b + 4 g + i.
      f32x4 s[HALVES] = {};
#pragma unroll
      for (int b = 0; b < HALVES; ++b) {
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          Frag k;
          if constexpr (kF32) {
            // the halves in turn, whose sums do not wait for each other
            if (b == 1) continue;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
#pragma unroll
              for (int half = 0; half < HALVES; ++half) {
                const float x = kFp8 ? code<C>(kw[half][i / 4][i % 4], w)
                                     : bits_f32(kw[half][kFp8 ? 0 : i][w]);
                s[half] = mma4(x, bits_f32(q[i].w[w]), s[half]);
              }
            }
            continue;
          } else if constexpr (kFp8) {
#pragma unroll
            for (int w = 0; w < 4; ++w)
              k.w[w] = widen<IO, C>(kw[b][i / 2][2 * (i % 2) + w / 2], w % 2);
          } else {
#pragma unroll
            for (int w = 0; w < 4; ++w) k.w[w] = kw[b][i][w];
          }
          s[b] = mma<IO>(k, q[i], s[b]);
        }
      }
      const bool more = base + kStride < to;
      if (more) load_keys(next);

      const bool whole = now.there == kAll && base >= last_lo && base + kFewStep <= first_hi;
      float x[4 * HALVES], p[4 * HALVES], top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4 * HALVES; ++e) {
        x[e] = s[e / 4][e % 4];
        if constexpr (INDEXED) x[e] *= token_scale(now, now.rows.ks, e);
      }
      if (a.softcap != 0.0f) {
        if constexpr (kF32) {
#pragma unroll
          for (int e = 0; e < 4 * HALVES; ++e) x[e] = capped_part(a, x[e] * ks);
        } else {
          cap_logits<IO, STREAM, decltype(x), 4 * HALVES>(a, ks, x);
        }
      }
      uint32_t hidden = 0;  // bit e: this lane's row does not see its token e
      if (!whole) {
        const uint32_t there = now.there >> (4 * g);
        const int start = base + 4 * g;
#pragma unroll
        for (int e = 0; e < 4 * HALVES; ++e) {
          const int at = start + place_of(e);
          const bool seen = ((there >> place_of(e)) & 1) & (at >= rlo) & (at < rhi);
          x[e] = seen ? x[e] : -INFINITY;
          hidden |= seen ? 0u : 1u << e;
        }
      }
#pragma unroll
      for (int e = 0; e < 4 * HALVES; ++e) top = fmaxf(top, x[e]);  // NaN does not move it
      top = fmaxf(top, __shfl_xor(top, 16));
      top = reference_maximum<IO>(fmaxf(top, __shfl_xor(top, 32)) * scale, 0);
      top = fmaxf(top, m);
      const float shift = top == -INFINITY ? 0.0f : top;
      if (__any(top > m)) {
        const float alpha = __builtin_amdgcn_exp2f(m - shift);
        l *= alpha;
        if constexpr (kRelative) {
          unit *= alpha;
        } else {
#pragma unroll
          for (int j = 0; j < NV; ++j) acc[j] *= alpha;
        }
      }
      m = top;
#pragma unroll
      for (int e = 0; e < 4 * HALVES; ++e) {
        float y = fmaf(x[e], scale, -shift);
        if constexpr (kF32) y += fmaxf(x[e], -3e38f) * scale_rest;  // no infinity by 0
        p[e] = __builtin_amdgcn_exp2f(y);
        l += p[e];
      }
      if constexpr (INDEXED) {
        // Values stay codes; weights carry the tokens' scales.  A page in front of
        // the window may have slid out of it and its scale be anything: one that
        // the row does not see counts as 0, by selection.
#pragma unroll
        for (int e = 0; e < 4 * HALVES; ++e) {
          const float by = token_scale(now, now.rows.vs, e);
          p[e] *= (hidden >> e) & 1 ? 0.0f : by;
        }
        if constexpr (kRelative) {
          float most = 0.0f;
#pragma unroll
          for (int e = 0; e < 4 * HALVES; ++e) most = fmaxf(most, fabsf(p[e]));
          most = fmaxf(most, __shfl_xor(most, 16));
          most = fmaxf(most, __shfl_xor(most, 32));
          const float fresh = reference_of(unit, most);
          if (__any(fresh != unit)) {
            const float ratio = unit / fresh;
#pragma unroll
            for (int j = 0; j < NV; ++j) acc[j] *= ratio;
            unit = fresh;
          }
          const float inv = __builtin_amdgcn_rcpf(unit);
#pragma unroll
          for (int e = 0; e < 4 * HALVES; ++e) p[e] *= inv;
        }
      }
      if (now.there != kAll) clear_values(now.there);
      if (t.count > 1 && (base < last_lo || base + kFewStep > first_hi)) {
        uint32_t odd = 0;  // some rows do not see some tokens
#pragma unroll
        for (int e = 0; e < (VT ? HALVES * NV : 4 * HALVES); ++e)
#pragma unroll
          for (int i = 0; i < (VT ? E : VW); ++i) {
            odd |= not_finite<C>(vw[e][i]);
            vw[e][i] = only_finite<C>(vw[e][i]);
          }
        if (odd != 0) infinities = 1;
      }
      if constexpr (kF32) {
#pragma unroll
        for (int e = 0; e < 4 * HALVES; ++e)
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            float x;
            if constexpr (VT)
              x = kFp8 ? code<C>(vw[(e / 4) * NV + j][0], e % 4)
                       : bits_f32(vw[(e / 4) * NV + j][kFp8 ? 0 : e % 4]);
            else
              x = kFp8 ? code<C>(vw[e][j / 4], j % 4) : bits_f32(vw[e][kFp8 ? 0 : j]);
            acc[j] = mma4(x, p[e], acc[j]);
          }
      } else {
        Frag w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w.w[i] = pair_of<IO>(p[2 * i], p[2 * i + 1]);
        // Values by element: v[j], token order of the weights.
        auto by_element = [&](int d, Frag *v) {  // v[2 d] and v[2 d + 1]
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (VT) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int at = (i / 2) * NV + 2 * d + k;
                v[k].w[i] = kFp8 ? widen<IO, C>(vw[at][0], i % 2) : vw[at][kFp8 ? 0 : i % 2];
              }
            } else {
              uint32_t t0, t1;
              if constexpr (kFp8) {
                t0 = widen<IO, C>(vw[2 * i][d / 2], d % 2);
                t1 = widen<IO, C>(vw[2 * i + 1][d / 2], d % 2);
              } else {
                t0 = vw[2 * i][d];
                t1 = vw[2 * i + 1][d];
              }
              v[0].w[i] = __builtin_amdgcn_perm(t1, t0, 0x05040100u);
              v[1].w[i] = __builtin_amdgcn_perm(t1, t0, 0x07060302u);
            }
          }
        };
#pragma unroll
        for (int d = 0; d < NV / 2; ++d) {
          Frag v[2];
          by_element(d, v);
          acc[2 * d] = mma<IO>(v[0], w, acc[2 * d]);
          acc[2 * d + 1] = mma<IO>(v[1], w, acc[2 * d + 1]);
        }
      }
      if (!more) break;
      load_values(next);
      now = next;
      base += kStride;
      next = advance(base + kStride);
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if constexpr (kRelative) {
#pragma unroll
    for (int j = 0; j < NV; ++j) acc[j] *= unit;
  }

  // Join the waves: every wave brings its sums to the common maximum, then two
  // and two add up.
  if (g == 0) {
    states[wave][0][c] = m;
    states[wave][1][c] = l;
  }
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i) top = fmaxf(top, states[i][0][c]);
  const float shift = top == -INFINITY ? 0.0f : top;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < kFewWaves; ++i)
    l += states[i][1][c] * __builtin_amdgcn_exp2f(states[i][0][c] - shift);
  const float mine = __builtin_amdgcn_exp2f(m - shift);
#pragma unroll
  for (int j = 0; j < NV; ++j) acc[j] *= mine;
  // Element of the head that acc[j][i] is.
  auto element = [&](int j, int i) { return VT ? 16 * j + 4 * g + i : NV * (4 * g + i) + j; };
#pragma unroll
  for (int half = kFewWaves / 2; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[wave - half][c][element(j, i)] = acc[j][i];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] += sums[wave][c][element(j, i)];
    }
    __syncthreads();
  }
  if (wave == 0) {
    // Through LDS once more, so that rows leave as whole lines.
    const bool none = top == -INFINITY && l == 0.0f;
    const float norm = a.splits > 1 ? vs : none ? 0.0f : vs / l;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sums[0][c][element(j, i)] = a.splits == 1 && none ? 0.0f : acc[j][i] * norm;
    const int64_t line = t.begin + t.first + tok;
    if (row && g == 0) {
      if (a.splits > 1) {
        const int64_t at = part_index(a, t, t.first + tok, qh) * a.splits + z;
        a.part_ml[2 * at] = top;
        a.part_ml[2 * at + 1] = l;
      } else if (a.lse != nullptr) {
        a.lse[line * (a.heads * a.group) + qh] = none ? -INFINITY : (top + log2f(l)) * kLn2;
      }
    }
    wave_sync();
    const int rows = t.count * a.tile_heads;
    constexpr int kLanes = DP / 8;  // lanes of a row
#pragma unroll
    for (int r0 = 0; r0 < kRowTile; r0 += kWave / kLanes) {
      const int r = r0 + lane / kLanes, d = (lane % kLanes) * 8;
      const int rt = r / a.tile_heads, rh = r - rt * a.tile_heads;
      if (r >= rows || rh >= nheads || d >= D) continue;
      const int64_t out_row = t.begin + t.first + rt;
      const int head = kvh * a.group + head0 + rh;
      const float *x = &sums[0][r][d];
      if (a.splits > 1) {
        const int64_t at = part_index(a, t, t.first + rt, head) * a.splits + z;
        float *o = a.part_o + at * D + d;
        *reinterpret_cast<f32x4 *>(o) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4 *>(o + 4) = f32x4{x[4], x[5], x[6], x[7]};
      } else {
        char *to_row =
            a.out + out_row * a.o_tok + (int64_t)head * a.o_head + d * bytes_of_type<IO>();
        Raw<16> o;
        if constexpr (kF32) {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o.w[i] = f32_bits(x[4 * b + i]);
            st<16>(to_row + 16 * b, o);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) o.w[i] = pack_pair<IO>(f32x2{x[2 * i], x[2 * i + 1]});
          st<16>(to_row, o);
        }
      }
    }
  }
  if (infinities == 0) return;
  __syncthreads();
  add_infinities<IO, C, kFewStep, false>(args_address(args_at), tile, z, y);
}

template <int IO, int C, int DP, bool VT, bool INDEXED, bool GROUPED, bool STREAM>
__global__ void __launch_bounds__(kFewThreads, DP == 256 ? 1 : 2)
    attention_few_kernel(AttentionArgs a) {
  __shared__ FewShared<DP> shared;
  attention_few<IO, C, DP, VT, INDEXED, GROUPED, STREAM>(a, 0, blockIdx.x, shared);
}

// go(DP, VT, INDEXED, GROUPED) with the constants that a call needs.
template <int IO, int C, typename F>
void with_variant(const AttentionArgs &a, bool vt, bool grouped, const F &go) {
  const bool indexed = C != IO && (a.ks.s_block != 0 || a.vs.s_block != 0);
  auto by_dim = [&](auto vt_, auto indexed_, auto grouped_) {
    if (a.head_dim <= 64) go(std::integral_constant<int, 64>{}, vt_, indexed_, grouped_);
    else if (a.head_dim <= 128) go(std::integral_constant<int, 128>{}, vt_, indexed_, grouped_);
    else go(std::integral_constant<int, 256>{}, vt_, indexed_, grouped_);
  };
  auto by_scale = [&](auto vt_, auto grouped_) {
    if constexpr (C != IO) {
      if (indexed) return by_dim(vt_, std::true_type{}, grouped_);
    }
    by_dim(vt_, std::false_type{}, grouped_);
  };
  auto by_values = [&](auto grouped_) {
    if (vt) by_scale(std::true_type{}, grouped_);
    else by_scale(std::false_type{}, grouped_);
  };
  if (grouped) by_values(std::true_type{});
  else by_values(std::false_type{});
}

template <int IO, int C>
void launch_few(const AttentionPart &p, bool vt, bool grouped, hipStream_t s) {
  with_variant<IO, C>(p.a, vt, grouped, [&](auto dp, auto vt_, auto indexed_, auto grouped_) {
    constexpr int kDim = decltype(dp)::value;
    constexpr bool kVt = decltype(vt_)::value, kIndexed = decltype(indexed_)::value;
    constexpr bool kGrouped = decltype(grouped_)::value;
    if constexpr (IO == KVX_DTYPE_F32) {  // others: launch_many
      if (!p.stream)
        return attention_few_kernel<IO, C, kDim, kVt, kIndexed, kGrouped, false>
            <<<dim3(p.grid), kFewThreads, 0, s>>>(p.a);
    }
    attention_few_kernel<IO, C, kDim, kVt, kIndexed, kGrouped, true>
        <<<dim3(p.grid), kFewThreads, 0, s>>>(p.a);
  });
}

}  // namespace dev
}  // namespace kvx
