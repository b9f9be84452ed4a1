// Attention of many rows over a paged cache: tiles of 32 to 256 rows
// (dsr_attention.h has the work split and the kernel for few rows).
#pragma once

#include <type_traits>

#include "dsr_attention.h"

namespace dsr {

typedef float attn_f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ attn_f32x16 attn_mfma32(AttnType<__bf16>::x8 a, AttnType<__bf16>::x8 b, attn_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ attn_f32x16 attn_mfma32(AttnType<_Float16>::x8 a, AttnType<_Float16>::x8 b,
                                                   attn_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <int DP, int WR>
struct AttnWideShared {
  static constexpr int WK = kAttnWaves / WR;   // waves along the tokens
  static constexpr int NT = kAttnTile * WK;    // tokens per step
  static constexpr int KS = DP + 8, VS = DP + 16;  // LDS rows: 16-byte reads of 32 keys, and the transposing
                                                   // reads of 4 x 32 bytes, both spread over all banks
  static constexpr int kKeys = 2 * NT * KS, kVals = 2 * NT * VS;  // elements, double-buffered
};

// The four waves are WR along the rows and WK = 4 / WR along the tokens: wave
// (wr, wk) multiplies rows 32 RB wr .. of the tile by tokens 32 wk .. of each
// step's 32 WK.  RB 32-row blocks per wave set how often a key or value read
// from LDS is used: at one block the LDS reads (128 bytes a cycle) take as
// long as the products, at two half as long.
//
// As in k_tree_attention the scores are computed transposed, S^T = K Q^T: a
// lane holds 16 tokens of one row (row lane % 32, tokens 8 (e / 4) +
// 4 (lane / 32) + e % 4), which are the second product's operand as they lie.
//
// One step of the loop multiplies tile t + 1's keys and tile t's values: the
// products of the one do not wait for the exponentials of the other, so the
// matrix cores and the vector units work side by side in one wave.  Keys and
// values pass from memory through registers (two steps in flight) into LDS.
template <class T, int DP, int RB, int WR>
__global__ __launch_bounds__(kAttnThreads, RB == 1 && DP <= 128 ? 2 : 1) void k_tree_attention_wide(
    AttnCall) {
  typedef typename AttnType<T>::x4 x4;
  typedef typename AttnType<T>::x8 x8;
  typedef AttnWideShared<DP, WR> Sh;
  typedef float f32x8 __attribute__((ext_vector_type(8)));
  constexpr int WK = Sh::WK, NT = Sh::NT, KS = Sh::KS, VS = Sh::VS;
  constexpr int QS = DP / 16;                         // k steps of the score product
  constexpr int DB = DP / 32;                         // 32-wide output blocks
  constexpr int CH = DP / 8;                          // 16-byte chunks of a row
  constexpr int NL = NT * CH / kAttnThreads;          // chunks a thread stages per step, of keys and of values
  static_assert(NT * CH % kAttnThreads == 0, "every thread stages as much");
  constexpr int SETS = NL <= 2 && RB == 1 ? 2 : 1;               // steps in flight in registers: 16 KB or more per workgroup
  __shared__ __align__(16) char attn_lds[(Sh::kKeys + Sh::kVals) * sizeof(T)];
  T* keys = (T*)attn_lds;             // [2][NT][KS]
  T* vals = keys + Sh::kKeys;         // [2][NT][VS]
  __shared__ float sm[kAttnWaves][32 * RB], sl[kAttnWaves][32 * RB];
  __shared__ float sbase[32 * RB * WR];
  __shared__ uint32_t sbits[4][WK];  // of a step's tokens, those whose page id is outside the cache
  __shared__ int sbad, spoison;  // a page id outside the cache; a value left out (attn_poison)

  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, n = l & 31, h = l >> 5;
  const int wr = w / WK, wk = w % WK;
  AttnWork<false> work(attn_call().a, attn_call().p, 0);
  AttnSegment u;
  AttnRequest q;
  while (work.next(attn_call().a, attn_call().p, u, q)) {  // the same for the whole workgroup
  const dsr_tree_attention_args_t& a = attn_call().a;
  const AttnPlan& p = attn_call().p;
  const int group = p.group, dim = a.head_dim, row_shift = p.tile_shift;
  __syncthreads();  // the last segment's LDS is read
  if (threadIdx.x < 4 * WK) sbits[threadIdx.x / WK][threadIdx.x % WK] = 0;
  if (threadIdx.x == 0) sbad = spoison = 0;
  const int ctx = q.kv - q.n, begin = u.begin, end = u.end;
  const int clear = min(ctx, end);  // every row sees the tokens before
  const int steps = end > begin ? (end - begin + NT - 1) / NT : 0;
  const int row0 = (u.tile << row_shift) + 32 * RB * wr;

  // A negative scale changes the queries' sign, so that scores only grow
  // with their products; scale 0 is queries of 0.
  const float scale = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  x8 qv[RB][QS];
  int tok[RB];
  uint64_t mask[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int row = row0 + 32 * b + n;
    const bool in = row < q.rows;
    const int t = in ? attn_token(p, row) : 0, hh = in ? row - t * group : 0;
    tok[b] = t;
    mask[b] = in && a.visible ? a.visible[q.lo + t] : 0;
    const T* src = (const T*)a.q + (int64_t)(q.lo + t) * a.q_token + (int64_t)(u.head * group + hh) * a.q_head;
#pragma unroll
    for (int s = 0; s < QS; ++s) {
      const int d = 16 * s + 8 * h;
      x8 v = in && d < dim && a.scale != 0.f ? *(const x8*)(src + d) : x8{};
      qv[b][s] = a.scale < 0.f ? -v : v;
    }
  }

  constexpr int SB = RB == 1 ? 2 : 1;  // scores of two steps, or of one where registers are short
  attn_f32x16 acc[RB][DB], sc[SB][RB];
  float m[RB], sum[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    m[b] = -INFINITY;
    sum[b] = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[b][d] = attn_f32x16{};
  }
  const dsr_tree_attention_args_t& c = attn_call().a;
  const int32_t* pages = c.table + u.r * c.table_ld;
  const T* kb = (const T*)c.k_cache + u.head * c.k_head;
  const T* vb = (const T*)c.v_cache + u.head * c.v_head;
  const int shift = attn_call().p.page_shift, page = c.page;
  const unsigned blocks = c.blocks;
  const uint32_t k_block = c.k_block, k_token = c.k_token, v_block = c.v_block, v_token = c.v_token;
  const bool masks = c.visible != nullptr;
  bool any_bad = false;

  // Staging: chunk c of token t of a step's NT; the step's places past the
  // last token read the last token (their scores are masked).  Steps past
  // the last read the last step again and are never used.
  x8 kr[SETS][NL], vr[SETS][NL];
  int kid[SETS][NL], vid[SETS][NL], nid[SETS][NL];  // page ids: of the keys and values in registers, of the next keys
  auto place_of = [&](int step, int i) __attribute__((always_inline)) {
    const int t = (int)(threadIdx.x + kAttnThreads * i) / CH;
    return min(begin + step * NT + t, end - 1);
  };
  auto load_ids = [&](int* id, int step) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NL; ++i) id[i] = pages[place_of(step, i) >> shift];
  };
  auto load = [&](x8* r, const int* id, int step, const T* base, uint32_t block, uint32_t token)
                  __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int c = (int)(threadIdx.x + kAttnThreads * i) % CH;
      const uint32_t b = (unsigned)id[i] < blocks ? id[i] : 0, place = place_of(step, i) & (page - 1);
      r[i] = *(const x8*)(base + min(8 * c, dim - 8) + ((uint64_t)b * block + (uint64_t)place * token));
    }
  };
  auto store = [&](T* rows, int stride, int buf, const x8* r, bool pad) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int x = (int)threadIdx.x + kAttnThreads * i, c = x % CH;
      *(x8*)&rows[(buf * NT + x / CH) * stride + 8 * c] = !pad || 8 * c < dim ? r[i] : x8{};
    }
  };
  auto outside = [&](const int* id) __attribute__((always_inline)) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < NL; ++i) bad |= (unsigned)id[i] >= blocks;
    return bad;
  };
  // Keys on pages outside the cache are noted, a bit each (rare).
  auto check_keys = [&](const int* id, int step) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if ((unsigned)id[i] >= blocks) {
        const int x = ((int)threadIdx.x + kAttnThreads * i) / CH;
        atomicOr(&sbits[step & 3][x / 32], 1u << (x % 32));
        any_bad = true;
      }
  };
  // Values that some row may not see have to be finite to be multiplied by
  // 0: where they are not, 0 takes their place (attn_poison adds them in the end).
  auto check_vals = [&](x8* r) __attribute__((always_inline)) {
    bool poison = false;
#pragma unroll
    for (int i = 0; i < NL; ++i) poison |= attn_make_finite<T>(r[i]);
    if (poison) spoison = 1;
  };
  // Scores of a step's keys.
  auto scores = [&](attn_f32x16* s, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < RB; ++b) s[b] = attn_f32x16{};
#pragma unroll
    for (int k = 0; k < QS; ++k) {
      const x8 key = *(const x8*)&keys[(buf * NT + 32 * wk + n) * KS + 16 * k + 8 * h];
#pragma unroll
      for (int b = 0; b < RB; ++b) s[b] = attn_mfma32(key, qv[b][k], s[b]);
    }
  };
  // The largest of a lane's row among a step's scores.
  auto largest = [&](attn_f32x16* s, float* top) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      float x = s[b][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) x = fmaxf(x, s[b][e]);
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      const u32x2 y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      top[b] = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
    }
  };
  // What rows may not see becomes -inf (rare); then the running maximum.
  auto settle = [&](attn_f32x16* s, float* top, int step, uint32_t bad) __attribute__((always_inline)) {
    const int p0 = begin + step * NT + 32 * wk;
    if (p0 + kAttnTile > clear || bad) {
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const uint32_t see = attn_sees(masks, mask[b], tok[b], p0, ctx, end, bad) >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[b][e] = see >> (8 * (e >> 2) + (e & 3)) & 1 ? s[b][e] : -INFINITY;
      }
      largest(s, top);
    }
    bool raise = false;
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      top[b] = __builtin_fmaf(top[b], scale, -AttnType<T>::kLift);
      raise |= top[b] > m[b] + 8.f;
    }
    if (__ballot(raise)) {
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const float next = fmaxf(m[b], top[b]), f = m[b] == next ? 1.f : __builtin_amdgcn_exp2f(m[b] - next);
        m[b] = next;
        sum[b] *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[b][d] *= f;
      }
    }
  };
  // Weights of a settled step: the values' operand.
  auto weigh = [&](attn_f32x16* s, x8 (*pv)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const float base = m[b] == -INFINITY ? 0.f : -m[b];
      float part = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f32x8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * k + e], scale, base));
          part += x[e];
        }
        pv[b][k] = __builtin_convertvector(x, x8);
      }
      sum[b] += part;
    }
  };
  auto weighted = [&](x8 (*pv)[2], int buf) __attribute__((always_inline)) {
    const T* rows = &vals[(buf * NT + 32 * wk) * VS];
    const T* at = rows + (4 * (l >> 5) + ((l & 15) >> 2)) * VS + 16 * (l >> 4 & 1) + 4 * (l & 3);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const x4 lo = attn_read_tr<T>(at + 16 * k * VS + 32 * d), hi = attn_read_tr<T>(at + (16 * k + 8) * VS + 32 * d);
        const x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b][d] = attn_mfma32(v, pv[b][k], acc[b][d]);
      }
  };

  if (steps > 0) {
    // Step t finds keys t + 1 and values t in LDS and keys t + 2 .. t + 1 +
    // SETS and values t + 1 .. t + SETS on their way to registers.
    const int last = steps - 1;
    auto keys_of = [&](auto S, int step) __attribute__((always_inline)) {  // registers of keys `step`, ids ahead
      constexpr int c = decltype(S)::value % SETS;
      load(kr[c], kid[c], min(step, last), kb, k_block, k_token);
      load_ids(nid[c], min(step + SETS, last));
    };
    auto vals_of = [&](auto S, int step) __attribute__((always_inline)) {  // values: on the pages of those keys
      constexpr int c = decltype(S)::value % SETS;
#pragma unroll
      for (int i = 0; i < NL; ++i) vid[c][i] = kid[c][i];
      load(vr[c], vid[c], min(step, last), vb, v_block, v_token);
    };
    auto next_ids = [&](auto S) __attribute__((always_inline)) {
      constexpr int c = decltype(S)::value % SETS;
#pragma unroll
      for (int i = 0; i < NL; ++i) kid[c][i] = nid[c][i];
    };
    constexpr std::integral_constant<int, 0> even{};
    constexpr std::integral_constant<int, 1> odd{};
    load_ids(kid[0], 0);
    if constexpr (SETS == 2) load_ids(kid[1], min(1, last));
    keys_of(even, 0);
    vals_of(even, 0);
    if constexpr (SETS == 2) {
      keys_of(odd, 1);
      vals_of(odd, 1);
    }
    __syncthreads();  // the flags
    if (__ballot(outside(kid[0]))) check_keys(kid[0], 0);
    if (begin + NT > clear || __ballot(outside(vid[0]))) check_vals(vr[0]);
    store(keys, KS, 0, kr[0], true);
    store(vals, VS, 0, vr[0], false);
    next_ids(even);
    if constexpr (SETS == 2) {
      keys_of(even, 2);
      vals_of(even, 2);
      if (__ballot(outside(kid[1]))) check_keys(kid[1], 1);
      store(keys, KS, 1, kr[1], true);
      next_ids(odd);
      keys_of(odd, 3);
    } else {
      keys_of(even, 1);
      vals_of(even, 1);
      if (__ballot(outside(kid[0]))) check_keys(kid[0], 1);
      store(keys, KS, 1, kr[0], true);
      next_ids(even);
      keys_of(even, 2);
    }
    __syncthreads();
    float top[RB];
    scores(sc[0], 0);
    largest(sc[0], top);
    settle(sc[0], top, 0, sbits[0][wk]);
    __syncthreads();  // keys 0 are read
    auto step = [&](auto S, int t) __attribute__((always_inline)) {
      constexpr int c = decltype(S)::value;  // t % 2
      constexpr std::integral_constant<int, c> now{};
      constexpr std::integral_constant<int, c ^ 1> next{};
      constexpr int kc = c % SETS, vc = (c ^ 1) % SETS;
      const bool odd = outside(kid[kc]) || outside(vid[vc]);
      if (begin + (t + 2) * NT > clear || __ballot(odd)) {
        check_keys(kid[kc], t + 2);
        check_vals(vr[vc]);
      }
      // From here on no branch: the compiler places the products among the
      // vector instructions that do not wait for them.
      sbits[(t + 3) & 3][threadIdx.x & (WK - 1)] = 0;  // last read two steps ago
      store(keys, KS, c, kr[kc], true);
      store(vals, VS, c ^ 1, vr[vc], false);
      vals_of(next, t + 1 + SETS);
      next_ids(now);
      keys_of(now, t + 2 + SETS);
      const uint32_t bad = sbits[(t + 1) & 3][wk];
      x8 pv[RB][2];
      constexpr int s0 = c % SB, s1 = (c ^ 1) % SB;
      weigh(sc[s0], pv);
      scores(sc[s1], c ^ 1);
      weighted(pv, c);
      largest(sc[s1], top);
      settle(sc[s1], top, t + 1, bad);
      __syncthreads();
    };
    // An odd count's last step lies past the end, where no row sees anything.
    for (int t = 0; t < steps; t += 2) {
      step(even, t);
      step(odd, t + 1);
    }
  }

  // The waves along the tokens join: all but the first hand theirs on through LDS.
#pragma unroll
  for (int b = 0; b < RB; ++b) sum[b] += __shfl_xor(sum[b], 32);
  if (any_bad) sbad = 1;
  if constexpr (WK > 1) {
    static_assert((WK - 1) * WR * RB * 32 * DP * 4 <= (Sh::kKeys + Sh::kVals) * (int)sizeof(T), "outputs fit");
    float* outs = (float*)attn_lds;
    __syncthreads();
    if (wk > 0) {
      float* mine = outs + (int64_t)(wr * (WK - 1) + wk - 1) * RB * 32 * DP;
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        if (h == 0) {
          sm[w][32 * b + n] = m[b];
          sl[w][32 * b + n] = sum[b];
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) mine[((b * DB + d) * 16 + e) * 64 + l] = acc[b][d][e];
      }
    }
    __syncthreads();
    if (wk == 0) {
#pragma unroll
      for (int k = 1; k < WK; ++k) {
        const float* theirs = outs + (int64_t)(wr * (WK - 1) + k - 1) * RB * 32 * DP;
#pragma unroll
        for (int b = 0; b < RB; ++b) {
          const float m2 = sm[w + k][32 * b + n], s2 = sl[w + k][32 * b + n];
          const float top = fmaxf(m[b], m2);
          const float f = m[b] == top ? 1.f : __builtin_amdgcn_exp2f(m[b] - top);
          const float f2 = m2 == top ? 1.f : __builtin_amdgcn_exp2f(m2 - top);
          m[b] = top;
          sum[b] = sum[b] * f + s2 * f2;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e)
              acc[b][d][e] = acc[b][d][e] * f + theirs[((b * DB + d) * 16 + e) * 64 + l] * f2;
        }
      }
    }
  }
  const AttnCall& e = attn_call();
  const bool split = !u.whole;
  const int64_t part = u.part;
  if (wk == 0) {
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int in_tile = 32 * RB * wr + 32 * b + n, row = row0 + 32 * b + n;
      if (row >= q.rows) continue;
      if (h == 0) sbase[in_tile] = m[b];
      if (split) {
        float* o = &e.p.part_o[(((int64_t)part << row_shift) + in_tile) * DP];
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *(attn_f32x4*)&o[32 * d + 8 * e + 4 * h] =
                attn_f32x4{acc[b][d][4 * e], acc[b][d][4 * e + 1], acc[b][d][4 * e + 2], acc[b][d][4 * e + 3]};
        if (h == 0) e.p.part_ml[((int64_t)part << row_shift) + in_tile] = float2{m[b], sum[b]};
      } else {
        const int t = attn_token(e.p, row), hh = row - t * group;
        const float inv = sum[b] == 0.f ? 0.f : 1.f / sum[b];
        T* o = (T*)e.a.out + (int64_t)(q.lo + t) * e.a.out_token + (int64_t)(u.head * group + hh) * e.a.out_head;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = 32 * d + 8 * e + 4 * h;
            x4 y;
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = (T)(acc[b][d][4 * e + i] * inv);
            if (at < dim) *(x4*)(o + at) = y;
          }
        if (e.a.lse && h == 0)
          e.a.lse[(int64_t)(q.lo + t) * e.a.q_heads + u.head * group + hh] =
              sum[b] == 0.f ? -INFINITY : (m[b] + log2f(sum[b])) * kLn2;
      }
    }
  }
  __threadfence_block();
  __syncthreads();
  if (spoison) attn_poison<T, DP>(e.a, e.p, u, q, sbad ? begin : max(begin, clear - NT), sbase);
  attn_report(e.a, e.p, u, q, sbad);
  }
}

}  // namespace dsr
