// Attention of many rows over a paged cache: tiles of 32 rows (up to 128
// dimensions), 64 (more dimensions) or 128 (dsr_attention.h has the work split
// and the kernel for few rows).
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

// Tokens that one round of the workgroup's 16-byte loads covers, where that is a whole number.
constexpr int attn_round(int DP) { return kAttnThreads / (DP / 8); }

// The four waves are WR along the rows and WK = 4 / WR along the tokens: wave
// (wr, wk) multiplies rows 32 wr .. of the tile by tokens 32 wk .. of each
// step's 32 WK.
//
// As in k_tree_attention the scores are computed transposed, S^T = K Q^T: a
// lane holds 16 tokens of one row (row lane % 32, tokens 8 (e / 4) +
// 4 (lane / 32) + e % 4), which are the second product's operand as they lie.
//
// One step of the loop multiplies tile t + 1's keys and tile t's values: the
// products of the one do not wait for the exponentials of the other, and a
// wave's vector instructions go on while the matrix cores work.  Keys and
// values pass from memory through registers into LDS.
//
// What bounds a step: the instructions a SIMD has to issue for its two waves
// (a 32 x 32 x 16 product takes 16 of the issue cycles and 32 of the matrix
// core's, an exponential 13, others 4), not the products themselves.  8 trees
// of 64 nodes over 32,001 tokens, 64 and 8 heads of 128: 681 to 705 us, 760 to
// 787 TFLOP/s; 32 ragged trees over up to 8,192 tokens 196 to 200.  64 rows
// a wave, with half the LDS reads a row, came out no faster (8 trees of 64
// nodes over 32,065 tokens: 710 us against 706 then) and wasted more on ragged
// rows.
//
// FLAT: a page holds every token of a round of loads, so that a round's page
// id and address are the same for the workgroup and a lane adds one offset.
template <class T, int DP, int WR>
constexpr int attn_wide_lds() {
  return 2 * kAttnTile * (kAttnWaves / WR) * (DP + 8 + DP + 16) * (int)sizeof(T);
}
template <class T, int DP, int WR, bool FLAT, bool BRANCH>
__device__ __forceinline__ void attn_wide_rows(char* attn_lds, int pass) {
  typedef typename AttnArgs<BRANCH>::type Call;
  typedef typename AttnType<T>::x4 x4;
  typedef typename AttnType<T>::x8 x8;
  typedef float f32x8 __attribute__((ext_vector_type(8)));
  constexpr int WK = kAttnWaves / WR;                 // waves along the tokens
  constexpr int NT = kAttnTile * WK;                  // tokens per step
  constexpr int KS = DP + 8, VS = DP + 16;            // LDS rows: 16-byte reads of 32 keys, and the transposing
                                                      // reads of 4 x 32 bytes, both spread over all banks
  constexpr int QS = DP / 16;                         // k steps of the score product
  constexpr int DB = DP / 32;                         // 32-wide output blocks
  constexpr int CH = DP / 8;                          // 16-byte chunks of a row
  constexpr int NL = NT * CH / kAttnThreads;          // chunks a thread stages per step, of keys and of values
  static_assert(NT * CH % kAttnThreads == 0, "every thread stages as much");
  static_assert(!FLAT || kAttnThreads % CH == 0, "a round is a whole number of tokens");
  constexpr int kKeys = 2 * NT * KS, kVals = 2 * NT * VS;  // elements, double-buffered
  T* keys = (T*)attn_lds;        // [2][NT][KS]
  T* vals = keys + kKeys;        // [2][NT][VS]
  __shared__ float sm[kAttnWaves][32], sl[kAttnWaves][32];
  __shared__ float sbase[32 * WR];
  __shared__ uint32_t sbits[4][WK];  // of a step's tokens, those whose page id is outside the cache
  __shared__ int sbad, spoison;      // a page id outside the cache; a value left out (attn_poison)

  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, n = l & 31, h = l >> 5;
  const int wr = w / WK, wk = w % WK;
  AttnWork<false, Call> work(attn_call<BRANCH>(pass), 0);
  AttnSegment u;
  AttnRequest q;
  while (work.next(attn_call<BRANCH>(pass), u, q)) {  // the same for the whole workgroup
    const dsr_tree_attention_args_t& a = attn_call<BRANCH>(pass).a;
    const AttnPlan& p = attn_call<BRANCH>(pass).p;
    const int group = p.group, dim = a.head_dim, row_shift = p.tile_shift;
    __syncthreads();  // the last segment's LDS is read
    if (threadIdx.x < 4 * WK) sbits[threadIdx.x / WK][threadIdx.x % WK] = 0;
    if (threadIdx.x == 0) sbad = spoison = 0;
    const int ctx = attn_context(attn_call<BRANCH>(pass), q), begin = u.begin, end = u.end;
    const int clear = min(ctx, end);  // every row sees the tokens before
    const int steps = end > begin ? (end - begin + NT - 1) / NT : 0;

    // This lane's row: token index, mask, query operand.  A negative scale
    // changes the queries' sign, so that scores only grow with their products;
    // scale 0 is queries of 0.
    const int in_tile = 32 * wr + n, row = (u.tile << row_shift) + in_tile;
    const bool live = row < q.rows;
    const int tok = live ? attn_token(p, row) : 0, head = u.head * group + (live ? row - tok * group : 0);
    const uint64_t mask = live && a.visible ? a.visible[q.lo + tok] : 0;
    const float scale = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
    x8 qv[QS];
    {
      const T* src = (const T*)a.q + (int64_t)(q.lo + tok) * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
      for (int s = 0; s < QS; ++s) {
        const int d = 16 * s + 8 * h;
        const x8 v = live && d < dim && a.scale != 0.f ? *(const x8*)(src + d) : x8{};
        qv[s] = a.scale < 0.f ? -v : v;
      }
    }

    attn_f32x16 acc[DB], sc[2];
    float m = -INFINITY, sum = 0.f, top;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = attn_f32x16{};
    const dsr_tree_attention_args_t& c = attn_call<BRANCH>(pass).a;
    const int32_t* pages = attn_pages(attn_call<BRANCH>(pass), u.r);
    const T* kb = (const T*)c.k_cache + u.head * c.k_head;
    const T* vb = (const T*)c.v_cache + u.head * c.v_head;
    const int shift = attn_call<BRANCH>(pass).p.page_shift, page = c.page;
    const unsigned blocks = c.blocks;
    const uint32_t k_block = c.k_block, k_token = c.k_token, v_block = c.v_block, v_token = c.v_token;
    const bool masks = c.visible != nullptr;
    bool any_bad = false;

    // Staging: thread x takes chunk (x + 256 i) % CH of token (x + 256 i) / CH
    // of a step's NT.  Steps past the last read the last one again and are
    // never used.  Places past the last token read that token, or, FLAT, what
    // lies behind it in the page: their scores are masked either way.
    x8 kr[NL], vr[NL];
    int kid[NL], vid[NL], nid[NL];  // page ids: of the keys and values in registers, of the next keys
    const uint32_t my_token = threadIdx.x / CH, my_dim = min(8 * (int)(threadIdx.x % CH), dim - 8);
    const uint32_t k_lane = (my_token * k_token + my_dim) * sizeof(T), v_lane = (my_token * v_token + my_dim) * sizeof(T);
    auto place_of = [&](int step, int i) __attribute__((always_inline)) {
      const int at = begin + step * NT;
      if constexpr (FLAT) return at + attn_round(DP) * i;  // the round's first
      return min(at + (int)(threadIdx.x + kAttnThreads * i) / CH, end - 1);
    };
    auto load_ids = [&](int* id, int step) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NL; ++i) id[i] = pages[min(place_of(step, i), end - 1) >> shift];
    };
    auto load = [&](x8* r, const int* id, int step, const T* base, uint32_t block, uint32_t token, uint32_t lane)
                    __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const uint32_t b = (unsigned)id[i] < blocks ? id[i] : 0, place = place_of(step, i) & (page - 1);
        const T* at = base + ((uint64_t)b * block + (uint64_t)place * token);
        if constexpr (FLAT)
          r[i] = *(const x8*)((const char*)at + lane);
        else
          r[i] = *(const x8*)(at + min(8 * ((int)(threadIdx.x + kAttnThreads * i) % CH), dim - 8));
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
      return FLAT ? bad : __ballot(bad) != 0;
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
    // 0: where they are not, 0 takes their place (attn_poison adds them in the
    // end, but for what lies behind the last token).
    auto check_vals = [&](x8* r, int step) __attribute__((always_inline)) {
      bool poison = false;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int x = ((int)threadIdx.x + kAttnThreads * i) / CH;
        poison |= attn_make_finite<T>(r[i]) && begin + step * NT + x < end;
      }
      if (poison) spoison = 1;
    };
    // Scores of a step's keys.
    auto scores = [&](attn_f32x16& s, int buf) __attribute__((always_inline)) {
      s = attn_f32x16{};
#pragma unroll
      for (int k = 0; k < QS; ++k)
        s = attn_mfma32(*(const x8*)&keys[(buf * NT + 32 * wk + n) * KS + 16 * k + 8 * h], qv[k], s);
    };
    // The largest of a lane's row among a step's scores.
    auto largest = [&](const attn_f32x16& s) __attribute__((always_inline)) {
      float x = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) x = fmaxf(x, s[e]);
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      const u32x2 y = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      top = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
    };
    // What rows may not see becomes -inf (rare); then the running maximum.
    auto settle = [&](attn_f32x16& s, int step, uint32_t bad) __attribute__((always_inline)) {
      const int p0 = begin + step * NT + 32 * wk;
      if (p0 + kAttnTile > clear || bad || (BRANCH && p0 < q.low)) {
        uint32_t see = attn_sees(masks, mask, tok, p0, ctx, end, bad);
        if constexpr (BRANCH) see &= ~attn_low_bits(q.low - p0);
        see >>= 4 * h;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = see >> (8 * (e >> 2) + (e & 3)) & 1 ? s[e] : -INFINITY;
        largest(s);
      }
      top = __builtin_fmaf(top, scale, -attn_lift<T, BRANCH>());
      if (__ballot(top > m + 8.f)) {
        const float next = fmaxf(m, top), f = m == next ? 1.f : __builtin_amdgcn_exp2f(m - next);
        m = next;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] *= f;
      }
    };
    // Weights of a settled step: the values' operand.
    auto weigh = [&](const attn_f32x16& s, x8* pv) __attribute__((always_inline)) {
      const float base = m == -INFINITY ? 0.f : -m;
      float part = 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        f32x8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * k + e], scale, base));
          part += x[e];
        }
        pv[k] = __builtin_convertvector(x, x8);
      }
      sum += part;
    };
    auto weighted = [&](const x8* pv, int buf) __attribute__((always_inline)) {
      const T* at = &vals[(buf * NT + 32 * wk + 4 * h + ((l & 15) >> 2)) * VS + 16 * (l >> 4 & 1) + 4 * (l & 3)];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const x4 lo = attn_read_tr<T>(at + 16 * k * VS + 32 * d), hi = attn_read_tr<T>(at + (16 * k + 8) * VS + 32 * d);
          acc[d] = attn_mfma32(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pv[k], acc[d]);
        }
    };

    if (steps > 0) {
      // Step t finds keys t + 1 and values t in LDS and keys t + 2 and values
      // t + 1 on their way to registers.  Page ids are read a step ahead of
      // their rows, and before that step's rows: waiting for them then leaves
      // the rows in flight.
      const int last = steps - 1;
      auto keys_of = [&](int step) __attribute__((always_inline)) {  // keys, and the ids of the next
        load_ids(nid, min(step + 1, last));
        load(kr, kid, min(step, last), kb, k_block, k_token, k_lane);
      };
      auto vals_of = [&](int step) __attribute__((always_inline)) {  // values: on the pages of those keys
#pragma unroll
        for (int i = 0; i < NL; ++i) vid[i] = kid[i];
        load(vr, vid, min(step, last), vb, v_block, v_token, v_lane);
      };
      auto next_ids = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NL; ++i) kid[i] = FLAT ? __builtin_amdgcn_readfirstlane(nid[i]) : nid[i];
      };
      load_ids(nid, 0);
      next_ids();
      keys_of(0);
      vals_of(0);
      __syncthreads();  // the flags
      if (outside(kid)) check_keys(kid, 0);
      if (begin + NT > clear || outside(vid) || (BRANCH && begin < q.low)) check_vals(vr, 0);
      store(keys, KS, 0, kr, true);
      store(vals, VS, 0, vr, false);
      next_ids();
      keys_of(1);
      vals_of(1);
      if (outside(kid)) check_keys(kid, 1);
      store(keys, KS, 1, kr, true);
      next_ids();
      keys_of(2);
      __syncthreads();
      scores(sc[0], 0);
      largest(sc[0]);
      settle(sc[0], 0, sbits[0][wk]);
      __syncthreads();  // keys 0 are read
      auto step = [&](auto C, int t) __attribute__((always_inline)) {
        constexpr int c = decltype(C)::value;  // t % 2
        if (begin + (t + 2) * NT > clear || outside(kid) || outside(vid)) {
          check_keys(kid, t + 2);
          check_vals(vr, t + 1);
        }
        // From here on no branch: the compiler places the products among the
        // vector instructions that do not wait for them.
        sbits[(t + 3) & 3][threadIdx.x & (WK - 1)] = 0;  // last read two steps ago
        const uint32_t bad = sbits[(t + 1) & 3][wk];
        x8 pv[2];
        weigh(sc[c], pv);
        scores(sc[c ^ 1], c ^ 1);
        weighted(pv, c);
        largest(sc[c ^ 1]);
        settle(sc[c ^ 1], t + 1, bad);
        // The rows in flight are waited for only now, behind the products.
        // (Stored before the products, with two steps of them in registers:
        // 706 us on 8 trees of 64 nodes over 32,065 tokens, so 682.)
        store(keys, KS, c, kr, true);
        store(vals, VS, c ^ 1, vr, false);
        vals_of(t + 2);
        next_ids();
        keys_of(t + 3);
        __syncthreads();
      };
      constexpr std::integral_constant<int, 0> even{};
      constexpr std::integral_constant<int, 1> odd{};
      // An odd count's last step lies past the end, where no row sees anything.
      for (int t = 0; t < steps; t += 2) {
        step(even, t);
        step(odd, t + 1);
      }
    }

    // The waves along the tokens join: all but the first hand theirs on through LDS.
    sum += __shfl_xor(sum, 32);
    if (any_bad) sbad = 1;
    if constexpr (WK > 1) {
      static_assert((WK - 1) * WR * 32 * DP * 4 <= (kKeys + kVals) * (int)sizeof(T), "outputs fit");
      float* outs = (float*)attn_lds + (int64_t)wr * (WK - 1) * 32 * DP;
      __syncthreads();
      if (wk > 0) {
        float* mine = outs + (wk - 1) * 32 * DP;
        if (h == 0) {
          sm[w][n] = m;
          sl[w][n] = sum;
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) mine[(d * 16 + e) * 64 + l] = acc[d][e];
      }
      __syncthreads();
      if (wk == 0) {
#pragma unroll
        for (int k = 1; k < WK; ++k) {
          const float* theirs = outs + (k - 1) * 32 * DP;
          const float m2 = sm[w + k][n], s2 = sl[w + k][n];
          const float both = fmaxf(m, m2);
          const float f = m == both ? 1.f : __builtin_amdgcn_exp2f(m - both);
          const float f2 = m2 == both ? 1.f : __builtin_amdgcn_exp2f(m2 - both);
          m = both;
          sum = sum * f + s2 * f2;
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[d][e] = acc[d][e] * f + theirs[(d * 16 + e) * 64 + l] * f2;
        }
      }
    }
    const Call& e = attn_call<BRANCH>(pass);
    if (wk == 0 && live) {
      if (h == 0) sbase[in_tile] = m;
      if (BRANCH || !u.whole) {
        int64_t at = ((int64_t)u.part << row_shift) + in_tile;
        float* o = &e.p.part_o[at * DP];
        float2* ml = &e.p.part_ml[at];
        if constexpr (BRANCH)
          if (u.whole) {
            at = (int64_t)(q.lo + tok) * e.a.q_heads + head;
            o = &e.b.row_o[at * DP];
            ml = &e.b.row_ml[at];
          }
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          // The join reads no more (trees of 96 dimensions, in a kernel of 128: 83 us with all columns, 79 so).
          if (BRANCH && 32 * d >= dim) break;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *(attn_f32x4*)&o[32 * d + 8 * i + 4 * h] =
                attn_f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
        }
        if (h == 0) *ml = float2{m, sum};
      } else {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T* o = (T*)e.a.out + (int64_t)(q.lo + tok) * e.a.out_token + (int64_t)head * e.a.out_head;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = 32 * d + 8 * i + 4 * h;
            x4 y;
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = (T)(acc[d][4 * i + k] * inv);
            if (at < dim) *(x4*)(o + at) = y;
          }
        if (e.a.lse && h == 0)
          e.a.lse[(int64_t)(q.lo + tok) * e.a.q_heads + head] = sum == 0.f ? -INFINITY : (m + log2f(sum)) * kLn2;
      }
    }
    __threadfence_block();
    __syncthreads();
    if (__builtin_expect(spoison, 0))
      attn_poison<T, DP>(e, u, q, sbad || (BRANCH && begin < q.low) ? begin : max(begin, clear - NT), sbase);
    attn_report(e, u, q, sbad);
  }
}

template <class T, int DP, int WR, bool FLAT>
__global__ __launch_bounds__(kAttnThreads, DP * (4 / WR) < 512 ? 2 : 1) void k_tree_attention_wide(AttnCall) {
  __shared__ __align__(16) char lds[attn_wide_lds<T, DP, WR>()];
  if ((int)blockIdx.x >= attn_call().p.groups) return attn_clear<T>(attn_call().p.groups, kAttnThreads);
  attn_wide_rows<T, DP, WR, FLAT, false>(lds, 0);
}

}  // namespace dsr
