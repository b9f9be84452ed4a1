// Attention of requests that share a prefix (dsr_prefix_attention).
//
// softmax over a prefix and over what lies behind it join as parts of any
// other cut do: with base m, sum l = sum_j 2^(s_j - m) and o = sum_j
// 2^(s_j - m) v_j of each, M the largest m,
//   out = sum 2^(m - M) o / sum 2^(m - M) l.
// So the kernels of dsr_tree_attention go over the rows twice, over the
// prefixes with all of a group's rows in tiles of up to 128, and over each
// request's own tokens, and k_prefix_join joins what both leave for a row.
//
// What it saves: 64 requests of a token over a prefix of 32,768 read 134 MB of
// keys and values in place of 8.6 GB, and have 16 times the rows a tile.
#pragma once

#include "dsr_attention.h"
#include "dsr_attention_wide.h"
#include "dsr_branch.h"

namespace dsr {

// The kernels' argument: the groups' pass and the requests'.
struct PrefixCall {
  AttnBranchCall c[2];
};

// Both passes in one launch.  Tiles of the groups' pass have A rows, of the
// requests' B.  Prefixes are bound by the matrix cores, the tokens of single
// requests by memory, so one half of the workgroups (64 in turn) begins with the
// prefixes and the other with the requests.  64 requests over one prefix of
// 32,768 tokens, up to 1,024 of their own: 158 us so, 164 with the prefixes first
// everywhere, 168 with the requests, 160 where every other one does, 169 where 256
// in turn do (in two launches 190, 163 then in one); 8 prefixes of 8 requests 92,
// and 94 in each of the other orders.
//
// What bounds it: long prefixes by the issue of the products' instructions (650 to
// 700 TFLOP/s of 128-row tiles), few and short tokens by a share's beginning and
// end, which are each a chain of reads.
template <int ROWS, class T, int DP, bool FLAT>
__device__ __forceinline__ void prefix_pass(char* lds, int pass) {
  if constexpr (ROWS == 16)
    attn_few<T, DP, kAttnWaves, true>(lds, pass);
  else
    attn_wide_rows<T, DP, ROWS / 32, FLAT, true>(lds, pass);
}
template <int ROWS, class T, int DP>
constexpr int prefix_lds() {
  if constexpr (ROWS == 16)
    return attn_few_lds<T, DP, kAttnWaves>();
  else
    return attn_wide_lds<T, DP, ROWS / 32>();
}
template <int ROWS, int DP>
constexpr bool prefix_two() {  // registers for two workgroups a CU (above 128 dimensions one is launched)
  return ROWS == 16 ? DP <= 128 : DP * (128 / ROWS) < 512;
}
template <class T, int DP, int A, int B, bool FLAT>
__global__ __launch_bounds__(kAttnThreads, (prefix_two<A, DP>() && prefix_two<B, DP>() ? 2 : 1)) void
k_prefix_attention(PrefixCall) {
  constexpr int kA = prefix_lds<A, T, DP>(), kB = prefix_lds<B, T, DP>(), kLds = kA > kB ? kA : kB;
  static_assert(kLds >= (kAttnLows + 1) * 4, "the groups fit");
  __shared__ __align__(16) char lds[kLds];
  const int shares = attn_call<true>(0).p.groups;
  const bool few = attn_call<true>(0).a.requests <= kAttnLows;
  if ((int)blockIdx.x >= shares) {
    const AttnBranchCall& c = attn_call<true>(0);
    const bool none = few ? attn_branch_wrong(c, kAttnThreads, nullptr) : c.b.low[0] == kAttnNone;
    return attn_clear<T, true>(shares, kAttnThreads, none);
  }
  if (few)
    attn_branch_lows(attn_call<true>(0), attn_call<true>(1), kAttnThreads, (int*)lds);
  const int first = blockIdx.x >> 6 & 1;
  if constexpr (A == B) {
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      __syncthreads();
      prefix_pass<A, T, DP, FLAT>(lds, first ^ i);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      __syncthreads();
      if ((first ^ i) == 0)
        prefix_pass<A, T, DP, FLAT>(lds, 0);
      else
        prefix_pass<B, T, DP, FLAT>(lds, 1);
    }
  }
}

// More requests than every workgroup looks over for itself, a thread each: their
// groups, then who leads these.
__global__ __launch_bounds__(kAttnThreads) void k_prefix_lows(PrefixCall) {
  attn_branch_lows(attn_call<true>(0), attn_call<true>(1), kAttnThreads, nullptr);
}
__global__ __launch_bounds__(kAttnThreads) void k_prefix_leads(PrefixCall) {
  const AttnBranchCall& c = attn_call<true>(0);
  const int r = (int)blockIdx.x * kAttnThreads + (int)threadIdx.x;
  attn_lead_of(c.b.lead, r < c.a.requests ? c.b.group_of[r] : -1, r);
}

struct PrefixJoin {
  dsr_tree_attention_args_t a;
  AttnPlan p[2];    // of the groups' pass and of the requests'
  AttnBranch b[2];
};

// The request of token t: how many end at or before it (a whole wave, 64 a round).
__device__ __forceinline__ int prefix_owner(const dsr_tree_attention_args_t& a, int t) {
  const int l = threadIdx.x & 63;
  int lo = 0, n = (int)a.requests;
  while (n > 0) {
    const int stride = (n + 63) / 64, end = lo + n, at = lo + l * stride + stride - 1;
    lo += __popcll(__ballot(at < end && a.offsets[at < end ? at + 1 : 0] <= t)) * stride;
    n = end - lo < stride - 1 ? end - lo : stride - 1;
  }
  return lo;
}

// Where the shares of the tile of row `row` (of a request's, or group's, rows
// of key head `head`; its first token is `lo`) are told: the first and their number.
__device__ __forceinline__ int2 prefix_tile(const PrefixJoin& j, int pass, int lo, int head, int row) {
  return j.b[pass].tiles[((int64_t)head * j.a.tokens + lo) * j.p[0].group + (row & -j.p[pass].tile_rows)];
}

// An item is a token and `each` blocks of JR of its rows (heads), a block at a
// time.  The threads left over take every SLOTS-th part each, summed in a fixed
// order (none are where a block has 192 or more dimensions, whose threads are no
// power of two); a thread has FLIGHT parts in flight.  A refused request's rows are one
// part without weight.
// What bounds it: a chain of reads (the token's request, its tiles' shares, the
// parts; 4 tokens of 32 heads 6.2 us), then the parts' way through the caches of
// other XCDs (64 tokens of 64 heads and 17 parts a row 12 us, 2,900 of 32 and few
// parts 38).
template <class T, int DP, int JR, int FLIGHT>
__global__ __launch_bounds__(kAttnThreads) void k_prefix_join(PrefixJoin j, int each) {
  typedef typename AttnType<T>::x4 x4;
  constexpr int E = JR * DP / 4;  // four dimensions of a row each
  constexpr int SLOTS = E < kAttnThreads ? kAttnThreads / E : 1;
  __shared__ float sm[SLOTS][JR], sl[SLOTS][JR];
  __shared__ attn_f32x4 so[SLOTS][SLOTS > 1 ? E : 1];
  const dsr_tree_attention_args_t& a = j.a;
  const int heads = a.q_heads, group = j.p[0].group;
  static_assert(SLOTS == 1 || SLOTS * E == kAttnThreads, "every thread has a slot");
  const int slot = SLOTS > 1 ? threadIdx.x / E : 0;
  const int chunk = blockIdx.y;
  const bool none = j.b[1].low[0] == kAttnNone;  // rows and statuses are written
  for (int64_t item = blockIdx.x; item < a.tokens; item += gridDim.x) {
    const int t = (int)item;
    const int r = prefix_owner(a, t);
    if (r >= a.requests || none) continue;
    const int g = j.b[1].group_of[r], g_lo = j.b[1].group_lo[r];
    const int lo = max(a.offsets[r], 0);
    if (t < lo) continue;  // a row of no request
    const int h_end = min(heads, (chunk + 1) * JR * each);
    for (int h0 = chunk * JR * each; h0 < h_end; h0 += JR) {
#pragma unroll
      for (int x = SLOTS > 1 ? threadIdx.x % E : threadIdx.x; x < E; x += kAttnThreads) {
        const int in = x / (DP / 4), h = h0 + in, d = x % (DP / 4) * 4;
        const bool live = h < heads && d < a.head_dim;
        const int64_t row = (int64_t)t * heads + h;
        float M = -INFINITY, L = 0.f;
        attn_f32x4 o = {};
        auto add = [&](float m, float l, attn_f32x4 x) {
          const float both = fmaxf(M, m), f = M == both ? 1.f : __builtin_amdgcn_exp2f(M - both);
          const float g = m == both ? 1.f : __builtin_amdgcn_exp2f(m - both);
          M = both;
          L = L * f + l * g;
          o = o * f + x * g;
        };
        if (live) {
          const int kv_head = attn_token(j.p[0], h), of_group = h - kv_head * group;
          const int row0 = (t - g_lo) * group + of_group, row1 = (t - lo) * group + of_group;
          const int2 s0 = g >= 0 ? prefix_tile(j, 0, g_lo, kv_head, row0) : int2{0, 0};
          const int2 s1 = prefix_tile(j, 1, lo, kv_head, row1);
          const int in0 = row0 & (j.p[0].tile_rows - 1), in1 = row1 & (j.p[1].tile_rows - 1);
          const int count = s0.y + s1.y;
          for (int i0 = slot; i0 < count; i0 += FLIGHT * SLOTS) {
            float2 ml[FLIGHT];
            attn_f32x4 v[FLIGHT];
#pragma unroll
            for (int k = 0; k < FLIGHT; ++k) {
              const int i = min(i0 + k * SLOTS, count - 1);
              const bool second = i >= s0.y;
              const int c = second ? i - s0.y : i, first = second ? s1.x : s0.x;
              const bool whole = (second ? s1.y : s0.y) == 1;
              // The first part is its workgroup's last (an odd place), the others their workgroups' first.
              const int place = 2 * (first + c) + (c == 0);
              const int64_t part = second ? ((int64_t)place << j.p[1].tile_shift) + in1
                                          : ((int64_t)place << j.p[0].tile_shift) + in0;
              const int64_t at = whole ? row : part;
              const float2* m_at = second ? (whole ? j.b[1].row_ml : j.p[1].part_ml)
                                          : (whole ? j.b[0].row_ml : j.p[0].part_ml);
              const float* o_at = second ? (whole ? j.b[1].row_o : j.p[1].part_o)
                                         : (whole ? j.b[0].row_o : j.p[0].part_o);
              ml[k] = m_at[at];
              v[k] = *(const attn_f32x4*)&o_at[at * DP + d];
            }
#pragma unroll
            for (int k = 0; k < FLIGHT; ++k)
              if (i0 + k * SLOTS < count) add(ml[k].x, ml[k].y, v[k]);
          }
        }
        if constexpr (SLOTS > 1) {
          so[slot][x] = o;
          if (d == 0) {
            sm[slot][in] = M;
            sl[slot][in] = L;
          }
          __syncthreads();
          if (slot == 0) {
#pragma unroll
            for (int i = 1; i < SLOTS; ++i) add(sm[i][in], sl[i][in], so[i][x]);
          }
          __syncthreads();  // the next block's
        }
        if (slot > 0 || !live) continue;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (T)(o[i] * inv);
        *(x4*)((T*)a.out + (int64_t)t * a.out_token + (int64_t)h * a.out_head + d) = y;
        if (a.lse && d == 0) a.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
      }
    }
    if (t == lo && chunk == 0 && threadIdx.x == 0) {
      // A request's (a group's) last tile of its first head speaks for its page ids.
      const AttnRequest own = attn_own(a, j.p[1], r, j.b[1].low[r]);
      int bad = 0;
      if (own.fine)
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
          if (pass == 0 && g < 0) continue;
          const int q_lo = pass == 0 ? g_lo : own.lo;
          const int end = pass == 0 ? min(a.offsets[j.b[0].groups[g + 1]], (int)a.tokens) : own.lo + own.n;
          const int2 s = prefix_tile(j, pass, q_lo, 0, (end - q_lo) * group - 1);
          if (s.y == 1) bad |= j.b[pass].bad[pass == 0 ? g : r];
          for (int c = 0; s.y > 1 && c < s.y; ++c) bad |= j.p[pass].part_bad[2 * (s.x + c) + (c == 0)];
        }
      a.status[r] = !own.fine ? DSR_E_LENGTH : bad ? DSR_E_BLOCK : DSR_OK;
    }
  }
}

}  // namespace dsr
