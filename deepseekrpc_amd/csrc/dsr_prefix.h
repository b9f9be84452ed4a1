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

// The shares that hold a tile of head `head` of request (or group) r.
__device__ __forceinline__ void prefix_shares(const AttnPlan& p, const AttnBranch& b, const AttnRequest& q, int r,
                                              int head, int tile, int& first, int& last) {
  const uint32_t quota = attn_quota(p, b.begin[b.count]);
  const uint32_t steps = AttnWork<false, AttnBranchCall>::steps_of(p, q);
  const uint32_t from = b.begin[r] + (head * (uint32_t)q.tiles + tile) * steps;
  first = from / quota;
  last = (from + steps - 1) / quota;
}

// JR rows (heads of a token) at a time; the threads left over take every
// SLOTS-th part each, summed in a fixed order.
template <class T, int DP, int JR>
__global__ __launch_bounds__(kAttnThreads) void k_prefix_join(PrefixJoin j) {
  typedef typename AttnType<T>::x4 x4;
  constexpr int E = JR * DP / 4;  // four dimensions of a row each
  constexpr int SLOTS = E < kAttnThreads ? kAttnThreads / E : 1;
  __shared__ float sm[SLOTS][JR], sl[SLOTS][JR];
  __shared__ attn_f32x4 so[SLOTS][SLOTS > 1 ? E : 1];
  const dsr_tree_attention_args_t& a = j.a;
  const int heads = a.q_heads, group = j.p[0].group, blocks = (heads + JR - 1) / JR;
  const int slot = SLOTS > 1 ? threadIdx.x / E : 0;
  const bool spare = slot >= SLOTS;  // 192 dimensions
  const int64_t items = a.tokens * blocks;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int t = (int)(item / blocks), h0 = (int)(item - (int64_t)t * blocks) * JR;
    const int r = prefix_owner(a, t);
    if (r >= a.requests) continue;
    const AttnRequest own = attn_request(a, j.p[1], j.b[1], r);
    if (t < own.lo || t >= own.lo + own.n) continue;  // a row of no request
    int g = own.fine ? j.b[1].group_of[r] : -1;
    AttnRequest all{};
    if (g >= 0) {
      all = attn_request(a, j.p[0], j.b[0], g);
      if (t < all.lo || t >= all.lo + all.n) g = -1;  // offsets that do not ascend
    }
#pragma unroll
    for (int x = SLOTS > 1 ? threadIdx.x % E : threadIdx.x; x < E; x += kAttnThreads) {
      const int in = x / (DP / 4), h = h0 + in, d = x % (DP / 4) * 4;
      const bool live = h < heads && !spare;
      const int kv_head = h / group, of_group = h - kv_head * group;
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
      if (live && own.fine) {
        int at = slot;  // parts of both passes, counted on
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
          if (pass == 0 && g < 0) continue;
          const AttnPlan& p = j.p[pass];
          const AttnBranch& b = j.b[pass];
          const AttnRequest& q = pass == 0 ? all : own;
          const int in_tiles = (t - q.lo) * group + of_group, tile = in_tiles >> p.tile_shift;
          const int in_tile = in_tiles - (tile << p.tile_shift);
          int first, last;
          prefix_shares(p, b, q, pass == 0 ? g : r, kv_head, tile, first, last);
          if (first == last) {
            if (at == 0) {
              const float2 ml = b.row_ml[row];
              add(ml.x, ml.y, *(const attn_f32x4*)&b.row_o[row * DP + d]);
              at += SLOTS;
            }
            at -= 1;
          } else {
            const int n = last - first + 1;
#pragma unroll 4
            for (; at < n; at += SLOTS) {
              // The first part is its workgroup's last (an odd place), the others their workgroups' first.
              const int64_t place = ((int64_t)(2 * (first + at) + (at == 0)) << p.tile_shift) + in_tile;
              const float2 ml = p.part_ml[place];
              add(ml.x, ml.y, *(const attn_f32x4*)&p.part_o[place * DP + d]);
            }
            at -= n;
          }
        }
      }
      if constexpr (SLOTS > 1) {
        if (!spare) so[slot][x] = o;
        if (d == 0 && !spare) {
          sm[slot][in] = M;
          sl[slot][in] = L;
        }
        __syncthreads();
        if (slot == 0) {
#pragma unroll
          for (int i = 1; i < SLOTS; ++i) add(sm[i][in], sl[i][in], so[i][x]);
        }
        __syncthreads();  // the next item's
      }
      if (slot > 0 || !live || d >= a.head_dim) continue;
      const float inv = L == 0.f ? 0.f : 1.f / L;
      x4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = (T)(o[i] * inv);
      *(x4*)((T*)a.out + (int64_t)t * a.out_token + (int64_t)h * a.out_head + d) = y;
      if (a.lse && d == 0) a.lse[row] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
    }
    if (t == own.lo && h0 == 0 && threadIdx.x == 0) {
      // A request's (a group's) last tile of its first head speaks for its page ids.
      int bad = 0;
      if (own.fine)
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
          if (pass == 0 && g < 0) continue;
          const AttnRequest& q = pass == 0 ? all : own;
          int first, last;
          prefix_shares(j.p[pass], j.b[pass], q, pass == 0 ? g : r, 0, q.tiles - 1, first, last);
          if (first == last)
            bad |= j.b[pass].bad[pass == 0 ? g : r];
          else
            for (int c = first; c <= last; ++c) bad |= j.p[pass].part_bad[2 * c + (c == first)];
        }
      a.status[r] = !own.fine ? DSR_E_LENGTH : bad ? DSR_E_BLOCK : DSR_OK;
    }
  }
}

}  // namespace dsr
