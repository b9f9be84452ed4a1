// Acceptance of drafted trees and their cache rows moved together
// (dsr_commit_tree).  What a step refused keeps its length and pending token.
//
// A workgroup takes one request and a few caches.  Its first wave walks the
// tree with one node per lane: the children of the current node whose token
// is the one sampled there are a ballot, the first of them its lowest bit, so
// a step costs a few cycles and no memory access.  Every workgroup of a
// request walks again rather than wait for another launch; the first writes
// the decision.
//
// The move is in place: path node j's row goes to place j, and path[j] >= j
// grows with j, so no row is overwritten before it is read as long as each
// byte's moves run in path order, or a batch of reads before its writes.  A
// thread owns a 16-byte column of the rows and does just that.
// What bounds it: a chain of a few dependent reads (tree, page ids, rows),
// then 2 x row bytes per move and cache.  64 trees, 48 layers of keys and
// values, about 35 MB moved: 10.5 to 11.5 us, 3.1 to 3.4 TB/s, on caches that
// change from call to call; 8 trees, 4 layers, 3.8 to 4.3.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dsr_tree.h"

namespace dsr {

constexpr int kCommitThreads = 256;
// Rows in flight per thread (64 trees, the same caches again and again: 10.1 us with two, 9.6 with four, 9.7 with eight).
constexpr int kCommitBatch = 4;

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// Caches per workgroup: as many as its threads cover with one 16-byte column
// each, at most 8 (64 trees, as above: 11.9 us with one, 9.6 with two to
// sixteen; the fewer, the more often a request's tree is walked).
__host__ __device__ inline int commit_caches(const dsr_commit_args_t& a) {
  const int columns = a.heads * (a.row_bytes / 16);
  const int c = columns > 0 ? kCommitThreads / columns : 1;
  return c < 1 ? 1 : c > 8 ? 8 : c;
}

// Caches of one launch whose pointers are its arguments (COUNT 0: they lie in
// device memory).  8 trees, 8 caches 4.5 us so and 4.4 from device memory; 64
// trees, 128 caches 11.0 and 11.1; 8 trees, 320 caches, three launches, 12.3
// and 3.9.
constexpr int kCommitInline = 128;
template <int COUNT>
struct CommitCaches {
  void* at[COUNT];
};
template <>
struct CommitCaches<0> {};

template <int COUNT>
__global__ __launch_bounds__(kCommitThreads) void k_commit_tree(dsr_commit_args_t a, CommitCaches<COUNT> caches) {
  __shared__ int64_t from[DSR_TREE_MAX_NODES], to[DSR_TREE_MAX_NODES];
  __shared__ int moves;
  const int r = blockIdx.x, l = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    int lo = a.offsets[r], hi = a.offsets[r + 1];
    lo = lo < 0 ? 0 : lo > a.tokens ? (int)a.tokens : lo;
    hi = hi < lo ? lo : hi > a.tokens ? (int)a.tokens : hi;
    const int n = hi - lo, kv = a.kv_lengths[r], limit = a.output_limit[r];
    const bool before = a.lengths_in != nullptr;
    const int old = before ? a.lengths_in[r] : 0, waiting = before ? a.pending_in[r] : -1;
    const int planned = before ? a.plan_status[r] : DSR_OK;
    int par = -1, token = -1, target = -1;
    if (l < n) {
      par = a.parents[lo + l];
      token = a.tokens_in[lo + l];
      target = a.sampled[lo + l];
    }
    const int64_t eos_lo = a.eos_off ? a.eos_off[r] : 0, eos_hi = a.eos_off ? a.eos_off[r + 1] : 0;
    int status = DSR_OK;
    if (n > DSR_TREE_MAX_NODES || __ballot(l < n && (par >= l || par < -1))) status = DSR_E_TREE;
    if (kv < n || kv > (int64_t)a.width * a.page || (limit < 1 && !(before && n == 0))) status = DSR_E_LENGTH;
    if (planned != DSR_OK) status = planned;
    int kept = 0, said = 0, pending = waiting, stop = DSR_STOP_NONE;
    int mine_path = -1, mine_id = -1;
    if (status == DSR_OK && n > 0) {
      int cur = 0;
      kept = 1;
      if (l == 0) mine_path = 0;
      for (;;) {  // at most n rounds: every round but the last moves to a later node
        const int t = __shfl(target, cur);
        if (t < 0) {
          status = DSR_E_TOKEN;
          break;
        }
        if (l == said) mine_id = t;
        ++said;
        bool end = false;
        for (int64_t e = eos_lo; e < eos_hi; e += 64) end |= __ballot(e + l < eos_hi && a.eos_ids[e + l] == t) != 0;
        const int reason = end ? DSR_STOP_EOS : said >= limit ? DSR_STOP_LENGTH : DSR_STOP_NONE;
        const uint64_t child = __ballot(l > 0 && l < n && par == cur && token == t);
        if (!child) {
          pending = t;
          stop = reason;
          break;
        }
        cur = __ffsll((unsigned long long)child) - 1;
        if (l == kept) mine_path = cur;
        ++kept;
        if (reason != DSR_STOP_NONE) {
          stop = reason;
          break;
        }
      }
    }
    const int ctx = kv - n;
    // Lane j: where path node j's row is and goes.
    int64_t src = 0, dst = 0;
    bool bad = false;
    if (status == DSR_OK && l < kept) {
      const int p = ctx + mine_path, q = ctx + l;
      const int ip = a.table[r * a.table_ld + p / a.page], iq = a.table[r * a.table_ld + q / a.page];
      bad = (unsigned)ip >= (unsigned)a.blocks || (unsigned)iq >= (unsigned)a.blocks;
      src = ip * a.c_block + (p & (a.page - 1)) * a.c_token;
      dst = iq * a.c_block + (q & (a.page - 1)) * a.c_token;
    }
    if (status == DSR_OK && __ballot(bad)) status = DSR_E_BLOCK;
    if (status != DSR_OK) {
      kept = said = 0;
      mine_path = mine_id = -1;
      pending = waiting;
      stop = DSR_STOP_NONE;
    }
    if (blockIdx.y == 0) {
      a.path[(int64_t)r * DSR_TREE_MAX_NODES + l] = mine_path;
      a.ids[(int64_t)r * DSR_TREE_MAX_NODES + l] = mine_id;
      if (l == 0) {
        a.accepted[r] = kept;
        a.count[r] = said;
        a.pending[r] = pending;
        a.stop[r] = stop;
        a.lengths[r] = before && status != DSR_OK ? old : status == DSR_E_LENGTH ? 0 : ctx + kept;
        a.status[r] = status;
      }
    }
    // The moves in path order: nodes already in place are none.
    const bool move = l < kept && mine_path != l;
    const uint64_t which = __ballot(move);
    if (move) {
      const int at = __popcll(which & ((1ull << l) - 1));
      from[at] = src;
      to[at] = dst;
    }
    if (l == 0) moves = __popcll(which);
  }
  __syncthreads();
  const int m = moves;
  if (m == 0) return;
  const int columns = a.heads * (a.row_bytes / 16), per_row = a.row_bytes / 16;
  const int per_group = commit_caches(a), first = blockIdx.y * per_group;
  for (int x = threadIdx.x; x < per_group * columns; x += kCommitThreads) {
    const int c = first + x / columns, col = x % columns;
    if (c >= a.cache_count) break;
    char* base;
    if constexpr (COUNT > 0)
      base = (char*)caches.at[c];
    else
      base = (char*)a.caches[c];
    base += (int64_t)(col / per_row) * a.c_head + (col % per_row) * 16;
    for (int j = 0; j < m; j += kCommitBatch) {
      u32x4_t v[kCommitBatch];
#pragma unroll
      for (int b = 0; b < kCommitBatch; ++b)
        if (j + b < m) v[b] = *(const u32x4_t*)(base + from[j + b]);
#pragma unroll
      for (int b = 0; b < kCommitBatch; ++b)
        if (j + b < m) *(u32x4_t*)(base + to[j + b]) = v[b];
    }
  }
}

}  // namespace dsr
