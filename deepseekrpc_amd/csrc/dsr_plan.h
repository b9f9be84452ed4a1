// Block tables, slot maps, positions and tree masks of a step's new tokens
// (dsr_plan_blocks), from request lengths that only the device knows.
//
// Two parts.  plan_scan: one workgroup turns lengths and counts into
// offsets, grants and the pool's ring index of each request's first new page
// by prefix sums.
// plan_token / plan_tree: every token's slot and position, 64 tokens to a
// wave, and every new table entry, written by the token that first touches
// the page (a new page lies wholly past the old tokens, so its first slot is
// always a new token's).
//
// What bounds it is latency: a call reads and writes a few KB to a few MB,
// and its chain is load -> three scans -> offset search -> table entry ->
// store.  64 requests of one token 6.0 us in one launch; 256 trees of 9 to 33
// nodes 7.7 to 8.2 in two; 1,024 prompts with 523,000 tokens (6.3 MB written)
// 12.6: 6.1 the one workgroup's scan, 6.0 the rest.
#pragma once

#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "dsr_tree.h"

namespace dsr {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

// What plan_scan leaves for the second part, per request (a.workspace; a
// PlanTail lies behind).
struct PlanRow {
  int32_t ring;  // granted: pool index of the first page taken; ended: of the first page given back
  int32_t old;   // pages held before
  int32_t held;  // and after
  int32_t mode;  // kPlanRefused / kPlanGranted / kPlanEnded
};
constexpr int kPlanRefused = 0, kPlanGranted = 1, kPlanEnded = 2;
constexpr int kPlanCheckers = 64;  // workgroups; a flag for each lane of a wave
struct PlanTail {
  int32_t flags[kPlanCheckers];  // a page outside the cache (plan_check)
  int32_t state[2];              // the pool's afterwards
};
__device__ __forceinline__ PlanTail* plan_tail(const dsr_plan_args_t& a) {
  return (PlanTail*)((PlanRow*)a.workspace + a.requests);
}

// Sums of counts that are at most 2^30 each: they stop at 2^31 - 1, above
// every bound they are compared with, so that 32 bits are enough for counts
// that come unchecked from device memory.
__device__ __forceinline__ int plan_add(int x, int y) { return __builtin_elementwise_add_sat(x, y); }

// Inclusive sums over the lanes of a wave (row shifts, then the rows' last
// lanes handed on), without LDS.
__device__ __forceinline__ int plan_wave_scan(int x) {
  x = plan_add(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // lane - 1 in its row of 16
  x = plan_add(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = plan_add(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = plan_add(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = plan_add(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // rows 1 and 3 get the row before
  x = plan_add(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));  // rows 2 and 3 get lane 31
  return x;
}

constexpr int kPlanSums = 3;  // tokens, pages wanted, pages given back

// One workgroup of 1,024 threads, a request per thread and round.  `checked`:
// other workgroups are reading pages held and pool state, whose new values,
// which may replace them, wait in the workspace for the second part.
//
// One scan of the three counts serves every decision.  A request that does
// not fit the token arrays, or finds the pool short, still counts in the sums
// of those behind it: by then no later request with tokens, or without its
// pages, can be granted either, and the others want none.
__device__ __forceinline__ void plan_scan(const dsr_plan_args_t& a, bool checked) {
  __shared__ int part[kPlanSums][kPlanWaves];
  __shared__ int done[2];  // pages taken and given back in all
  const int R = (int)a.requests;
  const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int shift = __ffs(a.page) - 1;
  const uint32_t most = (uint32_t)a.width << shift;
  const int capacity = (int)a.capacity, pool_size = a.pool_size;
  PlanRow* rows = (PlanRow*)a.workspace;
  int head = a.pool_state_in[0], count = a.pool_state_in[1];
  if (head < 0 || head >= pool_size || count < 0 || count > pool_size) head = count = 0;  // not a pool: empty
  auto wrap = [&](int x) { return x >= pool_size ? x - pool_size : x; };
  if (threadIdx.x < 2) done[threadIdx.x] = 0;
  if (threadIdx.x == 0) a.offsets[0] = 0;
  int base[kPlanSums] = {0, 0, 0};  // sums over the requests before these 1,024
  for (int r0 = 0; r0 < R; r0 += kPlanThreads) {
    const int r = r0 + (int)threadIdx.x;
    const bool in = r < R;
    const int L = in ? a.lengths[r] : 0, A = in ? a.added[r] : 0, held = in ? a.held_in[r] : 0;
    const bool ended = A == -1;
    const int take = A > 0 ? A : 0;
    int status = DSR_OK;
    if (L < 0 || A < -1 || (uint32_t)held > (uint32_t)a.width || (uint32_t)L > (uint32_t)held << shift ||
        (uint32_t)L + (uint32_t)take > most)
      status = DSR_E_LENGTH;
    const int wants = (int)(((uint32_t)L + (uint32_t)take + (uint32_t)a.page - 1) >> shift) - held;
    const int need = status == DSR_OK && !ended && wants > 0 ? wants : 0;
    const int give = status == DSR_OK && ended ? held : 0;
    int sum[kPlanSums] = {plan_wave_scan(take <= capacity ? take : capacity + 1), plan_wave_scan(need),
                          plan_wave_scan(give)};
    __syncthreads();  // the last round's readers are done
    if (l == 63)
#pragma unroll
      for (int k = 0; k < kPlanSums; ++k) part[k][w] = sum[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPlanSums; ++k) {
      const int waves_to = plan_wave_scan(l < kPlanWaves ? part[k][l] : 0);  // lane i: waves 0 .. i
      const int before = w > 0 ? __builtin_amdgcn_readlane(waves_to, w - 1) : 0;
      sum[k] = plan_add(sum[k], plan_add(base[k], before));
      base[k] = plan_add(base[k], __builtin_amdgcn_readlane(waves_to, 63));
    }
    if (status == DSR_OK && take > 0 && sum[0] > capacity) status = DSR_E_CAPACITY;
    if (status == DSR_OK && need > 0 && sum[1] > count) status = DSR_E_BLOCKS;
    if (status == DSR_OK && give > 0 && sum[2] > pool_size - count) status = DSR_E_BLOCKS;
    const bool granted = status == DSR_OK && !ended, frees = status == DSR_OK && ended;
    if (in) {
      PlanRow p;
      p.ring = granted && need > 0 ? wrap(head + sum[1] - need)
                                   : frees && give > 0 ? wrap(wrap(head + count) + sum[2] - give) : 0;
      p.old = held;
      p.held = granted ? held + need : frees ? 0 : held;
      p.mode = granted ? kPlanGranted : frees ? kPlanEnded : kPlanRefused;
      rows[r] = p;
      a.offsets[r + 1] = sum[0] < capacity ? sum[0] : capacity;
      a.kv_lengths[r] = granted ? L + take : 0;
      if (!checked) a.held_out[r] = p.held;
      a.status[r] = status;
    }
    if (granted && need > 0) atomicMax(&done[0], sum[1]);
    if (frees && give > 0) atomicMax(&done[1], sum[2]);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int32_t* state = checked ? plan_tail(a)->state : a.pool_state_out;
    state[0] = wrap(head + done[0]);
    state[1] = count - done[0] + done[1];
  }
}

// A request that touches a page outside the cache gets no slot at all, but its
// tokens are spread over waves that know nothing of each other.  So workgroups
// beside the scan's look through all pages that the step may touch; only if
// they find one do the waves look through their requests' pages.
__device__ __forceinline__ void plan_check(const dsr_plan_args_t& a, int checker) {
  __shared__ int found;
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  const int R = (int)a.requests, shift = __ffs(a.page) - 1, l = threadIdx.x & 63;
  const unsigned blocks = a.blocks;
  bool bad = false;
  // The pages held already, a request a wave.
  for (int r = checker * kPlanWaves + (int)(threadIdx.x >> 6); r < R; r += kPlanCheckers * kPlanWaves) {
    const int L = a.lengths[r], A = a.added[r], held = a.held_in[r];
    if (L < 0 || A <= 0 || (uint32_t)held > (uint32_t)a.width) continue;
    const uint32_t end = ((uint32_t)L + (uint32_t)A + (uint32_t)a.page - 1) >> shift;
    for (uint32_t b = ((uint32_t)L >> shift) + l; b < end && b < (uint32_t)held; b += 64)
      bad |= (unsigned)a.table[r * a.table_ld + b] >= blocks;
  }
  // The pool's first pages: a granted request takes at most one more than its tokens fill.
  const int head = a.pool_state_in[0], count = a.pool_state_in[1], size = a.pool_size;
  if (head >= 0 && head < size && count <= size) {
    const int most = (int)(a.capacity >> shift) + R;
    for (int i = checker * kPlanThreads + (int)threadIdx.x; i < count && i < most; i += kPlanCheckers * kPlanThreads)
      bad |= (unsigned)a.pool[head + i >= size ? head + i - size : head + i] >= blocks;
  }
  if (bad) found = 1;
  __syncthreads();
  if (threadIdx.x == 0) plan_tail(a)->flags[checker] = found;
}

// The slot of place `p` of request r, and, if this is the first slot of a
// new page, the page's table entry.
__device__ __forceinline__ int plan_slot(const dsr_plan_args_t& a, const PlanRow& row, int64_t r, int p) {
  const int shift = __ffs(a.page) - 1, b = p >> shift, o = p & (a.page - 1);
  int id;
  if (b < row.old) {
    id = a.table[r * a.table_ld + b];
  } else {
    const int at = row.ring + b - row.old;
    id = a.pool[at >= a.pool_size ? at - a.pool_size : at];
    if (o == 0) a.table[r * a.table_ld + b] = id;
  }
  if ((unsigned)id >= (unsigned)a.blocks) {
    a.status[r] = DSR_E_BLOCK;
    a.kv_lengths[r] = 0;
    return -1;
  }
  return (id << shift) + o;
}

__device__ __forceinline__ void plan_write(const dsr_plan_args_t& a, int64_t i, int slot, int position, int owner,
                                           uint64_t mask) {
  a.slots[i] = slot;
  a.positions[i] = position;
  if (a.owners) a.owners[i] = owner;
  if (a.visible) a.visible[i] = mask;
}

// The number of requests whose tokens end at or before token i (its owner),
// for a whole wave at once: 64 offsets per round.
__device__ __forceinline__ int plan_owner(const dsr_plan_args_t& a, int i) {
  const int l = threadIdx.x & 63;
  int lo = 0, n = (int)a.requests;
  while (n > 0) {
    const int stride = (n + 63) / 64, end = lo + n;
    const int at = lo + l * stride + stride - 1;
    const uint64_t le = __ballot(at < end && a.offsets[at < end ? at + 1 : 0] <= i);
    lo += __popcll(le) * stride;
    n = end - lo < stride - 1 ? end - lo : stride - 1;
  }
  return lo;
}

// How many of the wave's 64 non-decreasing x are <= i, for each lane's own i.
__device__ __forceinline__ int plan_count(int x, int i) {
  int c = 0;
#pragma unroll
  for (int s = 32; s > 0; s >>= 1)
    if (__shfl(x, c + s - 1) <= i) c += s;
  return __shfl(x, c) <= i ? c + 1 : c;
}

// Whether request r's new tokens touch a page outside the cache (one wave).
__device__ __forceinline__ bool plan_outside(const dsr_plan_args_t& a, int r) {
  const int shift = __ffs(a.page) - 1, n = a.offsets[r + 1] - a.offsets[r];
  const PlanRow row = ((const PlanRow*)a.workspace)[r];
  const int begin = a.lengths[r] >> shift, end = n > 0 ? ((a.lengths[r] + n - 1) >> shift) + 1 : begin;
  for (int b0 = begin; b0 < end; b0 += 64) {
    const int b = b0 + (int)(threadIdx.x & 63), at = row.ring + b - row.old;
    int id = 0;
    if (b < end) id = b < row.old ? a.table[r * a.table_ld + b] : a.pool[at >= a.pool_size ? at - a.pool_size : at];
    if (__ballot((unsigned)id >= (unsigned)a.blocks)) return true;
  }
  return false;
}

struct PlanToken {
  int owner, slot, position;
  bool granted;  // its request is served
};

// Token i0 + lane (one wave).
__device__ __forceinline__ PlanToken plan_token(const dsr_plan_args_t& a, int i0) {
  const int l = threadIdx.x & 63, R = (int)a.requests;
  const int i = i0 + l;
  // Each token's owner lies as many requests behind token i0's as end at or
  // before the token; 64 requests a round (empty ones can make it more).
  int base = plan_owner(a, i0), r = base, c;
  do {
    c = plan_count(base + l < R ? a.offsets[base + l + 1] : INT_MAX, i);
    r += r == base ? c : 0;
    base += 64;
  } while (__ballot(c == 64));
  PlanToken t{-1, -1, 0, false};
  if (i >= a.capacity || r >= R || i >= a.offsets[R]) return t;
  t.owner = r;
  const PlanRow row = ((const PlanRow*)a.workspace)[r];
  if (row.mode != kPlanGranted) return t;
  t.granted = true;
  t.position = a.lengths[r] + i - a.offsets[r];
  t.slot = plan_slot(a, row, r, t.position);
  return t;
}

// ... and its results.  `doubt`: some request may touch a page outside the cache.
__device__ __forceinline__ void plan_store(const dsr_plan_args_t& a, int i0, PlanToken t, bool doubt) {
  const int i = i0 + (int)(threadIdx.x & 63);
  if (doubt) {
    uint64_t left = __ballot(t.granted);
    while (left) {
      const int r = __shfl(t.owner, __ffsll((unsigned long long)left) - 1);
      const bool mine = t.granted && t.owner == r;
      left &= ~__ballot(mine);
      if (plan_outside(a, r) && mine) t.slot = -1;
    }
  }
  if (i < a.capacity) plan_write(a, i, t.slot, t.slot < 0 ? 0 : t.position, t.owner, 0);
}

// Request r's pages back to the pool, if it ended (one wave).
__device__ __forceinline__ void plan_release(const dsr_plan_args_t& a, int r) {
  const PlanRow row = ((const PlanRow*)a.workspace)[r];
  if (row.mode != kPlanEnded) return;
  for (int b = threadIdx.x & 63; b < row.old; b += 64) {
    const int at = row.ring + b;
    a.pool[at >= a.pool_size ? at - a.pool_size : at] = a.table[r * a.table_ld + b];
  }
}

// Request r's tree, one node per lane: masks and depths by pointer doubling
// (after round k a node knows its nearest 2^k ancestors).
__device__ __forceinline__ void plan_tree(const dsr_plan_args_t& a, int r) {
  const int l = threadIdx.x & 63;
  const PlanRow row = ((const PlanRow*)a.workspace)[r];
  const int lo = a.offsets[r], n = a.offsets[r + 1] - lo;
  if (row.mode != kPlanGranted) {
    for (int i = l; i < n; i += 64) plan_write(a, lo + i, -1, 0, r, 0);
    return;
  }
  const int par = l < n ? a.parents[lo + l] : -1;
  if (__ballot(par >= l || par < -1) || n > DSR_TREE_MAX_NODES) {
    for (int i = l; i < n; i += 64) {
      plan_write(a, lo + i, -1, 0, r, 0);
      // Pages already taken stay with the request, table entries included.
      const int p = a.lengths[r] + i;
      if (p >= row.old * a.page && (p & (a.page - 1)) == 0) plan_slot(a, row, r, p);
    }
    if (l == 0) {
      a.status[r] = DSR_E_TREE;
      a.kv_lengths[r] = 0;
    }
    return;
  }
  uint64_t mask = 1ull << l;
  int depth = par >= 0 ? 1 : 0, up = par;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const int at = up < 0 ? l : up;
    const uint64_t m = __shfl(mask, at);
    const int d = __shfl(depth, at), u = __shfl(up, at);
    if (up >= 0) {
      mask |= m;
      depth += d;
      up = u;
    }
  }
  const int slot = l < n ? plan_slot(a, row, r, a.lengths[r] + l) : 0;
  const bool outside = __ballot(slot < 0) != 0;  // then no node has a slot
  if (l < n) plan_write(a, lo + l, outside ? -1 : slot, outside ? 0 : a.lengths[r] + depth, r, outside ? 0 : mask);
}

// Tokens past the last request's (tree plans: the trees write their own).
__device__ __forceinline__ void plan_padding(const dsr_plan_args_t& a, int i) {
  if (i < a.capacity && i >= a.offsets[a.requests]) plan_write(a, i, -1, 0, -1, 0);
}

// The first workgroup scans, the others (for tokens without trees) check.
__global__ __launch_bounds__(kPlanThreads) void k_plan_scan(dsr_plan_args_t a) {
  if (blockIdx.x > 0)
    plan_check(a, blockIdx.x - 1);
  else
    plan_scan(a, gridDim.x > 1);
}

// 256 threads: workgroups [0, token_groups) take 256 tokens each, the others four requests each.
__global__ __launch_bounds__(256) void k_plan_fill(dsr_plan_args_t a, int token_groups, bool checked) {
  const int w = threadIdx.x >> 6, b = blockIdx.x;
  if (b < token_groups) {
    if (a.parents) {
      plan_padding(a, b * 256 + (int)threadIdx.x);
    } else {
      const bool doubt = checked && __ballot(plan_tail(a)->flags[threadIdx.x & (kPlanCheckers - 1)] != 0) != 0;
      plan_store(a, b * 256 + w * 64, plan_token(a, b * 256 + w * 64), doubt);
    }
    return;
  }
  const int r = (b - token_groups) * 4 + w;
  if (r >= a.requests) return;
  if (checked) {  // new values that waited
    if ((threadIdx.x & 63) == 0) a.held_out[r] = ((const PlanRow*)a.workspace)[r].held;
    if (r == 0 && threadIdx.x < 2) a.pool_state_out[threadIdx.x] = plan_tail(a)->state[threadIdx.x];
  }
  if (a.parents) plan_tree(a, r);
  plan_release(a, r);
}

// The whole plan in one workgroup, for calls that fit it.
__global__ __launch_bounds__(kPlanThreads) void k_plan_small(dsr_plan_args_t a) {
  __shared__ int doubt;
  if (threadIdx.x == 0) doubt = 0;
  plan_scan(a, false);
  __threadfence_block();
  __syncthreads();
  const int w = threadIdx.x >> 6;
  if (a.parents) {
    for (int i = threadIdx.x; i < a.capacity; i += kPlanThreads) plan_padding(a, i);
    for (int r = w; r < a.requests; r += kPlanWaves) plan_tree(a, r);
  } else {
    const PlanToken t = plan_token(a, w * 64);  // a token a thread
    if (t.granted && t.slot < 0) doubt = 1;
    __syncthreads();
    plan_store(a, w * 64, t, doubt != 0);
  }
  for (int r = w; r < a.requests; r += kPlanWaves) plan_release(a, r);
}

}  // namespace dsr
