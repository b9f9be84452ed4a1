// C ABI of dsr_tree.h: argument checks and launches.
#include "dsr_tree.h"

#include "dsr_attention.h"
#include "dsr_attention_wide.h"
#include "dsr_commit.h"
#include "dsr_plan.h"
#include "dsr_rotary.h"

using namespace dsr;

namespace {

int32_t launched() { return hipGetLastError() == hipSuccess ? 0 : DSR_ERR_LAUNCH; }

bool page_ok(int32_t page, int32_t blocks) {
  return page >= 1 && page <= DSR_TREE_MAX_PAGE && (page & (page - 1)) == 0 && blocks >= 1 &&
         (int64_t)blocks * page <= INT_MAX;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

// Plans of at most this many tokens and requests (trees) run in one workgroup
// and launch.  Us a call in one launch against two: 64 requests of 1 token 6.6
// and 7.1, of 16 8.3 and 8.8; 128 of 8 8.3 and 8.2, 256 of 2 8.9 and 7.9; 16
// trees of 8 nodes 6.5 and 7.1, of 32 6.9 and 7.3, 24 of 8 7.5 and 7.3.
constexpr int kPlanSmallTokens = 1024, kPlanSmallRequests = 128, kPlanSmallTrees = 16;
static_assert(kPlanSmallTokens <= kPlanThreads, "a token a thread");

// Whether every row, part and pair of a rotary call can be taken VE elements at a time.
template <class T>
bool rotary_fits(const dsr_rotary_args_t& a, int VE) {
  auto rows = [&](const void* p, int64_t t, int64_t h) {
    return !p || ((uintptr_t)p % (VE * sizeof(T)) == 0 && t % VE == 0 && h % VE == 0);
  };
  return a.head_dim % VE == 0 && a.rot_start % VE == 0 &&
         (a.interleaved ? a.rot_dim % VE == 0 : a.rot_dim / 2 % VE == 0) && (!a.v || a.v_dim % VE == 0) &&
         rows(a.q, a.q_token, a.q_head) && rows(a.q_out, a.qo_token, a.qo_head) && rows(a.k, a.k_token, a.k_head) &&
         rows(a.k_out, a.ko_token, a.ko_head) && rows(a.v, a.v_token, a.v_head) &&
         (!a.k_cache || (rows(a.k_cache, a.kc_token, a.kc_head) && a.kc_block % VE == 0)) &&
         (!a.v_cache || (rows(a.v_cache, a.vc_token, a.vc_head) && a.vc_block % VE == 0));
}

// Tokens of one launch: a workgroup each, and a launch has less than 2^32 threads.
constexpr int64_t kRotaryTokens = 1 << 23;

template <class T, int VE>
void rotary_launch(const dsr_rotary_args_t& a, hipStream_t s) {
  const int64_t items = (int64_t)(a.q_heads + a.kv_heads) * a.head_dim / VE;
  // Few tokens: a token's rows are shared by several workgroups, so that the
  // chip is filled (256 tokens of 80 rows of 128: 5.3 us with one each, 4.8 so;
  // 64 tokens 4.9 and 4.5; from 1,024 on the same).
  int64_t parts = (1024 + a.tokens - 1) / a.tokens, most = (items + kRotaryThreads - 1) / kRotaryThreads;
  if (parts > most) parts = most;
  if (parts < 1) parts = 1;
  const dim3 grid((unsigned)a.tokens, (unsigned)parts);
  const dim3 threads(kRotaryThreads);
  if (a.interleaved)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_rotary<T, VE, true>), grid, threads, 0, s, a);
  else
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_rotary<T, VE, false>), grid, threads, 0, s, a);
}

template <class T>
int32_t rotary_typed(const dsr_rotary_args_t& a, hipStream_t s) {
  constexpr int VE = 16 / sizeof(T);
  const bool wide = rotary_fits<T>(a, VE);
  const bool half = rotary_fits<T>(a, 4);  // halves of 12 or 20, say (float32 rows are wide then)
  for (int64_t first = 0; first < a.tokens; first += kRotaryTokens) {
    dsr_rotary_args_t part = a;
    part.tokens = a.tokens - first < kRotaryTokens ? a.tokens - first : kRotaryTokens;
    part.positions += first;
    if (a.slots) part.slots += first;
    if (a.status) part.status += first;
    if (a.q) part.q = (const T*)a.q + first * a.q_token, part.q_out = (T*)a.q_out + first * a.qo_token;
    if (a.k) part.k = (const T*)a.k + first * a.k_token;
    if (a.k_out) part.k_out = (T*)a.k_out + first * a.ko_token;
    if (a.v) part.v = (const T*)a.v + first * a.v_token;
    if (wide)
      rotary_launch<T, VE>(part, s);
    else if (half)
      rotary_launch<T, 4>(part, s);
    else
      rotary_launch<T, 1>(part, s);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  }
  return 0;
}

// Dimensions of the kernel that takes a head dimension (the rest are zeros in LDS).
int attn_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256; }

// Host part of the work split, from sizes alone.  The figures are us a call in
// bf16 with 8 key heads of 128, contexts about as long as the table's rows.
AttnPlan attn_plan(const dsr_tree_attention_args_t& a) {
  AttnPlan p{};
  const int64_t group = a.q_heads / a.kv_heads;
  const int64_t rows = a.requests > 0 ? (a.tokens * group + a.requests - 1) / a.requests : 0;  // of a usual request
  const bool big = a.head_dim > 128;
  const int64_t span = (int64_t)a.width * a.page;
  auto tiles_of = [&](int r) { return (a.tokens * group / r + a.requests) * a.kv_heads; };
  // Where a whole table row is a short way for one workgroup, a longer one if
  // there are tiles for more of the chip, a tile is one step: nothing is cut,
  // no parts are written and no joining launch follows.  Uncut against cut, a
  // token a request: 1 request over 500 tokens 11.9 and 14.2, over 1,000 15.8 and
  // 15.4; 16 over 1,000 19.9 and 27.8; 32 over 2,000 55 and 65.
  auto is_short = [&](int64_t tiles) { return span <= (tiles < 64 ? 512 : tiles > 256 ? 2048 : 8 * tiles); };
  // A tile for the rows of a usual request, so that its keys and values are
  // read once.  32 requests over 8,064 tokens: 16 rows 200 in tiles of 16, 210
  // of 32; 32 rows 228 of 16, 209 of 32, 229 of 64.  64 rows: 237 of 64 and 236
  // of 128, and 199 and 177 on 100 ragged requests, so that 128 take them.  With
  // 256 dimensions 32 rows 724 in tiles of 16, 384 of 64, 504 of 128.  Whole
  // tiles of 32 have a CU each, of 128 two share one: 200 requests of 24 rows over
  // 480 tokens 111 and 66.
  //
  // The kernel for 16 rows has the shortest way from start to end (9 us; 20 in
  // tiles of 32, 10 of 128; 14 with 256 dimensions, 26 of 64), and takes calls of
  // any rows whose tiles the chip holds about at once, as long as reading keys
  // and values again for each costs less.  16 against the other: 4 requests of 64
  // rows over 2,200 tokens 27 and 36, over 6,000 50 and 42; 16 of 24 over 6,000 96
  // and 107; 40 of 24 over 30 tokens 11 and 21 (10 of 128), of 64 17 and 10; 256
  // dimensions, 2 key heads: 16 of 64 over 3,000 50 and 80, 32 of 48 over 8,064 291
  // and 165; 192 dimensions, one key head: 3 of 200 over up to 19,500 94 and 74.
  const int64_t again = big && rows <= 64 ? 3 << 19 : rows <= 32 ? 1 << 21 : 5 << 17;
  const bool few = tiles_of(16) <= (big ? 384 : 512) && tiles_of(16) * span <= again;
  if (rows <= 16 || few)
    p.tile_rows = 16;
  else if (big)
    p.tile_rows = rows <= 64 ? 64 : 128;
  else
    p.tile_rows = rows <= 32 && !is_short(tiles_of(32)) ? 32 : 128;
  p.tokens = p.tile_rows == 16 || p.tile_rows == 32 ? 128 : p.tile_rows == 64 ? 64 : 32;
  p.min_steps = 128 / p.tokens;
  const int64_t tiles = tiles_of(p.tile_rows);
  p.cut = !is_short(tiles);
  // Chunks of prompts have many tiles, and causal ones of unlike lengths.  They
  // go uncut, the longest first, if no tile can be longer than half as much
  // again as a workgroup's share of the chunks alone: 16 chunks of 512 tokens 210
  // and 262, 2 of 512 39 and 116, one of 2,048 130 and 258.
  if (!a.visible && a.tokens > 64 * a.requests && span <= 1 << 20 &&
      span * a.requests * 2048 <= 3 * tiles * a.tokens)
    p.cut = false;
  if (!p.cut) {
    while (p.tokens < span) p.tokens *= 2;
    p.min_steps = 1;
    p.groups = 1 << 14;
  } else {
    // Workgroups that the chip holds at once: 256 CUs, one or two each.  One
    // where a CU has room for one or waits for memory anyway (a token for each
    // of 64 requests over 8,192: 370 with 256, 391 with 512), two where a CU's
    // matrix cores have more to do (8 trees of 64 nodes over 32,000: 822 and 693).
    p.groups = p.tile_rows < 128 || big ? 256 : 512;
  }
  while (((int64_t)a.width * a.page / p.tokens + 1) * tiles >= INT_MAX) p.tokens *= 2;  // steps are counted in 32 bits
  auto log2_of = [](int64_t x) { return x & (x - 1) ? -1 : __builtin_ctzll(x); };
  p.group = (int)group;
  p.tile_shift = log2_of(p.tile_rows), p.token_shift = log2_of(p.tokens), p.group_shift = log2_of(group);
  p.page_shift = a.page > 0 ? log2_of(a.page) : 0;
  // No more workgroups than shares of the fewest steps.
  const int64_t shares = tiles * ((span + p.tokens - 1) / p.tokens) / p.min_steps + 1;
  if (shares < p.groups) p.groups = (int)((shares + 7) / 8 * 8);
  return p;
}

int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

struct AttnSizes {
  int64_t o, ml, all;
};
AttnSizes attn_sizes(const dsr_tree_attention_args_t& a, const AttnPlan& p) {
  AttnSizes s;
  const int64_t parts = p.cut ? 2 * (int64_t)p.groups : 1;
  s.o = round256(parts * p.tile_rows * attn_dim(a.head_dim) * 4);
  s.ml = round256(parts * p.tile_rows * 8);
  s.all = s.o + s.ml + round256(parts * 4);
  return s;
}

bool attn_shape_ok(const dsr_tree_attention_args_t& a) {
  return (a.dtype == DSR_BF16 || a.dtype == DSR_F16) && a.q_heads >= 1 && a.kv_heads >= 1 &&
         a.q_heads % a.kv_heads == 0 && a.head_dim >= 8 && a.head_dim <= DSR_ATTENTION_MAX_DIM &&
         a.head_dim % 8 == 0 && a.requests >= 0 && a.requests <= DSR_TREE_MAX_REQUESTS && a.tokens >= 0 &&
         a.tokens <= INT_MAX &&
         (a.tokens + a.requests) * a.q_heads <= INT_MAX / 4 && a.page >= 1 && a.page <= DSR_TREE_MAX_PAGE &&
         a.width >= 1 && (int64_t)a.width * a.page <= INT_MAX;  // tiles and steps are counted in 32 bits
}

template <class T, int DP, int WR>
void attn_wide(dim3 grid, hipStream_t s, const AttnCall& call) {
  const dsr_tree_attention_args_t& a = call.a;
  // A round's tokens on one page, and their offsets in 32 bits (8 trees of 64
  // nodes over 32,000 tokens, pages of 32: 685 us, 713 without).
  constexpr bool whole = kAttnThreads % (DP / 8) == 0;
  const bool flat = whole && a.page >= attn_round(DP) && a.k_token <= 1 << 24 && a.v_token <= 1 << 24;
  if (flat)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_tree_attention_wide<T, DP, WR, whole>), grid, dim3(kAttnThreads), 0, s, call);
  else
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_tree_attention_wide<T, DP, WR, false>), grid, dim3(kAttnThreads), 0, s, call);
}

template <class T, int DP>
int32_t attn_launch(const dsr_tree_attention_args_t& a, const AttnPlan& p, hipStream_t s) {
  // Workgroups for rows of no request: one for each 256 KB that all rows have, so that a long padding is spread too.
  const int64_t clear = (a.tokens * a.q_heads * a.head_dim * 2 + (1 << 18) - 1) >> 18;
  const dim3 grid((unsigned)p.groups + (unsigned)(clear > 256 ? 256 : clear < 8 ? 8 : clear)), threads(kAttnThreads);
  const AttnCall call{a, p};
  switch (p.tile_rows) {
    case 16:
      if constexpr (DP <= 128)
        if (!p.cut && p.groups < 128) {
          hipLaunchKernelGGL(HIP_KERNEL_NAME(k_tree_attention<T, DP, 8>), grid, dim3(512), 0, s, call);
          break;
        }
      hipLaunchKernelGGL(HIP_KERNEL_NAME(k_tree_attention<T, DP, 4>), grid, threads, 0, s, call);
      break;
    case 128: attn_wide<T, DP, 4>(grid, s, call); break;
    case 64: if constexpr (DP > 128) attn_wide<T, DP, 2>(grid, s, call); break;
    default: if constexpr (DP <= 128) attn_wide<T, DP, 1>(grid, s, call);
  }
  if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  if (p.cut && p.groups > 1) {
    const unsigned borders = (unsigned)p.groups - 1;
    // Two rows a joining workgroup leave threads over for long rows of parts (256
    // dimensions, one request over 10,000 tokens: 34 us a call, 52 with sixteen;
    // one row each: 64 requests of a token 373, 370 with two); tiles of 128 rows
    // would be too many workgroups (4 requests: 53 with sixteen, 89 with two).
    if (p.tile_rows == 16)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(k_tree_join<T, DP, 2>), dim3(borders, (unsigned)(p.tile_rows / 2)), threads, 0, s,
                         call);
    else
      hipLaunchKernelGGL(HIP_KERNEL_NAME(k_tree_join<T, DP, 16>), dim3(borders, (unsigned)(p.tile_rows / 16)), threads, 0,
                         s, call);
  }
  return launched();
}

template <class T>
int32_t attn_typed(const dsr_tree_attention_args_t& a, const AttnPlan& p, hipStream_t s) {
  switch (attn_dim(a.head_dim)) {
    case 64: return attn_launch<T, 64>(a, p, s);
    case 128: return attn_launch<T, 128>(a, p, s);
    case 192: return attn_launch<T, 192>(a, p, s);
    default: return attn_launch<T, 256>(a, p, s);
  }
}

}  // namespace

extern "C" {

size_t dsr_plan_workspace_bytes(int64_t requests) {
  return requests > 0 && requests <= DSR_TREE_MAX_REQUESTS
             ? (size_t)requests * sizeof(PlanRow) + sizeof(PlanTail)
             : 0;
}

int32_t dsr_plan_blocks(const dsr_plan_args_t* args, void* stream) {
  if (!args) return DSR_ERR_ARG;
  const dsr_plan_args_t& a = *args;
  if (a.requests < 0 || a.requests > DSR_TREE_MAX_REQUESTS || a.capacity < 1 || a.capacity > (1 << 30) ||
      !page_ok(a.page, a.blocks) || a.width < 1 || (int64_t)a.width * a.page > INT_MAX || a.table_ld < a.width ||
      a.pool_size < 1 || a.pool_size > (1 << 30))
    return DSR_ERR_ARG;
  if (!a.pool_state_in || !a.pool || !a.pool_state_out || !a.offsets || !a.slots || !a.positions ||
      (a.parents && !a.visible) || (!a.parents && a.visible))
    return DSR_ERR_ARG;
  if (a.requests > 0 && (!a.lengths || !a.added || !a.held_in || !a.table || !a.held_out || !a.kv_lengths || !a.status))
    return DSR_ERR_ARG;
  if (a.requests > 0 && (!a.workspace || ((uintptr_t)a.workspace & 3u) ||
                         a.workspace_bytes < dsr_plan_workspace_bytes(a.requests)))
    return DSR_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  if (a.capacity <= kPlanSmallTokens && a.requests <= (a.parents ? kPlanSmallTrees : kPlanSmallRequests)) {
    hipLaunchKernelGGL(k_plan_small, dim3(1), dim3(kPlanThreads), 0, s, a);
    return launched();
  }
  const unsigned checkers = a.parents || a.requests == 0 ? 0 : kPlanCheckers;
  hipLaunchKernelGGL(k_plan_scan, dim3(1 + checkers), dim3(kPlanThreads), 0, s, a);
  if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  const int token_groups = (int)((a.capacity + 255) / 256);
  hipLaunchKernelGGL(k_plan_fill, dim3((unsigned)(token_groups + (a.requests + 3) / 4)), dim3(256), 0, s, a,
                     token_groups, checkers > 0);
  return launched();
}

int32_t dsr_rotary(const dsr_rotary_args_t* args, void* stream) {
  if (!args) return DSR_ERR_ARG;
  const dsr_rotary_args_t& a = *args;
  if ((a.dtype != DSR_BF16 && a.dtype != DSR_F16 && a.dtype != DSR_F32) || a.reserved != 0 || a.tokens < 0 ||
      a.tokens > (1 << 30) || a.q_heads < 0 || a.kv_heads < 0 || a.q_heads > 65536 || a.kv_heads > 65536 ||
      a.q_heads + a.kv_heads < 1 || a.head_dim < 2 || a.head_dim > DSR_ROTARY_MAX_DIM || a.rot_dim < 2 ||
      a.rot_dim % 2 != 0 || a.rot_start < 0 || a.rot_start + a.rot_dim > a.head_dim ||
      !(a.magnitude > 0.0 && a.magnitude < 1e30))
    return DSR_ERR_ARG;
  if (a.tokens == 0) return 0;
  if (!a.positions || !a.freqs) return DSR_ERR_ARG;
  if ((a.q_heads > 0) != (a.q != nullptr) || (a.q != nullptr) != (a.q_out != nullptr) ||
      (a.kv_heads > 0) != (a.k != nullptr) || (a.k != nullptr) != (a.k_out || a.k_cache) ||
      (a.v != nullptr) != (a.v_cache != nullptr) || (a.v && !a.k) ||
      (a.v && (a.v_dim < 1 || a.v_dim > DSR_ROTARY_MAX_DIM)))
    return DSR_ERR_ARG;
  if ((a.k_cache || a.v_cache) && (!page_ok(a.page, a.blocks) || !a.slots)) return DSR_ERR_ARG;
  if (!(a.k_cache || a.v_cache) && a.slots) return DSR_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  switch (a.dtype) {
    case DSR_BF16: return rotary_typed<__bf16>(a, s);
    case DSR_F16: return rotary_typed<_Float16>(a, s);
    default: return rotary_typed<float>(a, s);
  }
}

size_t dsr_tree_attention_workspace_bytes(const dsr_tree_attention_args_t* args) {
  if (!args || !attn_shape_ok(*args)) return 0;
  return (size_t)attn_sizes(*args, attn_plan(*args)).all;
}

int32_t dsr_tree_attention(const dsr_tree_attention_args_t* args, void* stream) {
  if (!args) return DSR_ERR_ARG;
  const dsr_tree_attention_args_t& a = *args;
  if (!attn_shape_ok(a) || !page_ok(a.page, a.blocks) || a.table_ld < a.width || !(a.scale == a.scale) || a.scale - a.scale != 0.f)
    return DSR_ERR_ARG;
  if (a.requests == 0) return a.tokens == 0 ? 0 : DSR_ERR_ARG;
  if (!a.table || !a.offsets || !a.kv_lengths || !a.status || !a.k_cache || !a.v_cache ||
      (a.tokens > 0 && (!a.q || !a.out)))
    return DSR_ERR_ARG;
  if (!aligned16(a.q) || !aligned16(a.out) || !aligned16(a.k_cache) || !aligned16(a.v_cache)) return DSR_ERR_ARG;
  for (int64_t st : {a.q_token, a.q_head, a.out_token, a.out_head, a.k_block, a.k_token, a.k_head, a.v_block,
                     a.v_token, a.v_head})
    if (st % 8 != 0 || st < 0) return DSR_ERR_ARG;
  for (int64_t st : {a.k_block, a.k_token, a.v_block, a.v_token})
    if (st > INT_MAX) return DSR_ERR_ARG;  // multiplied in 32 x 32 bits
  AttnPlan p = attn_plan(a);
  const AttnSizes z = attn_sizes(a, p);
  if (!a.workspace || ((uintptr_t)a.workspace & 255u) || a.workspace_bytes < (size_t)z.all) return DSR_ERR_WORKSPACE;
  p.part_o = (float*)a.workspace;
  p.part_ml = (float2*)((char*)a.workspace + z.o);
  p.part_bad = (int32_t*)((char*)a.workspace + z.o + z.ml);
  hipStream_t s = (hipStream_t)stream;
  return a.dtype == DSR_BF16 ? attn_typed<__bf16>(a, p, s) : attn_typed<_Float16>(a, p, s);
}

int32_t dsr_commit_tree(const dsr_commit_args_t* args, void* stream) {
  if (!args) return DSR_ERR_ARG;
  const dsr_commit_args_t& a = *args;
  if (a.requests < 0 || a.requests > DSR_TREE_MAX_REQUESTS || a.tokens < 0 || a.tokens > INT_MAX ||
      !page_ok(a.page, a.blocks) || a.width < 1 || (int64_t)a.width * a.page > INT_MAX || a.table_ld < a.width ||
      a.cache_count < 0 || a.cache_count > 65535)
    return DSR_ERR_ARG;
  if (a.cache_count > 0 && (!a.caches == !a.host_caches || a.heads < 1 || a.heads > 65536 || a.row_bytes < 16 || a.row_bytes > 65536 ||
                            a.row_bytes % 16 != 0 || a.c_block % 16 != 0 || a.c_token % 16 != 0 || a.c_head % 16 != 0))
    return DSR_ERR_ARG;
  if (a.requests == 0) return 0;
  if (!a.offsets || !a.kv_lengths || !a.table || !a.output_limit || !a.path || !a.ids || !a.accepted || !a.count ||
      !a.pending || !a.stop || !a.lengths || !a.status || a.lengths == a.kv_lengths ||
      (a.tokens > 0 && (!a.parents || !a.tokens_in || !a.sampled)) || (a.eos_off && !a.eos_ids))
    return DSR_ERR_ARG;
  // What was so before the step is read by every workgroup of a request, and one of them writes what is so after it.
  if (!a.lengths_in != !a.pending_in || !a.lengths_in != !a.plan_status)
    return DSR_ERR_ARG;
  if (a.lengths_in && (a.lengths == a.lengths_in || a.pending == a.pending_in || a.status == a.plan_status))
    return DSR_ERR_ARG;
  const int per = commit_caches(a);
  auto grid = [&](int count) { return dim3((unsigned)a.requests, count > 0 ? (unsigned)((count + per - 1) / per) : 1u); };
  hipStream_t s = (hipStream_t)stream;
  if (!a.host_caches || a.cache_count == 0) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_commit_tree<0>), grid(a.cache_count), dim3(kCommitThreads), 0, s, a,
                       CommitCaches<0>{});
    return launched();
  }
  // Each launch decides anew: its inputs are no launch's outputs.
  for (int first = 0; first < a.cache_count; first += kCommitInline) {
    dsr_commit_args_t part = a;
    CommitCaches<kCommitInline> caches;
    part.cache_count = a.cache_count - first < kCommitInline ? a.cache_count - first : kCommitInline;
    for (int c = 0; c < kCommitInline; ++c) caches.at[c] = c < part.cache_count ? a.host_caches[first + c] : nullptr;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_commit_tree<kCommitInline>), grid(part.cache_count), dim3(kCommitThreads), 0, s,
                       part, caches);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  }
  return 0;
}

}  // extern "C"
