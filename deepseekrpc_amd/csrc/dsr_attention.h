// Attention of a step's new tokens over a paged cache (dsr_tree_attention).
//
// For one request and key head the rows are (new token, query head of the
// group) pairs: rows = new x group.  They share the head's keys and values, so
// a workgroup takes a tile of rows and reads each key and value once for all
// of them.  How tiles and tokens are dealt out is at AttnWork.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dsr_tree.h"

namespace dsr {

typedef float attn_f32x4 __attribute__((ext_vector_type(4)));

// Rows of bf16 or f16: vector types and matrix products.
template <class T>
struct AttnType;
template <>
struct AttnType<__bf16> {
  typedef __bf16 x4 __attribute__((ext_vector_type(4)));
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExponent = 0x7F80u;  // all ones: infinity or NaN
  static constexpr float kLift = 0.f;
  static __device__ __forceinline__ attn_f32x4 mfma16(x8 a, x8 b, attn_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct AttnType<_Float16> {
  typedef _Float16 x4 __attribute__((ext_vector_type(4)));
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  static constexpr uint32_t kExponent = 0x7C00u;
  // Weights are 2^7 times larger (at most 2^15), so that those of a long
  // context's many small terms keep their bits: f16 has no normal number
  // below 2^-14.
  static constexpr float kLift = 7.f;
  static __device__ __forceinline__ attn_f32x4 mfma16(x8 a, x8 b, attn_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// Transposing LDS read: of the 16 lanes of a group, lane i points at four
// elements of row i / 4 (columns 4 (i % 4) ...) of a 4 x 16 block and gets the
// four rows' elements of column i.
template <class T>
__device__ __forceinline__ typename AttnType<T>::x4 attn_read_tr(const T* p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(typename AttnType<T>::x4,
                            __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = 4;
constexpr int kAttnTile = 32;             // tokens a wave takes at a time
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// What the host decides for one call.
struct AttnPlan {
  int tile_rows;      // rows of a tile, a power of two
  int tile_shift, token_shift, page_shift, group_shift;  // their logarithms; -1: not a power of two
  int group;          // query heads per key head
  int groups;         // workgroups, a multiple of 8
  int tokens;         // of a step of the work split: a power of two times the kernel's own
  int min_steps;      // fewest steps worth a workgroup
  bool cut;           // some tile may be cut into parts
  float* part_o;      // [2 groups, tile_rows, head dim of the kernel]
  float2* part_ml;    // [2 groups, tile_rows]: base (log2) and sum
  int32_t* part_bad;  // [2 groups]: a page id outside the cache
};

// The kernels' argument, read anew where a part of it begins: kept in
// scalar registers from its start to its end they would not fit, and a third
// of the few-row kernel's instructions were moves of spilled ones.
struct AttnCall {
  dsr_tree_attention_args_t a;
  AttnPlan p;
};
__device__ __forceinline__ const AttnCall& attn_call() {
  typedef const AttnCall __attribute__((address_space(4))) * Args;
  Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(args));
  return *(const AttnCall*)args;
}

struct AttnRequest {
  int lo, n, kv;  // first new token, new tokens, cached tokens (0: nothing to read)
  int rows, tiles;
  bool fine;
};

// A row's token among the request's new ones.
__device__ __forceinline__ int attn_token(const AttnPlan& p, int row) {
  return p.group_shift >= 0 ? row >> p.group_shift : row / p.group;
}

__device__ __forceinline__ AttnRequest attn_request(const dsr_tree_attention_args_t& a, const AttnPlan& p, int r) {
  AttnRequest q;
  int lo = a.offsets[r], hi = a.offsets[r + 1];
  const int N = (int)a.tokens;
  lo = lo < 0 ? 0 : lo > N ? N : lo;
  hi = hi < lo ? lo : hi > N ? N : hi;
  q.lo = lo;
  q.n = hi - lo;
  const int kv = a.kv_lengths[r];
  q.fine = kv >= q.n && kv <= (int64_t)a.width * a.page && !(a.visible && q.n > DSR_TREE_MAX_NODES);
  q.rows = q.n * p.group;
  q.kv = q.fine && q.n > 0 ? kv : 0;
  q.tiles = q.rows > p.tile_rows ? (q.rows + p.tile_rows - 1) >> p.tile_shift : 1;
  return q;
}

// Inclusive sums over the lanes of a wave, without LDS (row shifts, then the
// rows' last lanes handed on).  Sums stop at 2^31 - 1.
__device__ __forceinline__ int attn_wave_scan(int x) {
  x = __builtin_elementwise_add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = __builtin_elementwise_add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = __builtin_elementwise_add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = __builtin_elementwise_add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = __builtin_elementwise_add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  x = __builtin_elementwise_add_sat(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return x;
}

// One segment of a workgroup's work: the rows of a tile against tokens begin .. end - 1.
struct AttnSegment {
  int r, head, tile, begin, end;
  bool whole;         // all of the tile's tokens
  int part;           // else: where its result goes
  uint32_t from, to;  // the tile's place in the order of all steps
};

// A workgroup's share of the work.
//
// All work is put in one order of steps (p.tokens tokens of a tile): request
// by request, head by head, tile by tile, token by token.  Each workgroup
// takes an equal, contiguous part of it, so that requests of any lengths
// load the chip evenly; a tile that crosses a border is written in parts,
// which k_tree_join joins.  (Joining in this launch, by the workgroup that
// finishes a tile last, needs the parts made visible across the XCDs' caches:
// with the fences for that, 32 requests of 8,064 tokens and 128 rows took
// 447 us instead of 274.)  Every wave finds the place for itself from the
// requests' lengths, 64 at a time.  Neighbouring shares, which often have
// keys and values in common, go to one XCD.
// The host chooses p.tokens so that the steps of a call number less than 2^31.
// HOLD: each lane keeps its request of the 64 looked at last (for kernels with
// registers to spare), else a segment's request is read again.
template <bool HOLD>
struct AttnWork {
  uint32_t at, stop, quota;  // steps
  uint32_t base;             // steps of the requests before r
  int r, me;
  int r0;                    // lane l holds request r0 + l:
  AttnRequest mine;

  __device__ __forceinline__ int steps_of(const AttnPlan& p, const AttnRequest& q) {
    return q.rows == 0 ? 0 : q.kv > p.tokens ? (q.kv + p.tokens - 1) >> p.token_shift : 1;
  }

  // Steps of the lane's request of the 64 from `first` on.
  __device__ __forceinline__ int hold(const dsr_tree_attention_args_t& a, const AttnPlan& p, int first) {
    const int l = threadIdx.x & 63, R = (int)a.requests;
    r0 = first;
    mine = attn_request(a, p, first + l < R ? first + l : R - 1);
    return first + l < R ? mine.tiles * steps_of(p, mine) * a.kv_heads : 0;
  }

  // `border` 0: this workgroup's share.  Else the work from where share `border` begins.
  __device__ __forceinline__ AttnWork(const dsr_tree_attention_args_t& a, const AttnPlan& p, int border) {
    const int R = (int)a.requests;
    int upto = 0, steps = 0;
    uint32_t total = 0;
    for (int first = 0; first < R; first += 64) {
      steps = hold(a, p, first);
      upto = attn_wave_scan(steps);
      total += (uint32_t)__builtin_amdgcn_readlane(upto, 63);
      // Requests without rows have no work: the first workgroup tells their status.
      const int l = threadIdx.x & 63;
      if (blockIdx.x == 0 && border == 0 && threadIdx.x < 64 && first + l < R && mine.rows == 0)
        a.status[first + l] = mine.fine ? DSR_OK : DSR_E_LENGTH;
    }
    // Most calls of one step per tile have a workgroup for each: no division then.
    quota = total <= (uint32_t)p.groups ? 1 : (total + p.groups - 1) / (uint32_t)p.groups;
    if (quota < (uint32_t)p.min_steps) quota = p.min_steps;
    const uint32_t each = quota == 1 ? (total + 7) / 8 : (total + 8 * quota - 1) / (8 * quota);  // workgroups, per XCD
    if (border == 0) {
      me = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
      at = (blockIdx.x >> 3) < each ? me * quota : total;
    } else {
      me = border;
      at = (uint32_t)border < 8 * each ? border * quota : total;
    }
    stop = at + quota < total ? at + quota : total;
    r = R;
    base = 0;
    if (at >= stop) return;
    for (int first = 0; first < R; first += 64) {
      if (R > 64) {
        steps = hold(a, p, first);
        upto = attn_wave_scan(steps);
      }
      const uint64_t past = __ballot(base + (uint32_t)upto > at);
      if (past) {
        const int hit = __ffsll((unsigned long long)past) - 1;
        base += (uint32_t)__builtin_amdgcn_readlane(upto - steps, hit);
        r = first + hit;
        return;
      }
      base += (uint32_t)__builtin_amdgcn_readlane(upto, 63);
    }
  }

  // The next segment and its request; false at the end.
  __device__ __forceinline__ bool next(const dsr_tree_attention_args_t& a, const AttnPlan& p, AttnSegment& s,
                                       AttnRequest& q) {
    if (at >= stop) return false;
    uint32_t steps, length;
    for (;;) {  // past requests that end here or have no rows
      if (r >= a.requests) return false;
      if (!HOLD || r - r0 >= 64) {
        r0 = r;
        mine = attn_request(a, p, HOLD && r + (int)(threadIdx.x & 63) < a.requests ? r + (threadIdx.x & 63) : r);
      }
      const int l = r - r0;
      q.lo = __builtin_amdgcn_readlane(mine.lo, l);
      q.n = __builtin_amdgcn_readlane(mine.n, l);
      q.kv = __builtin_amdgcn_readlane(mine.kv, l);
      q.rows = __builtin_amdgcn_readlane(mine.rows, l);
      q.tiles = __builtin_amdgcn_readlane(mine.tiles, l);
      q.fine = __builtin_amdgcn_readlane((int)mine.fine, l);
      steps = steps_of(p, q);
      length = q.tiles * steps * a.kv_heads;
      if (at - base < length) break;
      base += length;
      ++r;
    }
    const uint32_t unit = steps == 1 ? at - base : (at - base) / steps, s0 = at - base - unit * steps;
    const uint32_t s1 = stop - at < steps - s0 ? s0 + stop - at : steps;
    s.r = r;
    s.head = q.tiles == 1 ? unit : unit / (uint32_t)q.tiles;
    s.tile = unit - (uint32_t)s.head * q.tiles;
    if (!p.cut && !a.visible) s.tile = q.tiles - 1 - s.tile;  // a chunk's longest tiles first
    s.begin = s0 * p.tokens;
    s.end = s1 == steps ? q.kv : s1 * p.tokens;
    if (!a.visible && q.kv > 0) {  // causal rows: nothing past the tile's last one
      const int last = attn_token(p, (s.tile + 1) * p.tile_rows - 1);
      if (s.end - (q.kv - q.n) > last + 1) s.end = q.kv - q.n + last + 1;
    }
    s.whole = s0 == 0 && s1 == steps;
    s.part = 2 * me + (s0 > 0 ? 0 : 1);  // a tile begun elsewhere can only be a workgroup's first
    s.from = base + unit * steps;
    s.to = s.from + steps;
    at += s1 - s0;
    return true;
  }
};

// Rows of no request, before the first one's and past the last one's, give 0
// and -inf.  The workgroups past p.groups take them in turn: looked for by the
// workgroups that have shares, they cost every small call 0.2 us of 8.5.
template <class T>
__device__ __forceinline__ void attn_clear(int groups, int threads) {
  typedef typename AttnType<T>::x8 x8;
  const dsr_tree_attention_args_t& a = attn_call().a;
  const int N = (int)a.tokens, lo = a.offsets[0], hi = a.offsets[a.requests];
  const int lead = lo < 0 ? 0 : lo > N ? N : lo, rest = hi < lead ? lead : hi > N ? N : hi;
  const int none = lead + N - rest, chunks = a.head_dim / 8;
  for (int i = blockIdx.x - groups; i < none; i += gridDim.x - groups) {
    const int64_t t = i < lead ? i : rest + i - lead;
    for (int x = threadIdx.x; x < a.q_heads * chunks; x += threads) {
      const int h = x / chunks, d = x - h * chunks;
      *(x8*)((T*)a.out + t * a.out_token + h * a.out_head + 8 * d) = x8{};
      if (a.lse && d == 0) a.lse[t * a.q_heads + h] = -INFINITY;
    }
  }
}

// v with 0 in the place of infinities and NaN; whether there were any.
template <class T>
__device__ __forceinline__ bool attn_make_finite(typename AttnType<T>::x8& v) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 w = __builtin_bit_cast(u32x4, v);
  constexpr uint32_t E = AttnType<T>::kExponent;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = (w[i] & E) == E, hi = ((w[i] >> 16) & E) == E;
    bad |= lo || hi;
    w[i] = w[i] & ((lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u));
  }
  v = __builtin_bit_cast(typename AttnType<T>::x8, w);
  return bad;
}

// Infinities and NaN among values that some row must not see were taken out
// of the products (0 x infinity would be NaN).  Here, after the workgroup's
// results are written, the rows that do see such a value get weight x value
// added in memory: what they hold becomes infinite or NaN as the sum would
// have.  Adding a term that was in the product already changes nothing, so the
// tokens from `from` on are all looked at.  A thread takes a row; `base` is
// its scores' base.  Nothing of this runs for ordinary values.
template <class T, int DP>
__device__ __forceinline__ void attn_poison(const dsr_tree_attention_args_t& a, const AttnPlan& p, const AttnSegment& u,
                                            const AttnRequest& q, int from, const float* base) {
  typedef typename AttnType<T>::x8 x8;
  const int r = threadIdx.x, row = u.tile * p.tile_rows + r, group = p.group, ctx = q.kv - q.n;
  if (r >= p.tile_rows || row >= q.rows) return;
  const int t = attn_token(p, row), h = u.head * group + row - t * group;
  const T* query = (const T*)a.q + (int64_t)(q.lo + t) * a.q_token + (int64_t)h * a.q_head;
  T* out = (T*)a.out + (int64_t)(q.lo + t) * a.out_token + (int64_t)h * a.out_head;
  float* o = &p.part_o[((int64_t)u.part * p.tile_rows + r) * DP];
#pragma unroll 1
  for (int at = from; at < u.end; ++at) {
    const int id = a.table[u.r * a.table_ld + (at >> p.page_shift)], place = at & (a.page - 1);
    if ((unsigned)id >= (unsigned)a.blocks) continue;
    const T* v = (const T*)a.v_cache + id * a.v_block + place * a.v_token + u.head * a.v_head;
    const T* k = (const T*)a.k_cache + id * a.k_block + place * a.k_token + u.head * a.k_head;
    const int j = at - ctx;
    if (j >= 0 && !(a.visible ? a.visible[q.lo + t] >> j & 1 : j <= t)) continue;
    float weight = -1.f;
#pragma unroll 1
    for (int d = 0; d < a.head_dim; d += 8) {
      x8 x = *(const x8*)(v + d);
      const x8 whole = x;
      if (!attn_make_finite<T>(x)) continue;
      if (weight < 0.f) {  // this row's weight of the token, once
        float dot = 0.f;
#pragma unroll 1
        for (int i = 0; i < a.head_dim; ++i) dot += (float)query[i] * (float)k[i];
        weight = __builtin_amdgcn_exp2f(dot * a.scale * kLog2e - base[r]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if ((float)x[i] == (float)whole[i]) continue;
        if (!u.whole)
          o[d + i] += weight * (float)whole[i];
        else
          out[d + i] = (T)((float)out[d + i] + weight * (float)whole[i]);
      }
    }
  }
}

// What a segment says of its page ids: the request's status, or its part's
// (its last tile of its first head speaks for all: causal tiles see all of the
// pages that the ones before them see).
__device__ __forceinline__ void attn_report(const dsr_tree_attention_args_t& a, const AttnPlan& p,
                                            const AttnSegment& u, const AttnRequest& q, int bad) {
  if (threadIdx.x != 0) return;
  if (!u.whole)
    p.part_bad[u.part] = bad;
  else if (u.head == 0 && u.tile == q.tiles - 1)
    a.status[u.r] = !q.fine ? DSR_E_LENGTH : bad ? DSR_E_BLOCK : DSR_OK;
}

__device__ __forceinline__ uint32_t attn_low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u;
}

// Which of the 32 tokens from place p0 on a row sees, a bit each: the
// context, of the new tokens those of `mask` (or, without masks, those up to
// the row's own token `tok`), none at or past `end`, none of `bad`.
__device__ __forceinline__ uint32_t attn_sees(bool masks, uint64_t mask, int tok, int p0, int ctx, int end,
                                              uint32_t bad) {
  const int s = p0 - ctx;  // the first token's index among the new ones
  uint32_t see;
  if (masks)
    see = attn_low_bits(-s) | (uint32_t)(s >= 64 || s <= -32 ? 0ull : s >= 0 ? mask >> s : mask << -s);
  else
    see = attn_low_bits(tok + 1 - s);
  return see & attn_low_bits(end - p0) & ~bad;
}

// Few rows (16 of a tile): the waves take the segment's 32-token tiles in
// turn, each for itself, and join their results at the end.
//
// S^T = K Q^T and O^T = V^T P^T, so that a lane holds one row's scores (row
// lane % 16) and outputs: statistics and rescaling stay in the lane, and the
// scores are the second product's operand as they lie, with the k index of
// both operands permuted alike (lane group g takes tokens 4 g + i and
// 16 + 4 g + i).  Keys and values pass through the wave's own LDS rows, from
// which the transposing read hands each lane four tokens of a value's
// dimension.  The next tile's keys and values are in flight while a tile is
// worked on, and no wave waits for another.
//
// The running maximum is raised only when a score passes it by 8 (log2): the
// weights then stay below 2^8, far inside every type's range, and most tiles
// need no rescaling.
//
// WAVES: eight where fewer than 128 workgroups take whole short contexts and
// their latency counts (a request of 64 query heads over 500 tokens: 11.9 us
// with eight, 12.8 with four), else four (from 16 requests on the same to
// 0.2 us).
//
// What bounds it: the cache's read.  64 requests of one token over 8,192
// tokens, 8 heads of 128: 370 us, 5.8 TB/s.
template <class T, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, DP <= 128 || WAVES > 4 ? 2 : 1) void k_tree_attention(AttnCall) {
  constexpr int kThreads = 64 * WAVES;
  typedef typename AttnType<T>::x4 x4;
  typedef typename AttnType<T>::x8 x8;
  constexpr int KS = DP / 32;   // k steps of the score product
  constexpr int DB = DP / 16;   // 16-wide output blocks
  constexpr int VS = DP + 16;   // LDS row of values: 32 bytes of padding spread the transposing reads over the banks
  __shared__ __align__(16) T keys[WAVES][kAttnTile][DP + 8];  // 16 bytes of padding for the 16-byte reads of 16 keys
  __shared__ __align__(16) T vals[WAVES][kAttnTile][VS];
  __shared__ float sm[WAVES][16], sl[WAVES][16];
  __shared__ float sbase[16];
  __shared__ int sbad, spoison;  // a page id outside the cache; a value left out (attn_poison)

  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63, n = l & 15, g = l >> 4;
  if ((int)blockIdx.x >= attn_call().p.groups) return attn_clear<T>(attn_call().p.groups, kThreads);
  AttnWork<DP <= 128> work(attn_call().a, attn_call().p, 0);
  AttnSegment u;
  AttnRequest q;
  while (work.next(attn_call().a, attn_call().p, u, q)) {  // the same for the whole workgroup
    const dsr_tree_attention_args_t& a = attn_call().a;
    const AttnPlan& p = attn_call().p;
    const int group = p.group, dim = a.head_dim, row_shift = p.tile_shift;
    __syncthreads();  // the last segment's LDS is read
    if (threadIdx.x == 0) sbad = spoison = 0;
    const int ctx = q.kv - q.n, begin = u.begin, end = u.end;
    const int row0 = u.tile << row_shift;

    attn_f32x4 acc[DB];
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = attn_f32x4{};
    const dsr_tree_attention_args_t& c = attn_call().a;
    const int32_t* pages = c.table + u.r * c.table_ld;
    const T* kb = (const T*)c.k_cache + u.head * c.k_head;
    const T* vb = (const T*)c.v_cache + u.head * c.v_head;
    const int shift = attn_call().p.page_shift, page = c.page;
    const unsigned blocks = c.blocks;
    const uint32_t k_block = c.k_block, k_token = c.k_token, v_block = c.v_block, v_token = c.v_token;
    const bool masks = c.visible != nullptr;
    bool any_bad = false;

    // Tiles of this wave: 32 tokens from begin + 32 (WAVES i + w) on.  LPR lanes
    // read a token's row, 16 bytes each side by side (lanes next to each other
    // on different rows, as the product wants them, would take a cache access
    // each: 16 bytes a cycle and CU in place of 64), and each of them NI tokens
    // in a row, which share a page unless it is smaller.  Places past the last
    // token read the last token (their scores are masked).
    constexpr int LPR = DP / 8 <= 8 ? 8 : DP / 8 <= 16 ? 16 : 32;
    constexpr int NI = kAttnTile / (64 / LPR);
    const int sub = l / LPR * NI, chunk = 8 * (l & (LPR - 1)), d0 = min(chunk, dim - 8);
    const bool stores = chunk < DP;  // 192 dimensions: 24 of 32 lanes
    const bool tiny = page < NI;   // several pages: their ids are read with the rows
    int id_next = 0;
    uint32_t bad_next = 0;
    x8 kr[NI], vr[NI];
    auto load_id = [&](int p0) __attribute__((always_inline)) { id_next = pages[min(p0 + sub, end - 1) >> shift]; };
    auto load_rows = [&](int p0) __attribute__((always_inline)) {
      bad_next = 0;
      auto load = [&](int i, int id, int place) __attribute__((always_inline)) {
        const uint32_t at = (unsigned)id < blocks ? id : 0, in = place & (page - 1);
        kr[i] = *(const x8*)(kb + d0 + ((uint64_t)at * k_block + (uint64_t)in * k_token));
        vr[i] = *(const x8*)(vb + d0 + ((uint64_t)at * v_block + (uint64_t)in * v_token));
      };
      if (!tiny) {
        const bool outside = (unsigned)id_next >= blocks;
        const uint64_t bad = __ballot(outside);
        if (bad)
#pragma unroll
          for (int j = 0; j < 64 / LPR; ++j)
            if (bad >> (j * LPR) & 1) bad_next |= ((1u << NI) - 1u) << (NI * j);
        if (p0 + kAttnTile <= end) {
          const uint32_t at = outside ? 0 : id_next, in = (p0 + sub) & (page - 1);
          const T* k = kb + d0 + ((uint64_t)at * k_block + (uint64_t)in * k_token);
          const T* v = vb + d0 + ((uint64_t)at * v_block + (uint64_t)in * v_token);
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            kr[i] = *(const x8*)k;
            vr[i] = *(const x8*)v;
            k += k_token;
            v += v_token;
          }
        } else {
#pragma unroll
          for (int i = 0; i < NI; ++i) load(i, id_next, min(p0 + sub + i, end - 1));
        }
      } else {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int place = min(p0 + sub + i, end - 1), id = pages[place >> shift];
          const uint64_t bad = __ballot((unsigned)id >= blocks);
#pragma unroll
          for (int j = 0; j < 64 / LPR; ++j) bad_next |= (uint32_t)(bad >> (j * LPR) & 1) << (NI * j + i);
          load(i, id, place);
        }
      }
    };
    const int first = begin + kAttnTile * w, step = kAttnTile * WAVES;
    if (first < end) {
      load_id(first);
      load_rows(first);
      load_id(first + step);
    }
    // This lane's rows: token index, mask, query operand.  A negative scale
    // changes the queries' sign, so that scores only grow with their products;
    // scale 0 is queries of 0.
    const float scale = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
    x8 qv[KS];
    const bool in = row0 + n < q.rows;
    const int tok = in ? attn_token(p, row0 + n) : 0, head = in ? row0 + n - tok * group : 0;
    const uint64_t mask = in && a.visible ? a.visible[q.lo + tok] : 0;
    const T* src = (const T*)a.q + (int64_t)(q.lo + tok) * a.q_token + (int64_t)(u.head * group + head) * a.q_head;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 32 * s + 8 * g;
      const x8 v = in && d < dim && a.scale != 0.f ? *(const x8*)(src + d) : x8{};
      qv[s] = a.scale < 0.f ? -v : v;
    }
    __syncthreads();  // the flags
    for (int p0 = first; p0 < end; p0 += step) {
      const uint32_t bad = bad_next;
      const bool masked = p0 + kAttnTile > ctx || bad;  // some row may not see some token
      any_bad |= bad != 0;
      if (masked) {
        bool poison = false;
#pragma unroll
        for (int i = 0; i < NI; ++i) poison |= attn_make_finite<T>(vr[i]);
        if (poison) spoison = 1;
      }
      // Keys and values to the wave's LDS rows; then the next tile's loads.
      __builtin_amdgcn_wave_barrier();
      if (DP == 8 * LPR || stores) {
        if (chunk >= dim)  // dimensions past the head's
#pragma unroll
          for (int i = 0; i < NI; ++i) kr[i] = x8{};
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          *(x8*)&keys[w][sub + i][chunk] = kr[i];
          *(x8*)&vals[w][sub + i][chunk] = vr[i];
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (p0 + step < end) {
        load_rows(p0 + step);
        load_id(p0 + 2 * step);
      }
      // Scores.
      attn_f32x4 sc[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) sc[k] = attn_f32x4{};
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const x8 key = *(const x8*)&keys[w][16 * k + n][32 * s + 8 * g];
          sc[k] = AttnType<T>::mfma16(key, qv[s], sc[k]);
        }
      // Softmax.  A lane's scores: tokens p0 + 16 k + 4 g + e of its row.
      x8 pv;
      float top = -INFINITY;
      if (masked) {
        const uint32_t see = attn_sees(masks, mask, tok, p0, ctx, end, bad) >> (4 * g);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[k][e] = see >> (16 * k + e) & 1 ? sc[k][e] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, sc[k][e]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32)) * scale - AttnType<T>::kLift;
      if (__ballot(top > m + 8.f)) {
        const float next = fmaxf(m, top);
        const float f = m == next ? 1.f : __builtin_amdgcn_exp2f(m - next);
        m = next;
        sum *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] *= f;
      }
      const float base = m == -INFINITY ? 0.f : -m;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[k][e], scale, base));
          sum += x;
          pv[4 * k + e] = (T)x;
        }
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const T* at = &vals[w][4 * g + (n >> 2)][16 * d + 4 * (n & 3)];
        const x4 lo = attn_read_tr<T>(at), hi = attn_read_tr<T>(at + 16 * VS);
        const x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        acc[d] = AttnType<T>::mfma16(v, pv, acc[d]);
      }
    }

    // The waves' results: statistics, then the rows.
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (g == 0) sm[w][n] = m;
    if (any_bad && l == 0) sbad = 1;
    __syncthreads();
    const AttnCall& e = attn_call();
    const bool split = !u.whole;
    const int64_t part = u.part;
    constexpr int OS = DP + 4;  // LDS row of outputs
    static_assert(16 * OS * sizeof(float) <= kAttnTile * VS * sizeof(T), "a wave's outputs fit its rows of values");
    float top = sm[0][n];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) top = fmaxf(top, sm[i][n]);
    const float f = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);  // a wave without tokens: 0
    if (g == 0) sl[w][n] = sum * f;
    if (w == 0 && g == 0) sbase[n] = top;
    float* mine = (float*)&vals[w][0][0];
#pragma unroll
    for (int d = 0; d < DB; ++d) *(attn_f32x4*)&mine[n * OS + 16 * d + 4 * g] = acc[d] * f;
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * (DP / 4); x += kThreads) {
      const int row = x / (DP / 4), d = x % (DP / 4) * 4;
      const float M = sbase[row];
      float L = 0.f;
      attn_f32x4 o = {};
#pragma unroll
      for (int i = 0; i < WAVES; ++i) {
        L += sl[i][row];
        o += *(const attn_f32x4*)((const float*)&vals[i][0][0] + row * OS + d);
      }
      if (split) {
        *(attn_f32x4*)&e.p.part_o[(((int64_t)part << row_shift) + row) * DP + d] = o;
        if (d == 0) e.p.part_ml[((int64_t)part << row_shift) + row] = float2{M, L};
      } else if (row0 + row < q.rows && d < dim) {
        const int t = attn_token(e.p, row0 + row), head = u.head * group + row0 + row - t * group;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (T)(o[i] * inv);
        *(x4*)((T*)e.a.out + (int64_t)(q.lo + t) * e.a.out_token + (int64_t)head * e.a.out_head + d) = y;
        if (e.a.lse && d == 0)
          e.a.lse[(int64_t)(q.lo + t) * e.a.q_heads + head] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
      }
    }
    __threadfence_block();
    __syncthreads();
    if (spoison) attn_poison<T, DP>(e.a, e.p, u, q, sbad ? begin : max(begin, min(ctx, end) - kAttnTile), sbase);
    attn_report(e.a, e.p, u, q, sbad);
  }
}

// Joins the parts of the tiles that borders between shares cut:
// out = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c.  Workgroup (x, y) takes
// rows JR y .. of the tile whose first border is the one before share x + 1.
// Few rows leave threads over: these take every SLOTS-th part each (a single
// long request has a part for each of 64 shares), summed in a fixed order.
// One pass with a running maximum: a part's outputs are not waited for behind
// all parts' maxima (a single request over 1,001 tokens 14.4 us a call, so 13.8).
// What bounds it: the call's second launch, and the parts' way through the
// caches (5 us of that call's 14; 67 MB in 22 us for 512 shares of 128 rows).
template <class T, int DP, int JR>
__global__ __launch_bounds__(kAttnThreads) void k_tree_join(AttnCall) {
  typedef typename AttnType<T>::x4 x4;
  constexpr int E = JR * DP / 4;  // four dimensions of a row each
  constexpr int SLOTS = E < kAttnThreads ? kAttnThreads / E : 1;
  __shared__ float sm[SLOTS][JR], sl[SLOTS][JR];
  __shared__ attn_f32x4 so[SLOTS][SLOTS > 1 ? E : 1];
  const int border = blockIdx.x + 1;
  AttnWork<true> work(attn_call().a, attn_call().p, border);
  AttnSegment u;
  AttnRequest q;
  const uint32_t at = work.at;
  if (!work.next(attn_call().a, attn_call().p, u, q) || u.from == at) return;  // no work there; a tile begins there
  const int first = u.from / work.quota, last = (u.to - 1) / work.quota;
  if (first != border - 1) return;
  const dsr_tree_attention_args_t& a = attn_call().a;
  const AttnPlan& p = attn_call().p;
  const int row0 = u.tile << p.tile_shift, slot = SLOTS > 1 ? threadIdx.x / E : 0;
  const bool spare = slot >= SLOTS;  // 192 dimensions: 64 threads
  const int rows = min(p.tile_rows, q.rows - row0);
  if ((int)blockIdx.y * JR >= rows) return;
#pragma unroll
  for (int x = SLOTS > 1 ? threadIdx.x % E : threadIdx.x; x < E; x += kAttnThreads) {
    const int in = x / (DP / 4), row = blockIdx.y * JR + in, d = x % (DP / 4) * 4;
    // The first part is its workgroup's last (an odd place), the others their workgroups' first.
    auto part = [&](int c) { return ((int64_t)(2 * c + (c == first)) << p.tile_shift) + row; };
    float M = -INFINITY, L = 0.f;
    attn_f32x4 o = {};
    auto add = [&](float m, float l, attn_f32x4 x) {
      const float both = fmaxf(M, m), f = M == both ? 1.f : __builtin_amdgcn_exp2f(M - both);
      const float g = m == both ? 1.f : __builtin_amdgcn_exp2f(m - both);
      M = both;
      L = L * f + l * g;
      o = o * f + x * g;
    };
#pragma unroll 4
    for (int c = spare ? last + 1 : first + slot; c <= last; c += SLOTS) {
      const float2 ml = p.part_ml[part(c)];
      add(ml.x, ml.y, *(const attn_f32x4*)&p.part_o[part(c) * DP + d]);
    }
    if constexpr (SLOTS > 1) {
      if (!spare) so[slot][x] = o;
      if (d == 0 && !spare) {
        sm[slot][in] = M;
        sl[slot][in] = L;
      }
      __syncthreads();
      if (slot > 0) break;
#pragma unroll
      for (int i = 1; i < SLOTS; ++i) add(sm[i][in], sl[i][in], so[i][x]);
    }
    if (row >= rows || d >= a.head_dim) continue;
    const int t = attn_token(p, row0 + row), h = row0 + row - t * p.group;
    const float inv = L == 0.f ? 0.f : 1.f / L;
    x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (T)(o[i] * inv);
    *(x4*)((T*)a.out + (int64_t)(q.lo + t) * a.out_token + (int64_t)(u.head * p.group + h) * a.out_head + d) = y;
    if (a.lse && d == 0)
      a.lse[(int64_t)(q.lo + t) * a.q_heads + u.head * p.group + h] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
  }
  if (u.head == 0 && u.tile == q.tiles - 1 && blockIdx.y == 0 && threadIdx.x == 0) {
    int bad = 0;
    for (int c = first; c <= last; ++c) bad |= p.part_bad[2 * c + (c == first)];
    a.status[u.r] = !q.fine ? DSR_E_LENGTH : bad ? DSR_E_BLOCK : DSR_OK;
  }
}

}  // namespace dsr
