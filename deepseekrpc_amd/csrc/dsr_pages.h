// Pages that several rows hold: rows that continue other rows
// (dsr_fork_pages), and held pages moved to the front (dsr_compact_pages).
//
// Every decision is made from counts and prefix sums, so that no result
// depends on timing: pages are taken from the pool in row order and given
// back in ascending order, which a bit per page makes a matter of counting
// the bits before it.
//
// What bounds both, beside a few launches that each wait for the one before,
// is the moved rows of the caches, read and written once.
#pragma once

#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "dsr_branch.h"

namespace dsr {

constexpr int kPagesThreads = 256;
constexpr int kForkThreads = 1024;
constexpr int kBitsChunk = kPagesThreads;      // words of 32 pages that a workgroup counts
constexpr int kPagesInline = 128;              // caches whose pointers are a launch's arguments

typedef uint32_t pages_u32x4 __attribute__((ext_vector_type(4)));

template <int COUNT>
struct PagesCaches {
  void* at[COUNT];
};
template <>
struct PagesCaches<0> {};

// Tokens [0, tokens) of page `from` go to page `to`, in every cache.
struct PageCopy {
  int32_t from, to, tokens;
};

__host__ __device__ inline int64_t pages_words(int32_t blocks) { return ((int64_t)blocks + 31) / 32; }
__host__ __device__ inline int pages_chunks(int32_t blocks) {
  return (int)((pages_words(blocks) + kBitsChunk - 1) / kBitsChunk);
}

// A place in a ring: x < 2 size <= 2^31.
__device__ __forceinline__ int pages_wrap(int x, int size) { return x >= size ? x - size : x; }

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int pages_scan(int x) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int y = __shfl_up(x, s);
    if ((int)(threadIdx.x & 63) >= s) x += y;
  }
  return x;
}

// Sums over the workgroup's threads before this one and over all of them;
// `part` is LDS of a number a wave.
template <int THREADS>
__device__ __forceinline__ int pages_before(int x, int* part, int& all) {
  const int upto = pages_scan(x), w = threadIdx.x >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[w] = upto;
  __syncthreads();
  int before = upto - x;
  all = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    if (i < w) before += part[i];
    all += part[i];
  }
  return before;
}
__device__ __forceinline__ int pages_total(int x, int* part) {
  int all;
  pages_before<kPagesThreads>(x, part, all);
  return all;
}

// One page's tokens of one cache, by a workgroup.  Units of 16 bytes; the
// rows of a page that lies in one piece are one run.
struct PageShape {
  int32_t heads, row_bytes;
  int64_t c_block, c_token, c_head;
};
constexpr int kPagesFlight = 8;  // reads of a thread in flight
__device__ __forceinline__ void pages_copy(const PageShape& s, char* cache, const PageCopy& c) {
  const char* src = cache + c.from * s.c_block;
  char* dst = cache + c.to * s.c_block;
  // A page of a cache is less than 2^31 bytes.
  const uint32_t cols = s.row_bytes / 16, per = cols * s.heads, units = c.tokens * per;
  const bool flat = (s.heads == 1 || s.c_head == s.row_bytes) && (c.tokens == 1 || s.c_token == (int64_t)per * 16);
  auto offset = [&](uint32_t u) __attribute__((always_inline)) -> int64_t {
    if (flat) return (int64_t)u * 16;
    const uint32_t t = u / per, in = u - t * per, h = in / cols;
    return t * s.c_token + h * s.c_head + (in - h * cols) * 16;
  };
  for (uint32_t u = threadIdx.x; u < units; u += kPagesFlight * kPagesThreads) {
    pages_u32x4 v[kPagesFlight];
    int64_t at[kPagesFlight];
#pragma unroll
    for (int i = 0; i < kPagesFlight; ++i)
      if (u + i * kPagesThreads < units) {
        at[i] = offset(u + i * kPagesThreads);
        v[i] = *(const pages_u32x4*)(src + at[i]);
      }
#pragma unroll
    for (int i = 0; i < kPagesFlight; ++i)
      if (u + i * kPagesThreads < units) *(pages_u32x4*)(dst + at[i]) = v[i];
  }
}

// Items (copy, cache), a workgroup each in turn.  What bounds it: memory (224 copies
// of 63 tokens at most, 32 caches of 8 heads of 256 bytes: 516 MB written in 140 us,
// and the 74 MB of the sources' tails, which each of seven copies reads anew from the
// caches; whole pages of 64 tokens, 2.3 GB in 447 us, 5.1 TB/s).
template <int COUNT>
__device__ __forceinline__ void pages_copies(const PageShape& s, const PageCopy* copies, int count,
                                             void* const* device, const PagesCaches<COUNT>& caches, int cache_count,
                                             int group, int groups) {
  const int64_t items = (int64_t)count * cache_count;
  for (int64_t i = group; i < items; i += groups) {
    const int k = (int)(i / cache_count), c = (int)(i - (int64_t)k * cache_count);
    char* cache;
    if constexpr (COUNT > 0)
      cache = (char*)caches.at[c];
    else
      cache = (char*)device[c];
    pages_copy(s, cache, copies[k]);
  }
}

// ---------------------------------------------------------------------------
// Fork.

struct ForkRow {
  int32_t source;  // -1: the row is empty
  int32_t full;    // pages shared with its siblings
  int32_t pages;   // pages in all
  int32_t fresh;   // the page from the pool that comes behind the shared ones, with `copied`
  int32_t copied;
};
struct ForkHead {
  int32_t first, count, taken;  // the pool's first free entry, their number, pages taken
};
// a.workspace: head, rows, children of each source, copies, a bit per page that is freed.
struct ForkSpace {
  ForkHead* head;
  ForkRow* rows;
  int32_t* children;  // rows that continue a source; -1: its length or pages are out of bounds
  PageCopy* copies;
  uint32_t* freed;
};
__host__ __device__ inline int64_t fork_space(const dsr_fork_args_t& a, ForkSpace& s) {
  char* p = (char*)a.workspace;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* q = p + at;
    at += (bytes + 15) / 16 * 16;
    return q;
  };
  s.head = (ForkHead*)take(sizeof(ForkHead));
  s.rows = (ForkRow*)take(a.rows * sizeof(ForkRow));
  s.children = (int32_t*)take(a.sources * 4);
  s.copies = (PageCopy*)take(a.rows * sizeof(PageCopy));
  s.freed = (uint32_t*)take(pages_words(a.blocks) * 4);
  return at;
}

// What each row gets, by one workgroup of kForkThreads.  `heir` and `children`
// are LDS for a number a source.
__device__ __forceinline__ void fork_decide(const dsr_fork_args_t& a, const ForkSpace& space, int32_t* heir,
                                            int32_t* children) {
  __shared__ int part[kForkThreads / 64];
  __shared__ int taken;
  const int S = (int)a.sources, R = (int)a.rows;
  for (int s = threadIdx.x; s < S; s += kForkThreads) {
    heir[s] = INT_MAX;  // the first row that continues a source
    children[s] = 0;
  }
  if (threadIdx.x == 0) taken = 0;
  __syncthreads();
  for (int r = threadIdx.x; r < R; r += kForkThreads) {
    const int s = a.parents[r];
    if ((unsigned)s < (unsigned)S) atomicMin(&heir[s], r);
  }
  __syncthreads();
  const int shift = __ffs(a.page) - 1, size = a.pool_size;
  int head = a.pool_state[0], count = a.pool_state[1];
  if (head < 0 || head >= size || count < 0 || count > size) head = count = 0;  // not a pool: empty
  auto fine = [&](int length, int held) {
    return length >= 0 && (uint32_t)held <= (uint32_t)a.width && (uint32_t)length <= (uint32_t)held << shift;
  };
  int base = 0;  // pages wanted by the rows before these
  for (int r0 = 0; r0 < R; r0 += kForkThreads) {
    const int r = r0 + (int)threadIdx.x;
    int status = DSR_OK, s = r < R ? a.parents[r] : -1, length = 0, held = 0;
    if (s < -1 || s >= S) {
      status = DSR_E_PARENT;
      s = -1;
    }
    if (s >= 0) {
      length = a.lengths[s];
      held = a.held[s];
      if (!fine(length, held)) {
        status = DSR_E_LENGTH;
        s = -1;
      }
    }
    const bool first = s >= 0 && heir[s] == r;
    const int want = s >= 0 && !first && (length & (a.page - 1)) != 0;
    int all;
    const int upto = base + pages_before<kForkThreads>(want, part, all) + want;
    base += all;
    if (want && upto > count) {
      status = DSR_E_BLOCKS;
      s = -1;
    }
    if (r >= R) continue;  // no barrier is passed over: the others of the round have none left
    ForkRow row{s, 0, 0, -1, 0};
    if (s >= 0) {
      row.full = length >> shift;
      row.pages = first ? held : row.full + want;
      atomicAdd(&children[s], 1);
      if (want) {
        row.fresh = a.pool[pages_wrap(head + upto - 1, size)];
        row.copied = 1;
        const int from = a.table[s * a.table_ld + row.full];
        const bool in = (unsigned)from < (unsigned)a.blocks && (unsigned)row.fresh < (unsigned)a.blocks;
        if (!in) status = DSR_E_BLOCK;  // a page of its own, but not its tokens
        space.copies[upto - 1] = PageCopy{in ? from : 0, in ? row.fresh : 0, in ? length & (a.page - 1) : 0};
        atomicMax(&taken, upto);
      }
    }
    space.rows[r] = row;
    a.held_out[r] = row.pages;
    a.lengths_out[r] = s >= 0 ? length : 0;
    a.status[r] = status;
  }
  __syncthreads();
  for (int s = threadIdx.x; s < S; s += kForkThreads)
    space.children[s] = fine(a.lengths[s], a.held[s]) ? children[s] : -1;
  if (threadIdx.x == 0) *space.head = ForkHead{head, count, taken};
}

// One entry of a row's table; whether its page id is outside the cache.
__device__ __forceinline__ bool fork_entry(const dsr_fork_args_t& a, const ForkRow& row, int64_t r, int c) {
  int id = -1;
  if (c < row.pages) id = row.copied && c == row.full ? row.fresh : a.table[row.source * a.table_ld + c];
  a.table_out[r * a.table_out_ld + c] = id;
  return c < row.pages && (unsigned)id >= (unsigned)a.blocks;
}

// A source's page gains the rows that share it besides one, or loses its row.
// `freed` has a bit per page, which changes as often as the count passes 0: in
// the end it says whether the count is below, whatever the order of the sources
// (it matters where `shared` knows less holders than there are).
// Returns whether the page id is outside the cache.
__device__ __forceinline__ bool fork_count(const dsr_fork_args_t& a, int64_t s, int c, int children, int full,
                                           uint32_t* freed) {
  const int id = a.table[s * a.table_ld + c], change = c < full ? children - 1 : children > 0 ? 0 : -1;
  if ((unsigned)id >= (unsigned)a.blocks) return true;
  if (change != 0) {
    const int before = atomicAdd(&a.shared_out[id], change);
    if ((before < 0) != (before + change < 0)) atomicXor(&freed[id >> 5], 1u << (id & 31));
  }
  return false;
}

// A freed page to the pool, behind `at` others.
__device__ __forceinline__ void fork_free(const dsr_fork_args_t& a, const ForkHead& head, int id, int at) {
  const int size = a.pool_size, room = size - head.count + head.taken;
  a.shared_out[id] = 0;
  if (at < room) a.pool[pages_wrap(pages_wrap(head.first + head.count, size) + at, size)] = id;
}
__device__ __forceinline__ void fork_state(const dsr_fork_args_t& a, const ForkHead& head, int freed) {
  const int size = a.pool_size, room = size - head.count + head.taken;
  a.pool_state_out[0] = pages_wrap(head.first + head.taken, size);
  a.pool_state_out[1] = head.count - head.taken + (freed < room ? freed : room);
}

// Everything but the copies in one workgroup, for batches whose tables it goes
// over about as fast as the launches begin that it spares (entries of rows and
// sources, in one workgroup and in three launches: 1,024 7.9 and 8.9 us a call;
// 1,728 10.8 to 11.0, and 10.1 to 12.2 with how fast the host launches; 2,688 11.6
// and 9.7).
constexpr int kForkSmallRows = 1024, kForkSmallEntries = 2048, kForkSmallBlocks = 32 * kForkThreads;
__global__ __launch_bounds__(kForkThreads) void k_fork_small(dsr_fork_args_t a) {
  __shared__ int32_t heir[kForkSmallRows], children[kForkSmallRows];
  __shared__ uint32_t freed[kForkThreads];
  __shared__ int base[kForkThreads], part[kForkThreads / 64];
  ForkSpace space;
  fork_space(a, space);
  freed[threadIdx.x] = 0;
  if (a.shared_out != a.shared)
    for (int i = threadIdx.x; i < a.blocks; i += kForkThreads) a.shared_out[i] = a.shared[i];
  fork_decide(a, space, heir, children);
  __syncthreads();
  const uint32_t width = a.width, rows = (uint32_t)a.rows * width, all = rows + (uint32_t)a.sources * width;
  for (uint32_t s = threadIdx.x; s < a.sources; s += kForkThreads)
    a.source_status[s] = space.children[s] < 0 ? DSR_E_LENGTH : DSR_OK;
  const int shift = __ffs(a.page) - 1;
  bool outside = false;
  for (uint32_t e = threadIdx.x; e < all; e += kForkThreads) {
    const bool row = e < rows;
    const uint32_t in = row ? e : e - rows, r = in / width, c = in - r * width;
    if (row) {
      outside |= fork_entry(a, space.rows[r], r, c);
    } else {
      const int n = space.children[r];
      if (n >= 0 && (int)c < a.held[r]) outside |= fork_count(a, r, c, n, a.lengths[r] >> shift, freed);
    }
  }
  if (__syncthreads_or(outside))  // rare: their statuses, behind the ones that are written
    for (uint32_t e = threadIdx.x; e < all; e += kForkThreads) {
      const bool row = e < rows;
      const uint32_t in = row ? e : e - rows, r = in / width, c = in - r * width;
      if (row) {
        const int id = a.table_out[r * a.table_out_ld + c];
        if ((int)c < space.rows[r].pages && (unsigned)id >= (unsigned)a.blocks) a.status[r] = DSR_E_BLOCK;
      } else if (space.children[r] >= 0 && (int)c < a.held[r] &&
                 (unsigned)a.table[r * a.table_ld + c] >= (unsigned)a.blocks) {
        a.source_status[r] = DSR_E_BLOCK;
      }
    }
  int total;
  base[threadIdx.x] = pages_before<kForkThreads>(__popc(freed[threadIdx.x]), part, total);
  __syncthreads();
  const ForkHead head = *space.head;
  if (total > 0)
    for (int p = threadIdx.x; p < a.blocks; p += kForkThreads) {
      const uint32_t w = freed[p >> 5], bit = 1u << (p & 31);
      if (w & bit) fork_free(a, head, p, base[p >> 5] + __popc(w & (bit - 1)));
    }
  if (threadIdx.x == 0) fork_state(a, head, total);
}

// Larger batches: the first workgroup decides, the others clear the bits and
// copy the counts.
__global__ __launch_bounds__(kForkThreads) void k_fork_scan(dsr_fork_args_t a) {
  __shared__ int32_t heir[DSR_TREE_MAX_REQUESTS], children[DSR_TREE_MAX_REQUESTS];
  ForkSpace space;
  fork_space(a, space);
  if (blockIdx.x == 0) return fork_decide(a, space, heir, children);
  const int64_t step = (int64_t)(gridDim.x - 1) * kForkThreads, words = pages_words(a.blocks);
  const int64_t first = (int64_t)(blockIdx.x - 1) * kForkThreads + threadIdx.x;
  for (int64_t i = first; i < words; i += step) space.freed[i] = 0;
  if (a.shared_out != a.shared)
    for (int64_t i = first; i < a.blocks; i += step) a.shared_out[i] = a.shared[i];
}

// Table rows, a workgroup each; then the sources' pages gain and lose rows.
__global__ __launch_bounds__(kPagesThreads) void k_fork_rows(dsr_fork_args_t a) {
  ForkSpace space;
  fork_space(a, space);
  bool outside = false;
  if ((int64_t)blockIdx.x < a.rows) {
    const int64_t r = blockIdx.x;
    const ForkRow row = space.rows[r];
    for (int c = threadIdx.x; c < a.width; c += kPagesThreads) outside |= fork_entry(a, row, r, c);
    if (__syncthreads_or(outside) && threadIdx.x == 0) a.status[r] = DSR_E_BLOCK;
    return;
  }
  const int64_t s = (int64_t)blockIdx.x - a.rows;
  const int children = space.children[s];
  if (children >= 0) {
    const int full = a.lengths[s] / a.page, held = a.held[s];
    for (int c = threadIdx.x; c < held; c += kPagesThreads)
      outside |= fork_count(a, s, c, children, full, space.freed);
  }
  outside = __syncthreads_or(outside);
  if (threadIdx.x == 0) a.source_status[s] = children < 0 ? DSR_E_LENGTH : outside ? DSR_E_BLOCK : DSR_OK;
}

// Freed pages to the pool, a chunk of the bits a workgroup: each counts the
// bits before its own, then its threads take its pages, side by side.
__device__ __forceinline__ void fork_chunk(const dsr_fork_args_t& a, const ForkSpace& space, int chunk) {
  __shared__ int part[4], base[kBitsChunk];
  __shared__ uint32_t word[kBitsChunk];
  const int64_t words = pages_words(a.blocks), begin = (int64_t)chunk * kBitsChunk;
  int mine = 0, all;
  for (int64_t i = threadIdx.x; i < begin; i += kPagesThreads) mine += __popc(space.freed[i]);
  const int before = chunk > 0 ? pages_total(mine, part) : 0;
  const uint32_t bits = begin + threadIdx.x < words ? space.freed[begin + threadIdx.x] : 0;
  const ForkHead head = *space.head;
  word[threadIdx.x] = bits;
  base[threadIdx.x] = before + pages_before<kPagesThreads>(__popc(bits), part, all);
  __syncthreads();
  const int end = (int)(a.blocks - begin * 32 < kBitsChunk * 32 ? a.blocks - begin * 32 : kBitsChunk * 32);
  for (int p = threadIdx.x; p < end; p += kPagesThreads) {
    const uint32_t w = word[p >> 5], bit = 1u << (p & 31);
    if (w & bit) fork_free(a, head, (int)(begin * 32) + p, base[p >> 5] + __popc(w & (bit - 1)));
  }
  if (chunk == pages_chunks(a.blocks) - 1 && threadIdx.x == 0) fork_state(a, head, before + all);
}

// `chunks` workgroups free pages, the others copy.
template <int COUNT>
__global__ __launch_bounds__(kPagesThreads) void k_fork_finish(dsr_fork_args_t a, PagesCaches<COUNT> caches,
                                                               int chunks) {
  ForkSpace space;
  fork_space(a, space);
  if ((int)blockIdx.x < chunks) return fork_chunk(a, space, blockIdx.x);
  pages_copies<COUNT>(PageShape{a.heads, a.row_bytes, a.c_block, a.c_token, a.c_head}, space.copies,
                      space.head->taken, a.caches, caches, a.cache_count, blockIdx.x - chunks, gridDim.x - chunks);
}

// ---------------------------------------------------------------------------
// Compact.

struct CompactHead {
  int32_t refused;  // some row has a status
  int32_t limit;    // first page behind the held ones afterwards
  int32_t moves;
};
// a.workspace: head, a bit per held page, rank of each page that moves or is moved to, copies.
struct CompactSpace {
  CompactHead* head;
  uint32_t* held;
  int32_t* rank;
  PageCopy* copies;
};
__host__ __device__ inline int64_t compact_space(const dsr_compact_args_t& a, CompactSpace& s) {
  char* p = (char*)a.workspace;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* q = p + at;
    at += (bytes + 15) / 16 * 16;
    return q;
  };
  s.head = (CompactHead*)take(sizeof(CompactHead));
  s.held = (uint32_t*)take(pages_words(a.blocks) * 4);
  s.rank = (int32_t*)take((int64_t)a.blocks * 4);
  s.copies = (PageCopy*)take((int64_t)(a.blocks / 2 + 1) * sizeof(PageCopy));  // a move needs two pages
  return at;
}

__global__ __launch_bounds__(kPagesThreads) void k_compact_clear(dsr_compact_args_t a) {
  CompactSpace space;
  compact_space(a, space);
  const int64_t first = (int64_t)blockIdx.x * kPagesThreads + threadIdx.x;
  if (first == 0) *space.head = CompactHead{0, 0, 0};
  for (int64_t i = first; i < pages_words(a.blocks); i += (int64_t)gridDim.x * kPagesThreads) space.held[i] = 0;
}

// Rows, a workgroup each.
__global__ __launch_bounds__(kPagesThreads) void k_compact_mark(dsr_compact_args_t a) {
  __shared__ int outside;
  CompactSpace space;
  compact_space(a, space);
  const int64_t r = blockIdx.x;
  if (threadIdx.x == 0) outside = 0;
  __syncthreads();
  const int held = a.held[r];
  const bool fine = (uint32_t)held <= (uint32_t)a.width;
  const int32_t* pages = a.table + r * a.table_ld;
  bool bad = false;
  for (int c = threadIdx.x; fine && c < held; c += kPagesThreads) {
    const int id = pages[c];
    if ((unsigned)id >= (unsigned)a.blocks)
      bad = true;
    else
      atomicOr(&space.held[id >> 5], 1u << (id & 31));
  }
  if (bad) outside = 1;
  __syncthreads();
  if (threadIdx.x == 0) {
    a.status[r] = !fine ? DSR_E_LENGTH : outside ? DSR_E_BLOCK : DSR_OK;
    if (!fine || outside) space.head->refused = 1;
  }
}

// The pages from `lo` on and before `hi` that are among word i's 32, a bit each.
__device__ __forceinline__ uint32_t pages_range(int64_t i, int64_t lo, int64_t hi) {
  const int64_t a = lo - 32 * i, b = hi - 32 * i;
  const uint32_t from = a <= 0 ? ~0u : a >= 32 ? 0u : ~0u << a, to = b <= 0 ? 0u : b >= 32 ? ~0u : ~(~0u << b);
  return from & to;
}

// Which page moves where: the k-th held page from the limit on, to the k-th
// free one before it.  For the words `begin` .. of the bits, a word a thread, of
// which `held` is this thread's, behind `moved` and `open` pages of earlier
// words; returns the moves up to here.
template <int THREADS>
__device__ __forceinline__ int compact_moves(const dsr_compact_args_t& a, const CompactSpace& space, uint32_t held,
                                             int64_t begin, int64_t limit, int moved, int open) {
  __shared__ uint32_t from[THREADS], to[THREADS];
  __shared__ int from_base[THREADS], to_base[THREADS], part[THREADS / 64];
  const int x = threadIdx.x;
  int all, unused;
  from[x] = held & pages_range(begin + x, limit, a.blocks);
  to[x] = ~held & pages_range(begin + x, a.first, limit);
  from_base[x] = moved + pages_before<THREADS>(__popc(from[x]), part, all);
  to_base[x] = open + pages_before<THREADS>(__popc(to[x]), part, unused);
  __syncthreads();
  const int end = (int)(a.blocks - begin * 32 < THREADS * 32 ? a.blocks - begin * 32 : THREADS * 32);
  for (int p = x; p < end; p += THREADS) {
    const int w = p >> 5, id = (int)(begin * 32) + p;
    const uint32_t bit = 1u << (p & 31);
    if (from[w] & bit) {
      const int at = from_base[w] + __popc(from[w] & (bit - 1));
      space.rank[id] = at;
      space.copies[at].from = id;
    } else if (to[w] & bit) {
      const int at = to_base[w] + __popc(to[w] & (bit - 1));
      space.rank[id] = at;
      space.copies[at].to = id;
      space.copies[at].tokens = a.page;
    }
  }
  return moved + all;
}

__global__ __launch_bounds__(kPagesThreads) void k_compact_plan(dsr_compact_args_t a) {
  __shared__ int part[4];
  CompactSpace space;
  compact_space(a, space);
  const int64_t words = pages_words(a.blocks), begin = (int64_t)blockIdx.x * kBitsChunk;
  const int64_t first = a.first, blocks = a.blocks;
  int mine = 0;
  for (int64_t i = threadIdx.x; i < words; i += kPagesThreads)
    mine += __popc(space.held[i] & pages_range(i, first, blocks));
  const int64_t limit = first + pages_total(mine, part);
  int moved = 0, open = 0;  // held pages behind the limit, free ones before it
  for (int64_t i = threadIdx.x; i < begin; i += kPagesThreads) {
    const uint32_t held = space.held[i];
    moved += __popc(held & pages_range(i, limit, blocks));
    open += __popc(~held & pages_range(i, first, limit));
  }
  if (begin > 0) {
    moved = pages_total(moved, part);
    open = pages_total(open, part);
  }
  const uint32_t held = begin + threadIdx.x < words ? space.held[begin + threadIdx.x] : 0;
  const int moves = compact_moves<kPagesThreads>(a, space, held, begin, limit, moved, open);
  if (begin + kBitsChunk >= words && threadIdx.x == 0) {
    space.head->limit = (int32_t)limit;
    space.head->moves = space.head->refused ? 0 : moves;
  }
}

// Bits, statuses and moves of a small cache in one workgroup (table entries: 544
// 7.5 us a call, 10.9 in four launches; 8,032 13.7 and 19.3; 13,400 17.7 and 21.6;
// 26,800 the same).
constexpr int kCompactSmallEntries = 16384, kCompactSmallBlocks = 32 * kForkThreads;
__global__ __launch_bounds__(kForkThreads) void k_compact_small(dsr_compact_args_t a) {
  __shared__ uint32_t bits[kForkThreads];
  __shared__ int part[kForkThreads / 64];
  CompactSpace space;
  compact_space(a, space);
  const int x = threadIdx.x;
  bits[x] = 0;
  bool refused = false;
  for (uint32_t r = x; r < a.rows; r += kForkThreads) {
    const bool fine = (uint32_t)a.held[r] <= (uint32_t)a.width;
    a.status[r] = fine ? DSR_OK : DSR_E_LENGTH;
    refused |= !fine;
  }
  __syncthreads();
  const uint32_t width = a.width, entries = (uint32_t)a.rows * width;
  for (uint32_t e = x; e < entries; e += kForkThreads) {
    const uint32_t r = e / width, c = e - r * width;
    const int held = a.held[r];
    if ((uint32_t)held > width || (int)c >= held) continue;
    const int id = a.table[r * a.table_ld + c];
    if ((unsigned)id >= (unsigned)a.blocks) {
      a.status[r] = DSR_E_BLOCK;
      refused = true;
    } else {
      atomicOr(&bits[id >> 5], 1u << (id & 31));
    }
  }
  refused = __syncthreads_or(refused);
  const uint32_t held = bits[x];
  const bool inside = x < pages_words(a.blocks);
  if (inside) space.held[x] = held;
  int n;
  pages_before<kForkThreads>(__popc(held & pages_range(x, a.first, a.blocks)), part, n);
  const int moves = compact_moves<kForkThreads>(a, space, held, 0, (int64_t)a.first + n, 0, 0);
  if (x == 0) *space.head = CompactHead{refused, a.first + n, refused ? 0 : moves};
}

// `rows` workgroups write table rows, `others` what is kept per page and the
// pool, the rest copy.
template <int COUNT>
__global__ __launch_bounds__(kPagesThreads) void k_compact_apply(dsr_compact_args_t a, PagesCaches<COUNT> caches,
                                                                 int rows, int others) {
  CompactSpace space;
  compact_space(a, space);
  const CompactHead head = *space.head;
  if ((int)blockIdx.x < rows) {
    const int64_t r = blockIdx.x;
    const int held = head.refused ? 0 : a.held[r];
    for (int64_t c = threadIdx.x; c < a.width; c += kPagesThreads) {
      int id = a.table[r * a.table_ld + c];
      if (c < held && id >= head.limit) id = space.copies[space.rank[id]].to;
      a.table_out[r * a.table_out_ld + c] = id;
    }
    return;
  }
  if ((int)blockIdx.x < rows + others) {
    const int64_t step = (int64_t)others * kPagesThreads;
    const int64_t thread = (int64_t)((int)blockIdx.x - rows) * kPagesThreads + threadIdx.x;
    for (int64_t p = thread; p < a.blocks; p += step) {
      const bool held = space.held[p >> 5] >> (p & 31) & 1;
      if (head.refused || p < a.first || (held && p < head.limit)) {
        a.remap[p] = (int32_t)p;
        if (a.shared) a.shared_out[p] = a.shared[p];
      } else if (held) {  // moves: its place's thread writes its count
        a.remap[p] = space.copies[space.rank[p]].to;
      } else {
        a.remap[p] = -1;
        if (a.shared && p < head.limit) {
          const int from = space.copies[space.rank[p]].from;
          a.shared_out[p] = a.shared[from];
          a.shared_out[from] = 0;
        } else if (a.shared) {
          a.shared_out[p] = 0;
        }
      }
    }
    for (int64_t i = thread; i < a.pool_size; i += step)
      a.pool_out[i] = head.refused ? a.pool[i] : i < a.blocks - head.limit ? (int32_t)(head.limit + i) : -1;
    if (thread < 2)
      a.pool_state_out[thread] = head.refused ? a.pool_state[thread] : thread == 0 ? 0 : a.blocks - head.limit;
    return;
  }
  pages_copies<COUNT>(PageShape{a.heads, a.row_bytes, a.c_block, a.c_token, a.c_head}, space.copies, head.moves,
                      a.caches, caches, a.cache_count, blockIdx.x - rows - others, gridDim.x - rows - others);
}

}  // namespace dsr
