/*
 * dsr_branch.h - C ABI of decoding with several branches a request (parallel
 * samples, beams) over the paged cache of dsr_tree.h (MI355X, gfx950).
 *
 *   dsr_select_beams      the best continuations of each group of beams
 *   dsr_fork_pages        rows continue rows of the step before: whole pages
 *                         shared, the last one copied, unheld ones freed
 *   dsr_compact_pages     the held pages moved to the front of the cache
 *   dsr_prefix_attention  attention of requests that share a prefix, whose
 *                         keys and values are read once for all of them
 *
 * Conventions are those of dsr_tree.h: device pointers owned by the caller,
 * the caller's stream, no allocation, no synchronisation, 0 or a negative
 * DSR_ERR_* as the return value, data errors as status codes, strides of rows
 * in elements and of caches in bytes.  These entry points came without a
 * change of what was there, so DSR_ABI_VERSION is as it was; a library that
 * lacks them lacks the symbols.
 *
 * A page may be held by several rows.  shared[p] counts the rows that hold
 * page p besides one: 0 for a page that is free or held once, which is what
 * dsr_plan_blocks's pages are, and never less.  Only pages that are full are
 * shared, so the new tokens of a step, and dsr_commit_tree's moves, are always
 * in pages of their row's own.  A row with shared pages ends in dsr_fork_pages
 * (no row continues it), not in dsr_plan_blocks (added == -1), which would give
 * the shared pages back to the pool.
 */
#ifndef DSR_BRANCH_H
#define DSR_BRANCH_H

#include "dsr_tree.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DSR_BEAMS_MAX_KEEP 64
#define DSR_BEAMS_MAX_VOCAB 1048576
#define DSR_BEAMS_MAX_ROWS 65536

/* Status code, continuing those of dsr_tree.h. */
#define DSR_E_PARENT 21        /* a parent that is no row of the step before */

/* dsr_select_beams: group g is rows [offsets[g], offsets[g + 1]) of logits.
 * Row b offers each token v at scores[b] + logits[b][v] - lse_b, lse_b = log
 * sum_v exp logits[b][v]; with finished[b] != 0 it offers itself alone, as
 * token -1, at scores[b], and its logits are not read.  The group's `keep`
 * best offers, best first: equal ones go to the lowest row, then to the lowest
 * token (logits that differ, but whose sums round to one float64, come in any
 * order).  A score or logit of -inf offers nothing; places without an offer
 * get parent -1, token -1 and score -inf.
 * Sums of exponentials, scores and their order are float64.
 * Status per row: DSR_E_LOGITS (a NaN or +inf among its logits or in its
 * score: it offers nothing), DSR_E_MASKED (every logit -inf).  Rows of no
 * group get DSR_OK; rows of two groups are offered in both. */
typedef struct dsr_select_beams_args {
  const void* logits;          /* [rows, ld] */
  const double* scores;        /* [rows] sums of log probabilities so far */
  const int32_t* finished;     /* [rows] or NULL */
  const int32_t* offsets;      /* [groups + 1] rows of each group */
  int32_t* parents;            /* [groups, keep] rows */
  int32_t* tokens;             /* [groups, keep] */
  double* out_scores;          /* [groups, keep] */
  int32_t* status;             /* [rows] */
  int32_t dtype;               /* DSR_BF16 | DSR_F16 | DSR_F32 */
  int32_t keep;                /* 1 .. DSR_BEAMS_MAX_KEEP */
  int64_t rows;                /* 0 .. DSR_BEAMS_MAX_ROWS */
  int64_t groups;              /* 0 .. DSR_BEAMS_MAX_ROWS */
  int64_t vocab;               /* 1 .. DSR_BEAMS_MAX_VOCAB */
  int64_t ld;                  /* >= vocab */
  void* workspace;             /* >= dsr_select_beams_workspace_bytes(args), 16-byte aligned */
  size_t workspace_bytes;
} dsr_select_beams_args_t;

/* dsr_fork_pages: row r of the new step continues row s = parents[r] of the
 * step before (sources), or is empty (-1).
 *
 * Source s holds lengths[s] tokens in held[s] pages.  Its full pages, the
 * first lengths[s] / page, are shared by all rows that continue it.  The first
 * of these rows also takes over its other pages; each other one gets a page
 * from the pool, in row order, if the last token's page is not full, and the
 * tokens in it are copied there in every cache.  Rows that the pool cannot
 * serve are refused (DSR_E_BLOCKS), once one is also all later ones that want
 * a page; refused rows are empty.  A page that no row holds any more (its
 * sources ended, or spare pages of a source without a row: its count, less one
 * for each that is gone and more for each row that joins, is below 0) goes back
 * to the pool, whose entries are as in dsr_plan_blocks: in ascending order
 * behind the last one, to be taken by the next call.  (Pages that a ring shorter
 * than its pages has no room for are lost.)
 *
 * Table entries past a row's pages are -1.  table, held and lengths are new
 * arrays: rows may be more or fewer than sources.  shared_out and
 * pool_state_out may be shared and pool_state; no other arrays may overlap.
 * Status per row: DSR_E_PARENT (parents[r] is neither -1 nor a source),
 * DSR_E_LENGTH (its source's length or pages are out of bounds), DSR_E_BLOCKS:
 * the row is empty; DSR_E_BLOCK (a page id outside the cache, among the row's
 * or the one that it should have a copy of): the row is made, but such a page is
 * not copied and not counted, and the page that was to have its tokens holds
 * what it held.
 * Status per source: DSR_E_LENGTH (its pages stay as they are, in no row and
 * not in the pool), DSR_E_BLOCK. */
typedef struct dsr_fork_args {
  const int32_t* lengths;      /* [sources] */
  const int32_t* held;         /* [sources] */
  const int32_t* table;        /* [sources, table_ld] */
  const int32_t* parents;      /* [rows] */
  const int32_t* shared;       /* [blocks] */
  const int32_t* pool_state;   /* [2]: first free entry, free entries */
  int32_t* pool;               /* [pool_size] */
  int32_t* table_out;          /* [rows, table_out_ld] */
  int32_t* held_out;           /* [rows] */
  int32_t* lengths_out;        /* [rows] */
  int32_t* shared_out;         /* [blocks] */
  int32_t* pool_state_out;     /* [2] */
  int32_t* status;             /* [rows] */
  int32_t* source_status;      /* [sources] */
  void* const* caches;         /* device array of cache_count device pointers, or NULL with host_caches */
  void* const* host_caches;    /* the pointers in host memory instead: read during the call, passed with the launch */
  int64_t sources;             /* 0 .. DSR_TREE_MAX_REQUESTS */
  int64_t rows;                /* 0 .. DSR_TREE_MAX_REQUESTS */
  int64_t table_ld;            /* >= width */
  int64_t table_out_ld;        /* >= width */
  int32_t width;               /* pages per table row, >= 1; width * page < 2^31 */
  int32_t page, blocks;
  int32_t pool_size;           /* 1 .. 2^30 */
  int32_t cache_count;         /* 0 .. 65535 */
  int32_t heads;               /* rows per token */
  int32_t row_bytes;           /* bytes of one row, a multiple of 16 */
  int32_t reserved;            /* must be 0 */
  int64_t c_block, c_token, c_head; /* strides in bytes, multiples of 16 */
  void* workspace;             /* >= dsr_fork_workspace_bytes(args), 16-byte aligned */
  size_t workspace_bytes;
} dsr_fork_args_t;

/* dsr_compact_pages: of the pages first .. blocks - 1, the n that some row
 * holds come to lie at first .. first + n - 1: the k-th held page from
 * first + n on moves, in every cache, to the k-th page before it that is not
 * held; the others stay.  Tables and shared follow; every other page is free
 * afterwards, and the pool holds them in ascending order from its first entry
 * on (-1 behind them).  Pages before `first` are left alone.
 * remap[p] is page p's new id, -1 for a page that is free.
 * table_out, shared_out, pool_out and pool_state_out may be the inputs
 * themselves; no other arrays may overlap.
 * Status per row: DSR_E_LENGTH (held outside 0 .. width), DSR_E_BLOCK (a page
 * id outside the cache).  If any row has one nothing moves, the outputs are
 * copies of the inputs and remap[p] = p. */
typedef struct dsr_compact_args {
  const int32_t* held;         /* [rows] */
  const int32_t* table;        /* [rows, table_ld] */
  const int32_t* shared;       /* [blocks] or NULL (with shared_out) */
  const int32_t* pool;         /* [pool_size] */
  const int32_t* pool_state;   /* [2] */
  int32_t* table_out;          /* [rows, table_out_ld]: all `width` entries */
  int32_t* shared_out;         /* [blocks] */
  int32_t* pool_out;           /* [pool_size] */
  int32_t* pool_state_out;     /* [2] */
  int32_t* remap;              /* [blocks] */
  int32_t* status;             /* [rows] */
  void* const* caches;         /* as dsr_fork_args_t */
  void* const* host_caches;
  int64_t rows;                /* 0 .. DSR_TREE_MAX_REQUESTS */
  int64_t table_ld;            /* >= width */
  int64_t table_out_ld;        /* >= width */
  int32_t width;               /* as dsr_fork_args_t */
  int32_t page, blocks;
  int32_t first;               /* 0 .. blocks - 1 */
  int32_t pool_size;           /* blocks - first .. 2^30 */
  int32_t cache_count;
  int32_t heads;
  int32_t row_bytes;
  int64_t c_block, c_token, c_head;
  void* workspace;             /* >= dsr_compact_workspace_bytes(args), 16-byte aligned */
  size_t workspace_bytes;
} dsr_compact_args_t;

/* dsr_prefix_attention: dsr_tree_attention for requests in groups that share
 * a prefix.  Group g is requests [groups[g], groups[g + 1]); the first
 * prefix_lengths[g] tokens of their contexts are the same, on the same pages:
 * their keys and values are read once for all of the group's rows, from the
 * table row of its first request with new tokens, and may be from that of each.
 * Requests without new tokens may be anything, empty rows too.  Requests of no
 * group have no shared prefix.  out, lse and `visible` are as there, and so
 * is the rounding.
 * Status per request: as there, and DSR_E_LENGTH too where groups do not
 * ascend within 0 .. requests or offsets, held to 0 .. tokens, descend (every
 * request, and every row gives 0 and -inf), prefix_lengths[g] is negative or
 * more than width * page (requests of that group), or the context of a request
 * with new tokens (kv_lengths less these) is shorter than its group's prefix.
 * Values are summed in float32 before the sum is divided by that of the weights.
 * bf16 weights are at most 1: values near that type's largest in many places
 * overflow.  f16 ones are at most 2^15, and no sum of f16 values does: 2^15 x
 * 65504 x 2^31 tokens is below 2^62.
 * `a.workspace` holds dsr_prefix_attention_workspace_bytes(args). */
typedef struct dsr_prefix_attention_args {
  dsr_tree_attention_args_t a;
  const int32_t* groups;         /* [group_count + 1], ascending */
  const int32_t* prefix_lengths; /* [group_count] tokens */
  int64_t group_count;           /* 0 .. requests */
} dsr_prefix_attention_args_t;

size_t dsr_select_beams_workspace_bytes(const dsr_select_beams_args_t* args);
size_t dsr_fork_workspace_bytes(const dsr_fork_args_t* args);
size_t dsr_compact_workspace_bytes(const dsr_compact_args_t* args);
size_t dsr_prefix_attention_workspace_bytes(const dsr_prefix_attention_args_t* args);

int32_t dsr_select_beams(const dsr_select_beams_args_t* args, void* stream);
int32_t dsr_fork_pages(const dsr_fork_args_t* args, void* stream);
int32_t dsr_compact_pages(const dsr_compact_args_t* args, void* stream);
int32_t dsr_prefix_attention(const dsr_prefix_attention_args_t* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DSR_BRANCH_H */
