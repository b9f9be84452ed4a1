/*
 * dsr_tree.h - C ABI of a tree-speculative decoding step over a paged cache
 * (MI355X, gfx950), next to the sampling entry points of dsr_sampling.h.
 *
 * A step brings new tokens for each of R requests: one decoded token, a
 * chain, or a tree of drafted tokens whose node 0 is the pending token.
 *   dsr_plan_blocks     where they go: pages from a pool, block table, slot,
 *                       position and tree mask of every new token
 *   dsr_rotary          rotary positions of queries and keys; keys and values
 *                       written to their cache slots
 *   dsr_tree_attention  attention of the new tokens over the cache and each other
 *   dsr_commit_tree     the accepted path of each tree, given the target's
 *                       token at every node, and its cache rows moved together
 *
 * Conventions are those of dsr_sampling.h: device pointers owned by the
 * caller, the caller's stream, no allocation, no synchronisation, 0 or a
 * negative DSR_ERR_* as the return value, data errors as per-request (or
 * per-token) status codes.  New tokens of all requests lie one after the
 * other: request r owns tokens [offsets[r], offsets[r + 1]).  A cache is an
 * array of `blocks` pages of `page` tokens of `heads` rows, addressed by three
 * strides, so that token-major and head-major pages both work; slot s is
 * token s % page of page s / page.  Strides are in elements.
 */
#ifndef DSR_TREE_H
#define DSR_TREE_H

#include "dsr_sampling.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DSR_F16 4                     /* element type, next to DSR_BF16 / DSR_F32 / DSR_F64 */

#define DSR_TREE_MAX_NODES 64         /* nodes of one tree: a bit each in a 64-bit mask */
#define DSR_TREE_MAX_PAGE 1024        /* tokens per page, a power of two */
#define DSR_TREE_MAX_REQUESTS 16384
#define DSR_ROTARY_MAX_DIM 512
#define DSR_ATTENTION_MAX_DIM 256

/* Status codes, continuing DSR_E_*. */
#define DSR_E_LENGTH 16        /* a length, page count or offset outside its bounds */
#define DSR_E_BLOCKS 17        /* the page pool cannot serve (or take back) the request's pages */
#define DSR_E_CAPACITY 18      /* the new tokens do not fit the token arrays */
#define DSR_E_TREE 19          /* not a tree: a parent at or after its child, or too many nodes */
#define DSR_E_BLOCK 20         /* a page id or slot outside the cache */

/* dsr_plan_blocks: block tables and slot maps from request lengths.
 *
 * Request r holds lengths[r] tokens in held_in[r] pages (the first entries of
 * its table row) and brings added[r] new tokens, or ends (added[r] == -1: its
 * pages go back to the pool).  A request gets the pages it lacks for
 * lengths + added tokens; spare pages it already holds are used first.
 *
 * The pool is a ring of page ids, pool[0 .. pool_size), of which the
 * pool_state[1] entries from pool_state[0] on are free.  Pages are taken from
 * the front in request order, so the result does not depend on timing; pages
 * given back join behind the last entry and are first used by the next
 * call.  A request that lacks pages when the pages wanted up to and
 * including it exceed the free ones is refused (DSR_E_BLOCKS), and so is
 * every later request that lacks pages.
 * A request whose new tokens touch a page id outside the cache is refused
 * (DSR_E_BLOCK), and keeps the pages that it took.
 *
 * Per token: its slot, its position (lengths[r] + its index, or + its depth
 * in the tree), its request.  With `parents` (per token: the index of its
 * parent among its request's new tokens, -1 for none, always before its
 * child) also `visible`: bit i is set for the token's ancestors and itself.
 * Tokens of refused requests, and tokens past the last request's, get slot -1,
 * position 0 and mask 0, the latter also owner -1.  kv_lengths[r] is
 * lengths + added, or 0 for a refused or ended request.
 *
 * held_out / pool_state_out may be held_in / pool_state_in themselves; no
 * other arrays may overlap. */
typedef struct dsr_plan_args {
  const int32_t* lengths;      /* [requests] */
  const int32_t* added;        /* [requests] */
  const int32_t* parents;      /* [capacity] or NULL */
  const int32_t* held_in;      /* [requests] */
  const int32_t* pool_state_in;/* [2]: first free entry, free entries */
  int32_t* table;              /* [requests, table_ld] page ids; only new entries are written */
  int32_t* pool;               /* [pool_size] */
  int64_t requests;            /* 0 .. DSR_TREE_MAX_REQUESTS */
  int64_t table_ld;            /* >= width */
  int64_t capacity;            /* tokens in the per-token arrays, 1 .. 2^30 */
  int32_t width;               /* pages per table row, >= 1; width * page < 2^31 */
  int32_t page;
  int32_t pool_size;           /* 1 .. 2^30 */
  int32_t blocks;              /* pages of the cache; blocks * page < 2^31 */
  int32_t* held_out;           /* [requests] */
  int32_t* pool_state_out;     /* [2] */
  int32_t* offsets;            /* [requests + 1], clamped to capacity */
  int32_t* kv_lengths;         /* [requests] */
  int32_t* status;             /* [requests] DSR_OK or DSR_E_* */
  int32_t* slots;              /* [capacity] */
  int32_t* positions;          /* [capacity] */
  int32_t* owners;             /* [capacity] or NULL */
  uint64_t* visible;           /* [capacity], with parents */
  void* workspace;             /* >= dsr_plan_workspace_bytes(requests), 4-byte aligned */
  size_t workspace_bytes;
} dsr_plan_args_t;

/* dsr_rotary: for each token and head the pairs (a, b) of dimensions
 * [rot_start, rot_start + rot_dim) become
 *   (a cos - b sin, a sin + b cos) * magnitude,  angle = position * freqs[i]
 * (inverse: -sin, the transposed rotation: the gradient of the forward one).
 * Pair i is dimensions (i, i + rot_dim / 2) of the part, or (2 i, 2 i + 1)
 * when interleaved.  Other dimensions are copied.  Angles are reduced in
 * float64, so that positions of millions keep their accuracy; products are
 * float32, rounded once.  Keys go to k_out (if set) and to slot slots[n] of
 * k_cache (if set), values to that slot of v_cache.  Slot -1 writes no cache;
 * a slot outside the cache neither, and gives DSR_E_BLOCK. */
typedef struct dsr_rotary_args {
  const void* q;               /* [tokens, q_heads] rows of head_dim, or NULL (q_heads 0) */
  void* q_out;                 /* may be q */
  const void* k;               /* or NULL (kv_heads 0) */
  void* k_out;                 /* or NULL; may be k */
  const void* v;               /* [tokens, kv_heads] rows of v_dim, or NULL */
  const int32_t* positions;    /* [tokens], >= 0 */
  const double* freqs;         /* [rot_dim / 2] radians per position */
  const int32_t* slots;        /* [tokens], with a cache */
  void* k_cache;               /* or NULL */
  void* v_cache;               /* or NULL (exactly when v is NULL) */
  int32_t* status;             /* [tokens] DSR_OK or DSR_E_BLOCK, or NULL */
  int32_t dtype;               /* DSR_BF16 | DSR_F16 | DSR_F32, of all rows */
  int32_t q_heads, kv_heads;
  int32_t head_dim, v_dim;     /* 1 .. DSR_ROTARY_MAX_DIM */
  int32_t rot_start, rot_dim;  /* rot_dim even, 2 .. head_dim */
  int32_t interleaved, inverse;
  int32_t page, blocks;
  int32_t reserved;            /* must be 0 */
  double magnitude;
  int64_t tokens;              /* 0 .. 2^30 */
  int64_t q_token, q_head;     /* strides */
  int64_t qo_token, qo_head;
  int64_t k_token, k_head;
  int64_t ko_token, ko_head;
  int64_t v_token, v_head;
  int64_t kc_block, kc_token, kc_head;
  int64_t vc_block, vc_token, vc_head;
} dsr_rotary_args_t;

/* dsr_tree_attention: for each new token t of request r and query head h,
 *   s_j = scale * q . k_j,  out = sum_j softmax(s)_j v_j,  lse = log sum_j exp s_j
 * over the request's cached tokens j: all kv_lengths[r] - new of the context,
 * and of its own new tokens (the last ones in the cache) those whose bit is
 * set in visible[t], or without `visible` those up to t itself.  Query head h
 * reads key head h / (q_heads / kv_heads).  A row with no visible token gives
 * out 0 and lse -inf, and so do the rows of no request: those before
 * offsets[0] and from offsets[requests] on.  Values of tokens that a row does
 * not see never reach it, whatever they hold.
 * bf16 or f16 rows; products on the matrix cores, scores, softmax statistics
 * and sums in float32; the weights are rounded to the rows' type before
 * they multiply the values.
 * Status per request: DSR_E_LENGTH (kv_lengths[r] below its new tokens or
 * above width * page; or more than 64 new tokens with `visible`): its rows
 * give 0 and -inf; DSR_E_BLOCK: a page id outside the cache, whose tokens
 * are left out. */
typedef struct dsr_tree_attention_args {
  const void* q;               /* [tokens, q_heads] rows of head_dim */
  const void* k_cache;
  const void* v_cache;
  const int32_t* table;        /* [requests, table_ld] */
  const int32_t* offsets;      /* [requests + 1] */
  const int32_t* kv_lengths;   /* [requests] cached tokens, the new ones among them */
  const uint64_t* visible;     /* [tokens] or NULL */
  void* out;                   /* [tokens, q_heads] rows of head_dim */
  float* lse;                  /* [tokens, q_heads] or NULL */
  int32_t* status;             /* [requests] */
  int32_t dtype;               /* DSR_BF16 | DSR_F16 */
  int32_t q_heads, kv_heads;   /* q_heads a multiple of kv_heads */
  int32_t head_dim;            /* a multiple of 8 up to DSR_ATTENTION_MAX_DIM */
  int32_t page, width, blocks;
  float scale;
  int64_t requests;            /* 0 .. DSR_TREE_MAX_REQUESTS */
  int64_t tokens;              /* rows of q and out; (tokens + requests) * q_heads < 2^29 */
  int64_t table_ld;
  int64_t q_token, q_head;     /* strides: >= 0, multiples of 8; rows 16-byte aligned */
  int64_t out_token, out_head;
  int64_t k_block, k_token, k_head;  /* of pages and tokens less than 2^31 */
  int64_t v_block, v_token, v_head;
  void* workspace;             /* >= dsr_tree_attention_workspace_bytes(args), 256-byte aligned */
  size_t workspace_bytes;
} dsr_tree_attention_args_t;

/* dsr_commit_tree: after the target's token sampled[n] is known at every
 * node, each request's accepted path: from node 0 (the pending token, always
 * kept), the first child whose token is the one sampled at its parent, and so
 * on.  Each sampled token on the way is an output id; the last, which no child
 * matches, is the new pending token.  Stops are those of verify_drafts: an
 * accepted draft whose token is an EOS id or reaches output_limit ends the
 * path there, with no pending token (-1); a pending token can stop likewise.
 * Then, in each of the `caches` (no two of which overlap), the path's rows are
 * moved together: path node j's row to place lengths + j.
 * Status: DSR_E_TREE (parents, or more than 64 nodes), DSR_E_LENGTH
 * (kv_lengths below the new tokens or above width * page, output_limit < 1),
 * DSR_E_TOKEN (a negative sampled token on the path), DSR_E_BLOCK (a page id
 * outside the cache): nothing is accepted or moved then and the length is
 * that before the new tokens (0 with DSR_E_LENGTH).
 * A request without new tokens gives an empty path and no pending token.
 *
 * Given what was so before the step (lengths_in and plan_status: the plan's
 * input and result; pending_in: the pending tokens; all three or none), a
 * request that the plan refused, or that commit gives a status, keeps its
 * length and pending token, so that a later step can serve it; the status is
 * the plan's if it has one.  One without new tokens keeps its pending token,
 * whatever its output_limit, and has the length kv_lengths (0 if the plan
 * ended it).  Without the three a refused request's context is lost: the plan
 * gives kv_lengths 0 for it. */
typedef struct dsr_commit_args {
  const int32_t* parents;      /* [tokens] as dsr_plan_args_t */
  const int32_t* tokens_in;    /* [tokens] drafted token of each node */
  const int32_t* sampled;      /* [tokens] the target's token after each node */
  const int32_t* offsets;      /* [requests + 1] */
  const int32_t* kv_lengths;   /* [requests] */
  const int32_t* table;        /* [requests, table_ld] */
  const int32_t* output_limit; /* [requests], >= 1 */
  const int64_t* eos_off;      /* [requests + 1] CSR of EOS ids, or NULL */
  const int32_t* eos_ids;
  void* const* caches;         /* device array of cache_count device pointers, or NULL with host_caches */
  int32_t* path;               /* [requests, 64] kept nodes, -1 padded */
  int32_t* ids;                /* [requests, 64] output ids, -1 padded */
  int32_t* accepted;           /* [requests] kept nodes, the root among them */
  int32_t* count;              /* [requests] output ids */
  int32_t* pending;            /* [requests] pending token or -1 */
  int32_t* stop;               /* [requests] DSR_STOP_* */
  int32_t* lengths;            /* [requests] cached tokens afterwards; not kv_lengths itself */
  int32_t* status;             /* [requests] */
  int64_t requests;
  int64_t tokens;              /* length of the per-token arrays */
  int64_t table_ld;
  int32_t width, page, blocks;
  int32_t cache_count;         /* 0 .. 65535 */
  int32_t heads;               /* rows per token */
  int32_t row_bytes;           /* bytes of one row, a multiple of 16 */
  int64_t c_block, c_token, c_head; /* strides in bytes, multiples of 16 */
  const int32_t* lengths_in;   /* [requests] as dsr_plan_args_t.lengths, or NULL; none of these is an output */
  const int32_t* pending_in;   /* [requests] */
  const int32_t* plan_status;  /* [requests] as dsr_plan_args_t.status */
  void* const* host_caches;    /* the pointers in host memory instead: read during the call, passed with the launch */
} dsr_commit_args_t;

size_t dsr_plan_workspace_bytes(int64_t requests);
size_t dsr_tree_attention_workspace_bytes(const dsr_tree_attention_args_t* args);

int32_t dsr_plan_blocks(const dsr_plan_args_t* args, void* stream);
int32_t dsr_rotary(const dsr_rotary_args_t* args, void* stream);
int32_t dsr_tree_attention(const dsr_tree_attention_args_t* args, void* stream);
int32_t dsr_commit_tree(const dsr_commit_args_t* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DSR_TREE_H */
