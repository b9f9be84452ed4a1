// C ABI of dsr_prefix_attention: argument checks and launches.
#include "dsr_prefix.h"

using namespace dsr;

namespace {

int32_t launched() { return hipGetLastError() == hipSuccess ? 0 : DSR_ERR_LAUNCH; }

// Dimensions of the kernel that takes a head dimension.
int prefix_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256; }

// Rows of a tile for a usual group's, or request's, rows.  64 only above 128
// dimensions: 8 prefixes of 8 requests, 64 rows a head, 84 us in tiles of 128 rows
// and 112 in ones of 64, whose steps are of twice the tokens and leave room for one
// workgroup a CU.  Groups of 32 to 64 rows over 8,192 tokens and more, in tiles of 64
// and of 128: 192 dimensions 133 to 223 us and 156 to 278; 256 dimensions 308 and 550
// where requests have 32 rows, but 185 to 283 and 175 to 244 where they have 4 to 16.
int prefix_rows(const dsr_tree_attention_args_t& a, int64_t count) {
  const int64_t rows = count > 0 ? (a.tokens * (a.q_heads / a.kv_heads) + count - 1) / count : 0;
  return rows <= 16 ? 16 : a.head_dim > 128 && rows <= 64 ? 64 : 128;
}

// The work splits of both passes, from sizes alone.
void prefix_plan(const dsr_tree_attention_args_t& a, const int64_t* counts, AttnPlan* plans) {
  const int64_t group = a.q_heads / a.kv_heads, span = (int64_t)a.width * a.page;
  const bool big = a.head_dim > 128;
  int rows[2] = {prefix_rows(a, counts[0]), prefix_rows(a, counts[1])};
  if (rows[1] > 16) rows[1] = rows[0];  // the kernels that there are
  int64_t most = 0;
  for (int pass = 0; pass < 2; ++pass) {
    AttnPlan& p = plans[pass] = AttnPlan{};
    p.tile_rows = rows[pass];
    p.tokens = p.tile_rows == 16 ? 128 : p.tile_rows == 64 ? 64 : 32;
    p.min_steps = 128 / p.tokens;
    p.cut = true;
    const int64_t tiles = (a.tokens * group / p.tile_rows + counts[pass]) * a.kv_heads;
    while ((span / p.tokens + 1) * tiles >= INT_MAX) p.tokens *= 2;  // steps are counted in 32 bits
    auto log2_of = [](int64_t x) { return x & (x - 1) ? -1 : __builtin_ctzll(x); };
    p.group = (int)group;
    p.tile_shift = log2_of(p.tile_rows), p.token_shift = log2_of(p.tokens), p.group_shift = log2_of(group);
    p.page_shift = a.page > 0 ? log2_of(a.page) : 0;
    const int64_t cuts = (span + p.tokens - 1) / p.tokens / p.min_steps;  // shares of the fewest steps
    most += tiles * (cuts > 1 ? cuts : 1) + 1;
  }
  // Workgroups that the chip holds at once: 256 CUs, two each where there is room.
  int groups = big ? 256 : 512;
  if (most < groups) groups = (int)((most + 7) / 8 * 8);
  plans[0].groups = plans[1].groups = groups;
}

// Addresses in the workspace; their end.
int64_t prefix_space(const dsr_prefix_attention_args_t& x, PrefixJoin& j) {
  const dsr_tree_attention_args_t& a = x.a;
  const int64_t counts[2] = {x.group_count, a.requests}, dim = prefix_dim(a.head_dim);
  char* base = (char*)a.workspace;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = base + at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  int32_t* low = (int32_t*)take(a.requests * 4);
  int32_t* group_of = (int32_t*)take(a.requests * 4);
  int32_t* group_lo = (int32_t*)take(a.requests * 4);
  int32_t* lead = (int32_t*)take(x.group_count * 4);
  prefix_plan(a, counts, j.p);
  for (int pass = 0; pass < 2; ++pass) {
    AttnPlan& p = j.p[pass];
    AttnBranch& b = j.b[pass];
    const int64_t parts = 2 * (int64_t)p.groups * p.tile_rows;
    p.part_o = (float*)take(parts * dim * 4);
    p.part_ml = (float2*)take(parts * 8);
    p.part_bad = (int32_t*)take(2 * (int64_t)p.groups * 4);
    b.groups = x.groups;
    b.prefix = x.prefix_lengths;
    b.group_count = (int32_t)x.group_count;
    b.own = pass;
    b.count = counts[pass];
    b.tiles = (int2*)take(a.tokens * a.q_heads * 8);
    b.bad = (int32_t*)take(counts[pass] * 4);
    b.row_o = (float*)take(a.tokens * a.q_heads * dim * 4);
    b.row_ml = (float2*)take(a.tokens * a.q_heads * 8);
    b.low = low;
    b.group_of = group_of;
    b.group_lo = group_lo;
    b.lead = lead;
  }
  return at;
}

// Items of the join that the chip holds about at once (8 prefixes of 8 requests 84 us, 91 with 256; trees of 96
// dimensions 71.5 and 79.7; 4,096 as 1,024).
constexpr int64_t kPrefixItems = 1024;

template <class T, int DP>
int32_t prefix_launch(const dsr_prefix_attention_args_t& x, const PrefixJoin& j, hipStream_t s) {
  const dsr_tree_attention_args_t& a = x.a;
  PrefixCall c{{{a, j.p[0], j.b[0]}, {a, j.p[1], j.b[1]}}};
  c.c[0].a.visible = nullptr;  // every row sees the whole prefix
  const dim3 threads(kAttnThreads);
  if (a.requests > kAttnLows) {
    const int64_t lows = (a.requests + kAttnThreads - 1) / kAttnThreads;
    hipLaunchKernelGGL(k_prefix_lows, dim3((unsigned)lows), threads, 0, s, c);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
    hipLaunchKernelGGL(k_prefix_leads, dim3((unsigned)lows), threads, 0, s, c);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  }
  // Workgroups for rows of no request: one for each 256 KB that all rows have.
  const int64_t clear = (a.tokens * a.q_heads * a.head_dim * 2 + (1 << 18) - 1) >> 18;
  const dim3 grid((unsigned)(j.p[0].groups + (clear > 256 ? 256 : clear < 8 ? 8 : clear)));
  constexpr bool whole = kAttnThreads % (DP / 8) == 0;
  const bool flat = whole && a.page >= attn_round(DP) && a.k_token <= 1 << 24 && a.v_token <= 1 << 24;
  auto launch = [&](auto A, auto B) {
    constexpr int rows = decltype(A)::value, own = decltype(B)::value;
    if (flat && rows > 16)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(k_prefix_attention<T, DP, rows, own, whole && (rows > 16)>), grid, threads, 0,
                         s, c);
    else
      hipLaunchKernelGGL(HIP_KERNEL_NAME(k_prefix_attention<T, DP, rows, own, false>), grid, threads, 0, s, c);
  };
  constexpr std::integral_constant<int, 16> few{};
  constexpr std::integral_constant<int, 128> many{};
  // A group's rows are no fewer than a request's.
  switch (j.p[0].tile_rows) {
    case 16: launch(few, few); break;
    case 128: j.p[1].tile_rows == 16 ? launch(many, few) : launch(many, many); break;
    default:
      if constexpr (DP > 128) {
        constexpr std::integral_constant<int, 64> mid{};
        j.p[1].tile_rows == 16 ? launch(mid, few) : launch(mid, mid);
      }
  }
  if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  const int64_t rows = x.a.tokens * x.a.q_heads;
  if (rows == 0) return 0;
  // Parts of a row, about: the chip's workgroups over all tiles, or as many as the longest row has steps.
  const int64_t tiles = (rows + j.p[0].tile_rows - 1) / j.p[0].tile_rows, span = (int64_t)a.width * a.page;
  const int64_t cuts = j.p[0].groups / tiles, steps = span / 128, parts = 2 + (cuts < steps ? cuts : steps);
  // Many parts: four rows a block, so that more threads share a row's (a single call over 1,000 tokens 19.7 us, 21.0
  // with eight); few: eight (chunks of up to 400 tokens 591 us, 616 with four).
  const int jr = parts > 6 ? 4 : 8;
  // Blocks of rows of an item: one where there are few, else so many that the chip holds about all items at once.
  const int64_t blocks = (x.a.q_heads + jr - 1) / jr, most = x.a.tokens * blocks / kPrefixItems;
  const int64_t each = most < 1 ? 1 : most < blocks ? most : blocks, chunks = (blocks + each - 1) / each;
  const int64_t tokens = x.a.tokens < (1 << 20) / chunks ? x.a.tokens : (1 << 20) / chunks;
  const dim3 join((unsigned)tokens, (unsigned)chunks);
  if (jr == 4)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_prefix_join<T, DP, 4, 5>), join, threads, 0, s, j, (int)each);
  else
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_prefix_join<T, DP, 8, 4>), join, threads, 0, s, j, (int)each);
  return launched();
}

template <class T>
int32_t prefix_typed(const dsr_prefix_attention_args_t& x, const PrefixJoin& j, hipStream_t s) {
  switch (prefix_dim(x.a.head_dim)) {
    case 64: return prefix_launch<T, 64>(x, j, s);
    case 128: return prefix_launch<T, 128>(x, j, s);
    case 192: return prefix_launch<T, 192>(x, j, s);
    default: return prefix_launch<T, 256>(x, j, s);
  }
}

}  // namespace

extern "C" {

size_t dsr_prefix_attention_workspace_bytes(const dsr_prefix_attention_args_t* args) {
  if (!args || args->group_count < 0 || args->group_count > args->a.requests) return 0;
  const size_t tree = dsr_tree_attention_workspace_bytes(&args->a);
  if (tree == 0) return 0;
  PrefixJoin j;
  const size_t own = (size_t)prefix_space(*args, j);
  return own > tree ? own : tree;
}

int32_t dsr_prefix_attention(const dsr_prefix_attention_args_t* args, void* stream) {
  if (!args) return DSR_ERR_ARG;
  const dsr_prefix_attention_args_t& x = *args;
  const dsr_tree_attention_args_t& a = x.a;
  if (x.group_count < 0 || x.group_count > a.requests) return DSR_ERR_ARG;
  if (x.group_count == 0) return dsr_tree_attention(&x.a, stream);
  if (!x.groups || !x.prefix_lengths) return DSR_ERR_ARG;
  // What dsr_tree_attention asks.
  if (a.page < 1 || (a.page & (a.page - 1)) || a.blocks < 1 || (int64_t)a.blocks * a.page > INT_MAX ||
      a.table_ld < a.width || !(a.scale == a.scale) || a.scale - a.scale != 0.f)
    return DSR_ERR_ARG;
  const size_t need = dsr_prefix_attention_workspace_bytes(args);
  if (need == 0) return DSR_ERR_ARG;
  if (!a.table || !a.offsets || !a.kv_lengths || !a.status || !a.k_cache || !a.v_cache ||
      (a.tokens > 0 && (!a.q || !a.out)))
    return DSR_ERR_ARG;
  for (const void* p : {a.q, a.k_cache, a.v_cache, (const void*)a.out})
    if ((uintptr_t)p & 15u) return DSR_ERR_ARG;
  for (int64_t st : {a.q_token, a.q_head, a.out_token, a.out_head, a.k_block, a.k_token, a.k_head, a.v_block,
                     a.v_token, a.v_head})
    if (st % 8 != 0 || st < 0) return DSR_ERR_ARG;
  for (int64_t st : {a.k_block, a.k_token, a.v_block, a.v_token})
    if (st > INT_MAX) return DSR_ERR_ARG;  // multiplied in 32 x 32 bits
  if (!a.workspace || ((uintptr_t)a.workspace & 255u) || a.workspace_bytes < need) return DSR_ERR_WORKSPACE;
  PrefixJoin j;
  j.a = a;
  prefix_space(x, j);
  hipStream_t s = (hipStream_t)stream;
  return a.dtype == DSR_BF16 ? prefix_typed<__bf16>(x, j, s) : prefix_typed<_Float16>(x, j, s);
}

}  // extern "C"
