// C ABI of dsr_branch.h but for the attention (dsr_prefix.hip): argument
// checks and launches.
#include "dsr_branch.h"

#include "dsr_beams.h"
#include "dsr_pages.h"

using namespace dsr;

namespace {

int32_t launched() { return hipGetLastError() == hipSuccess ? 0 : DSR_ERR_LAUNCH; }

bool page_ok(int32_t page, int32_t blocks) {
  return page >= 1 && page <= DSR_TREE_MAX_PAGE && (page & (page - 1)) == 0 && blocks >= 1 &&
         (int64_t)blocks * page <= INT_MAX;
}

bool beams_shape_ok(const dsr_select_beams_args_t& a) {
  return (a.dtype == DSR_BF16 || a.dtype == DSR_F16 || a.dtype == DSR_F32) && a.keep >= 1 &&
         a.keep <= DSR_BEAMS_MAX_KEEP && a.rows >= 0 && a.rows <= DSR_BEAMS_MAX_ROWS && a.groups >= 0 &&
         a.groups <= DSR_BEAMS_MAX_ROWS && a.vocab >= 1 && a.vocab <= DSR_BEAMS_MAX_VOCAB;
}

template <class T, int EACH>
void beams_launch(const dsr_select_beams_args_t& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows * beam_slices(a))), threads(kBeamThreads);
  if ((uintptr_t)a.logits % 16 == 0 && (a.rows == 1 || a.ld * sizeof(T) % 16 == 0))
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_beam_slices<T, EACH, true>), grid, threads, 0, s, a);
  else
    hipLaunchKernelGGL(HIP_KERNEL_NAME(k_beam_slices<T, EACH, false>), grid, threads, 0, s, a);
}

template <class T>
void beams_typed(const dsr_select_beams_args_t& a, hipStream_t s) {
  switch (beam_each(a.rows, a.vocab)) {
    case 8: return beams_launch<T, 8>(a, s);
    case 32: return beams_launch<T, 32>(a, s);
    default: return beams_launch<T, 64>(a, s);
  }
}

// What fork and compact ask of caches; without caches the rest is free.
template <class A>
bool caches_ok(const A& a) {
  if (a.cache_count < 0 || a.cache_count > 65535) return false;
  if (a.cache_count == 0) return true;
  return !a.caches != !a.host_caches && a.heads >= 1 && a.heads <= 65536 && a.row_bytes >= 16 &&
         a.row_bytes <= 65536 && a.row_bytes % 16 == 0 && (int64_t)a.page * a.heads * a.row_bytes <= INT_MAX &&
         a.c_block % 16 == 0 && a.c_token % 16 == 0 && a.c_head % 16 == 0;
}

template <class A>
bool table_ok(const A& a) {
  return page_ok(a.page, a.blocks) && a.width >= 1 && (int64_t)a.width * a.page <= INT_MAX && a.table_ld >= a.width &&
         a.table_out_ld >= a.width && a.pool_size >= 1 && a.pool_size <= (1 << 30);
}

bool fork_shape_ok(const dsr_fork_args_t& a) {
  return a.sources >= 0 && a.sources <= DSR_TREE_MAX_REQUESTS && a.rows >= 0 && a.rows <= DSR_TREE_MAX_REQUESTS &&
         a.reserved == 0 && table_ok(a) && caches_ok(a);
}

bool compact_shape_ok(const dsr_compact_args_t& a) {
  return a.rows >= 0 && a.rows <= DSR_TREE_MAX_REQUESTS && table_ok(a) && caches_ok(a) && a.first >= 0 &&
         a.first < a.blocks && a.pool_size >= a.blocks - a.first;
}

// The last launch of a call: once with the caches' addresses on the device, or
// once for every kPagesInline caches whose addresses go with it (the first of
// these has also the work that is not copying).
// Workgroups that copy: as many as the chip holds a few times over.
constexpr int64_t kPagesCopiers = 2048;
template <class A, class Inline, class Device>
int32_t pages_launch(const A& a, int64_t most_copies, Inline with_inline, Device with_device) {
  auto copiers = [&](int count) {
    const int64_t items = most_copies * count;
    return (unsigned)(items < kPagesCopiers ? items : kPagesCopiers);
  };
  if (!a.host_caches || a.cache_count == 0) {
    with_device(a, copiers(a.cache_count));
    return launched();
  }
  for (int first = 0; first < a.cache_count; first += kPagesInline) {
    A part = a;
    PagesCaches<kPagesInline> caches;
    part.cache_count = a.cache_count - first < kPagesInline ? a.cache_count - first : kPagesInline;
    for (int c = 0; c < kPagesInline; ++c) caches.at[c] = c < part.cache_count ? a.host_caches[first + c] : nullptr;
    with_inline(part, caches, copiers(part.cache_count), first == 0);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  }
  return 0;
}

}  // namespace

extern "C" {

size_t dsr_select_beams_workspace_bytes(const dsr_select_beams_args_t* args) {
  if (!args || !beams_shape_ok(*args)) return 0;
  const int64_t slices = beam_slices(*args);
  const int64_t row = slices * (int64_t)sizeof(BeamPart) + (int64_t)sizeof(BeamTerm) + slices * args->keep * 8;
  return (size_t)(args->rows * row);
}

int32_t dsr_select_beams(const dsr_select_beams_args_t* args, void* stream) {
  if (!args) return DSR_ERR_ARG;
  const dsr_select_beams_args_t& a = *args;
  if (!beams_shape_ok(a) || a.ld < a.vocab) return DSR_ERR_ARG;
  if (a.rows > 0 && (!a.logits || !a.scores || !a.status)) return DSR_ERR_ARG;
  if (a.groups > 0 && (!a.offsets || !a.parents || !a.tokens || !a.out_scores)) return DSR_ERR_ARG;
  if (a.rows > 0 && (!a.workspace || ((uintptr_t)a.workspace & 15u) ||
                     a.workspace_bytes < dsr_select_beams_workspace_bytes(args)))
    return DSR_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  if (a.rows > 0) {
    switch (a.dtype) {
      case DSR_BF16: beams_typed<__bf16>(a, s); break;
      case DSR_F16: beams_typed<_Float16>(a, s); break;
      default: beams_typed<float>(a, s);
    }
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  }
  if (a.groups == 0) return 0;
  hipLaunchKernelGGL(k_beam_groups, dim3((unsigned)a.groups), dim3(kBeamGroupThreads), 0, s, a);
  return launched();
}

size_t dsr_fork_workspace_bytes(const dsr_fork_args_t* args) {
  if (!args || !fork_shape_ok(*args)) return 0;
  ForkSpace s;
  return (size_t)fork_space(*args, s);
}

int32_t dsr_fork_pages(const dsr_fork_args_t* args, void* stream) {
  if (!args) return DSR_ERR_ARG;
  const dsr_fork_args_t& a = *args;
  if (!fork_shape_ok(a)) return DSR_ERR_ARG;
  if (!a.shared || !a.shared_out || !a.pool || !a.pool_state || !a.pool_state_out ||
      (a.sources > 0 && (!a.lengths || !a.held || !a.table || !a.source_status)) ||
      (a.rows > 0 && (!a.parents || !a.table_out || !a.held_out || !a.lengths_out || !a.status)))
    return DSR_ERR_ARG;
  // The sources are read while rows are written.
  if (a.rows > 0 && a.sources > 0 &&
      (a.table_out == a.table || a.held_out == a.held || a.lengths_out == a.lengths || a.lengths_out == a.parents ||
       a.held_out == a.parents))
    return DSR_ERR_ARG;
  if (!a.workspace || ((uintptr_t)a.workspace & 15u) || a.workspace_bytes < dsr_fork_workspace_bytes(args))
    return DSR_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  int chunks = 0;  // of pages that the last launch frees
  if (a.rows <= kForkSmallRows && a.sources <= kForkSmallRows && a.blocks <= kForkSmallBlocks &&
      (a.rows + a.sources) * a.width <= kForkSmallEntries) {
    hipLaunchKernelGGL(k_fork_small, dim3(1), dim3(kForkThreads), 0, s, a);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
    if (a.cache_count == 0) return 0;
  } else {
    const int64_t words = a.shared_out != a.shared ? a.blocks : pages_words(a.blocks);
    const int64_t helpers = (words + 8 * kForkThreads - 1) / (8 * kForkThreads);
    hipLaunchKernelGGL(k_fork_scan, dim3(1 + (unsigned)(helpers < 256 ? helpers : 256)), dim3(kForkThreads), 0, s, a);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
    if (a.rows + a.sources > 0) {
      hipLaunchKernelGGL(k_fork_rows, dim3((unsigned)(a.rows + a.sources)), dim3(kPagesThreads), 0, s, a);
      if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
    }
    chunks = pages_chunks(a.blocks);
  }
  return pages_launch(
      a, a.rows,
      [&](const dsr_fork_args_t& part, const PagesCaches<kPagesInline>& caches, unsigned copiers, bool first) {
        const int free = first ? chunks : 0;
        if (free + copiers > 0)
          hipLaunchKernelGGL(HIP_KERNEL_NAME(k_fork_finish<kPagesInline>), dim3(free + copiers), dim3(kPagesThreads), 0,
                             s, part, caches, free);
      },
      [&](const dsr_fork_args_t& all, unsigned copiers) {
        if (chunks + copiers > 0)
          hipLaunchKernelGGL(HIP_KERNEL_NAME(k_fork_finish<0>), dim3(chunks + copiers), dim3(kPagesThreads), 0, s, all,
                           PagesCaches<0>{}, chunks);
      });
}

size_t dsr_compact_workspace_bytes(const dsr_compact_args_t* args) {
  if (!args || !compact_shape_ok(*args)) return 0;
  CompactSpace s;
  return (size_t)compact_space(*args, s);
}

int32_t dsr_compact_pages(const dsr_compact_args_t* args, void* stream) {
  if (!args) return DSR_ERR_ARG;
  const dsr_compact_args_t& a = *args;
  if (!compact_shape_ok(a)) return DSR_ERR_ARG;
  if (!a.pool || !a.pool_out || !a.pool_state || !a.pool_state_out || !a.remap || !a.shared != !a.shared_out ||
      (a.rows > 0 && (!a.held || !a.table || !a.table_out || !a.status)))
    return DSR_ERR_ARG;
  if (a.table_out == a.table && a.table_out_ld != a.table_ld) return DSR_ERR_ARG;
  if (!a.workspace || ((uintptr_t)a.workspace & 15u) || a.workspace_bytes < dsr_compact_workspace_bytes(args))
    return DSR_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  const dim3 threads(kPagesThreads);
  if (a.blocks <= kCompactSmallBlocks && a.rows * a.width <= kCompactSmallEntries) {
    hipLaunchKernelGGL(k_compact_small, dim3(1), dim3(kForkThreads), 0, s, a);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  } else {
    const int64_t clear = (pages_words(a.blocks) + 8 * kPagesThreads - 1) / (8 * kPagesThreads);
    hipLaunchKernelGGL(k_compact_clear, dim3((unsigned)(clear < 256 ? clear : 256)), threads, 0, s, a);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
    if (a.rows > 0) {
      hipLaunchKernelGGL(k_compact_mark, dim3((unsigned)a.rows), threads, 0, s, a);
      if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
    }
    hipLaunchKernelGGL(k_compact_plan, dim3((unsigned)pages_chunks(a.blocks)), threads, 0, s, a);
    if (hipGetLastError() != hipSuccess) return DSR_ERR_LAUNCH;
  }
  const int64_t entries = a.blocks > a.pool_size ? a.blocks : a.pool_size;
  const int64_t each = (entries + kPagesThreads - 1) / kPagesThreads;
  const int rows = (int)a.rows, others = (int)(each < 512 ? each : 512);
  return pages_launch(
      a, a.blocks / 2,
      [&](const dsr_compact_args_t& part, const PagesCaches<kPagesInline>& caches, unsigned copiers, bool first) {
        const int r = first ? rows : 0, o = first ? others : 0;
        if (r + o + copiers > 0)
          hipLaunchKernelGGL(HIP_KERNEL_NAME(k_compact_apply<kPagesInline>), dim3(r + o + copiers), threads, 0, s,
                             part, caches, r, o);
      },
      [&](const dsr_compact_args_t& all, unsigned copiers) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(k_compact_apply<0>), dim3(rows + others + copiers), threads, 0, s, all,
                           PagesCaches<0>{}, rows, others);
      });
}

}  // extern "C"
