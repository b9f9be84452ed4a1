// The best continuations of groups of beams (dsr_select_beams).
//
// Two launches.  k_beam_slices: a workgroup takes a slice of one row, reads it
// once into registers, and leaves its `keep` largest logits, in order, with
// the slice's largest value and sum of exponentials.  k_beam_groups: a
// workgroup takes a group, makes each row's log sum of its slices, and picks
// the best of their candidates.
//
// Which of two rows' candidates is better hangs on the difference of two log
// sums, so these, and the scores, are float64: an exponential costs a dozen
// float64 instructions (beam_exp).
#pragma once

#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "dsr_branch.h"

namespace dsr {

constexpr int kBeamThreads = 256, kBeamWaves = kBeamThreads / 64;
constexpr int kBeamList = 256;                            // candidates a wave sorts from LDS
constexpr int kBeamGroupThreads = 512, kBeamGroupWaves = kBeamGroupThreads / 64;

// One slice of a row.
struct BeamPart {
  double sum;  // of exp(logit - top)
  float top;   // -inf: nothing but -inf
  int32_t bad; // a NaN or +inf among the logits
};

// a.workspace: parts [rows, slices], terms [rows], candidates [rows, slices, keep].
// A row's candidates are worth (logit - top) - rest + score each, in this
// order: top + rest, their log sum, would lose `rest` where all of a row's
// logits are the type's lowest value.
struct BeamTerm {
  double top, rest;  // largest logit, log sum exp(logit - top)
  double score;      // NaN: the row offers nothing
};
struct BeamSpace {
  BeamPart* parts;
  BeamTerm* terms;
  uint64_t* found; // order of the logit, ~token; 0: none
};
// Logits of a thread: many where that leaves workgroups enough for the chip,
// because a wave's sorts cost as much as 30 logits of each thread.
__host__ __device__ inline int beam_each(int64_t rows, int64_t vocab) {
  auto groups = [&](int each) { return rows * ((vocab + kBeamThreads * each - 1) / (kBeamThreads * each)); };
  return groups(64) >= 512 ? 64 : groups(32) >= 512 ? 32 : 8;
}
__host__ __device__ inline int beam_slices(const dsr_select_beams_args_t& a) {
  const int slice = kBeamThreads * beam_each(a.rows, a.vocab);
  return (int)((a.vocab + slice - 1) / slice);
}
__host__ __device__ inline BeamSpace beam_space(const dsr_select_beams_args_t& a) {
  BeamSpace s;
  s.parts = (BeamPart*)a.workspace;
  s.terms = (BeamTerm*)(s.parts + a.rows * beam_slices(a));
  s.found = (uint64_t*)(s.terms + a.rows);
  return s;
}

// The value of lane ^ J.
template <int J>
__device__ __forceinline__ uint32_t beam_xor(uint32_t x) {
  if constexpr (J == 1) return __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xf, 0xf, true);   // quads 1 0 3 2
  if constexpr (J == 2) return __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xf, 0xf, true);   // quads 2 3 0 1
  if constexpr (J == 4) {                                                                  // 7 - i, then quads 3 2 1 0
    const uint32_t y = __builtin_amdgcn_update_dpp(0, x, 0x141, 0xf, 0xf, true);
    return __builtin_amdgcn_update_dpp(0, y, 0x1B, 0xf, 0xf, true);
  }
  if constexpr (J == 8) return __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, true);  // rows of 16 turned by 8
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  if constexpr (J == 16) {
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(x, x, false, false));
    return threadIdx.x & 16 ? y[0] : y[1];
  }
  if constexpr (J == 32) {
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(x, x, false, false));
    return threadIdx.x & 32 ? y[0] : y[1];
  }
}
template <int J>
__device__ __forceinline__ uint64_t beam_xor(uint64_t x) {
  return (uint64_t)beam_xor<J>((uint32_t)(x >> 32)) << 32 | beam_xor<J>((uint32_t)x);
}

// A candidate among all of a group's: the greater is better.
struct BeamOffer {
  uint64_t key;   // order of its score; 0: none
  uint32_t place; // ~place: of equal scores the earliest
  __device__ __forceinline__ bool operator<(const BeamOffer& o) const {
    return key < o.key || (key == o.key && place < o.place);
  }
};
template <int J>
__device__ __forceinline__ BeamOffer beam_xor(BeamOffer x) {
  return BeamOffer{beam_xor<J>(x.key), beam_xor<J>(x.place)};
}

// One step of a bitonic network over a wave's lanes: the greater of a pair goes to the lane where `up`.
template <int J, class K>
__device__ __forceinline__ void beam_step(K& x, bool up) {
  const K y = beam_xor<J>(x);
  if ((x < y) == up) x = y;
}
// Lanes of a bitonic sequence, the greatest first.
template <class K>
__device__ __forceinline__ void beam_merge(K& x) {
  const int l = threadIdx.x;
  beam_step<32>(x, !(l & 32));
  beam_step<16>(x, !(l & 16));
  beam_step<8>(x, !(l & 8));
  beam_step<4>(x, !(l & 4));
  beam_step<2>(x, !(l & 2));
  beam_step<1>(x, !(l & 1));
}
// Any lanes, the greatest first (Batcher's bitonic sort).
template <class K>
__device__ __forceinline__ void beam_sort(K& x) {
  const int l = threadIdx.x;
  beam_step<1>(x, !(l & 1) == !(l & 2));
  beam_step<2>(x, !(l & 2) == !(l & 4));
  beam_step<1>(x, !(l & 1) == !(l & 4));
  beam_step<4>(x, !(l & 4) == !(l & 8));
  beam_step<2>(x, !(l & 2) == !(l & 8));
  beam_step<1>(x, !(l & 1) == !(l & 8));
  beam_step<8>(x, !(l & 8) == !(l & 16));
  beam_step<4>(x, !(l & 4) == !(l & 16));
  beam_step<2>(x, !(l & 2) == !(l & 16));
  beam_step<1>(x, !(l & 1) == !(l & 16));
  beam_step<16>(x, !(l & 16) == !(l & 32));
  beam_step<8>(x, !(l & 8) == !(l & 32));
  beam_step<4>(x, !(l & 4) == !(l & 32));
  beam_step<2>(x, !(l & 2) == !(l & 32));
  beam_step<1>(x, !(l & 1) == !(l & 32));
  beam_merge(x);
}
// The lanes in the opposite order.
__device__ __forceinline__ uint32_t beam_turn(uint32_t x) { return __shfl(x, 63 - (int)(threadIdx.x & 63)); }
__device__ __forceinline__ uint64_t beam_turn(uint64_t x) { return __shfl(x, 63 - (int)(threadIdx.x & 63)); }
__device__ __forceinline__ BeamOffer beam_turn(BeamOffer x) {
  const int l = 63 - (int)(threadIdx.x & 63);
  return BeamOffer{(uint64_t)__shfl(x.key, l), (uint32_t)__shfl((int)x.place, l)};
}
// The 64 greatest of two sorted 64, `y` in the opposite order.
template <class K>
__device__ __forceinline__ void beam_join(K& x, const K& y) {
  if (x < y) x = y;
  beam_merge(x);
}

// Order of float values as unsigned numbers (both zeros alike), and back.
__device__ __forceinline__ uint32_t beam_order(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float beam_value(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ uint64_t beam_order(double x) {
  const uint64_t u = __double_as_longlong(x + 0.0);
  return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double beam_value(uint64_t u) {
  return __longlong_as_double(u & 0x8000000000000000ull ? u ^ 0x8000000000000000ull : ~u);
}

// A sum and exp(d), -700 <= d <= 0, to about 2^-52: 2^(n / 256) from a table times a
// polynomial of what is left, |r| <= ln 2 / 512, whose next term would be below
// 2^-54 (Tang, Table-driven implementation of the exponential function, 1989).
// n is rounded by adding 1.5 x 2^52, which leaves it in the low bits; the power
// of two goes to the table value's exponent, which d >= -700 keeps in range.
constexpr double kBeamFar = 700.0;  // what is farther below the largest counts as that far: e^-700
constexpr int kBeamTable = 256;
__device__ __forceinline__ void beam_table(double* table) {
  for (int i = threadIdx.x; i < kBeamTable; i += blockDim.x) table[i] = exp2(i / (double)kBeamTable);
}
__device__ __forceinline__ double beam_add(double sum, double d, const double* table) {  // sum + exp(d)
  constexpr double kRound = 6755399441055744.0;
  const double t = __builtin_fma(d, 369.3299304675746, kRound);  // 256 / ln 2
  const double r = __builtin_fma(t - kRound, -0.0027076061740622863, d);
  double p = __builtin_fma(r, 1.0 / 24, 1.0 / 6);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  const int k = (int)__double_as_longlong(t);
  const int64_t scale = (int64_t)((uint64_t)(uint32_t)(k >> 8) << 52);
  return __builtin_fma(p, __longlong_as_double(__double_as_longlong(table[k & (kBeamTable - 1)]) + scale), sum);
}
// exp(x - top); x may be -inf or NaN, top not.
__device__ __forceinline__ double beam_exp(float x, float top, const double* table) {
  return beam_add(0.0, __builtin_fmax((double)x - (double)top, -kBeamFar), table);
}

__device__ __forceinline__ double beam_sum(double x) {  // over the wave's lanes
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) x += __shfl_xor(x, s);
  return x;
}

// EACH: logits of a thread.  VEC: rows are 16-byte aligned and read 16 bytes at a time.
//
// What bounds it: the issue of vector instructions, 26 a logit, of which the
// exponential takes 17, most of them float64.  128 rows of 129,280 bf16 (33 MB)
// 18.2 us, 512 of float32 (265 MB) 68 us, 3.9 TB/s; 4 rows of 32,000 6.5 us, one
// wave's chain of a read and sorts.
template <class T, int EACH, bool VEC>
__global__ __launch_bounds__(kBeamThreads) void k_beam_slices(dsr_select_beams_args_t a) {
  constexpr int VE = VEC ? 16 / sizeof(T) : 1, C = EACH / VE;
  typedef T xv __attribute__((ext_vector_type(VE)));
  __shared__ double table[kBeamTable];
  __shared__ uint64_t list[kBeamWaves][kBeamList];
  __shared__ BeamPart part[kBeamWaves];
  const int V = (int)a.vocab, slices = (V + kBeamThreads * EACH - 1) / (kBeamThreads * EACH);
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t row = blockIdx.x / (unsigned)slices;
  const int slice = blockIdx.x - (unsigned)row * slices, first = slice * kBeamThreads * EACH;
  if (slice == 0 && threadIdx.x == 0) a.status[row] = DSR_OK;
  if (a.finished && a.finished[row]) return;
  const T* logits = (const T*)a.logits + row * a.ld;

  // Element e of the thread is token first + (e / VE * threads + thread) VE + e % VE.
  float x[EACH];
  auto token = [&](int e) { return first + (e / VE * kBeamThreads + (int)threadIdx.x) * VE + e % VE; };
  // No read stands behind a branch of its own (129,281 bf16 logits, which are read
  // one by one, 42 us where each did, 28 so), but in rows that end inside 16 bytes.
  if (V % VE == 0) {
    xv v[C];
#pragma unroll
    for (int c = 0; c < C; ++c) v[c] = *(const xv*)(logits + (token(c * VE) < V ? token(c * VE) : 0));
#pragma unroll
    for (int e = 0; e < EACH; ++e) x[e] = token(e / VE * VE) < V ? (float)v[e / VE][e % VE] : -INFINITY;
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = token(c * VE);
      if (at + VE <= V) {
        const xv v = *(const xv*)(logits + at);
#pragma unroll
        for (int i = 0; i < VE; ++i) x[c * VE + i] = (float)v[i];
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) x[c * VE + i] = at + i < V ? (float)logits[at + i] : -INFINITY;
      }
    }
  }
  beam_table(table);
  bool bad = false;
  float most = -INFINITY;
#pragma unroll
  for (int e = 0; e < EACH; e += 2) {
    bad |= __builtin_isunordered(x[e], x[e + 1]);
    most = fmaxf(most, fmaxf(x[e], x[e + 1]));
  }
  bad |= most == INFINITY;
  // The keep-th largest of the lanes' largest: at least `keep` of the wave's
  // logits are not below it, and few more.
  uint32_t tops = beam_order(most);
  beam_sort(tops);
  const float base = beam_value(__shfl(tops, 0)), least = fmaxf(beam_value(__shfl(tops, a.keep - 1)), -FLT_MAX);
  auto key_of = [&](float v, int e) { return (uint64_t)beam_order(v) << 32 | (uint32_t)~token(e); };
  int n = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const bool in = x[e] >= least;
    const uint64_t which = __ballot(in);
    if (which) {
      const int at = n + __popcll(which & ((1ull << l) - 1));
      if (in && at < kBeamList) list[w][at] = key_of(x[e], e);
      n += __popcll(which);
    }
  }
  uint64_t top = 0, floor = 0;
  auto take = [&](uint64_t key) __attribute__((always_inline)) {
    beam_sort(key);
    if (__ballot(top != 0))
      beam_join(top, beam_turn(key));
    else
      top = key;
    floor = __shfl(top, a.keep - 1);
  };
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  if (n <= kBeamList) {
#pragma unroll 1
    for (int i = 0; i < n; i += 64) take(i + l < n ? list[w][i + l] : 0);
  } else {
    // Hundreds of equal logits, or a few lanes with all the large ones: the
    // wave's logits once more, 64 at a time.
#pragma unroll 1
    for (int e = 0; e < EACH; ++e) {
      const int at = token(e);
      const float v = at < V ? (float)logits[at] : -INFINITY;
      const uint64_t key = v >= least ? key_of(v, e) : 0;
      if (__ballot(key > floor)) take(key);
    }
  }
  __syncthreads();  // the table
  double sum = 0.0;
  if (base > -INFINITY)
#pragma unroll
    for (int e = 0; e < EACH; ++e)
      sum = beam_add(sum, __builtin_fmax((double)x[e] - (double)base, -kBeamFar), table);
  sum = beam_sum(sum);
  const int wrong = __ballot(bad) != 0;
  list[w][l] = top;
  if (l == 0) part[w] = BeamPart{sum, base, wrong};
  __syncthreads();
  if (w > 0) return;
  const BeamSpace space = beam_space(a);
  const int64_t at = row * slices + slice;
#pragma unroll
  for (int i = 1; i < kBeamWaves; ++i) beam_join(top, list[i][63 - l]);
  if (l < a.keep) space.found[at * a.keep + l] = top;
  if (l == 0) {
    BeamPart p = part[0];
#pragma unroll
    for (int i = 1; i < kBeamWaves; ++i) {
      p.top = fmaxf(p.top, part[i].top);
      p.bad |= part[i].bad;
    }
    p.sum = 0.0;
    if (p.top > -INFINITY)
#pragma unroll
      for (int i = 0; i < kBeamWaves; ++i)
        p.sum += part[i].sum * beam_exp(part[i].top, p.top, table);
    space.parts[at] = p;
  }
}

// What bounds it: a chain of reads, a logarithm and sorts, with nothing to fill the
// chip beside (1 group of 4 rows 6.6 us, 64 of 8 9.8).  Eight waves share a group so
// that the chain is short: its rows' sums and the candidates go to all of them.
__global__ __launch_bounds__(kBeamGroupThreads) void k_beam_groups(dsr_select_beams_args_t a) {
  __shared__ double table[kBeamTable];
  __shared__ uint64_t keys[kBeamGroupWaves][64];
  __shared__ uint32_t places[kBeamGroupWaves][64];
  const int g = blockIdx.x, l = threadIdx.x & 63, w = threadIdx.x >> 6, slices = beam_slices(a), keep = a.keep;
  const int rows = (int)a.rows;
  int lo = a.offsets[g], hi = a.offsets[g + 1];
  lo = lo < 0 ? 0 : lo > rows ? rows : lo;
  hi = hi < lo ? lo : hi > rows ? rows : hi;
  const BeamSpace space = beam_space(a);
  beam_table(table);
  __syncthreads();
  // Candidates do not wait for the rows' sums: the first ones are on their way.
  const int each = slices * keep, count = (hi - lo) * each;
  const uint64_t* found = space.found + (int64_t)lo * each;
  uint64_t next = (int)threadIdx.x < count ? found[threadIdx.x] : 0;
  // A row's sum, a wave each, a slice a lane.
  for (int r = lo + w; r < hi; r += kBeamGroupWaves) {
    const double score = a.scores[r];
    const bool ended = a.finished && a.finished[r];
    int status = !(score < INFINITY) ? DSR_E_LOGITS : DSR_OK;
    BeamTerm term{0.0, 0.0, score};
    if (!ended) {
      const BeamPart* p = space.parts + (int64_t)r * slices;
      BeamPart mine{0.0, -INFINITY, 0};
      for (int s = l; s < slices; s += 64) {
        const BeamPart x = p[s];
        const float top = fmaxf(mine.top, x.top);
        if (top > -INFINITY && !(x.bad | mine.bad))
          mine.sum = mine.sum * beam_exp(mine.top, top, table) + x.sum * beam_exp(x.top, top, table);
        mine.top = top;
        mine.bad |= x.bad;
      }
      float top = mine.top;
#pragma unroll
      for (int s = 1; s < 64; s <<= 1) top = fmaxf(top, __shfl_xor(top, s));
      const bool bad = __ballot(mine.bad) != 0;
      if (bad)
        status = DSR_E_LOGITS;
      else if (top == -INFINITY && status == DSR_OK)
        status = DSR_E_MASKED;
      if (status == DSR_OK) {
        term.top = top;
        term.rest = log(beam_sum(mine.sum * beam_exp(mine.top, top, table)));
      }
    }
    if (status != DSR_OK) term.score = NAN;
    if (l == 0) {
      if (status != DSR_OK) a.status[r] = status;
      space.terms[r] = term;
    }
  }
  __threadfence_block();
  __syncthreads();

  // Candidates, 64 of a wave at a time, into its sorted `best`.
  BeamOffer best{0, 0}, last{0, 0};
#pragma unroll 1
  for (int i0 = 64 * w; i0 < count; i0 += kBeamGroupThreads) {
    const int i = i0 + l;
    const uint64_t now = next;
    next = i + kBeamGroupThreads < count ? found[i + kBeamGroupThreads] : 0;
    BeamOffer mine{0, 0};
    if (i < count) {
      const int r = (unsigned)i / (unsigned)each, in = i - r * each;
      const BeamTerm term = space.terms[lo + r];
      double score = NAN;
      if (a.finished && a.finished[lo + r]) {
        if (in == 0) score = term.score;
      } else if (now) {
        score = ((double)beam_value((uint32_t)(now >> 32)) - term.top) - term.rest + term.score;
      }
      if (score > -INFINITY) mine = BeamOffer{beam_order(score), ~(uint32_t)i};
    }
    if (!__ballot(last < mine)) continue;
    beam_sort(mine);
    if (__ballot(best.key != 0))
      beam_join(best, beam_turn(mine));
    else
      best = mine;
    last = BeamOffer{(uint64_t)__shfl(best.key, keep - 1), (uint32_t)__shfl((int)best.place, keep - 1)};
  }
#pragma unroll
  for (int half = kBeamGroupWaves / 2; half > 0; half /= 2) {
    if (w >= half && w < 2 * half) {
      keys[w][l] = best.key;
      places[w][l] = best.place;
    }
    __syncthreads();
    if (w < half) beam_join(best, BeamOffer{keys[w + half][63 - l], places[w + half][63 - l]});
  }
  if (w > 0 || l >= keep) return;
  const int64_t at = (int64_t)g * keep + l;
  int parent = -1, token = -1;
  if (best.key) {
    const uint32_t i = ~best.place, r = i / each;
    parent = lo + (int)r;
    if (!(a.finished && a.finished[parent]))
      token = (int)~(uint32_t)found[i];
  }
  a.parents[at] = parent;
  a.tokens[at] = token;
  a.out_scores[at] = best.key ? beam_value(best.key) : -INFINITY;
}

}  // namespace dsr
