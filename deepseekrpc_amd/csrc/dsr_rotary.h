// Rotary positions of a step's queries and keys, keys and values written to
// their cache slots (dsr_rotary).
//
// One pass: every row is read once and written once (keys twice if both an
// array and a cache take them).  A workgroup takes one token, or a share of
// its rows when there are few tokens; it computes the token's cosines and
// sines once into LDS for all heads, each angle reduced to (-1, 1] half turns
// in float64 first, so that the sine of a position in the millions is as
// good as that of a small one (float32 angles are 0.06 radians apart there).
// What bounds it is memory traffic; the trigonometry is one sincospi per
// pair and token against 2 x heads x 2 rows of traffic.  A thread reads its
// first rows before the angles and each further ones before it writes: 8,192
// tokens of 64 + 8 + 8 heads of 128 in bf16 take 65 us (5.2 TB/s; 85 us when
// rows are read behind the angles, 64 to 66 with two or three items ahead).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dsr_tree.h"

namespace dsr {

constexpr int kRotaryThreads = 256;

template <class T, int N>
struct RotaryVec {
  typedef T type __attribute__((ext_vector_type(N)));
  static __device__ __forceinline__ float get(const type& x, int e) { return (float)x[e]; }
  static __device__ __forceinline__ void set(type& x, int e, float y) { x[e] = (T)y; }
};
template <class T>
struct RotaryVec<T, 1> {
  typedef T type;
  static __device__ __forceinline__ float get(const T& x, int) { return (float)x; }
  static __device__ __forceinline__ void set(T& x, int, float y) { x = (T)y; }
};

// VE elements per access: 16 bytes' worth when every row and part allows it,
// else 8 bytes' worth, else one (8,192 tokens of 80 rows of 128 in bf16: 64 us,
// one by one 125; with the first 24 dimensions turned by halves 85 in 8 bytes,
// 182 one by one).
template <class T, int VE, bool PAIRS>
__global__ __launch_bounds__(kRotaryThreads) void k_rotary(dsr_rotary_args_t a) {
  typedef RotaryVec<T, VE> V;
  typedef typename V::type Vec;
  constexpr int IP = PAIRS ? (VE < 2 ? 1 : VE / 2) : VE;  // pairs per item
  constexpr bool ONE = PAIRS && VE >= 2;                  // an item's pairs lie in one access
  __shared__ float cs[DSR_ROTARY_MAX_DIM / 2], sn[DSR_ROTARY_MAX_DIM / 2];
  const int64_t n = blockIdx.x;
  const int half = a.rot_dim / 2;
  const int position = a.positions[n];
  const int slot = a.slots ? a.slots[n] : -1;
  const bool bad = slot < -1 || slot >= (int64_t)a.blocks * a.page;
  const bool cached = slot >= 0 && !bad;
  const int block = cached ? slot / a.page : 0, place = cached ? slot & (a.page - 1) : 0;
  if (a.status && blockIdx.y == 0 && threadIdx.x == 0) a.status[n] = bad ? DSR_E_BLOCK : DSR_OK;

  const int turned = half / IP;  // items of a row that turn
  const int per = turned + (a.head_dim - a.rot_dim) / VE;
  const int per_v = a.v ? a.v_dim / VE : 0;
  const int q_items = a.q_heads * per, k_items = a.kv_heads * per;
  const int all = q_items + k_items + (a.v && cached ? a.kv_heads * per_v : 0);
  struct Item {
    Vec x, y;
    T *dst, *dst2;  // null: not written
    int item, d, d2;
  };
  auto fetch = [&](Item& u, int i) __attribute__((always_inline)) {
    const T* src;
    u.dst2 = nullptr;
    if (i < q_items) {
      const int h = i / per;
      u.item = i - h * per;
      src = (const T*)a.q + n * a.q_token + h * a.q_head;
      u.dst = (T*)a.q_out + n * a.qo_token + h * a.qo_head;
    } else if (i < q_items + k_items) {
      const int j = i - q_items, h = j / per;
      u.item = j - h * per;
      src = (const T*)a.k + n * a.k_token + h * a.k_head;
      u.dst = a.k_out ? (T*)a.k_out + n * a.ko_token + h * a.ko_head : nullptr;
      if (cached && a.k_cache) u.dst2 = (T*)a.k_cache + block * a.kc_block + place * a.kc_token + h * a.kc_head;
    } else {
      const int j = i - q_items - k_items, h = j / per_v;
      u.item = per + j - h * per_v;
      src = (const T*)a.v + n * a.v_token + h * a.v_head;
      u.dst = (T*)a.v_cache + block * a.vc_block + place * a.vc_token + h * a.vc_head;
    }
    if (u.item >= per) {
      u.d = (u.item - per) * VE;
    } else if (u.item >= turned) {  // dimensions that do not turn
      u.d = (u.item - turned) * VE;
      if (u.d >= a.rot_start) u.d += a.rot_dim;
    } else {
      u.d = a.rot_start + (PAIRS ? (VE < 2 ? 2 : VE) : VE) * u.item;
    }
    u.d2 = u.d + (PAIRS ? 1 : half);
    u.x = *(const Vec*)(src + u.d);
    if (!ONE && u.item < turned) u.y = *(const Vec*)(src + u.d2);
  };
  auto finish = [&](Item& u) __attribute__((always_inline)) {
    if (u.item < turned) {
#pragma unroll
      for (int e = 0; e < IP; ++e) {
        const float c = cs[u.item * IP + e], s = sn[u.item * IP + e];
        if constexpr (ONE) {
          const float p = V::get(u.x, 2 * e), q = V::get(u.x, 2 * e + 1);
          V::set(u.x, 2 * e, p * c - q * s);
          V::set(u.x, 2 * e + 1, p * s + q * c);
        } else {
          const float p = V::get(u.x, e), q = V::get(u.y, e);
          V::set(u.x, e, p * c - q * s);
          V::set(u.y, e, p * s + q * c);
        }
      }
    }
    const bool both = !ONE && u.item < turned;
    if (u.dst) {
      *(Vec*)(u.dst + u.d) = u.x;
      if (both) *(Vec*)(u.dst + u.d2) = u.y;
    }
    if (u.dst2) {
      *(Vec*)(u.dst2 + u.d) = u.x;
      if (both) *(Vec*)(u.dst2 + u.d2) = u.y;
    }
  };

  // Every item is read before the last one is written, the first before the angles.
  const int step = gridDim.y * kRotaryThreads;
  int i = blockIdx.y * kRotaryThreads + threadIdx.x;
  Item now, next;
  if (i < all) fetch(now, i);
  for (int k = threadIdx.x; k < half; k += kRotaryThreads) {
    const double x = (double)position * a.freqs[k] * 0.31830988618379067154;  // half turns
    const double r = x - 2.0 * rint(0.5 * x);
    float s, c;
    sincospif((float)r, &s, &c);
    const float m = (float)a.magnitude;
    cs[k] = c * m;
    sn[k] = (a.inverse ? -s : s) * m;
  }
  __syncthreads();
  for (; i < all; i += step) {
    if (i + step < all) fetch(next, i + step);
    finish(now);
    now = next;
  }
}

}  // namespace dsr
