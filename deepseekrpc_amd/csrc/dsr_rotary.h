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
// pair and token against 2 x heads x 2 rows of traffic.
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

// VE elements per access: 16 bytes' worth when every row and part allows it, else one.
template <class T, int VE, bool PAIRS>
__global__ __launch_bounds__(kRotaryThreads) void k_rotary(dsr_rotary_args_t a) {
  typedef RotaryVec<T, VE> V;
  typedef typename V::type Vec;
  constexpr int IP = PAIRS ? (VE < 2 ? 1 : VE / 2) : VE;  // pairs per item
  __shared__ float cs[DSR_ROTARY_MAX_DIM / 2], sn[DSR_ROTARY_MAX_DIM / 2];
  const int64_t n = blockIdx.x;
  const int half = a.rot_dim / 2;
  const int position = a.positions[n];
  const int slot = a.slots ? a.slots[n] : -1;
  for (int i = threadIdx.x; i < half; i += kRotaryThreads) {
    const double x = (double)position * a.freqs[i] * 0.31830988618379067154;  // half turns
    const double r = x - 2.0 * rint(0.5 * x);
    float s, c;
    sincospif((float)r, &s, &c);
    const float m = (float)a.magnitude;
    cs[i] = c * m;
    sn[i] = (a.inverse ? -s : s) * m;
  }
  const bool bad = slot < -1 || slot >= (int64_t)a.blocks * a.page;
  const bool cached = slot >= 0 && !bad;
  const int block = cached ? slot / a.page : 0, place = cached ? slot & (a.page - 1) : 0;
  if (a.status && blockIdx.y == 0 && threadIdx.x == 0) a.status[n] = bad ? DSR_E_BLOCK : DSR_OK;
  __syncthreads();

  const int turned = half / IP;  // items of a row that turn
  const int per = turned + (a.head_dim - a.rot_dim) / VE;
  const int per_v = a.v ? a.v_dim / VE : 0;
  const int q_items = a.q_heads * per, k_items = a.kv_heads * per;
  const int all = q_items + k_items + (a.v && cached ? a.kv_heads * per_v : 0);
  for (int i = blockIdx.y * kRotaryThreads + threadIdx.x; i < all; i += gridDim.y * kRotaryThreads) {
    const T* src;
    T *dst, *dst2 = nullptr;
    int item;
    if (i < q_items) {
      const int h = i / per;
      item = i - h * per;
      src = (const T*)a.q + n * a.q_token + h * a.q_head;
      dst = (T*)a.q_out + n * a.qo_token + h * a.qo_head;
    } else if (i < q_items + k_items) {
      const int j = i - q_items, h = j / per;
      item = j - h * per;
      src = (const T*)a.k + n * a.k_token + h * a.k_head;
      dst = a.k_out ? (T*)a.k_out + n * a.ko_token + h * a.ko_head : nullptr;
      if (cached && a.k_cache) dst2 = (T*)a.k_cache + block * a.kc_block + place * a.kc_token + h * a.kc_head;
    } else {
      const int j = i - q_items - k_items, h = j / per_v;
      item = per + j - h * per_v;
      src = (const T*)a.v + n * a.v_token + h * a.v_head;
      dst = (T*)a.v_cache + block * a.vc_block + place * a.vc_token + h * a.vc_head;
    }
    if (item >= turned) {  // dimensions that do not turn: one access
      int d = (item - turned) * VE;
      if (item >= per)
        d = (item - per) * VE;
      else if (d >= a.rot_start)
        d += a.rot_dim;
      const Vec x = *(const Vec*)(src + d);
      if (dst) *(Vec*)(dst + d) = x;
      if (dst2) *(Vec*)(dst2 + d) = x;
      continue;
    }
    if constexpr (PAIRS && VE >= 2) {
      const int d = a.rot_start + item * VE;
      const Vec x = *(const Vec*)(src + d);
      Vec y;
#pragma unroll
      for (int e = 0; e < IP; ++e) {
        const float c = cs[item * IP + e], s = sn[item * IP + e];
        const float p = V::get(x, 2 * e), q = V::get(x, 2 * e + 1);
        V::set(y, 2 * e, p * c - q * s);
        V::set(y, 2 * e + 1, p * s + q * c);
      }
      if (dst) *(Vec*)(dst + d) = y;
      if (dst2) *(Vec*)(dst2 + d) = y;
    } else {
      const int d = a.rot_start + (PAIRS ? 2 : VE) * item, d2 = d + (PAIRS ? 1 : half);
      Vec x = *(const Vec*)(src + d), y = *(const Vec*)(src + d2);
#pragma unroll
      for (int e = 0; e < IP; ++e) {
        const float c = cs[item * IP + e], s = sn[item * IP + e];
        const float p = V::get(x, e), q = V::get(y, e);
        V::set(x, e, p * c - q * s);
        V::set(y, e, p * s + q * c);
      }
      if (dst) {
        *(Vec*)(dst + d) = x;
        *(Vec*)(dst + d2) = y;
      }
      if (dst2) {
        *(Vec*)(dst2 + d) = x;
        *(Vec*)(dst2 + d2) = y;
      }
    }
  }
}

}  // namespace dsr
