// Element types, vector access and lane-group sums of the sequence-block kernels.
#pragma once
#include <algorithm>
#include <type_traits>

#include "../sb_common.h"
#include "../../../include/sound_bubble_seq.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// V elements behind one pointer that is aligned to its element only: gfx950 takes unaligned global accesses, so rows of odd
// lengths and sliced tensors keep their 16-byte loads
template <class T, int V> struct Vec { T v[V]; };
template <class T, int V> SB_DEVINL Vec<T, V> vload(const T* p) {
  Vec<T, V> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <class T, int V> SB_DEVINL void vstore(T* p, const Vec<T, V>& r) { __builtin_memcpy(p, &r, sizeof(r)); }
// the first n of V elements, n in 0 .. V (rest: zero / not written)
template <class T, int V> SB_DEVINL Vec<T, V> vload_n(const T* p, int n) {
  if (n >= V) return vload<T, V>(p);
  Vec<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
  return r;
}
template <class T, int V> SB_DEVINL void vstore_n(T* p, const Vec<T, V>& r, int n) {
  if (n >= V) {
    vstore<T, V>(p, r);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) p[i] = r.v[i];
}
template <class T> constexpr int vec_of() { return 16 / (int)sizeof(T); }

// sum over groups of L lanes (L a power of two up to 64), every lane gets it: the order of additions is the lanes' alone
template <int L> SB_DEVINL float lane_sum(float v) {
  if constexpr (L >= 2) v = dpp_add<0xB1>(v);     // quad_perm [1,0,3,2]
  if constexpr (L >= 4) v = dpp_add<0x4E>(v);     // quad_perm [2,3,0,1]
  if constexpr (L >= 8) v = dpp_add<0x141>(v);    // row_half_mirror
  if constexpr (L >= 16) v = dpp_add<0x140>(v);   // row_mirror
  if constexpr (L >= 32) v += __shfl_xor(v, 16, 64);
  if constexpr (L >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// calls f(type tag) for an element type; -1000-x is the caller's
template <class F> static int sb_with_type(int t, F&& f) {
  switch (t) {
    case SB_F32: return f((float*)nullptr);
    case SB_BF16: return f((bf16_t*)nullptr);
    case SB_F16: return f((f16_t*)nullptr);
    default: return -1001;
  }
}
