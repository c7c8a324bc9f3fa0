// 8 neighbouring elements of a row that may start at any element, or the first n
// of them.  The vector types carry the alignment of one element, so the compiler
// may use wide accesses only as the target allows them unaligned (gfx950's
// global memory does), and rows of odd widths need no kernel of their own.
//
// A row's ragged end: where lanes of one wave take different paths in load(),
// the element path writes registers that the other lanes' wide load still has
// to fill, and the wave waits for it -- one load in flight instead of many.  So
// n should be the same for all lanes: kernels that keep many rows in flight let
// the last chunk of a row overlap the one before it instead (rows of 8 and more).
#pragma once
#include "zk_common.h"

namespace zk {

template <typename T>
struct Part8 {
  typedef T V8 __attribute__((ext_vector_type(8)));
  typedef V8 V8u __attribute__((aligned(sizeof(T))));
  V8 u;
  template <bool kOnce>  // kOnce: read once, not worth a place in the caches
  __device__ __forceinline__ void get(const T* p, int n) {
    if (kOnce && n >= 8) u = __builtin_nontemporal_load(reinterpret_cast<const V8u*>(p));
    else load(p, n);
  }
  // the first n (<= 8) elements at p; the others are zero
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= 8) {
      u = *reinterpret_cast<const V8u*>(p);
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = i < n ? p[i] : static_cast<T>(0.f);
  }
  __device__ __forceinline__ float operator[](int i) const { return static_cast<float>(u[i]); }
  static __device__ __forceinline__ void store(T* p, const float (&v)[8], int n) {
    if (n >= 8) {
      V8 w;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = static_cast<T>(v[i]);
      *reinterpret_cast<V8u*>(p) = w;
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = static_cast<T>(v[i]);
  }
};

}  // namespace zk
