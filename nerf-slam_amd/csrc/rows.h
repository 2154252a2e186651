// rows.h -- pieces shared by the row operators (embedding.hip, layer_norm.hip): a row of features is D elements of f16, bf16 or f32
// that follow each other in memory; rows are `stride` elements apart.  Every lane moves 16 bytes of a row at a time.
#pragma once
#include "common.h"

typedef __bf16 rw_bf16;

// elements of T in 16 bytes: what a lane holds of a row
template <typename T>
constexpr int row_vec() { return 16 / (int)sizeof(T); }

// N elements of T as they lie in memory.  Loads and stores go through memcpy, so that they only assume the alignment of an element:
// gfx950 takes 16-byte accesses at any address, and rows of an odd length need no kernel of their own.
template <typename T, int N>
struct RowPiece {
  T e[N];
};

template <typename T, int N>
__device__ __forceinline__ RowPiece<T, N> row_get(const T* __restrict__ at) {
  RowPiece<T, N> v;
  __builtin_memcpy(&v, at, sizeof(v));
  return v;
}

// STREAM: stores that are not kept in the caches, for outputs that nothing reads while the kernel runs
template <typename T, int N, bool STREAM>
__device__ __forceinline__ void row_put(T* __restrict__ at, const float* f) {
  typedef int v4i __attribute__((ext_vector_type(4), aligned(2)));     // (an element may be 2 bytes)
  RowPiece<T, N> v;
#pragma unroll
  for (int i = 0; i < N; i++) v.e[i] = (T)f[i];
  if constexpr (STREAM && sizeof(v) % 16 == 0) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(v) / 16; i++) {
      v4i q;
      __builtin_memcpy(&q, (const char*)&v + 16 * i, 16);
      __builtin_nontemporal_store(q, reinterpret_cast<v4i*>(at) + i);
    }
  } else {
    __builtin_memcpy(at, &v, sizeof(v));
  }
}

// the 16 bytes become opaque to the compiler: what is computed from them again is not kept from the first time
template <typename T, int N>
__device__ __forceinline__ void row_pin(RowPiece<T, N>& v) {
  typedef int v4i __attribute__((ext_vector_type(4)));
  if constexpr (sizeof(v) == sizeof(v4i)) {
    v4i q;
    __builtin_memcpy(&q, &v, sizeof(q));
    asm volatile("" : "+v"(q));
    __builtin_memcpy(&v, &q, sizeof(q));
  }
}

static inline bool row_aligned(const void* p, int dtype) { return (uintptr_t)p % (dtype == NS_F32 ? 4 : 2) == 0; }

// lanes that share a row: the power of two that covers its 16-byte pieces, at least 1, at most 64
static inline int row_lanes_log2(int D, int vec) {
  const int pieces = (D + vec - 1) / vec;
  int s = 0;
  while (s < 6 && (1 << s) < pieces) s++;
  return s;
}
