// Element types of the operators that take rows in 32 or 16 bits (GS_TYPE_* of gslim.h), and how their kernels read and write them.
#pragma once
#include "gs_common.h"

template <int T>
struct GsElt;
template <>
struct GsElt<GS_TYPE_F32> {
  typedef float type;
};
template <>
struct GsElt<GS_TYPE_F16> {
  typedef _Float16 type;
};
template <>
struct GsElt<GS_TYPE_BF16> {
  typedef __bf16 type;
};

// N elements that are aligned to one element only: a row of odd width starts anywhere, and the global memory path takes 16-byte
// accesses at any element's address (a wave's access then touches one cache line more).
template <typename E, int N>
struct GsVec {
  typedef E type __attribute__((ext_vector_type(N), aligned(sizeof(E))));
};
template <typename E>
struct GsVec<E, 1> {
  typedef E type;
};

// p[0 .. N) as floats, the elements from `n` on as `fill`
template <typename E, int N>
__device__ __forceinline__ void gs_load(const E* __restrict__ p, long n, float fill, float* __restrict__ v) {
  if (n >= N) {
    const typename GsVec<E, N>::type r = *(const typename GsVec<E, N>::type*)p;
    if constexpr (N == 1) {
      v[0] = (float)r;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (float)r[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : fill;
  }
}

template <typename E, int N>
__device__ __forceinline__ void gs_store(E* __restrict__ p, long n, const float* __restrict__ v) {
  if (n >= N) {
    typename GsVec<E, N>::type r;
    if constexpr (N == 1) {
      r = (E)v[0];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = (E)v[i];
    }
    *(typename GsVec<E, N>::type*)p = r;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (E)v[i];
  }
}

// the same past the caches, for what is read again only after more than they hold
template <typename E, int N>
__device__ __forceinline__ void gs_store_past(E* __restrict__ p, long n, const float* __restrict__ v) {
  if (n >= N) {
    typename GsVec<E, N>::type r;
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (E)v[i];
    __builtin_nontemporal_store(r, (typename GsVec<E, N>::type*)p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (E)v[i];
  }
}

// N elements that are read once, past the caches
template <typename E, int N>
__device__ __forceinline__ typename GsVec<E, N>::type gs_load_past(const E* __restrict__ p) {
  return __builtin_nontemporal_load((const typename GsVec<E, N>::type*)p);
}

// A matrix in memory, in bytes.  What a call writes must not lie on what it reads: workgroups run in any order.
struct GsSpan {
  const void* p;
  long rows, ld, cols;
};
static inline GsSpan gs_span(const void* p, long rows, long ld, long cols, int bytes) { return {p, rows, ld * bytes, cols * bytes}; }
static inline GsSpan gs_span(const void* p, long n, int bytes) { return {p, 1, n * bytes, n * bytes}; }

static inline bool gs_overlap(const GsSpan& a, const GsSpan& b) {
  if (!a.p || !b.p || a.rows < 1 || b.rows < 1 || a.cols < 1 || b.cols < 1) return false;
  const long d = (long)((size_t)b.p - (size_t)a.p);
  if (d >= (a.rows - 1) * a.ld + a.cols || -d >= (b.rows - 1) * b.ld + b.cols) return false;
  if ((a.rows > 1 && b.rows > 1 && a.ld != b.ld) || (a.rows == 1 && b.rows == 1)) return true;
  const long ld = a.rows > 1 ? a.ld : b.ld, at = (d % ld + ld) % ld;     // columns of one matrix side by side lie apart
  return at < a.cols || at + b.cols > ld;
}

static inline int gs_type_bytes(int t) { return t == GS_TYPE_F32 ? 4 : (t == GS_TYPE_F16 || t == GS_TYPE_BF16 ? 2 : 0); }
