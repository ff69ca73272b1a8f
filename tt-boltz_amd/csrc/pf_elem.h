// Element types of the operators that work in the caller's own type (fp32, fp16, bf16) rather than
// in the build's operand type: these sources are compiled once and linked into both libraries.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pf_internal.h"

#define PF_DEV __device__ __forceinline__

typedef _Float16 half_t;
typedef __bf16 bhalf_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// 16 bytes of elements: the widest global access
template <typename T>
struct Vec16 {
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(N)));
};

// N consecutive elements as floats; N is 1, or 4 or 8 of at most 16 bytes, aligned to their size
template <typename T, int N>
PF_DEV void load_elems(const T* p, float (&x)[N]) {
  if constexpr (N == 1) {
    x[0] = (float)p[0];
  } else {
    typedef T vec_t __attribute__((ext_vector_type(N)));
    const vec_t v = *reinterpret_cast<const vec_t*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)v[i];
  }
}

template <typename T, int N>
PF_DEV void store_elems(T* p, const float (&x)[N]) {
  if constexpr (N == 1) {
    p[0] = (T)x[0];
  } else {
    typedef T vec_t __attribute__((ext_vector_type(N)));
    vec_t v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
    *reinterpret_cast<vec_t*>(p) = v;
  }
}

inline bool pf_aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
inline int pf_elem_size(int dtype) { return dtype == PF_FP32 ? 4 : 2; }
