// dpt_dev.h - types and small device helpers shared by the training kernels (gfx950, 64-wide waves).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../../include/train/diffphore_train.h"

namespace dpt {

typedef __attribute__((ext_vector_type(4))) float f4;
typedef __attribute__((ext_vector_type(16))) float f16v;
typedef __attribute__((ext_vector_type(4))) short s4;
typedef __attribute__((ext_vector_type(4))) __bf16 b4;
typedef __attribute__((ext_vector_type(8))) __bf16 b8;

// N consecutive elements as floats, by loads of up to 16 bytes (the caller has checked the alignment) or one by one
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* __restrict__ p, float* o) {
  typedef __attribute__((ext_vector_type(N))) T vec;
  if constexpr (N == 1) {
    o[0] = (float)*p;
  } else if constexpr (N * sizeof(T) > 16) {
    load_n<T, N / 2>(p, o);
    load_n<T, N / 2>(p + N / 2, o + N / 2);
  } else {
    const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (float)v[i];
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* __restrict__ p, const float* o) {
  typedef __attribute__((ext_vector_type(N))) T vec;
  if constexpr (N == 1) {
    *p = (T)o[0];
  } else if constexpr (N * sizeof(T) > 16) {
    store_n<T, N / 2>(p, o);
    store_n<T, N / 2>(p + N / 2, o + N / 2);
  } else {
    vec v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)o[i];
    *reinterpret_cast<vec*>(p) = v;
  }
}

// sum over groups of L lanes (L a power of two up to 64), the same bits in every lane
template <int L>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int d = 1; d < L; d <<= 1) x += __shfl_xor(x, d, 64);
  return x;
}

}  // namespace dpt
