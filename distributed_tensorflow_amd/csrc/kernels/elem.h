// Elements of fp32, bf16 and fp16 arrays in vectors at any alignment.
#pragma once

#include "common.h"

struct dtf_bf16 {
  unsigned short v;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(dtf_bf16 v) { return dtf_bf16_to_f32(v.v); }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ dtf_bf16 from_f32<dtf_bf16>(float v) { return dtf_bf16{dtf_f32_to_bf16(v)}; }
template <>
__device__ __forceinline__ _Float16 from_f32<_Float16>(float v) { return (_Float16)v; }

// 16 bytes at element alignment: rows of an odd width start anywhere, and the memory pipe takes
// such vectors as they are
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[N];
};

// elements [c, c + N) of a row of n: zero behind its end
template <int N, typename T>
__device__ __forceinline__ void load_part(const T* __restrict__ row, int c, int n, float* out) {
  if (c + N <= n) {
    const Pack<T, N> p = *reinterpret_cast<const Pack<T, N>*>(row + c);
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] = to_f32(p.v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) out[k] = c + k < n ? to_f32(row[c + k]) : 0.f;
  }
}

template <int N, typename T>
__device__ __forceinline__ void store_part(T* __restrict__ row, int c, int n, const float* v) {
  if (c + N <= n) {
    Pack<T, N> p;
#pragma unroll
    for (int k = 0; k < N; ++k) p.v[k] = from_f32<T>(v[k]);
    *reinterpret_cast<Pack<T, N>*>(row + c) = p;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (c + k < n) row[c + k] = from_f32<T>(v[k]);
  }
}
