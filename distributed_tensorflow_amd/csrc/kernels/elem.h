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

// N elements as fp32 and back, rounded to nearest even. The 16-bit types go two to a register:
// one operation per bf16 element in, one per two out (v_cvt_pk_bf16_f32).
template <typename T, int N>
__device__ __forceinline__ void unpack(const Pack<T, N>& p, float* out) {
#pragma unroll
  for (int k = 0; k < N; ++k) out[k] = to_f32(p.v[k]);
}
template <int N>
__device__ __forceinline__ void unpack(const Pack<dtf_bf16, N>& p, float* out) {
  static_assert(N % 2 == 0, "pairs");
  struct Words {
    unsigned w[N / 2];
  };
  const Words q = __builtin_bit_cast(Words, p);
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    out[2 * k] = __uint_as_float(q.w[k] << 16);
    out[2 * k + 1] = __uint_as_float(q.w[k] & 0xffff0000u);
  }
}
template <int N>
__device__ __forceinline__ Pack<float, N> pack(const float* v, float) {
  Pack<float, N> p;
#pragma unroll
  for (int k = 0; k < N; ++k) p.v[k] = v[k];
  return p;
}
template <int N>
__device__ __forceinline__ Pack<_Float16, N> pack(const float* v, _Float16) {
  Pack<_Float16, N> p;
#pragma unroll
  for (int k = 0; k < N; ++k) p.v[k] = (_Float16)v[k];
  return p;
}
template <int N>
__device__ __forceinline__ Pack<dtf_bf16, N> pack(const float* v, dtf_bf16) {
  static_assert(N % 2 == 0, "pairs");
  struct Words {
    unsigned w[N / 2];
  } q;
#pragma unroll
  for (int k = 0; k < N / 2; ++k) q.w[k] = dtf_f32x2_to_bf16x2(v[2 * k], v[2 * k + 1]);
  return __builtin_bit_cast(Pack<dtf_bf16, N>, q);
}

// elements [c, c + N) of a row of n: zero behind its end
template <int N, typename T>
__device__ __forceinline__ Pack<T, N> load_raw(const T* __restrict__ row, int c, int n) {
  Pack<T, N> p;
  if (c + N <= n) {
    p = *reinterpret_cast<const Pack<T, N>*>(row + c);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) p.v[k] = c + k < n ? row[c + k] : T();
  }
  return p;
}
template <int N, typename T>
__device__ __forceinline__ void load_part(const T* __restrict__ row, int c, int n, float* out) {
  unpack(load_raw<N>(row, c, n), out);
}

template <int N, typename T>
__device__ __forceinline__ void store_part(T* __restrict__ row, int c, int n, const float* v) {
  if (c + N <= n) {
    *reinterpret_cast<Pack<T, N>*>(row + c) = pack<N>(v, T());
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (c + k < n) row[c + k] = from_f32<T>(v[k]);
  }
}
