// Element types of the kernels that take fp32, bf16 and fp16: fp32 <-> T, and
// four or eight elements at a time.
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"

namespace pvb2 {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

// one rounding, to nearest even
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}

template <int BYTES>
struct RawVec;
template <>
struct RawVec<32> {
  uint4 a, b;
};
template <>
struct RawVec<16> {
  uint4 a;
};
template <>
struct RawVec<8> {
  uint2 a;
};

// N consecutive elements from an address aligned to min(16, N * sizeof(T))
template <int N, typename T>
__device__ __forceinline__ void load_vec(const T* p, float* v) {
  union {
    RawVec<N * sizeof(T)> raw;
    T e[N];
  } u;
  u.raw = *reinterpret_cast<const RawVec<N * sizeof(T)>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = to_f32(u.e[i]);
}

template <int N, typename T>
__device__ __forceinline__ void unpack_vec(const RawVec<N * sizeof(T)>& raw, float* v) {
  union U {
    RawVec<N * sizeof(T)> raw;
    T e[N];
    __device__ U() {}
  } u;
  u.raw = raw;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = to_f32(u.e[i]);
}

template <int N, typename T>
__device__ __forceinline__ void store_vec(T* p, const float* v) {
  union U {
    RawVec<N * sizeof(T)> raw;
    T e[N];
    __device__ U() {}
  } u;
#pragma unroll
  for (int i = 0; i < N; ++i) u.e[i] = from_f32<T>(v[i]);
  *reinterpret_cast<RawVec<N * sizeof(T)>*>(p) = u.raw;
}

}  // namespace pvb2
