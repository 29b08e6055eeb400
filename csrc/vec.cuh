// Element types and vector accesses shared by the bandwidth-bound kernels whose operands
// come in fp32, bf16 or fp16 and at any alignment.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace revpp {

template <int BYTES>
struct RawOf;
template <>
struct RawOf<16> { using type = uint4; };
template <>
struct RawOf<8> { using type = uint2; };
template <>
struct RawOf<4> { using type = uint32_t; };
template <>
struct RawOf<2> { using type = unsigned short; };

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// V elements in one access; p is aligned to V * sizeof(T) <= 16 bytes.
template <typename T, int V>
struct Pack {
  using Raw = typename RawOf<V * static_cast<int>(sizeof(T))>::type;
  Raw raw;
  __device__ __forceinline__ static Pack load(const T* p) { return Pack{*reinterpret_cast<const Raw*>(p)}; }
  __device__ __forceinline__ static Pack load_ro(const T* p) { return Pack{__ldg(reinterpret_cast<const Raw*>(p))}; }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void get(float (&f)[V]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f32(e[i]);
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f32<T>(f[i]);
  }
};

// V floats from / to an address aligned to min(V, 4) * 4 bytes.
template <int V>
__device__ __forceinline__ void load_f32(const float* p, float (&f)[V]) {
  constexpr int C = V < 4 ? V : 4;
#pragma unroll
  for (int i = 0; i < V; i += C) {
    float t[C];
    Pack<float, C>::load_ro(p + i).get(t);
#pragma unroll
    for (int j = 0; j < C; ++j) f[i + j] = t[j];
  }
}
template <int V>
__device__ __forceinline__ void store_f32(float* p, const float (&f)[V]) {
  constexpr int C = V < 4 ? V : 4;
#pragma unroll
  for (int i = 0; i < V; i += C) {
    float t[C];
#pragma unroll
    for (int j = 0; j < C; ++j) t[j] = f[i + j];
    Pack<float, C> v;
    v.set(t);
    v.store(p + i);
  }
}

}  // namespace revpp
