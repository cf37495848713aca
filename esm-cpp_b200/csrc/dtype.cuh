// Element types of the serving kernels: float, half and bfloat16 rows read as
// float32 and rounded to nearest even once when written.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace esmb200 {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Element i of an array whose type is known at run time (DType).
__device__ __forceinline__ float load_typed(const void* p, long i, int type) {
  if (type == 0) return __ldg(static_cast<const float*>(p) + i);
  if (type == 1) return to_f32(static_cast<const __half*>(p)[i]);
  return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
}

// V consecutive elements, as 16-byte (or smaller) accesses; p is aligned to
// min(16, V * sizeof(T)).
template <typename T, int V>
struct Vec {
  static constexpr int kBytes = V * static_cast<int>(sizeof(T));
  static constexpr int kWord = kBytes >= 16 ? 16 : kBytes;
  static constexpr int kWords = kBytes / kWord;
  alignas(kWord) T e[V];

  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWord == 16) {
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (kWord == 8) {
      *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kWord == 16) {
#pragma unroll
      for (int i = 0; i < kWords; ++i)
        reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
    } else if constexpr (kWord == 8) {
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) p[i] = e[i];
    }
  }
};

}  // namespace esmb200
