// Rows in 16 or 32 bits (KMB_F32, KMB_F16, KMB_BF16), computed with in 32 bits.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kmb_common.cuh"

namespace kmb {

// Runs `body` with T bound to float, __half or __nv_bfloat16.
#define KMB_DISPATCH_ROWS(dtype, ...)                                                           \
  do {                                                                                          \
    if ((dtype) == KMB_F32) {                                                                   \
      using T = float;                                                                          \
      __VA_ARGS__                                                                               \
    } else if ((dtype) == KMB_F16) {                                                            \
      using T = __half;                                                                         \
      __VA_ARGS__                                                                               \
    } else if ((dtype) == KMB_BF16) {                                                           \
      using T = __nv_bfloat16;                                                                  \
      __VA_ARGS__                                                                               \
    } else {                                                                                    \
      kmb::set_error("dtype must be KMB_F32, KMB_F16 or KMB_BF16, got %d", (int)(dtype));       \
      return KMB_ERR_INVALID;                                                                   \
    }                                                                                           \
  } while (0)

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Whether rows of d elements can be read in 16-byte pieces.
template <typename T>
inline bool rows_are_vec(const T* x, int64_t d) {
  return ((uintptr_t)x & 15) == 0 && (d * sizeof(T)) % 16 == 0;
}

// v[j] = p[f + j] for f + j < d, else 0; `vec`: rows_are_vec holds and f is a multiple of 8.
template <typename T>
__device__ __forceinline__ void load_vec8(const T* __restrict__ p, int f, int d, bool vec, float (&v)[8]) {
  if (vec && f + 8 <= d) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p + f);
      const float4 b = *reinterpret_cast<const float4*>(p + f + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      union { uint4 u; T t[8]; } r;
      r.u = *reinterpret_cast<const uint4*>(p + f);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_float(r.t[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f + j < d ? to_float(p[f + j]) : 0.f;
  }
}

// p[f + j] = v[j] for f + j < d, rounded to T.
template <typename T>
__device__ __forceinline__ void store_vec8(T* __restrict__ p, int f, int d, bool vec, const float (&v)[8]) {
  if (vec && f + 8 <= d) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p + f) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + f + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      union { uint4 u; T t[8]; } r;
#pragma unroll
      for (int j = 0; j < 8; ++j) r.t[j] = from_float<T>(v[j]);
      *reinterpret_cast<uint4*>(p + f) = r.u;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (f + j < d) p[f + j] = from_float<T>(v[j]);
  }
}

}  // namespace kmb
