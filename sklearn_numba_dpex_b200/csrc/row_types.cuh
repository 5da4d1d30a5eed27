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

}  // namespace kmb
