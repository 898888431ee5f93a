// Elements of the arrays that entry points take by type: fp32, bf16 or fp16 in memory, fp32 in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/pssa_b200.h"

namespace pssa {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

inline size_t dtype_size(int dtype) { return dtype == PSSA_B200_F32 ? 4 : 2; }

// f(T()) for the type that `dtype` names
template <typename F>
inline auto with_dtype(int dtype, F f) {
    if (dtype == PSSA_B200_F32) return f(float());
    if (dtype == PSSA_B200_BF16) return f(__nv_bfloat16());
    return f(__half());
}

}  // namespace pssa
