// Element types of the operators that take activations in more than one type (B200_F32, B200_BF16, B200_F16): loads give
// fp32, stores round once to nearest even.  All arithmetic in between is fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include "../../include/b200conv.h"

namespace b200 {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

inline size_t type_size(int type) { return type == B200_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == B200_F32 || type == B200_BF16 || type == B200_F16; }
// a tensor of this type may start at any multiple of its element size
inline bool element_aligned(const void *p, int type) { return (reinterpret_cast<uintptr_t>(p) & (type_size(type) - 1)) == 0; }

}  // namespace b200
