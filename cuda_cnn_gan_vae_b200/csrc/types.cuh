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

// V neighbouring values (V = 1, or the number in 16 bytes: the address is then a multiple of 16)
template <typename T, int V> struct alignas(V == 1 ? sizeof(T) : 16) Pack { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T *p)
{
    Pack<T, V> r;
    if constexpr (V == 1) r.v[0] = *p;
    else *reinterpret_cast<uint4 *>(r.v) = *reinterpret_cast<const uint4 *>(p);
    return r;
}
template <typename T, int V> __device__ __forceinline__ void store_pack(T *p, const float *f)
{
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; i++) r.v[i] = from_float<T>(f[i]);
    if constexpr (V == 1) *p = r.v[0];
    else *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(r.v);
}
template <typename T> constexpr int kWide = 16 / (int)sizeof(T);

inline size_t type_size(int type) { return type == B200_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == B200_F32 || type == B200_BF16 || type == B200_F16; }
// a tensor of this type may start at any multiple of its element size
// whether rows of n values can be read in 16-byte pieces
inline bool wide_rows(const void *p, int type, size_t n, size_t pitch)
{
    const size_t per = 16 / type_size(type);
    return !(reinterpret_cast<uintptr_t>(p) & 15) && n % per == 0 && pitch % per == 0;
}
inline bool element_aligned(const void *p, int type) { return (reinterpret_cast<uintptr_t>(p) & (type_size(type) - 1)) == 0; }

}  // namespace b200
