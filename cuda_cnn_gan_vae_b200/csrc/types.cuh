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

// Two fp32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}

// two values rounded in one instruction, the first in the lower half
__device__ __forceinline__ uint32_t from_float2(float2 v, __nv_bfloat16)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t from_float2(float2 v, __half)
{
    const __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// V neighbouring values: one, or 8 or 16 bytes of them at a multiple of that
template <typename T, int V> struct alignas(V * sizeof(T)) Pack { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T *p)
{
    Pack<T, V> r;
    if constexpr (V == 1) r.v[0] = *p;
    else if constexpr (V * sizeof(T) == 8) *reinterpret_cast<uint2 *>(r.v) = *reinterpret_cast<const uint2 *>(p);
    else *reinterpret_cast<uint4 *>(r.v) = *reinterpret_cast<const uint4 *>(p);
    return r;
}
template <typename T, int V> __device__ __forceinline__ void store_pack(T *p, const float *f)
{
    if constexpr (V == 1) {
        *p = from_float<T>(f[0]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
        uint32_t w[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; i++) w[i] = from_float2(make_float2(f[2 * i], f[2 * i + 1]), T());
        if constexpr (V == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
template <typename T> constexpr int kWide = 16 / (int)sizeof(T);

inline size_t type_size(int type) { return type == B200_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == B200_F32 || type == B200_BF16 || type == B200_F16; }
// whether rows of n values can be read in 16-byte pieces
inline bool wide_rows(const void *p, int type, size_t n, size_t pitch)
{
    const size_t per = 16 / type_size(type);
    return !(reinterpret_cast<uintptr_t>(p) & 15) && n % per == 0 && pitch % per == 0;
}
// a tensor of this type may start at any multiple of its element size
inline bool element_aligned(const void *p, int type) { return (reinterpret_cast<uintptr_t>(p) & (type_size(type) - 1)) == 0; }

}  // namespace b200
