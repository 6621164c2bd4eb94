// The 8-bit form of an activation tensor as device functions: a row is cut into blocks of 32 values, a block has one exponent
// byte b and a signed byte q per value, and q stands for q/64 * 2^(b-127).
//
// The step 2^(b-133) is a power of two, so x / step is exact in fp32 and the code is the correctly rounded quotient: no
// division, and the same codes from any correct implementation.  A value has 8 significant bits, so it is exact in bf16 (and
// tf32): a tensor-core product over a checkpoint needs no separate scale.  A block of 32 keeps the shared exponent close to
// the values it serves; the exponents cost one byte in 33.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>
#include "types.cuh"

namespace b200 {

constexpr int kCkptBlock = 32;
__host__ __device__ inline size_t ckpt8_blocks(size_t n) { return (n + kCkptBlock - 1) / kCkptBlock; }

// top: the largest magnitude of the block as the bits of a non-negative float (any NaN compares above infinity)
__device__ __forceinline__ uint32_t ckpt8_exponent(uint32_t top)
{
    if (top >= 0x7f800000u) return 255u;                     // the block reads as NaN
    const uint32_t e = top >> 23;
    // magnitudes from 127.5 steps on would round to 128: the next exponent (the largest finite one saturates at 127 instead)
    const uint32_t up = ((top & 0x7fffffu) >= 0x7f0000u && e >= 1u && e < 254u) ? 1u : 0u;
    return max(e, 1u) + up;                                  // subnormals share the exponent of the smallest normal numbers
}

// Codes of V values.  x * 2^(133-b) + 1.5 * 2^23 in one fused step rounds the quotient to nearest, ties to even, and leaves it in the
// low byte of the sum.  Three kinds of blocks need more, and are rare enough for a branch: b < 6, where the factor is not a
// finite number; b = 254, where a code may have to be held at 127; and b = 255, all of whose codes are 0.
template <int V> __device__ __forceinline__ void ckpt8_codes(uint32_t *q, const float *x, uint32_t b, bool keep_sign)
{
    const float scale = __uint_as_float((260u - max(b, 6u)) << 23);            // 2^(133-b) for b = 6 .. 255
    if (b >= 6u && b < 254u) {
        if constexpr (V == 1) {
            q[0] = __float_as_uint(fmaf(x[0], scale, 12582912.f));
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 v = fma2(make_float2(x[i], x[i + 1]), make_float2(scale, scale), make_float2(12582912.f, 12582912.f));
                q[i] = __float_as_uint(v.x);
                q[i + 1] = __float_as_uint(v.y);
            }
        }
    } else {
        const float more = __uint_as_float((127u + max(b, 6u) - b) << 23);     // 2^(6-b) below 6, else 1
#pragma unroll
        for (int i = 0; i < V; i++) q[i] = b == 255u ? 0u : (uint32_t)max(-127, min(127, __float2int_rn(x[i] * more * scale)));
    }
    if (keep_sign) {
#pragma unroll
        for (int i = 0; i < V; i++)
            if ((q[i] & 0xffu) == 0u && x[i] < 0.f && b != 255u) q[i] = 0xffu;
    }
}

// b = 255: 0 * infinity = NaN
__device__ __forceinline__ float ckpt8_unit(uint32_t b) { return __uint_as_float(b << 23); }
__device__ __forceinline__ float ckpt8_value(int q, float unit) { return ((float)q * 0.015625f) * unit; }

// The largest of three magnitudes; a NaN if one of them is
__device__ __forceinline__ float largest(float a, float b, float c)
{
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A group of lanes that hold V neighbouring values each shares a block: its largest magnitude.
template <int V> __device__ __forceinline__ uint32_t ckpt8_top(const float *f)
{
    if constexpr (V == 1) {
        return __reduce_max_sync(0xffffffffu, __float_as_uint(f[0]) & 0x7fffffffu);
    } else {
        float most = largest(f[0], f[1], f[2]);
#pragma unroll
        for (int i = 3; i < V; i += 2) most = largest(most, f[i], i + 1 < V ? f[i + 1] : 0.f);
        uint32_t top = __float_as_uint(most);
#pragma unroll
        for (int o = 1; o < kCkptBlock / V; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        return top;
    }
}

// codes of V values at dst (a multiple of V bytes), and the values of V codes
template <int V> __device__ __forceinline__ void ckpt8_put(int8_t *dst, const float *f, uint32_t b, bool keep_sign)
{
    uint32_t q[V];
    ckpt8_codes<V>(q, f, b, keep_sign);
    if constexpr (V == 1) {
        *dst = (int8_t)q[0];
    } else {
        uint32_t w[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; i++)
            w[i] = __byte_perm(__byte_perm(q[4 * i], q[4 * i + 1], 0x0040), __byte_perm(q[4 * i + 2], q[4 * i + 3], 0x0040), 0x5410);
        if constexpr (V == 4) *reinterpret_cast<uint32_t *>(dst) = w[0];
        else *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
    }
}
template <int V> struct CkptCodes { uint32_t w[V <= 4 ? 1 : V / 4]; };
template <int V> __device__ __forceinline__ CkptCodes<V> ckpt8_get(const int8_t *src)
{
    CkptCodes<V> c;
    if constexpr (V == 1) c.w[0] = (uint32_t)(int)*src;
    else if constexpr (V == 4) c.w[0] = *reinterpret_cast<const uint32_t *>(src);
    else { const uint2 u = *reinterpret_cast<const uint2 *>(src); c.w[0] = u.x; c.w[1] = u.y; }
    return c;
}
template <int V> __device__ __forceinline__ void ckpt8_values(float *f, CkptCodes<V> c, uint32_t b)
{
    // the byte u = q + 128 under the exponent of 2^23 is the float 2^23 + u: no conversion instruction; the step may be subnormal
    const float step = ckpt8_unit(b) * 0.015625f;
    auto byte = [&](int i) { return __uint_as_float(__byte_perm(c.w[i / 4] ^ 0x80808080u, 0x4b000000u, 0x7540 | (i & 3))); };
    if constexpr (V == 1) {
        f[0] = (byte(0) - 8388736.f) * step;
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 v = mul2(add2(make_float2(byte(i), byte(i + 1)), make_float2(-8388736.f, -8388736.f)), make_float2(step, step));
            f[i] = v.x;
            f[i + 1] = v.y;
        }
    }
}

}  // namespace b200
