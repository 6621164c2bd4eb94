// 8-bit activation checkpoints (format: ckpt8.cuh): storing a tensor, reading it back, and the backward pass of a function
// layer whose input was kept that way.
#include "common.cuh"
#include "types.cuh"
#include "ckpt8.cuh"
#include "act.cuh"
#include "norm.h"

namespace b200 {

// One warp per block of 32 values, one value per lane.
template <typename T>
__global__ void __launch_bounds__(256) ckpt8_store_kernel(int8_t *__restrict__ codes, uint8_t *__restrict__ exponents, const T *__restrict__ x,
                                                          size_t total, size_t blocks, size_t n, size_t pitch, int keep_sign)
{
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const size_t step = (size_t)gridDim.x * (blockDim.x >> 5);
    for (size_t i = (size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < total; i += step) {
        const size_t row = i / blocks, col = (i - row * blocks) * kCkptBlock + lane;
        const float v = col < n ? to_float(x[row * pitch + col]) : 0.f;
        const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu);
        const uint32_t b = ckpt8_exponent(top);
        codes[i * kCkptBlock + lane] = (int8_t)ckpt8_code(v, ckpt8_scale(b), b, keep_sign != 0);
        if (lane == 0) exponents[i] = (uint8_t)b;
    }
}

// A value beyond the range of fp16 reads as the largest finite number (only the rounding of the code can bring it there).
template <typename T> __device__ __forceinline__ T ckpt8_out(float v) { return from_float<T>(v); }
template <> __device__ __forceinline__ __half ckpt8_out<__half>(float v)
{
    if (fabsf(v) > 65504.f && !isinf(v)) v = copysignf(65504.f, v);
    return __float2half_rn(v);
}

// FUNC < 0 reads the values back; otherwise out = f'(value) * error
template <typename T>
__global__ void __launch_bounds__(256) ckpt8_load_kernel(T *out, const int8_t *__restrict__ codes, const uint8_t *__restrict__ exponents,
                                                         const T *error, size_t total, size_t blocks, size_t n, size_t pitch,
                                                         size_t error_pitch, int func, double slope)
{
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const size_t step = (size_t)gridDim.x * (blockDim.x >> 5);
    for (size_t i = (size_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); i < total; i += step) {
        const size_t row = i / blocks, col = (i - row * blocks) * kCkptBlock + lane;
        if (col >= n) continue;
        const float v = ckpt8_value(codes[i * kCkptBlock + lane], ckpt8_unit(exponents[i]));
        if (func < 0) out[row * pitch + col] = ckpt8_out<T>(v);
        else out[row * pitch + col] = from_float<T>(act_derivative(v, func, slope) * to_float(error[row * error_pitch + col]));
    }
}

int check_ckpt8(const void *codes, const void *exponents)
{
    if (!codes || !exponents) return fail(B200_E_ARG, "null checkpoint pointer");
    if (reinterpret_cast<uintptr_t>(codes) & 15) return fail(B200_E_ARG, "the codes of a checkpoint must start at a 16-byte boundary");
    return B200_OK;
}

int check_rows(int rows, size_t n)
{
    if (rows < 0 || (size_t)rows > kMaxRow) return fail(B200_E_SHAPE, "the number of rows must be 0 to %zu", kMaxRow);
    if (n == 0 || n > kMaxRow) return fail(B200_E_SHAPE, "a row must have 1 to %zu values", kMaxRow);
    return B200_OK;
}

int check_matrix(const void *p, int type, int rows, size_t n, size_t pitch, const char *name)
{
    if (!p) return fail(B200_E_ARG, "null tensor pointer (%s)", name);
    if (!element_aligned(p, type)) return fail(B200_E_ARG, "%s is not aligned to its element size", name);
    if (rows > 1 && pitch < n) return fail(B200_E_SHAPE, "%s: the pitch is smaller than a row", name);
    return B200_OK;
}

static unsigned ckpt8_grid(size_t total)
{
    const size_t want = (total + 7) / 8, most = (size_t)sm_count() * 8;
    return (unsigned)(want < most ? want : most);
}

template <typename T>
static void launch_load(T *out, const int8_t *codes, const uint8_t *exponents, const T *error, int rows, size_t n, size_t pitch, size_t error_pitch,
                        int func, double slope, cudaStream_t s)
{
    const size_t blocks = ckpt8_blocks(n), total = (size_t)rows * blocks;
    Launch(ckpt8_grid(total), 256, 0, s)(ckpt8_load_kernel<T>, out, codes, exponents, error, total, blocks, n, pitch, error_pitch, func, slope);
}

}  // namespace b200

using namespace b200;
#define ST(s) ((cudaStream_t)(s))

extern "C" {

int b200_ckpt8_store(int8_t *codes, uint8_t *exponents, const void *x, int type, int rows, size_t n, size_t x_pitch, int keep_sign, void *stream)
{
    if (!known_type(type)) return fail(B200_E_ARG, "unknown element type %d", type);
    int r = check_rows(rows, n);
    if (r || rows == 0) return r;
    if ((r = check_ckpt8(codes, exponents)) || (r = check_matrix(x, type, rows, n, x_pitch, "x"))) return r;
    const size_t blocks = ckpt8_blocks(n), total = (size_t)rows * blocks;
    const Launch launch(ckpt8_grid(total), 256, 0, ST(stream));
    if (type == B200_F32) launch(ckpt8_store_kernel<float>, codes, exponents, (const float *)x, total, blocks, n, x_pitch, keep_sign);
    else if (type == B200_BF16) launch(ckpt8_store_kernel<__nv_bfloat16>, codes, exponents, (const __nv_bfloat16 *)x, total, blocks, n, x_pitch, keep_sign);
    else launch(ckpt8_store_kernel<__half>, codes, exponents, (const __half *)x, total, blocks, n, x_pitch, keep_sign);
    B200_LAUNCH_CHECK();
    return B200_OK;
}

static int load_impl(void *out, const int8_t *codes, const uint8_t *exponents, const void *error, int type, int rows, size_t n, size_t out_pitch,
                     size_t error_pitch, int func, double slope, void *stream)
{
    cudaStream_t s = ST(stream);
    if (type == B200_F32) launch_load((float *)out, codes, exponents, (const float *)error, rows, n, out_pitch, error_pitch, func, slope, s);
    else if (type == B200_BF16) launch_load((__nv_bfloat16 *)out, codes, exponents, (const __nv_bfloat16 *)error, rows, n, out_pitch, error_pitch, func, slope, s);
    else launch_load((__half *)out, codes, exponents, (const __half *)error, rows, n, out_pitch, error_pitch, func, slope, s);
    B200_LAUNCH_CHECK();
    return B200_OK;
}

int b200_ckpt8_load(void *out, const int8_t *codes, const uint8_t *exponents, int type, int rows, size_t n, size_t out_pitch, void *stream)
{
    if (!known_type(type)) return fail(B200_E_ARG, "unknown element type %d", type);
    int r = check_rows(rows, n);
    if (r || rows == 0) return r;
    if ((r = check_ckpt8(codes, exponents)) || (r = check_matrix(out, type, rows, n, out_pitch, "out"))) return r;
    return load_impl(out, codes, exponents, nullptr, type, rows, n, out_pitch, 0, -1, 0.0, stream);
}

int b200_ckpt8_activation_backward(void *out, const int8_t *codes, const uint8_t *exponents, const void *error, int type, int rows, size_t n,
                                   size_t out_pitch, size_t error_pitch, int func, double leaky_slope, void *stream)
{
    if (!known_type(type)) return fail(B200_E_ARG, "unknown element type %d", type);
    if (func < B200_ACT_SIGMOID || func > B200_ACT_GELU) return fail(B200_E_ARG, "unknown neuron function");
    int r = check_rows(rows, n);
    if (r || rows == 0) return r;
    if ((r = check_ckpt8(codes, exponents)) || (r = check_matrix(out, type, rows, n, out_pitch, "out")) || (r = check_matrix(error, type, rows, n, error_pitch, "error"))) return r;
    return load_impl(out, codes, exponents, error, type, rows, n, out_pitch, error_pitch, func, leaky_slope, stream);
}

}  // extern "C"
