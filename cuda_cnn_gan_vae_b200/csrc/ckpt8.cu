// 8-bit activation checkpoints (format: ckpt8.cuh): storing a tensor, reading it back, and the backward pass of a function
// layer whose input was kept that way.
#include "common.cuh"
#include "types.cuh"
#include "ckpt8.cuh"
#include "act.cuh"
#include "norm.h"

namespace b200 {

// Store and load are bound by memory.  A warp takes kSpans spans at a time, a span being V neighbouring values per lane (16
// bytes, or one value where the rows cannot be read in 16-byte pieces); a block's lanes find its largest magnitude by shuffles.  All
// loads of the kSpans spans are under way before the first is used.  A dense tensor whose rows are whole blocks is one long
// row, so the division that finds a span's row is left to ragged ones.
// Measured on 128 x 524288 fp32 values: store 63 us (5.4 TB/s; 90 us with conversion instructions, clamps and two factors
// for every code), load 53 us (6.4 TB/s), backward of LeakyReLU 91 us (6.7 TB/s).
constexpr int kSpans = 4;

struct CkptShape {
    size_t total, spans, n, blocks, pitch;      // spans in all and per row
    int one_row;
};
__device__ __forceinline__ void span_at(const CkptShape &g, size_t i, size_t &row, size_t &span)
{
    if (g.one_row) { row = 0; span = i; }
    else if (g.total <= 0xffffffffu) { row = (uint32_t)i / (uint32_t)g.spans; span = i - row * g.spans; }
    else { row = i / g.spans; span = i - row * g.spans; }
}

template <typename T, int V>
__global__ void __launch_bounds__(256) ckpt8_store_kernel(int8_t *__restrict__ codes, uint8_t *__restrict__ exponents, const T *__restrict__ x,
                                                          const __grid_constant__ CkptShape g, int keep_sign)
{
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const size_t warps = (size_t)gridDim.x * 8;
    for (size_t first = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); first * kSpans < g.total; first += warps) {
        Pack<T, V> in[kSpans];
        size_t row[kSpans], col[kSpans];
#pragma unroll
        for (int k = 0; k < kSpans; k++) {
            size_t span;
            const size_t i = first * kSpans + k;
            span_at(g, i < g.total ? i : g.total - 1, row[k], span);
            col[k] = (span * 32 + lane) * V;
            if (i < g.total && col[k] < g.n) {
                in[k] = load_pack<T, V>(x + row[k] * g.pitch + col[k]);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) in[k].v[j] = from_float<T>(0.f);
            }
        }
#pragma unroll
        for (int k = 0; k < kSpans; k++) {
            if (first * kSpans + k >= g.total) break;
            float f[V];
#pragma unroll
            for (int j = 0; j < V; j++) f[j] = to_float(in[k].v[j]);
            const uint32_t b = ckpt8_exponent(ckpt8_top<V>(f));
            const size_t block = col[k] / kCkptBlock;
            if (block < g.blocks) {
                ckpt8_put<V>(codes + row[k] * g.blocks * kCkptBlock + col[k], f, b, keep_sign != 0);
                if (col[k] % kCkptBlock == 0) exponents[row[k] * g.blocks + block] = (uint8_t)b;
            }
        }
    }
}

// A value beyond the range of fp16 reads as the largest finite number (only the rounding of the code can bring it there).
template <typename T> __device__ __forceinline__ float ckpt8_clip(float v) { return v; }
template <> __device__ __forceinline__ float ckpt8_clip<__half>(float v) { return fabsf(v) > 65504.f && !isinf(v) ? copysignf(65504.f, v) : v; }

// FUNC < 0 reads the values back; otherwise out = f'(value) * error
template <typename T, int V, int FUNC>
__global__ void __launch_bounds__(256) ckpt8_load_kernel(T *out, const int8_t *__restrict__ codes, const uint8_t *__restrict__ exponents,
                                                         const T *error, const __grid_constant__ CkptShape g, size_t error_pitch, double slope)
{
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const size_t warps = (size_t)gridDim.x * 8;
    for (size_t first = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); first * kSpans < g.total; first += warps) {
        CkptCodes<V> c[kSpans];
        uint32_t b[kSpans];
        Pack<T, V> e[kSpans];
        size_t row[kSpans], col[kSpans];
#pragma unroll
        for (int k = 0; k < kSpans; k++) {
            size_t span;
            const size_t i = first * kSpans + k;
            span_at(g, i < g.total ? i : g.total - 1, row[k], span);
            col[k] = i < g.total ? (span * 32 + lane) * V : g.n;
            if (col[k] < g.n) {
                c[k] = ckpt8_get<V>(codes + row[k] * g.blocks * kCkptBlock + col[k]);
                b[k] = exponents[row[k] * g.blocks + col[k] / kCkptBlock];
                if (FUNC >= 0) e[k] = load_pack<T, V>(error + row[k] * error_pitch + col[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < kSpans; k++) {
            if (col[k] >= g.n) continue;
            float f[V];
            ckpt8_values<V>(f, c[k], b[k]);
#pragma unroll
            for (int j = 0; j < V; j++) {
                if (FUNC < 0) f[j] = ckpt8_clip<T>(f[j]);
                else f[j] = act_derivative(f[j], FUNC, slope) * to_float(e[k].v[j]);
                // a NaN is not above zero: without this the finite neighbours of an infinity would pass for negative values
                if ((FUNC == B200_ACT_RELU || FUNC == B200_ACT_LEAKY_RELU) && b[k] == 255u) f[j] = __int_as_float(0x7fffffff);
            }
            store_pack<T, V>(out + row[k] * g.pitch + col[k], f);
        }
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

static CkptShape ckpt8_shape(int rows, size_t n, size_t pitch, int v, bool same_pitch)
{
    CkptShape g;
    g.one_row = rows == 1 || (pitch == n && same_pitch && n % kCkptBlock == 0);
    g.n = g.one_row ? n * (size_t)rows : n;
    g.blocks = ckpt8_blocks(g.n);
    g.pitch = pitch;
    g.spans = (g.blocks * kCkptBlock + 32 * v - 1) / (32 * v);      // whole blocks: the last one is filled up with zeros
    g.total = g.one_row ? g.spans : g.spans * (size_t)rows;
    return g;
}
static unsigned ckpt8_grid(const CkptShape &g)
{
    const size_t want = (g.total + 8 * kSpans - 1) / (8 * kSpans), most = (size_t)sm_count() * 8;
    return (unsigned)(want < most ? want : most);
}

template <typename T, int V>
static void launch_load(const Launch &launch, T *out, const int8_t *codes, const uint8_t *exponents, const T *error, const CkptShape &g, size_t error_pitch,
                        int func, double slope)
{
#define B200_CKPT8_LOAD(F) launch(ckpt8_load_kernel<T, V, F>, out, codes, exponents, error, g, error_pitch, slope)
    switch (func) {
    case B200_ACT_SIGMOID: B200_CKPT8_LOAD(B200_ACT_SIGMOID); break;
    case B200_ACT_RELU: B200_CKPT8_LOAD(B200_ACT_RELU); break;
    case B200_ACT_LEAKY_RELU: B200_CKPT8_LOAD(B200_ACT_LEAKY_RELU); break;
    case B200_ACT_LINEAR: B200_CKPT8_LOAD(B200_ACT_LINEAR); break;
    case B200_ACT_TANH: B200_CKPT8_LOAD(B200_ACT_TANH); break;
    case B200_ACT_GELU: B200_CKPT8_LOAD(B200_ACT_GELU); break;
    default: B200_CKPT8_LOAD(-1); break;
    }
#undef B200_CKPT8_LOAD
}

template <typename T>
static int load_typed(T *out, const int8_t *codes, const uint8_t *exponents, const T *error, int type, int rows, size_t n, size_t pitch, size_t error_pitch,
                      int func, double slope, cudaStream_t s)
{
    const bool wide = wide_rows(out, type, n, pitch) && (!error || wide_rows(error, type, n, error_pitch));
    const CkptShape g = ckpt8_shape(rows, n, pitch, wide ? kWide<T> : 1, !error || error_pitch == pitch);
    const Launch launch(ckpt8_grid(g), 256, 0, s);
    if (wide) launch_load<T, kWide<T>>(launch, out, codes, exponents, error, g, error_pitch, func, slope);
    else launch_load<T, 1>(launch, out, codes, exponents, error, g, error_pitch, func, slope);
    B200_LAUNCH_CHECK();
    return B200_OK;
}

template <typename T>
static int store_typed(int8_t *codes, uint8_t *exponents, const T *x, int type, int rows, size_t n, size_t pitch, int keep_sign, cudaStream_t s)
{
    const bool wide = wide_rows(x, type, n, pitch);
    const CkptShape g = ckpt8_shape(rows, n, pitch, wide ? kWide<T> : 1, true);
    const Launch launch(ckpt8_grid(g), 256, 0, s);
    if (wide) launch(ckpt8_store_kernel<T, kWide<T>>, codes, exponents, x, g, keep_sign);
    else launch(ckpt8_store_kernel<T, 1>, codes, exponents, x, g, keep_sign);
    B200_LAUNCH_CHECK();
    return B200_OK;
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
    if (type == B200_F32) return store_typed(codes, exponents, (const float *)x, type, rows, n, x_pitch, keep_sign, ST(stream));
    if (type == B200_BF16) return store_typed(codes, exponents, (const __nv_bfloat16 *)x, type, rows, n, x_pitch, keep_sign, ST(stream));
    return store_typed(codes, exponents, (const __half *)x, type, rows, n, x_pitch, keep_sign, ST(stream));
}

static int load_impl(void *out, const int8_t *codes, const uint8_t *exponents, const void *error, int type, int rows, size_t n, size_t out_pitch,
                     size_t error_pitch, int func, double slope, void *stream)
{
    cudaStream_t s = ST(stream);
    if (type == B200_F32) return load_typed((float *)out, codes, exponents, (const float *)error, type, rows, n, out_pitch, error_pitch, func, slope, s);
    if (type == B200_BF16) return load_typed((__nv_bfloat16 *)out, codes, exponents, (const __nv_bfloat16 *)error, type, rows, n, out_pitch, error_pitch, func, slope, s);
    return load_typed((__half *)out, codes, exponents, (const __half *)error, type, rows, n, out_pitch, error_pitch, func, slope, s);
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
