// Layer normalisation over the rows of a matrix, forward and backward:
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = gamma xh + beta
//   backward  g = dy gamma, dx = r (g - mean(g) - xh mean(g xh)), dgamma = sum over rows of dy xh, dbeta = sum over rows of dy
// The normalised values can be kept in 8 bits by the forward pass (ckpt8.cuh) and the backward pass can read them from there.
// Statistics and sums are held in fp32; the variance is the mean of the squared deviations from the mean that was found first,
// so a large mean costs no digits.
#include "common.cuh"
#include "types.cuh"
#include "ckpt8.cuh"
#include "norm.h"

namespace b200 {

constexpr int kRowThreads = 256;

// Sum over the block; every thread receives it.  `scratch` holds one float per warp and may be used again after the call.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float *scratch)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < THREADS / 32 ? scratch[threadIdx.x & 31] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    return v;
}

// One block per row, one value per lane: a warp holds whole blocks of the checkpoint.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) ln_forward_kernel(T *y, float *mean, float *rstd, int8_t *codes, uint8_t *exponents, const T *x,
                                                                const float *__restrict__ gamma, const float *__restrict__ beta, int rows, size_t n,
                                                                size_t x_pitch, size_t y_pitch, float eps)
{
    __shared__ float scratch[kRowThreads / 32];
    grid_dependency_wait();
    const size_t blocks = ckpt8_blocks(n);
    for (int row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + (size_t)row * x_pitch;
        float s = 0.f;
        for (size_t i = threadIdx.x; i < n; i += kRowThreads) s += to_float(xr[i]);
        const float mu = block_sum<kRowThreads>(s, scratch) / (float)n;
        float q = 0.f;
        for (size_t i = threadIdx.x; i < n; i += kRowThreads) {
            const float d = to_float(xr[i]) - mu;
            q = fmaf(d, d, q);
        }
        const float r = 1.0f / sqrtf(block_sum<kRowThreads>(q, scratch) / (float)n + eps);
        if (threadIdx.x == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
        for (size_t i = threadIdx.x; i < blocks * kCkptBlock; i += kRowThreads) {
            const float xh = i < n ? (to_float(xr[i]) - mu) * r : 0.f;
            if (codes) {
                const uint32_t b = ckpt8_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(xh) & 0x7fffffffu));
                codes[(size_t)row * blocks * kCkptBlock + i] = (int8_t)ckpt8_code(xh, ckpt8_scale(b), b, false);
                if ((threadIdx.x & 31) == 0) exponents[(size_t)row * blocks + i / kCkptBlock] = (uint8_t)b;
            }
            if (i < n) y[(size_t)row * y_pitch + i] = from_float<T>(fmaf(xh, gamma[i], beta[i]));
        }
    }
}

template <typename T>
struct LnBackward {
    T *dx;
    const T *dy, *x;
    const float *mean, *rstd;
    const int8_t *codes;
    const uint8_t *exponents;
    const float *gamma;
    int rows;
    size_t n, blocks, dy_pitch, x_pitch, dx_pitch;
    float *part;                 // [groups][2][n] partial sums of dgamma and dbeta
    int groups;
};

template <typename T>
__device__ __forceinline__ float ln_xhat(const LnBackward<T> &p, int row, size_t i, float mu, float r)
{
    if (p.codes) return ckpt8_value(p.codes[(size_t)row * p.blocks * kCkptBlock + i], ckpt8_unit(p.exponents[(size_t)row * p.blocks + i / kCkptBlock]));
    return (to_float(p.x[(size_t)row * p.x_pitch + i]) - mu) * r;
}

// dgamma and dbeta of a group of rows: a thread owns a column
template <typename T>
__global__ void __launch_bounds__(256) ln_backward_columns_kernel(LnBackward<T> p)
{
    grid_dependency_wait();
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.n) return;
    const int begin = (int)((long long)p.rows * blockIdx.y / p.groups), end = (int)((long long)p.rows * (blockIdx.y + 1) / p.groups);
    float dg = 0.f, db = 0.f;
    for (int row = begin; row < end; row++) {
        const float d = to_float(p.dy[(size_t)row * p.dy_pitch + i]);
        dg = fmaf(d, ln_xhat(p, row, i, p.mean ? p.mean[row] : 0.f, p.rstd[row]), dg);
        db += d;
    }
    p.part[((size_t)blockIdx.y * 2) * p.n + i] = dg;
    p.part[((size_t)blockIdx.y * 2 + 1) * p.n + i] = db;
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) ln_backward_rows_kernel(LnBackward<T> p)
{
    __shared__ float scratch[kRowThreads / 32];
    grid_dependency_wait();
    for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const float mu = p.mean ? p.mean[row] : 0.f, r = p.rstd[row];
        const T *dy = p.dy + (size_t)row * p.dy_pitch;
        float s1 = 0.f, s2 = 0.f;
        for (size_t i = threadIdx.x; i < p.n; i += kRowThreads) {
            const float g = to_float(dy[i]) * p.gamma[i];
            s1 += g;
            s2 = fmaf(g, ln_xhat(p, row, i, mu, r), s2);
        }
        const float c1 = block_sum<kRowThreads>(s1, scratch) / (float)p.n, c2 = block_sum<kRowThreads>(s2, scratch) / (float)p.n;
        for (size_t i = threadIdx.x; i < p.n; i += kRowThreads) {
            const float g = to_float(dy[i]) * p.gamma[i];
            p.dx[(size_t)row * p.dx_pitch + i] = from_float<T>(r * (g - c1 - ln_xhat(p, row, i, mu, r) * c2));
        }
    }
}

// Sum of the groups' partial rows in their order: the result does not depend on how the groups were scheduled.
__global__ void __launch_bounds__(256) ln_backward_join_kernel(float *dgamma, float *dbeta, const float *__restrict__ part, int groups, size_t n, int accumulate)
{
    grid_dependency_wait();
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * n) return;
    float s = 0.f;
    for (int g = 0; g < groups; g++) s += part[(size_t)g * 2 * n + i];
    float *out = i < n ? dgamma + i : dbeta + (i - n);
    *out = accumulate ? *out + s : s;
}

static int ln_groups(int rows, size_t n)
{
    const size_t column_blocks = (n + 255) / 256;
    const int want = (int)((2 * (size_t)sm_count() + column_blocks - 1) / column_blocks);
    return rows < want ? (rows > 0 ? rows : 1) : want;
}

template <typename T>
static int ln_forward_launch(void *y, float *mean, float *rstd, int8_t *codes, uint8_t *exponents, const void *x, const float *gamma, const float *beta,
                             int rows, size_t n, size_t x_pitch, size_t y_pitch, float eps, cudaStream_t s)
{
    Launch((unsigned)min(rows, sm_count() * 8), kRowThreads, 0, s)(ln_forward_kernel<T>, (T *)y, mean, rstd, codes, exponents, (const T *)x, gamma, beta,
                                                                  rows, n, x_pitch, y_pitch, eps);
    B200_LAUNCH_CHECK();
    return B200_OK;
}

template <typename T>
static int ln_backward_launch(LnBackward<T> p, float *dgamma, float *dbeta, int create_delta_weight, int accumulate, cudaStream_t s)
{
    if (create_delta_weight) {
        Launch(dim3((unsigned)((p.n + 255) / 256), (unsigned)p.groups), 256, 0, s)(ln_backward_columns_kernel<T>, p);
        B200_LAUNCH_CHECK();
        Launch((unsigned)((2 * p.n + 255) / 256), 256, 0, s)(ln_backward_join_kernel, dgamma, dbeta, p.part, p.groups, p.n, accumulate);
        B200_LAUNCH_CHECK();
    }
    Launch((unsigned)min(p.rows, sm_count() * 8), kRowThreads, 0, s)(ln_backward_rows_kernel<T>, p);
    B200_LAUNCH_CHECK();
    return B200_OK;
}

}  // namespace b200

using namespace b200;
#define ST(s) ((cudaStream_t)(s))

extern "C" {

int b200_ln_forward(void *y, float *mean, float *rstd, int8_t *codes, uint8_t *exponents, const void *x, const float *gamma, const float *beta, int type,
                    int rows, size_t n, size_t x_pitch, size_t y_pitch, float eps, void *stream)
{
    if (!known_type(type)) return fail(B200_E_ARG, "unknown element type %d", type);
    if (!(eps > 0.f)) return fail(B200_E_ARG, "layer normalisation needs a positive epsilon");
    int r = check_rows(rows, n);
    if (r || rows == 0) return r;
    if (!gamma || !beta) return fail(B200_E_ARG, "null tensor pointer");
    if ((codes || exponents) && (r = check_ckpt8(codes, exponents))) return r;
    if ((r = check_matrix(x, type, rows, n, x_pitch, "x")) || (r = check_matrix(y, type, rows, n, y_pitch, "y"))) return r;
    if (type == B200_F32) return ln_forward_launch<float>(y, mean, rstd, codes, exponents, x, gamma, beta, rows, n, x_pitch, y_pitch, eps, ST(stream));
    if (type == B200_BF16) return ln_forward_launch<__nv_bfloat16>(y, mean, rstd, codes, exponents, x, gamma, beta, rows, n, x_pitch, y_pitch, eps, ST(stream));
    return ln_forward_launch<__half>(y, mean, rstd, codes, exponents, x, gamma, beta, rows, n, x_pitch, y_pitch, eps, ST(stream));
}

size_t b200_ln_backward_workspace(int rows, size_t n)
{
    if (rows <= 0 || n == 0 || n > kMaxRow) return 0;
    return sizeof(float) * 2 * n * (size_t)ln_groups(rows, n);
}

int b200_ln_backward(void *dx, float *dgamma, float *dbeta, const void *dy, const void *x, const float *mean, const float *rstd, const int8_t *codes,
                     const uint8_t *exponents, const float *gamma, int type, int rows, size_t n, size_t dx_pitch, size_t dy_pitch, size_t x_pitch,
                     int create_delta_weight, int accumulate, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!known_type(type)) return fail(B200_E_ARG, "unknown element type %d", type);
    int r = check_rows(rows, n);
    if (r) return r;
    if (create_delta_weight && (!dgamma || !dbeta)) return fail(B200_E_ARG, "null gradient pointer");
    if (rows == 0) {
        if (create_delta_weight && !accumulate) {
            B200_CUDA(cudaMemsetAsync(dgamma, 0, sizeof(float) * n, ST(stream)));
            B200_CUDA(cudaMemsetAsync(dbeta, 0, sizeof(float) * n, ST(stream)));
        }
        return B200_OK;
    }
    if (!rstd || !gamma) return fail(B200_E_ARG, "null tensor pointer");
    if ((x != nullptr) == (codes != nullptr)) return fail(B200_E_ARG, "the normalised rows come from x or from a checkpoint, one of the two");
    if (x ? ((r = check_matrix(x, type, rows, n, x_pitch, "x")) != 0) : ((r = check_ckpt8(codes, exponents)) != 0)) return r;
    if (x && !mean) return fail(B200_E_ARG, "null mean");
    if ((r = check_matrix(dx, type, rows, n, dx_pitch, "dx")) || (r = check_matrix(dy, type, rows, n, dy_pitch, "dy"))) return r;
    if (create_delta_weight) {
        if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)) return fail(B200_E_ARG, "the workspace must be given, aligned to 16 bytes");
        if (workspace_bytes < b200_ln_backward_workspace(rows, n))
            return fail(B200_E_NOMEM, "the workspace has %zu bytes, %zu are needed", workspace_bytes, b200_ln_backward_workspace(rows, n));
    }
    const size_t blocks = ckpt8_blocks(n);
    const int groups = ln_groups(rows, n);
    if (!x) mean = nullptr;
#define B200_LN_BWD(T) ln_backward_launch<T>(LnBackward<T>{(T *)dx, (const T *)dy, (const T *)x, mean, rstd, codes, exponents, gamma, rows, n, blocks, dy_pitch, x_pitch, dx_pitch, (float *)workspace, groups}, dgamma, dbeta, create_delta_weight, accumulate, ST(stream))
    if (type == B200_F32) return B200_LN_BWD(float);
    if (type == B200_BF16) return B200_LN_BWD(__nv_bfloat16);
    return B200_LN_BWD(__half);
#undef B200_LN_BWD
}

}  // extern "C"
