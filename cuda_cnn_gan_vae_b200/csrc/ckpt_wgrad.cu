// Weight and bias gradient of a Linear layer whose input was kept in 8 bits (ckpt8.cuh):
//   dweight[o][i] (+)= sum over rows of delta[row][o] * x[row][i],   dbias[o] (+)= sum over rows of delta[row][o]
#include "common.cuh"
#include "types.cuh"
#include "ckpt8.cuh"
#include "norm.h"

namespace b200 {

constexpr int kTile = 64, kDepth = 16;

// 64 x 64 outputs per block of 256 threads, 4 x 4 per thread, the checkpoint decoded while a slice of 16 rows is staged
template <typename T>
__global__ void __launch_bounds__(256) ckpt8_wgrad_simt_kernel(float *dweight, float *dbias, const T *__restrict__ delta, const int8_t *__restrict__ codes,
                                                               const uint8_t *__restrict__ exponents, int rows, int out, size_t in, size_t pitch, size_t blocks,
                                                               int accumulate)
{
    __shared__ float a[kDepth][kTile], b[kDepth][kTile];
    grid_dependency_wait();
    const size_t i0 = (size_t)blockIdx.x * kTile;
    const int o0 = (int)blockIdx.y * kTile;
    const int ti = threadIdx.x & 15, to = threadIdx.x >> 4;
    float acc[4][4] = {}, bias[4] = {};
    for (int r0 = 0; r0 < rows; r0 += kDepth) {
        for (int k = threadIdx.x; k < kDepth * kTile; k += 256) {
            const int kr = k / kTile, kc = k % kTile, row = r0 + kr;
            const bool in_range = row < rows;
            a[kr][kc] = in_range && o0 + kc < out ? to_float(delta[(size_t)row * pitch + o0 + kc]) : 0.f;
            const size_t i = i0 + kc;
            b[kr][kc] = in_range && i < in ? ckpt8_value(codes[(size_t)row * blocks * kCkptBlock + i], ckpt8_unit(exponents[(size_t)row * blocks + i / kCkptBlock])) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; k++) {
            float av[4], bv[4];
#pragma unroll
            for (int j = 0; j < 4; j++) { av[j] = a[k][to * 4 + j]; bv[j] = b[k][ti * 4 + j]; }
#pragma unroll
            for (int x = 0; x < 4; x++) {
                bias[x] += av[x];
#pragma unroll
                for (int y = 0; y < 4; y++) acc[x][y] = fmaf(av[x], bv[y], acc[x][y]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const int o = o0 + to * 4 + x;
        if (o >= out) break;
        if (dbias && blockIdx.x == 0 && ti == 0) dbias[o] = accumulate ? dbias[o] + bias[x] : bias[x];
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const size_t i = i0 + ti * 4 + y;
            if (i >= in) break;
            float *w = dweight + (size_t)o * in + i;
            *w = accumulate ? *w + acc[x][y] : acc[x][y];
        }
    }
}

}  // namespace b200

using namespace b200;
#define ST(s) ((cudaStream_t)(s))

extern "C" {

size_t b200_ckpt8_wgrad_workspace(int type, int rows, int out, size_t in)
{
    return 0;
}

int b200_ckpt8_wgrad(float *dweight, float *dbias, int accumulate, const void *delta, const int8_t *codes, const uint8_t *exponents, int type, int rows,
                     int out, size_t in, size_t delta_pitch, void *workspace, size_t workspace_bytes, void *stream)
{
    if (!known_type(type)) return fail(B200_E_ARG, "unknown element type %d", type);
    int r = check_rows(rows, in);
    if (r) return r;
    if (out <= 0) return fail(B200_E_SHAPE, "non-positive number of outputs");
    if (!dweight) return fail(B200_E_ARG, "null gradient pointer");
    if (rows == 0) {
        if (!accumulate) {
            B200_CUDA(cudaMemsetAsync(dweight, 0, sizeof(float) * in * (size_t)out, ST(stream)));
            if (dbias) B200_CUDA(cudaMemsetAsync(dbias, 0, sizeof(float) * (size_t)out, ST(stream)));
        }
        return B200_OK;
    }
    if ((r = check_ckpt8(codes, exponents)) || (r = check_matrix(delta, type, rows, (size_t)out, delta_pitch, "delta"))) return r;
    const size_t blocks = ckpt8_blocks(in);
    const Launch launch(dim3((unsigned)((in + kTile - 1) / kTile), (unsigned)ceil_div(out, kTile)), 256, 0, ST(stream));
    if (type == B200_F32) launch(ckpt8_wgrad_simt_kernel<float>, dweight, dbias, (const float *)delta, codes, exponents, rows, out, in, delta_pitch, blocks, accumulate);
    else if (type == B200_BF16) launch(ckpt8_wgrad_simt_kernel<__nv_bfloat16>, dweight, dbias, (const __nv_bfloat16 *)delta, codes, exponents, rows, out, in, delta_pitch, blocks, accumulate);
    else launch(ckpt8_wgrad_simt_kernel<__half>, dweight, dbias, (const __half *)delta, codes, exponents, rows, out, in, delta_pitch, blocks, accumulate);
    B200_LAUNCH_CHECK();
    set_path(B200_PATH_SIMT);
    return B200_OK;
}

}  // extern "C"
