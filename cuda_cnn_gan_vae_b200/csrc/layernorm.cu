// Layer normalisation over the rows of a matrix, forward and backward:
//   forward   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = gamma xh + beta
//   backward  g = dy gamma, dx = r (g - mean(g) - xh mean(g xh)), dgamma = sum over rows of dy xh, dbeta = sum over rows of dy
// The normalised values can be kept in 8 bits by the forward pass (ckpt8.cuh) and the backward pass can read them from there.
// Statistics and sums are held in fp32; the variance is the mean of the squared deviations from the mean that was found first,
// so a large mean costs no digits.  Everything here is bound by memory.
//
// Every form is chosen by the length of a row (and by whether rows can be read in 16-byte pieces), never by their number, so
// a row's result does not depend on the batch around it.
#include "common.cuh"
#include "types.cuh"
#include "ckpt8.cuh"
#include "norm.h"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace b200 {

__device__ __forceinline__ float warp_total(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sums over the THREADS threads of a team (a warp, or whole warps that share named barrier `id`); every thread receives them.
// `scratch` holds N floats per warp of the team and is free again after the call.
template <int THREADS, int N>
__device__ __forceinline__ void team_total(float *v, float *scratch, int id)
{
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = warp_total(v[k]);
    if constexpr (THREADS > 32) {
        constexpr int kWarps = THREADS / 32;
        const int lane = threadIdx.x & 31, warp = (threadIdx.x % THREADS) >> 5;
        if (lane == 0) {
#pragma unroll
            for (int k = 0; k < N; k++) scratch[k * kWarps + warp] = v[k];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
#pragma unroll
        for (int k = 0; k < N; k++) {
            v[k] = lane < kWarps ? scratch[k * kWarps + lane] : 0.f;
            v[k] = warp_total(v[k]);
        }
        asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
    }
}

// ---- forward -----------------------------------------------------------------------------------------------------------------

template <typename T>
struct LnForward {
    T *y;
    float *mean, *rstd;
    int8_t *codes;
    uint8_t *exponents;
    const T *x;
    const float *gamma, *beta;
    int rows;
    size_t n, x_pitch, y_pitch, share;      // share: values of a row per block (a multiple of 32 * V)
    float eps;
};

constexpr int kLnValues = 32;       // values of a row in a thread's registers

// writes V normalised values and keeps them; col < n may be false for lanes that fill up a block of the checkpoint
template <typename T, int V>
__device__ __forceinline__ void ln_put(const LnForward<T> &p, size_t row, size_t col, const float *xh)
{
    if (p.codes) {
        const uint32_t b = ckpt8_exponent(ckpt8_top<V>(xh));
        const size_t blocks = ckpt8_blocks(p.n);
        if (col < blocks * kCkptBlock) {
            ckpt8_put<V>(p.codes + row * blocks * kCkptBlock + col, xh, b, false);
            if (col % kCkptBlock == 0) p.exponents[row * blocks + col / kCkptBlock] = (uint8_t)b;
        }
    }
    if (col < p.n) {
        float y[V];
#pragma unroll
        for (int j = 0; j < V; j++) y[j] = fmaf(xh[j], __ldg(p.gamma + col + j), __ldg(p.beta + col + j));
        store_pack<T, V>(p.y + row * p.y_pitch + col, y);
    }
}

// A row in the registers of one team, or of CLUSTER blocks that hold a share each: read once, written once.  The blocks of a
// cluster exchange the mean and the squared deviations of their shares through distributed shared memory, one barrier a row.
template <typename T, int V, int TEAM, int BLOCK, bool CLUSTER>
__global__ void __launch_bounds__(BLOCK, 1024 / BLOCK) ln_forward_kernel(const __grid_constant__ LnForward<T> p)
{
    constexpr int K = kLnValues / V, kTeams = BLOCK / TEAM;
    __shared__ float scratch[kTeams][TEAM / 32];
    __shared__ float2 shares[2][8];
    grid_dependency_wait();
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    unsigned rank = 0, ranks = 1;
    if constexpr (CLUSTER) { rank = cg::this_cluster().block_rank(); ranks = cg::this_cluster().num_blocks(); }
    const size_t begin = CLUSTER ? (size_t)rank * p.share : 0;
    const size_t end = CLUSTER ? min(begin + p.share, p.n) : p.n;
    const float mine = CLUSTER ? (float)(begin < end ? end - begin : 0) : (float)p.n;
    const int step = CLUSTER ? (int)(gridDim.x / ranks) : (int)gridDim.x * kTeams;
    int turn = 0;
    for (int row = CLUSTER ? (int)(blockIdx.x / ranks) : (int)blockIdx.x * kTeams + team; row < p.rows; row += step, turn ^= 1) {
        const T *x = p.x + (size_t)row * p.x_pitch;
        float v[K][V];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const size_t col = begin + (size_t)(k * TEAM + t) * V;
            if (col < end) {
                const Pack<T, V> in = load_pack<T, V>(x + col);
#pragma unroll
                for (int j = 0; j < V; j++) v[k][j] = to_float(in.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) v[k][j] = 0.f;
            }
        }
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) s += v[k][j];
        }
        team_total<TEAM, 1>(&s, scratch[team], 1 + team);
        float mu = s / (CLUSTER ? fmaxf(mine, 1.f) : mine);
#pragma unroll
        for (int k = 0; k < K; k++) {
            const size_t col = begin + (size_t)(k * TEAM + t) * V;
            if (col < end) {
#pragma unroll
                for (int j = 0; j < V; j++) { const float d = v[k][j] - mu; q = fmaf(d, d, q); }
            }
        }
        team_total<TEAM, 1>(&q, scratch[team], 1 + team);
        if constexpr (CLUSTER) {
            // deviations about the mean of all: those about the share's own mean, and its distance
            cg::cluster_group cluster = cg::this_cluster();
            if (threadIdx.x < ranks) *cluster.map_shared_rank(&shares[turn][rank], threadIdx.x) = make_float2(mu, q);
            cluster.sync();
            float total = 0.f;
            for (unsigned k = 0; k < ranks; k++) {
                const size_t at = k * p.share;
                total += shares[turn][k].x * (float)(at < p.n ? min(p.share, p.n - at) : 0);
            }
            mu = total / (float)p.n;
            q = 0.f;
            for (unsigned k = 0; k < ranks; k++) {
                const size_t at = k * p.share;
                const float d = shares[turn][k].x - mu;
                q += shares[turn][k].y + d * d * (float)(at < p.n ? min(p.share, p.n - at) : 0);
            }
        }
        const float r = 1.0f / sqrtf(q / (float)p.n + p.eps);
        if (t == 0 && rank == 0) {
            if (p.mean) p.mean[row] = mu;
            if (p.rstd) p.rstd[row] = r;
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
            const size_t first = begin + (size_t)(k * TEAM + (t & ~31)) * V;       // of the warp
            if (first >= end) break;
            const size_t col = begin + (size_t)(k * TEAM + t) * V;
            float xh[V];
#pragma unroll
            for (int j = 0; j < V; j++) xh[j] = col < end ? (v[k][j] - mu) * r : 0.f;
            ln_put<T, V>(p, row, col, xh);
        }
    }
}

// Longer rows: a cluster per row that reads its share three times (from L2 the second and third time).
template <typename T, int V>
__global__ void __launch_bounds__(512) ln_forward_long_kernel(const __grid_constant__ LnForward<T> p)
{
    __shared__ float scratch[16];
    __shared__ float2 shares[2][8];
    grid_dependency_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), ranks = cluster.num_blocks();
    const size_t begin = rank * p.share, end = min(begin + p.share, p.n);
    const float mine = (float)(begin < p.n ? end - begin : 0);
    const int step = (int)(gridDim.x / ranks);
    constexpr int U = 4;
    int turn = 0;
    for (int row = (int)(blockIdx.x / ranks); row < p.rows; row += step, turn ^= 1) {
        const T *x = p.x + (size_t)row * p.x_pitch;
        auto total = [&](auto f) {
            float s[U] = {};
            for (size_t base = begin; base < end; base += 512 * V * U) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const size_t col = base + (size_t)(u * 512 + threadIdx.x) * V;
                    if (col < end) {
                        const Pack<T, V> in = load_pack<T, V>(x + col);
#pragma unroll
                        for (int j = 0; j < V; j++) s[u] += f(to_float(in.v[j]));
                    }
                }
            }
            float v = (s[0] + s[1]) + (s[2] + s[3]);
            team_total<512, 1>(&v, scratch, 1);
            return v;
        };
        float mu = total([](float v) { return v; }) / fmaxf(mine, 1.f);
        float q = total([&](float v) { const float d = v - mu; return d * d; });
        if (threadIdx.x < ranks) *cluster.map_shared_rank(&shares[turn][rank], threadIdx.x) = make_float2(mu, q);
        cluster.sync();
        float sum = 0.f;
        for (unsigned k = 0; k < ranks; k++) {
            const size_t at = k * p.share;
            sum += shares[turn][k].x * (float)(at < p.n ? min(p.share, p.n - at) : 0);
        }
        mu = sum / (float)p.n;
        q = 0.f;
        for (unsigned k = 0; k < ranks; k++) {
            const size_t at = k * p.share;
            const float d = shares[turn][k].x - mu;
            q += shares[turn][k].y + d * d * (float)(at < p.n ? min(p.share, p.n - at) : 0);
        }
        const float r = 1.0f / sqrtf(q / (float)p.n + p.eps);
        if (threadIdx.x == 0 && rank == 0) {
            if (p.mean) p.mean[row] = mu;
            if (p.rstd) p.rstd[row] = r;
        }
        for (size_t base = begin + (threadIdx.x & ~31u) * V; base < end; base += 512 * V) {      // whole warps: they share blocks
            const size_t col = base + (threadIdx.x & 31) * V;
            float xh[V];
            if (col < end) {
                const Pack<T, V> in = load_pack<T, V>(x + col);
#pragma unroll
                for (int j = 0; j < V; j++) xh[j] = (to_float(in.v[j]) - mu) * r;
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) xh[j] = 0.f;
            }
            ln_put<T, V>(p, row, col, xh);
        }
    }
}

template <typename T, int V>
static int ln_forward_launch(LnForward<T> p, cudaStream_t s)
{
    constexpr size_t kBlockRow = 512 * kLnValues;
    if (p.n <= kBlockRow) {
        // teams of one, four or sixteen warps: 1024, 4096 or 16384 values
        const int teams = p.n <= 32 * kLnValues ? 4 : 1;
        const Launch launch((unsigned)min((p.rows + teams - 1) / teams, sm_count() * 16), p.n <= 128 * kLnValues ? 128 : 512, 0, s);
        if (p.n <= 32 * kLnValues) launch(ln_forward_kernel<T, V, 32, 128, false>, p);
        else if (p.n <= 128 * kLnValues) launch(ln_forward_kernel<T, V, 128, 128, false>, p);
        else launch(ln_forward_kernel<T, V, 512, 512, false>, p);
    } else {
        const int ranks = p.n <= 2 * kBlockRow ? 2 : p.n <= 4 * kBlockRow ? 4 : 8;
        p.share = align_up((p.n + ranks - 1) / ranks, 32 * V);
        Launch launch((unsigned)(min(p.rows, sm_count() * 2) * ranks), 512, 0, s);
        launch.cluster((unsigned)ranks);
        if (p.n <= 8 * kBlockRow) launch(ln_forward_kernel<T, V, 512, 512, true>, p);
        else launch(ln_forward_long_kernel<T, V>, p);
    }
    B200_LAUNCH_CHECK();
    return B200_OK;
}

// ---- backward ----------------------------------------------------------------------------------------------------------------

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
    int weights;                 // form dgamma and dbeta
    float *part;                 // [groups][2][n] partial sums of dgamma and dbeta
    int groups;
    float2 *row_part;            // long rows: [rows][pieces] partial sums of g and g xh
    int pieces;
};

// V values of dy and of what xh comes from, as loaded
template <typename T, int V> struct LnRaw { Pack<T, V> dy, x; CkptCodes<V> c; uint32_t e; };

template <typename T, int V>
__device__ __forceinline__ void ln_load(const LnBackward<T> &p, int row, size_t col, LnRaw<T, V> &in)
{
    in.dy = load_pack<T, V>(p.dy + (size_t)row * p.dy_pitch + col);
    if (p.codes) {
        in.c = ckpt8_get<V>(p.codes + (size_t)row * p.blocks * kCkptBlock + col);
        in.e = p.exponents[(size_t)row * p.blocks + col / kCkptBlock];
    } else {
        in.x = load_pack<T, V>(p.x + (size_t)row * p.x_pitch + col);
    }
}
template <typename T, int V>
__device__ __forceinline__ void ln_values(const LnBackward<T> &p, const LnRaw<T, V> &in, float mu, float r, float *dy, float *xh)
{
    if (p.codes) {
        ckpt8_values<V>(xh, in.c, in.e);
    } else {
#pragma unroll
        for (int j = 0; j < V; j++) xh[j] = (to_float(in.x.v[j]) - mu) * r;
    }
#pragma unroll
    for (int j = 0; j < V; j++) dy[j] = to_float(in.dy.v[j]);
}

constexpr int kLnBack = 8;          // columns of a thread in the one-pass form

// Rows of up to 8192 values in one pass: a team holds a row, a thread the same columns of every row, so gamma stays in
// registers and dgamma, dbeta are summed there; the teams of a block join theirs in shared memory, the blocks in a second
// kernel.
template <typename T, int V, int TEAM, int BLOCK>
__global__ void __launch_bounds__(BLOCK, 1024 / BLOCK) ln_backward_rows_kernel(const __grid_constant__ LnBackward<T> p)
{
    constexpr int K = kLnBack / V, kTeams = BLOCK / TEAM, kColumns = TEAM * kLnBack;
    __shared__ float scratch[kTeams][2 * TEAM / 32];
    __shared__ float joined[kTeams > 1 ? 2 * kColumns : 1];
    grid_dependency_wait();
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    float gamma[K][V], dgamma[K][V], dbeta[K][V];
    bool in[K];
#pragma unroll
    for (int k = 0; k < K; k++) {
        const size_t col = (size_t)(k * TEAM + t) * V;
        in[k] = col < p.n;
#pragma unroll
        for (int j = 0; j < V; j++) { gamma[k][j] = in[k] ? __ldg(p.gamma + col + j) : 0.f; dgamma[k][j] = dbeta[k][j] = 0.f; }
    }
    const int step = (int)gridDim.x * kTeams;
    int row = (int)blockIdx.x * kTeams + team;
    for (; row < p.rows; row += step) {
        LnRaw<T, V> raw[K];
#pragma unroll
        for (int k = 0; k < K; k++)
            if (in[k]) ln_load<T, V>(p, row, (size_t)(k * TEAM + t) * V, raw[k]);
        const float r = p.rstd[row], mu = p.mean ? p.mean[row] : 0.f;
        float dy[K][V], xh[K][V], s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (in[k]) {
                ln_values<T, V>(p, raw[k], mu, r, dy[k], xh[k]);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) dy[k][j] = xh[k][j] = 0.f;
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                dgamma[k][j] = fmaf(dy[k][j], xh[k][j], dgamma[k][j]);
                dbeta[k][j] += dy[k][j];
                dy[k][j] *= gamma[k][j];                    // g
                s[0] += dy[k][j];
                s[1] = fmaf(dy[k][j], xh[k][j], s[1]);
            }
        }
        team_total<TEAM, 2>(s, scratch[team], 1 + team);
        const float c1 = s[0] / (float)p.n, c2 = s[1] / (float)p.n;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (!in[k]) continue;
            float dx[V];
#pragma unroll
            for (int j = 0; j < V; j++) dx[j] = r * (dy[k][j] - c1 - xh[k][j] * c2);
            store_pack<T, V>(p.dx + (size_t)row * p.dx_pitch + (size_t)(k * TEAM + t) * V, dx);
        }
    }
    if (!p.weights) return;
    if constexpr (kTeams > 1) {
        for (int w = 0; w < kTeams; w++) {                  // in the order of the teams
            if (team == w) {
#pragma unroll
                for (int k = 0; k < K; k++) {
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        float *a = joined + (k * TEAM + t) * V + j;
                        a[0] = w ? a[0] + dgamma[k][j] : dgamma[k][j];
                        a[kColumns] = w ? a[kColumns] + dbeta[k][j] : dbeta[k][j];
                    }
                }
            }
            __syncthreads();
        }
        float *out = p.part + (size_t)blockIdx.x * 2 * p.n;
        for (int c = threadIdx.x; c < (int)p.n; c += BLOCK) { out[c] = joined[c]; out[p.n + c] = joined[kColumns + c]; }
    } else {
        float *out = p.part + (size_t)blockIdx.x * 2 * p.n;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (!in[k]) continue;
#pragma unroll
            for (int j = 0; j < V; j++) {
                out[(size_t)(k * TEAM + t) * V + j] = dgamma[k][j];
                out[p.n + (size_t)(k * TEAM + t) * V + j] = dbeta[k][j];
            }
        }
    }
}

// Longer rows in two passes.  First: a thread owns V columns and walks a group of rows; it sums dgamma and dbeta of its columns, and
// its warp writes the partial sums of g and g xh of each row.  Second: a block joins a row's partial sums and forms a piece of dx.
constexpr int kLnSlice = 128;
template <typename T, int V>
__global__ void __launch_bounds__(kLnSlice) ln_backward_columns_kernel(const __grid_constant__ LnBackward<T> p)
{
    constexpr int U = 4;
    grid_dependency_wait();
    const size_t col = ((size_t)blockIdx.x * kLnSlice + threadIdx.x) * V;
    const int piece = (int)(blockIdx.x * (kLnSlice / 32) + (threadIdx.x >> 5)), lane = threadIdx.x & 31;
    const bool in = col < p.n;
    float gamma[V], dgamma[V], dbeta[V];
#pragma unroll
    for (int j = 0; j < V; j++) { gamma[j] = in ? __ldg(p.gamma + col + j) : 0.f; dgamma[j] = dbeta[j] = 0.f; }
    const int begin = (int)((long long)p.rows * blockIdx.y / p.groups), end = (int)((long long)p.rows * (blockIdx.y + 1) / p.groups);
    for (int row = begin; row < end; row += U) {
        LnRaw<T, V> raw[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (in && row + u < end) ln_load<T, V>(p, row + u, col, raw[u]);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (row + u >= end) break;
            float dy[V], xh[V], s1 = 0.f, s2 = 0.f;
            if (in) {
                ln_values<T, V>(p, raw[u], p.mean ? p.mean[row + u] : 0.f, p.rstd[row + u], dy, xh);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    dgamma[j] = fmaf(dy[j], xh[j], dgamma[j]);
                    dbeta[j] += dy[j];
                    const float g = dy[j] * gamma[j];
                    s1 += g;
                    s2 = fmaf(g, xh[j], s2);
                }
            }
            s1 = warp_total(s1);
            s2 = warp_total(s2);
            if (lane == 0) p.row_part[(size_t)(row + u) * p.pieces + piece] = make_float2(s1, s2);
        }
    }
    if (!p.weights || !in) return;
    float *out = p.part + (size_t)blockIdx.y * 2 * p.n + col;
#pragma unroll
    for (int j = 0; j < V; j++) { out[j] = dgamma[j]; out[p.n + j] = dbeta[j]; }
}

template <typename T, int V>
__global__ void __launch_bounds__(256) ln_backward_apply_kernel(const __grid_constant__ LnBackward<T> p)
{
    constexpr int K = 4;
    __shared__ float scratch[16];
    grid_dependency_wait();
    for (int row = blockIdx.y; row < p.rows; row += gridDim.y) {
        LnRaw<T, V> raw[K];
        const size_t base = (size_t)blockIdx.x * 256 * K * V;
#pragma unroll
        for (int k = 0; k < K; k++) {
            const size_t col = base + (size_t)(k * 256 + threadIdx.x) * V;
            if (col < p.n) ln_load<T, V>(p, row, col, raw[k]);
        }
        float s[2] = {0.f, 0.f};
        for (int i = threadIdx.x; i < p.pieces; i += 256) {
            const float2 v = p.row_part[(size_t)row * p.pieces + i];
            s[0] += v.x;
            s[1] += v.y;
        }
        team_total<256, 2>(s, scratch, 1);
        const float c1 = s[0] / (float)p.n, c2 = s[1] / (float)p.n, mu = p.mean ? p.mean[row] : 0.f, r = p.rstd[row];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const size_t col = base + (size_t)(k * 256 + threadIdx.x) * V;
            if (col >= p.n) continue;
            float dy[V], xh[V];
            ln_values<T, V>(p, raw[k], mu, r, dy, xh);
#pragma unroll
            for (int j = 0; j < V; j++) dy[j] = r * (dy[j] * __ldg(p.gamma + col + j) - c1 - xh[j] * c2);
            store_pack<T, V>(p.dx + (size_t)row * p.dx_pitch + col, dy);
        }
    }
}

// Sum of the groups' partial rows, in an order that does not depend on how they were scheduled: eight threads take every eighth group.
__global__ void __launch_bounds__(256) ln_backward_join_kernel(float *dgamma, float *dbeta, const float *__restrict__ part, int groups, size_t n, int accumulate)
{
    __shared__ float sums[8][33];
    grid_dependency_wait();
    const int c = threadIdx.x & 31, w = threadIdx.x >> 5;
    const size_t i = (size_t)blockIdx.x * 32 + c;
    float s = 0.f;
    if (i < 2 * n) {
#pragma unroll 4
        for (int g = w; g < groups; g += 8) s += part[(size_t)g * 2 * n + i];
    }
    sums[w][c] = s;
    __syncthreads();
    if (w || i >= 2 * n) return;
#pragma unroll
    for (int k = 1; k < 8; k++) s += sums[k][c];
    float *out = i < n ? dgamma + i : dbeta + (i - n);
    *out = accumulate ? *out + s : s;
}

constexpr size_t kLnOnePass = 8192;
struct LnPlan { bool one_pass; int team, block, groups, pieces; };
static LnPlan ln_plan(int rows, size_t n, int v)
{
    LnPlan w = {};
    w.one_pass = n <= kLnOnePass;
    if (w.one_pass) {
        w.team = n <= 256 ? 32 : n <= 1024 ? 128 : n <= 2048 ? 256 : n <= 4096 ? 512 : 1024;
        w.block = w.team <= 512 ? 512 : 1024;
        const int teams = w.block / w.team;
        w.groups = min((rows + teams - 1) / teams, sm_count() * (1024 / w.block));
    } else {
        const size_t slices = (n + (size_t)kLnSlice * v - 1) / ((size_t)kLnSlice * v);
        w.pieces = (int)slices * (kLnSlice / 32);
        // about sixteen blocks of 128 threads per SM, and eight rows each at least
        const long long want = ((long long)sm_count() * 16 + (long long)slices - 1) / (long long)slices;
        w.groups = (int)max(1ll, min(want, (long long)(rows + 7) / 8));
    }
    return w;
}

template <typename T, int V>
static int ln_backward_launch(LnBackward<T> p, float *dgamma, float *dbeta, int accumulate, char *workspace, cudaStream_t s)
{
    const LnPlan w = ln_plan(p.rows, p.n, V);
    p.groups = w.groups;
    p.pieces = w.pieces;
    p.row_part = reinterpret_cast<float2 *>(workspace);
    p.part = reinterpret_cast<float *>(workspace + align_up((size_t)p.rows * w.pieces * sizeof(float2), 16));
    if (w.one_pass) {
        const Launch launch((unsigned)w.groups, (unsigned)w.block, 0, s);
        switch (w.team) {
        case 32: launch(ln_backward_rows_kernel<T, V, 32, 512>, p); break;
        case 128: launch(ln_backward_rows_kernel<T, V, 128, 512>, p); break;
        case 256: launch(ln_backward_rows_kernel<T, V, 256, 512>, p); break;
        case 512: launch(ln_backward_rows_kernel<T, V, 512, 512>, p); break;
        default: launch(ln_backward_rows_kernel<T, V, 1024, 1024>, p); break;
        }
        B200_LAUNCH_CHECK();
    } else {
        Launch(dim3((unsigned)(w.pieces / (kLnSlice / 32)), (unsigned)w.groups), kLnSlice, 0, s)(ln_backward_columns_kernel<T, V>, p);
        B200_LAUNCH_CHECK();
        Launch(dim3((unsigned)((p.n + 1024 * V - 1) / (1024 * V)), (unsigned)min(p.rows, 65535)), 256, 0, s)(ln_backward_apply_kernel<T, V>, p);
        B200_LAUNCH_CHECK();
    }
    if (p.weights) {
        Launch((unsigned)((2 * p.n + 31) / 32), 256, 0, s)(ln_backward_join_kernel, dgamma, dbeta, p.part, p.groups, p.n, accumulate);
        B200_LAUNCH_CHECK();
    }
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
    const bool wide = wide_rows(x, type, n, x_pitch) && wide_rows(y, type, n, y_pitch);
#define B200_LN_FWD(T)                                                                                                                               \
    do {                                                                                                                                             \
        const LnForward<T> p = {(T *)y, mean, rstd, codes, exponents, (const T *)x, gamma, beta, rows, n, x_pitch, y_pitch, 0, eps};                 \
        return wide ? ln_forward_launch<T, kWide<T>>(p, ST(stream)) : ln_forward_launch<T, 1>(p, ST(stream));                                        \
    } while (0)
    if (type == B200_F32) B200_LN_FWD(float);
    if (type == B200_BF16) B200_LN_FWD(__nv_bfloat16);
    B200_LN_FWD(__half);
#undef B200_LN_FWD
}

size_t b200_ln_backward_workspace(int rows, size_t n)
{
    if (check_rows(rows, n) || rows == 0) return 0;
    // enough for either width of the loads
    size_t most = 0;
    for (int v = 1; v <= 8; v *= v == 1 ? 4 : 2) {
        const LnPlan w = ln_plan(rows, n, v);
        const size_t bytes = align_up((size_t)rows * w.pieces * sizeof(float2), 16) + sizeof(float) * 2 * n * (size_t)w.groups;
        most = bytes > most ? bytes : most;
    }
    return most;
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
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)) return fail(B200_E_ARG, "the workspace must be given, aligned to 16 bytes");
    if (workspace_bytes < b200_ln_backward_workspace(rows, n))
        return fail(B200_E_NOMEM, "the workspace has %zu bytes, %zu are needed", workspace_bytes, b200_ln_backward_workspace(rows, n));
    const bool wide = wide_rows(dx, type, n, dx_pitch) && wide_rows(dy, type, n, dy_pitch) && (!x || wide_rows(x, type, n, x_pitch));
    if (!x) mean = nullptr;
#define B200_LN_BWD(T)                                                                                                                               \
    do {                                                                                                                                             \
        const LnBackward<T> p = {(T *)dx, (const T *)dy, (const T *)x, mean, rstd, codes, exponents, gamma, rows, n, ckpt8_blocks(n), dy_pitch,      \
                                 x_pitch, dx_pitch, create_delta_weight != 0, nullptr, 0, nullptr, 0};                                               \
        return wide ? ln_backward_launch<T, kWide<T>>(p, dgamma, dbeta, accumulate, (char *)workspace, ST(stream))                                   \
                    : ln_backward_launch<T, 1>(p, dgamma, dbeta, accumulate, (char *)workspace, ST(stream));                                         \
    } while (0)
    if (type == B200_F32) B200_LN_BWD(float);
    if (type == B200_BF16) B200_LN_BWD(__nv_bfloat16);
    B200_LN_BWD(__half);
#undef B200_LN_BWD
}

}  // extern "C"
