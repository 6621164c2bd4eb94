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
#include "kernels.h"
#include "tc_ptx.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace b200 {

__device__ __forceinline__ float warp_total(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over the THREADS threads of a team (a warp, or whole warps that share named barrier `id`); every thread receives it.
// `scratch` holds a float per warp of the team and is free again after the call.
template <int THREADS>
__device__ __forceinline__ float team_total(float v, float *scratch, int id)
{
    v = warp_total(v);
    if constexpr (THREADS > 32) {
        constexpr int kWarps = THREADS / 32;
        const int lane = threadIdx.x & 31, warp = (threadIdx.x % THREADS) >> 5;
        if (lane == 0) scratch[warp] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
        v = warp_total(lane < kWarps ? scratch[lane] : 0.f);
        asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
    }
    return v;
}

// Two sums over a warp: the lower lanes finish the first, the upper ones the second
__device__ __forceinline__ float2 warp_totals(float2 v)
{
    const bool upper = threadIdx.x & 16;
    float mine = upper ? v.y : v.x;
    mine += __shfl_xor_sync(0xffffffffu, upper ? v.x : v.y, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    return make_float2(__shfl_sync(0xffffffffu, mine, 0), __shfl_sync(0xffffffffu, mine, 16));
}
// Two sums over a team with one barrier: the caller alternates between two `scratch` areas of a float2 per warp
template <int THREADS>
__device__ __forceinline__ float2 team_totals(float2 v, float2 *scratch, int id)
{
    v = warp_totals(v);
    if constexpr (THREADS > 32) {
        constexpr int kWarps = THREADS / 32;
        const int lane = threadIdx.x & 31, warp = (threadIdx.x % THREADS) >> 5;
        if (lane == 0) scratch[warp] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
        if constexpr (kWarps <= 8) {
            v = scratch[0];
#pragma unroll
            for (int k = 1; k < kWarps; k++) v = add2(v, scratch[k]);
        } else {
            v = warp_totals(lane < kWarps ? scratch[lane] : make_float2(0.f, 0.f));
        }
    }
    return v;
}

// V parameters from column `col` on (a multiple of V); wide: they start at a 16-byte boundary
template <int V>
__device__ __forceinline__ void load_params(float *f, const float *p, size_t col, bool wide)
{
    if constexpr (V >= 4) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < V / 4; i++) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(p + col) + i);
                f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = __ldg(p + col + i);
}

// (x - mu) r and xh gamma + beta of V values, in pairs
template <int V> __device__ __forceinline__ void normalise(float *xh, const float *x, float mu, float r)
{
    if constexpr (V == 1) {
        xh[0] = (x[0] - mu) * r;
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const float2 h = mul2(add2(make_float2(x[j], x[j + 1]), make_float2(-mu, -mu)), make_float2(r, r));
            xh[j] = h.x;
            xh[j + 1] = h.y;
        }
    }
}
template <int V> __device__ __forceinline__ void affine(float *y, const float *xh, const float *gamma, const float *beta)
{
    if constexpr (V == 1) {
        y[0] = fmaf(xh[0], gamma[0], beta[0]);
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const float2 v = fma2(make_float2(xh[j], xh[j + 1]), make_float2(gamma[j], gamma[j + 1]), make_float2(beta[j], beta[j + 1]));
            y[j] = v.x;
            y[j + 1] = v.y;
        }
    }
}
inline bool wide_params(const void *a, const void *b) { return !((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15); }

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
    size_t n, x_pitch, y_pitch;
    float eps;
    int wide;                    // gamma and beta can be read in 16-byte pieces
    size_t share;                // long rows: values of a row per block (a multiple of V)
    int groups;                  // and groups of rows
};

// writes V normalised values of a row and keeps them; col < n may be false for lanes that fill up a block of the checkpoint
template <typename T> struct LnOut { T *y; int8_t *codes; uint8_t *exponents; uint32_t padded; };
template <typename T>
__device__ __forceinline__ LnOut<T> ln_out(const LnForward<T> &p, int row)
{
    const size_t blocks = ckpt8_blocks(p.n);
    return {p.y + (size_t)row * p.y_pitch, p.codes ? p.codes + (size_t)row * blocks * kCkptBlock : nullptr, p.exponents + (size_t)row * blocks,
            (uint32_t)(blocks * kCkptBlock)};
}
template <typename T, int V>
__device__ __forceinline__ void ln_put(const LnForward<T> &p, const LnOut<T> &out, uint32_t col, const float *xh)
{
    if (out.codes) {
        const uint32_t b = ckpt8_exponent(ckpt8_top<V>(xh));
        if (col < out.padded) {
            ckpt8_put<V>(out.codes + col, xh, b, false);
            if (col % kCkptBlock == 0) out.exponents[col / kCkptBlock] = (uint8_t)b;
        }
    }
    if (col < (uint32_t)p.n) {
        float y[V], gamma[V], beta[V];
        load_params<V>(gamma, p.gamma, col, p.wide);
        load_params<V>(beta, p.beta, col, p.wide);
        affine<V>(y, xh, gamma, beta);
        store_pack<T, V>(out.y + col, y);
    }
}

// A row in the registers of one team: read once, written once.
template <typename T, int V, int VALUES, int TEAM, int BLOCK>
__global__ void __launch_bounds__(BLOCK, (VALUES <= 16 ? 1536 : 1024) / BLOCK) ln_forward_kernel(const __grid_constant__ LnForward<T> p)
{
    constexpr int K = VALUES / V, kTeams = BLOCK / TEAM;
    __shared__ float scratch[kTeams][TEAM / 32];
    grid_dependency_wait();
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM, n = (int)p.n;
    for (int row = (int)blockIdx.x * kTeams + team; row < p.rows; row += (int)gridDim.x * kTeams) {
        const T *x = p.x + (size_t)row * p.x_pitch;
        float v[K][V];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int col = (k * TEAM + t) * V;
#pragma unroll
            for (int j = 0; j < V; j++) v[k][j] = 0.f;
            if (col < n) {
                const Pack<T, V> in = load_pack<T, V>(x + col);
#pragma unroll
                for (int j = 0; j < V; j++) v[k][j] = to_float(in.v[j]);
            }
        }
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int j = 0; j < V; j++) s += v[k][j];
        }
        const float mu = team_total<TEAM>(s, scratch[team], 1 + team) / (float)n;
#pragma unroll
        for (int k = 0; k < K; k++) {
            if ((k * TEAM + t) * V < n) {
#pragma unroll
                for (int j = 0; j < V; j++) { const float d = v[k][j] - mu; q = fmaf(d, d, q); }
            }
        }
        const float r = 1.0f / sqrtf(team_total<TEAM>(q, scratch[team], 1 + team) / (float)n + p.eps);
        if (t == 0) {
            if (p.mean) p.mean[row] = mu;
            if (p.rstd) p.rstd[row] = r;
        }
        const LnOut<T> out = ln_out(p, row);
#pragma unroll
        for (int k = 0; k < K; k++) {
            if ((k * TEAM + (t & ~31)) * V >= n) break;     // whole warps: their lanes share blocks of the checkpoint
            const int col = (k * TEAM + t) * V;
            float xh[V];
#pragma unroll
            for (int j = 0; j < V; j++) xh[j] = col < n ? (v[k][j] - mu) * r : 0.f;
            ln_put<T, V>(p, out, (uint32_t)col, xh);
        }
    }
}

// Rows that no block holds in two kernels: the statistics, then the values, read a second time (from L2 where the tensor fits there).
// In one kernel, a cluster of blocks on a row, every block reads its share of gamma and beta for every row, which is twice
// the row itself in fp32: 55 us for 128 rows of 131072 values with a checkpoint.  Here a thread of the second kernel keeps those of
// its columns and walks down the rows.
//
// Statistics are joined pair by pair: values a of mean m_a and squared deviations q_a with values b give
// m = m_a + d b / (a + b), q = q_a + q_b + d^2 a b / (a + b), d = m_b - m_a.
struct Moments { float count, mean, q; };
__device__ __forceinline__ Moments join(Moments a, Moments b)
{
    const float count = a.count + b.count, part = count > 0.f ? b.count / count : 0.f, d = b.mean - a.mean;
    // (the mean of a row with an infinity is that infinity, on whichever side of the pair it is).  The counts come before the second
    // d: beside an empty side, where d is the other side's whole mean, the term is 0 times d and not infinity times 0.
    return {count, isfinite(d) ? fmaf(d, part, a.mean) : a.mean + b.mean, a.q + b.q + d * (a.count * part) * d};
}
__device__ __forceinline__ Moments warp_join(Moments m)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Moments other = {__shfl_xor_sync(0xffffffffu, m.count, o), __shfl_xor_sync(0xffffffffu, m.mean, o), __shfl_xor_sync(0xffffffffu, m.q, o)};
        m = join(m, other);
    }
    return m;
}

constexpr int kLnShares = 4;        // blocks of a cluster (four of 256 threads: 50 us for the case above, eight of 512: 56)
template <typename T, int V>
__global__ void __launch_bounds__(256, 4) ln_statistics_kernel(const __grid_constant__ LnForward<T> p)
{
    constexpr int U = 32 / V;
    __shared__ Moments warps[8], shares[kLnShares];
    grid_dependency_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank();
    const int row = (int)(blockIdx.x / kLnShares), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t begin = rank * p.share, end = min(begin + p.share, p.n);
    const T *x = p.x + (size_t)row * p.x_pitch;
    Moments m = {0.f, 0.f, 0.f};
    for (size_t base = begin; base < end; base += 256 * V * U) {
        float v[U][V], s = 0.f, q = 0.f, count = 0.f;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t col = base + (size_t)(u * 256 + threadIdx.x) * V;
            if (col < end) {
                const Pack<T, V> in = load_pack<T, V>(x + col);
#pragma unroll
                for (int j = 0; j < V; j++) v[u][j] = to_float(in.v[j]);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (base + (size_t)(u * 256 + threadIdx.x) * V < end) {
                count += (float)V;
#pragma unroll
                for (int j = 0; j < V; j++) s += v[u][j];
            }
        }
        const float mu = s / fmaxf(count, 1.f);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (base + (size_t)(u * 256 + threadIdx.x) * V < end) {
#pragma unroll
                for (int j = 0; j < V; j++) { const float d = v[u][j] - mu; q = fmaf(d, d, q); }
            }
        }
        m = join(m, {count, mu, q});
    }
    m = warp_join(m);
    if (lane == 0) warps[warp] = m;
    __syncthreads();
    if (warp == 0) {
        m = warp_join(lane < 8 ? warps[lane] : Moments{0.f, 0.f, 0.f});
        if (lane == 0) *cluster.map_shared_rank(&shares[rank], 0) = m;
    }
    cluster.sync();
    if (rank == 0 && threadIdx.x == 0) {
        m = shares[0];
#pragma unroll
        for (int k = 1; k < kLnShares; k++) m = join(m, shares[k]);
        p.mean[row] = m.mean;
        p.rstd[row] = 1.0f / sqrtf(m.q / (float)p.n + p.eps);
    }
}

constexpr int kLnSlice = 128;       // threads on a slice of columns, V each
template <typename T, int V>
__global__ void __launch_bounds__(kLnSlice) ln_normalise_kernel(const __grid_constant__ LnForward<T> p)
{
    // rows under way (of eight values four fill the registers: 400 x 20000 bf16 with a checkpoint took 35 us for 25)
    constexpr int U = V == 8 ? 2 : 4;
    grid_dependency_wait();
    const uint32_t n = (uint32_t)p.n, first = (blockIdx.x * kLnSlice + (threadIdx.x & ~31u)) * V, col = first + (threadIdx.x & 31) * V;
    if (first >= n) return;                                  // whole warps: their lanes share blocks of the checkpoint
    const bool in = col < n;
    float gamma[V], beta[V];
#pragma unroll
    for (int j = 0; j < V; j++) gamma[j] = beta[j] = 0.f;
    if (in) {
        load_params<V>(gamma, p.gamma, col, p.wide);
        load_params<V>(beta, p.beta, col, p.wide);
    }
    const size_t blocks = ckpt8_blocks(p.n);
    const bool in_block = p.codes && col < blocks * kCkptBlock, opens_block = in_block && col % kCkptBlock == 0;
    const int begin = (int)((long long)p.rows * blockIdx.y / p.groups), end = (int)((long long)p.rows * (blockIdx.y + 1) / p.groups);
    for (int row = begin; row < end; row += U) {
        Pack<T, V> raw[U];
        float mu[U], r[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (row + u >= end) break;
            if (in) raw[u] = load_pack<T, V>(p.x + (size_t)(row + u) * p.x_pitch + col);
            mu[u] = p.mean[row + u];
            r[u] = p.rstd[row + u];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (row + u >= end) break;
            float xh[V] = {}, y[V];
            if (in) {
#pragma unroll
                for (int j = 0; j < V; j++) y[j] = to_float(raw[u].v[j]);
                normalise<V>(xh, y, mu[u], r[u]);
            }
            if (p.codes) {
                const uint32_t b = ckpt8_exponent(ckpt8_top<V>(xh));
                if (in_block) ckpt8_put<V>(p.codes + (size_t)(row + u) * blocks * kCkptBlock + col, xh, b, false);
                if (opens_block) p.exponents[(size_t)(row + u) * blocks + col / kCkptBlock] = (uint8_t)b;
            }
            if (in) {
                affine<V>(y, xh, gamma, beta);
                store_pack<T, V>(p.y + (size_t)(row + u) * p.y_pitch + col, y);
            }
        }
    }
}

constexpr size_t kLnHeld = 16384;   // values of the longest row that a block holds
template <typename T, int V>
static int ln_forward_launch(LnForward<T> p, cudaStream_t s)
{
    if (p.n <= kLnHeld) {
        // teams of one, four or sixteen warps with 16 values a thread (more rows under way on an SM than with 32), or 32
        const int teams = p.n <= 512 ? 4 : 1;
        const Launch launch((unsigned)min((p.rows + teams - 1) / teams, sm_count() * 24), p.n <= 2048 ? 128 : 512, 0, s);
        if (p.n <= 512) launch(ln_forward_kernel<T, V, 16, 32, 128>, p);
        else if (p.n <= 2048) launch(ln_forward_kernel<T, V, 16, 128, 128>, p);
        else if (p.n <= 8192) launch(ln_forward_kernel<T, V, 16, 512, 512>, p);
        else launch(ln_forward_kernel<T, V, 32, 512, 512>, p);
        B200_LAUNCH_CHECK();
        return B200_OK;
    }
    if (!p.mean || !p.rstd) return fail(B200_E_ARG, "rows of more than %zu values need mean and rstd", kLnHeld);
    p.share = align_up((p.n + kLnShares - 1) / kLnShares, V);
    const int most = 0x7fffffff / kLnShares;
    for (int row = 0; row < p.rows; row += most) {           // a cluster per row
        LnForward<T> part = p;
        part.x += (size_t)row * p.x_pitch;
        part.mean += row;
        part.rstd += row;
        part.rows = min(most, p.rows - row);
        Launch(dim3((unsigned)part.rows * kLnShares), 256, 0, s).cluster(kLnShares)(ln_statistics_kernel<T, V>, part);
        B200_LAUNCH_CHECK();
    }
    // about sixteen blocks of 128 threads per SM, and four rows each at least
    const long long slices = (long long)((p.n + (size_t)kLnSlice * V - 1) / ((size_t)kLnSlice * V));
    p.groups = (int)max(1ll, min((long long)(p.rows + 3) / 4, min(65535ll, ((long long)sm_count() * 16 + slices - 1) / slices)));
    Launch(dim3((unsigned)slices, (unsigned)p.groups), kLnSlice, 0, s)(ln_normalise_kernel<T, V>, p);
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
    float2 *row_part;            // long rows: [rows][pieces] partial sums of g and g xh,
    float2 *row_mean;            // [rows] and their means
    int pieces;
    // one-pass form: shared memory of a team's slot for a row of dy, a row of x or codes, and its number of slots
    uint32_t dy_bytes, x_bytes;
    int depth;
    unsigned *status;
    float *dgamma, *dbeta;       // written directly where the blocks are one cluster
    int accumulate, one_cluster;
    int wide;                    // gamma can be read in 16-byte pieces
};

// V values of dy and of what xh comes from, as loaded
template <typename T, int V> struct LnRaw { Pack<T, V> dy, x; CkptCodes<V> c; uint32_t e; };

// where a row lies (64-bit address arithmetic once a row instead of once a load)
template <typename T> struct LnRow { const T *dy, *x; const int8_t *codes; const uint8_t *exponents; };
template <typename T>
__device__ __forceinline__ LnRow<T> ln_row(const LnBackward<T> &p, int row)
{
    LnRow<T> r;
    r.dy = p.dy + (size_t)row * p.dy_pitch;
    if (p.codes) { r.codes = p.codes + (size_t)row * p.blocks * kCkptBlock; r.exponents = p.exponents + (size_t)row * p.blocks; }
    else r.x = p.x + (size_t)row * p.x_pitch;
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void ln_load(const LnBackward<T> &p, const LnRow<T> &row, uint32_t col, LnRaw<T, V> &in)
{
    in.dy = load_pack<T, V>(row.dy + col);
    if (p.codes) {
        in.c = ckpt8_get<V>(row.codes + col);
        in.e = row.exponents[col / kCkptBlock];
    } else {
        in.x = load_pack<T, V>(row.x + col);
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

// Rows of up to 8192 values in one pass: a team holds a row, a thread the same sixteen columns of every row, so gamma stays in
// registers and dgamma, dbeta are summed there; the teams of a block join theirs in shared memory, the blocks (one per SM) in a
// second kernel, or, where the rows are few, in distributed shared memory.  Rows come into a ring of slots in shared memory by
// bulk copies, several rows ahead.  A bulk copy moves whole 16-byte pieces: of a row that starts anywhere also the neighbours'
// values in its first and its last piece, which nobody looks at.  Only pieces that lie whole in the tensor are copied; the values
// of the others (at most seven at either end of the tensor) are loaded by their threads.  (With each row's own whole pieces copied
// and its first and last values loaded a row ahead, 5003 x 1021 fp16 took 22.5 us.)
// Measured at 16384 x 2048 bf16 with the rows kept in 8 bits: 47 us, 3.6 TB/s, half the cycles issue (sixteen warps an SM wait for
// one another at a row's barrier); loads into registers, two blocks an SM, took 91 us, eight columns a thread with 1024 threads 80.  With the
// next row's sums formed before this row's are waited for, and the values formed again after it, 56.
constexpr int kLnBack = 16;
constexpr int kLnBlock = 512;
constexpr uint32_t kLnRing = 198656;
constexpr int kLnMostDepth = 8;

// The 16-byte pieces that a row of n values touches, as far as they lie whole in its tensor: address, bytes (may be 0), and how far
// behind the row's first piece they start
template <typename T>
__device__ __forceinline__ const T *row_pieces(const T *tensor, int rows, size_t pitch, int n, int row, uint32_t &bytes, uint32_t &skip)
{
    const uintptr_t first = reinterpret_cast<uintptr_t>(tensor), end = reinterpret_cast<uintptr_t>(tensor + (size_t)(rows - 1) * pitch + n);
    const uintptr_t at = reinterpret_cast<uintptr_t>(tensor + (size_t)row * pitch), piece = at & ~(uintptr_t)15;
    const uintptr_t lo = max(piece, (first + 15) & ~(uintptr_t)15), hi = min((at + (size_t)n * sizeof(T) + 15) & ~(uintptr_t)15, end & ~(uintptr_t)15);
    bytes = hi > lo ? (uint32_t)(hi - lo) : 0u;
    skip = (uint32_t)(lo - piece);
    return reinterpret_cast<const T *>(lo);
}
// the values of a row before `head` and from `tail` on lie in pieces that reach out of the tensor
template <typename T>
__device__ __forceinline__ void row_edges(const T *tensor, int rows, size_t pitch, int n, int row, int &head, int &tail)
{
    asm volatile("" : "+l"(tensor));                        // (not worked out ahead for every row, in registers that spill)
    const T *at = tensor + (size_t)row * pitch, *end = tensor + (size_t)(rows - 1) * pitch + n;
    const uintptr_t lo = (reinterpret_cast<uintptr_t>(tensor) + 15) & ~(uintptr_t)15, hi = reinterpret_cast<uintptr_t>(end) & ~(uintptr_t)15;
    const long long h = (long long)(lo - reinterpret_cast<uintptr_t>(at)) / (int)sizeof(T), l = (long long)(hi - reinterpret_cast<uintptr_t>(at)) / (int)sizeof(T);
    head = (int)max(0ll, h);
    tail = (int)min((long long)n, l);
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <int THREADS>
__device__ __forceinline__ void team_sync(int id)
{
    if constexpr (THREADS == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(THREADS) : "memory");
}

template <typename T, int V, int TEAM>
__global__ void __launch_bounds__(kLnBlock, 1) ln_backward_rows_kernel(const __grid_constant__ LnBackward<T> p)
{
    constexpr int K = kLnBack / V, kTeams = kLnBlock / TEAM, kColumns = TEAM * kLnBack;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float2 scratch[kTeams][2][TEAM / 32];
    __shared__ uint8_t exps[kTeams][2][kColumns / kCkptBlock];
    __shared__ __align__(8) uint64_t bars[kTeams][kLnMostDepth];
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM, n = (int)p.n, depth = p.depth;
    const uint32_t slot_bytes = p.dy_bytes + p.x_bytes;
    uint8_t *mine = ring + (size_t)team * depth * slot_bytes;
    const uint32_t bar0 = ptx::smem_u32(bars[team]);
    if (t == 0) {
        for (int d = 0; d < depth; d++) ptx::mbar_init(bar0 + 8u * d, 1);
        ptx::fence_barrier_init();
    }
    __syncthreads();
    grid_dependency_wait();

    const int step = (int)gridDim.x * kTeams;
    int row = (int)blockIdx.x * kTeams + team;
    // one thread: the pieces of a row into slot d
    auto issue = [&](int at, int d) {
        const uint32_t bar = bar0 + 8u * d, dst = ptx::smem_u32(mine + (size_t)d * slot_bytes);
        const T *dy = p.dy + (size_t)at * p.dy_pitch, *x = p.x + (size_t)at * p.x_pitch;
        uint32_t dy_size = (uint32_t)n * (uint32_t)sizeof(T), x_size = dy_size, dy_skip = 0, x_skip = 0;
        if constexpr (V == 1) {
            dy = row_pieces(p.dy, p.rows, p.dy_pitch, n, at, dy_size, dy_skip);
            if (!p.codes) x = row_pieces(p.x, p.rows, p.x_pitch, n, at, x_size, x_skip);
        }
        if (p.codes) x_size = (uint32_t)(p.blocks * kCkptBlock);
        ptx::mbar_arrive_expect_tx(bar, dy_size + x_size);
        if (V > 1 || dy_size) bulk_load(dst + dy_skip, dy, dy_size, bar);
        if (p.codes) bulk_load(dst + p.dy_bytes, p.codes + (size_t)at * p.blocks * kCkptBlock, x_size, bar);
        else if (V > 1 || x_size) bulk_load(dst + p.dy_bytes + x_skip, x, x_size, bar);
    };
    if (t < depth && row + (long long)t * step < p.rows) issue(row + t * step, t);
    // what does not come by bulk copies, a row ahead: statistics, and the row's place in its slot
    T *dx_row = p.dx + (size_t)row * p.dx_pitch;
    const size_t dx_step = (size_t)step * p.dx_pitch;
    uint32_t next_dy_at = (uint32_t)(reinterpret_cast<uintptr_t>(p.dy + (size_t)row * p.dy_pitch) & 15);
    uint32_t next_x_at = p.codes ? 0u : (uint32_t)(reinterpret_cast<uintptr_t>(p.x + (size_t)row * p.x_pitch) & 15);
    const uint32_t dy_turn = (uint32_t)step * (uint32_t)p.dy_pitch * (uint32_t)sizeof(T), x_turn = p.codes ? 0u : (uint32_t)step * (uint32_t)p.x_pitch * (uint32_t)sizeof(T);
    // the rows that may touch a piece that reaches out of the tensor, from its first row and from its last (16 bytes: eight values at most)
    const int edge = V > 1 ? 0 : n >= 8 ? 1 : 8;
    float next_mu = 0.f, next_r = 0.f;
    auto ahead = [&](int at) {
        next_r = p.rstd[at];
        if (p.mean) next_mu = p.mean[at];
    };
    // exponents: into a register two rows ahead, into shared memory one row ahead
    const bool has_exp = p.codes && t < (int)p.blocks;
    const uint8_t *exp_next = p.exponents + (size_t)row * p.blocks + t;
    const size_t exp_step = (size_t)step * p.blocks;
    uint8_t next_exp = 0;
    int turn = 0, limit = 1000000;
    if (row < p.rows) {
        ahead(row);
        if (has_exp) {
            exps[team][0][t] = *exp_next;
            exp_next += exp_step;
            if (row + step < p.rows) next_exp = *exp_next;
        }
    }
    team_sync<TEAM>(1 + team);

    constexpr int kPairs = kLnBack / 2;                      // values 2i and 2i + 1 of the thread's sixteen
    float2 gamma[kPairs], dgamma[kPairs], dbeta[kPairs];
    bool in[K];
#pragma unroll
    for (int k = 0; k < K; k++) in[k] = (k * TEAM + t) * V < n;
#pragma unroll
    for (int i = 0; i < kLnBack; i++) {
        const float g = in[i / V] ? __ldg(p.gamma + (i / V * TEAM + t) * V + i % V) : 0.f;
        if (i & 1) gamma[i / 2].y = g;
        else gamma[i / 2].x = g;
    }
#pragma unroll
    for (int i = 0; i < kPairs; i++) dgamma[i] = dbeta[i] = make_float2(0.f, 0.f);
    const float inverse_n = 1.0f / (float)n;
    int slot = 0;
    uint32_t phase = 0;
    for (; row < p.rows; row += step, turn ^= 1) {
        for (int polls = 0; !ptx::mbar_try_wait(bar0 + 8u * slot, phase); polls++) {
            if (polls >= limit) {                           // a second or so: the results are reported invalid, no later wait takes long
                atomicExch(p.status, 0xb00u + B200_E_TIMEOUT);
                __threadfence_system();
                limit = 0;
                break;
            }
        }
        const uint8_t *src = mine + (uint32_t)slot * slot_bytes;
        const T *dy_in = reinterpret_cast<const T *>(src + (V == 1 ? next_dy_at : 0u));
        const T *x_in = reinterpret_cast<const T *>(src + p.dy_bytes + (V == 1 ? next_x_at : 0u));
        const int8_t *code_in = reinterpret_cast<const int8_t *>(src + p.dy_bytes);
        const float r = next_r, mu = next_mu;
        float dy[kLnBack], xh[kLnBack];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int col = (k * TEAM + t) * V;
#pragma unroll
            for (int j = 0; j < V; j++) dy[k * V + j] = xh[k * V + j] = 0.f;
            if (in[k]) {
                const Pack<T, V> a = load_pack<T, V>(dy_in + col);
#pragma unroll
                for (int j = 0; j < V; j++) dy[k * V + j] = to_float(a.v[j]);
                if (p.codes) {
                    ckpt8_values<V>(xh + k * V, ckpt8_get<V>(code_in + col), exps[team][turn][col / kCkptBlock]);
                } else {
                    const Pack<T, V> b = load_pack<T, V>(x_in + col);
#pragma unroll
                    for (int j = 0; j < V; j++) xh[k * V + j] = to_float(b.v[j]);
#pragma unroll
                    for (int j = 0; j < V; j++) xh[k * V + j] = (xh[k * V + j] - mu) * r;
                }
            }
        }
        if (V == 1 && (row < edge || row >= p.rows - edge)) {
            int head, tail, x_head = 0, x_tail = n;
            row_edges(p.dy, p.rows, p.dy_pitch, n, row, head, tail);
            if (!p.codes) row_edges(p.x, p.rows, p.x_pitch, n, row, x_head, x_tail);
            const T *dy_at = p.dy + (size_t)row * p.dy_pitch + t, *x_at = p.x + (size_t)row * p.x_pitch + t;
#pragma unroll
            for (int k = 0; k < K; k++) {
                const int col = k * TEAM + t;
                if (in[k] && (col < head || col >= tail)) dy[k] = to_float(dy_at[k * TEAM]);
                if (in[k] && (col < x_head || col >= x_tail)) xh[k] = (to_float(x_at[k * TEAM]) - mu) * r;
            }
        }
        next_dy_at = (next_dy_at + dy_turn) & 15;
        next_x_at = (next_x_at + x_turn) & 15;
        float2 g[kPairs], s1 = make_float2(0.f, 0.f), s2 = s1;
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            const float2 d = make_float2(dy[2 * i], dy[2 * i + 1]), h = make_float2(xh[2 * i], xh[2 * i + 1]);
            dgamma[i] = fma2(d, h, dgamma[i]);
            dbeta[i] = add2(dbeta[i], d);
            g[i] = mul2(d, gamma[i]);
            s1 = add2(s1, g[i]);
            s2 = fma2(g[i], h, s2);
        }
        if (has_exp) {
            exps[team][turn ^ 1][t] = next_exp;
            exp_next += exp_step;
            if (row + 2ll * step < p.rows) next_exp = *exp_next;
        }
        if (row + step < p.rows) ahead(row + step);
        // after the barrier in here every thread has read the slot and written its exponents; the fence orders its reads and the copy
        // that then refills the slot (no time on any of the sizes measured)
        ptx::fence_proxy_async();
        const float2 s = team_totals<TEAM>(make_float2(s1.x + s1.y, s2.x + s2.y), scratch[team][turn], 1 + team);
        if (TEAM == 32) __syncwarp();
        if (t == 0 && row + (long long)depth * step < p.rows) issue(row + depth * step, slot);
        if (++slot == depth) { slot = 0; phase ^= 1u; }
        const float c1 = s.x * inverse_n, c2 = s.y * inverse_n;
        float dx[kLnBack];
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            const float2 d = add2(g[i], make_float2(-c1, -c1));
            const float2 v = mul2(fma2(make_float2(xh[2 * i], xh[2 * i + 1]), make_float2(-c2, -c2), d), make_float2(r, r));
            dx[2 * i] = v.x;
            dx[2 * i + 1] = v.y;
        }
#pragma unroll
        for (int k = 0; k < K; k++)
            if (in[k]) store_pack<T, V>(dx_row + (k * TEAM + t) * V, dx + k * V);
        dx_row += dx_step;
    }
    if (limit == 0) {                                       // copies still under way get time to land before the block ends
        for (int k = 0; k < 1000; k++) __nanosleep(200);
    }
    if (!p.weights) return;
    // the teams' sums, two by two (the ring is free: every copy has been waited for)
    __syncthreads();
    float2 *tree = reinterpret_cast<float2 *>(ring);
#pragma unroll
    for (int half = kTeams / 2; half > 0; half /= 2) {
        if (team >= half && team < 2 * half) {
            float2 *a = tree + (size_t)(team - half) * kColumns;
#pragma unroll
            for (int i = 0; i < kPairs; i++) { a[i * TEAM + t] = dgamma[i]; a[(kPairs + i) * TEAM + t] = dbeta[i]; }
        }
        __syncthreads();
        if (team < half) {
            const float2 *a = tree + (size_t)team * kColumns;
#pragma unroll
            for (int i = 0; i < kPairs; i++) { dgamma[i] = add2(dgamma[i], a[i * TEAM + t]); dbeta[i] = add2(dbeta[i], a[(kPairs + i) * TEAM + t]); }
        }
        __syncthreads();
    }
    if (!p.one_cluster) {
        if (team) return;
        float *out_g = p.part + (size_t)blockIdx.x * 2 * n, *out_b = out_g + n;
#pragma unroll
        for (int i = 0; i < kLnBack; i++) {
            if (!in[i / V]) continue;
            const int col = (i / V * TEAM + t) * V + i % V;
            out_g[col] = i & 1 ? dgamma[i / 2].y : dgamma[i / 2].x;
            out_b[col] = i & 1 ? dbeta[i / 2].y : dbeta[i / 2].x;
        }
        return;
    }
    // Few rows: the blocks are one cluster and join their sums through distributed shared memory, every block a share of the columns,
    // in the order of the blocks; no second kernel.
    float *sums = reinterpret_cast<float *>(ring);
    if (team == 0) {
#pragma unroll
        for (int i = 0; i < kLnBack; i++) {
            if (!in[i / V]) continue;
            const int col = (i / V * TEAM + t) * V + i % V;
            sums[col] = i & 1 ? dgamma[i / 2].y : dgamma[i / 2].x;
            sums[n + col] = i & 1 ? dbeta[i / 2].y : dbeta[i / 2].x;
        }
    }
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = (int)cluster.block_rank() * kLnBlock + (int)threadIdx.x; i < 2 * n; i += (int)cluster.num_blocks() * kLnBlock) {
        float v = 0.f;
        for (unsigned k = 0; k < cluster.num_blocks(); k++) v += *cluster.map_shared_rank(sums + i, k);
        float *out = i < n ? p.dgamma + i : p.dbeta + (i - n);
        *out = p.accumulate ? *out + v : v;
    }
    cluster.sync();                                         // no block leaves while another still reads its sums
}

// Longer rows in two passes.  First: a thread owns four columns (four single ones, where rows are not read in pieces) and walks a
// group of rows; it sums dgamma and dbeta of its columns, and its warp writes the partial sums of g and g xh of each row.
// Then a small kernel joins both kinds of sums, and the second pass, again a thread on its columns down a group of rows, forms
// dx.  512 x 16384 bf16: 33 us; with eight columns a thread and eight rows under way (140 registers) it took 49, with twice the groups
// 36.  (With the rows' sums joined by every block of the second pass, 300 x 40001 fp16 took 71 us, now 43.)
template <int V> constexpr int kLnRuns = V == 1 ? 4 : 1;      // runs of V columns of a thread, a slice apart
template <int V> constexpr int kLnLong = V == 1 ? 1 : 4;
template <typename T, int V>
__global__ void __launch_bounds__(kLnSlice) ln_backward_columns_kernel(const __grid_constant__ LnBackward<T> p)
{
    constexpr int C = kLnRuns<V>, U = V == 1 ? 1 : 2;          // rows under way
    grid_dependency_wait();
    const uint32_t first = (blockIdx.x * C * kLnSlice + threadIdx.x) * V, n = (uint32_t)p.n;
    const int piece = (int)(blockIdx.x * (kLnSlice / 32) + (threadIdx.x >> 5)), lane = threadIdx.x & 31;
    bool in[C];
    float gamma[C][V], dgamma[C][V], dbeta[C][V];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const uint32_t col = first + c * kLnSlice * V;
        in[c] = col < n;
#pragma unroll
        for (int j = 0; j < V; j++) gamma[c][j] = dgamma[c][j] = dbeta[c][j] = 0.f;
        if (in[c]) load_params<V>(gamma[c], p.gamma, col, p.wide);
    }
    const int begin = (int)((long long)p.rows * blockIdx.y / p.groups), end = (int)((long long)p.rows * (blockIdx.y + 1) / p.groups);
#pragma unroll(V == 1 ? 2 : 1)
    for (int row = begin; row < end; row += U) {
        LnRaw<T, V> raw[U][C];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (row + u >= end) break;
            const LnRow<T> at = ln_row(p, row + u);
#pragma unroll
            for (int c = 0; c < C; c++)
                if (in[c]) ln_load<T, V>(p, at, first + c * kLnSlice * V, raw[u][c]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (row + u >= end) break;
            const float mu = p.mean ? p.mean[row + u] : 0.f, r = p.rstd[row + u];
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int c = 0; c < C; c++) {
                if (!in[c]) continue;
                float dy[V], xh[V];
                ln_values<T, V>(p, raw[u][c], mu, r, dy, xh);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    dgamma[c][j] = fmaf(dy[j], xh[j], dgamma[c][j]);
                    dbeta[c][j] += dy[j];
                    const float g = dy[j] * gamma[c][j];
                    s1 += g;
                    s2 = fmaf(g, xh[j], s2);
                }
            }
            const float2 both = warp_totals(make_float2(s1, s2));
            if (lane == 0) p.row_part[(size_t)(row + u) * p.pieces + piece] = both;
        }
    }
    if (!p.weights) return;
#pragma unroll
    for (int c = 0; c < C; c++) {
        if (!in[c]) continue;
        float *out = p.part + (size_t)blockIdx.y * 2 * p.n + first + (size_t)c * kLnSlice * V;
#pragma unroll
        for (int j = 0; j < V; j++) { out[j] = dgamma[c][j]; out[p.n + j] = dbeta[c][j]; }
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kLnSlice) ln_backward_apply_kernel(const __grid_constant__ LnBackward<T> p)
{
    constexpr int C = kLnRuns<V>, U = V == 1 ? 1 : 2;
    grid_dependency_wait();
    const uint32_t first = (blockIdx.x * C * kLnSlice + threadIdx.x) * V, n = (uint32_t)p.n;
    bool in[C];
    float gamma[C][V];
#pragma unroll
    for (int c = 0; c < C; c++) {
        in[c] = first + c * kLnSlice * V < n;
        if (in[c]) load_params<V>(gamma[c], p.gamma, first + c * kLnSlice * V, p.wide);
    }
    const int begin = (int)((long long)p.rows * blockIdx.y / p.groups), end = (int)((long long)p.rows * (blockIdx.y + 1) / p.groups);
#pragma unroll(V == 1 ? 2 : 1)
    for (int row = begin; row < end; row += U) {
        LnRaw<T, V> raw[U][C];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (row + u >= end) break;
            const LnRow<T> at = ln_row(p, row + u);
#pragma unroll
            for (int c = 0; c < C; c++)
                if (in[c]) ln_load<T, V>(p, at, first + c * kLnSlice * V, raw[u][c]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (row + u >= end) break;
            const float2 m = p.row_mean[row + u];
            const float mu = p.mean ? p.mean[row + u] : 0.f, r = p.rstd[row + u];
            T *dx = p.dx + (size_t)(row + u) * p.dx_pitch;
#pragma unroll
            for (int c = 0; c < C; c++) {
                if (!in[c]) continue;
                float dy[V], xh[V];
                ln_values<T, V>(p, raw[u][c], mu, r, dy, xh);
#pragma unroll
                for (int j = 0; j < V; j++) dy[j] = r * (dy[j] * gamma[c][j] - m.x - xh[j] * m.y);
                store_pack<T, V>(dx + first + c * kLnSlice * V, dy);
            }
        }
    }
}

// Sum of the groups' partial rows, in an order that does not depend on how they were scheduled: SPLIT threads take every SPLIT-th
// group of a column.  The blocks from `column_blocks` on join the rows' partial sums instead, a warp to a row.
struct LnRows { const float2 *part; float2 *mean; int rows, pieces; };
template <int SPLIT>
__global__ void __launch_bounds__(1024) ln_backward_join_kernel(float *dgamma, float *dbeta, const float *__restrict__ part, int groups, size_t n, int accumulate,
                                                                unsigned column_blocks, LnRows r)
{
    constexpr int kWide = 1024 / SPLIT;
    __shared__ float sums[SPLIT][kWide + 1];
    grid_dependency_wait();
    if (blockIdx.x >= column_blocks) {
        const long long row = (long long)(blockIdx.x - column_blocks) * 32 + (threadIdx.x >> 5);
        if (row >= r.rows) return;
        const float2 *at = r.part + (size_t)row * r.pieces;
        float2 v = make_float2(0.f, 0.f);
#pragma unroll 4
        for (int k = threadIdx.x & 31; k < r.pieces; k += 32) v = add2(v, at[k]);
        v = warp_totals(v);
        if ((threadIdx.x & 31) == 0) r.mean[row] = make_float2(v.x / (float)n, v.y / (float)n);
        return;
    }
    const int c = threadIdx.x % kWide, w = threadIdx.x / kWide;
    const size_t i = (size_t)blockIdx.x * kWide + c;
    float s = 0.f;
    if (i < 2 * n) {
#pragma unroll 8
        for (int g = w; g < groups; g += SPLIT) s += part[(size_t)g * 2 * n + i];
    }
    if constexpr (SPLIT > 1) {
        sums[w][c] = s;
        __syncthreads();
        if (w == 0) {
#pragma unroll
            for (int k = 1; k < SPLIT; k++) s += sums[k][c];
        }
    }
    if (w || i >= 2 * n) return;
    float *out = i < n ? dgamma + i : dbeta + (i - n);
    *out = accumulate ? *out + s : s;
}

constexpr size_t kLnOnePass = 8192;
struct LnPlan { bool one_pass, one_cluster; int team, groups, pieces; };
static LnPlan ln_plan(int rows, size_t n, int v)
{
    LnPlan w = {};
    w.one_pass = n <= kLnOnePass;
    if (w.one_pass) {
        w.team = n <= 512 ? 32 : n <= 1024 ? 64 : n <= 2048 ? 128 : n <= 4096 ? 256 : 512;
        // A cluster of up to eight blocks where each team then has four rows at most: it joins the gradients itself.
        const int teams = kLnBlock / w.team;
        w.groups = min((rows + teams - 1) / teams, sm_count());
        w.one_cluster = rows <= 32 * teams;
        if (w.one_cluster) w.groups = w.groups > 4 ? 8 : w.groups > 2 ? 4 : w.groups;
    } else {
        const size_t slice = (size_t)kLnSlice * (v == 1 ? kLnRuns<1> : kLnRuns<4> * v), slices = (n + slice - 1) / slice;
        w.pieces = (int)slices * (kLnSlice / 32);
        // about eight blocks of 128 threads per SM (sixteen where single values need more loads under way), and eight rows each at
        // least: a group's partial sums are written and read once more
        const long long want = ((long long)sm_count() * (v == 1 ? 16 : 8) + (long long)slices - 1) / (long long)slices;
        w.groups = (int)max(1ll, min(want, (long long)(rows + 7) / 8));
    }
    return w;
}

static size_t row_bytes(const LnPlan &w, int rows) { return w.one_pass ? 0 : align_up((size_t)rows * (w.pieces + 1) * sizeof(float2), 16); }

template <typename T, int V>
static int ln_backward_launch(LnBackward<T> p, float *dgamma, float *dbeta, int accumulate, char *workspace, cudaStream_t s)
{
    constexpr int kLong = kLnLong<V>;
    const LnPlan w = ln_plan(p.rows, p.n, kLong);
    p.groups = w.groups;
    p.pieces = w.pieces;
    p.row_part = reinterpret_cast<float2 *>(workspace);
    p.row_mean = p.row_part + (size_t)p.rows * w.pieces;
    p.part = reinterpret_cast<float *>(workspace + row_bytes(w, p.rows));
    p.dgamma = dgamma;
    p.dbeta = dbeta;
    p.accumulate = accumulate;
    p.wide = wide_params(p.gamma, p.gamma);
    p.one_cluster = w.one_cluster;
    if (w.one_pass) {
        int r = status_word(&p.status);
        if (r) return r;
        const int teams = kLnBlock / w.team;
        p.dy_bytes = (uint32_t)align_up(p.n * sizeof(T) + 16, 16);
        p.x_bytes = p.codes ? (uint32_t)(p.blocks * kCkptBlock) : p.dy_bytes;
        p.depth = min(kLnMostDepth, (int)(kLnRing / (teams * (p.dy_bytes + p.x_bytes))));      // three at least: 8192 values of 4 bytes, twice
        // the ring, and after it the sums of the teams (32 KB) and of the block (two for every column)
        const uint32_t smem = max(max((uint32_t)(teams * p.depth) * (p.dy_bytes + p.x_bytes), 32768u), (uint32_t)(2 * sizeof(float) * p.n));
#define B200_LN_ROWS(TEAM)                                                                                                                           \
    do {                                                                                                                                             \
        if ((r = allow_shared<ln_backward_rows_kernel<T, V, TEAM>>((int)kLnRing))) return r;                                                         \
        Launch((unsigned)w.groups, kLnBlock, smem, s).cluster(w.one_cluster ? (unsigned)w.groups : 1u)(ln_backward_rows_kernel<T, V, TEAM>, p);      \
    } while (0)
        switch (w.team) {
        case 32: B200_LN_ROWS(32); break;
        case 64: B200_LN_ROWS(64); break;
        case 128: B200_LN_ROWS(128); break;
        case 256: B200_LN_ROWS(256); break;
        default: B200_LN_ROWS(512); break;
        }
#undef B200_LN_ROWS
        B200_LAUNCH_CHECK();
        if (w.one_cluster) return B200_OK;
    } else {
        Launch(dim3((unsigned)(w.pieces / (kLnSlice / 32)), (unsigned)w.groups), kLnSlice, 0, s)(ln_backward_columns_kernel<T, kLong>, p);
        B200_LAUNCH_CHECK();
    }
    const LnRows rows = {p.row_part, p.row_mean, w.one_pass ? 0 : p.rows, w.pieces};
    const unsigned row_blocks = (unsigned)((rows.rows + 31ll) / 32);
    // few columns need several threads each to fill the machine
    const int split = p.n <= 16384 && p.groups > 8 ? 32 : 1;
    const unsigned column_blocks = p.weights ? (unsigned)((2 * p.n * split + 1023) / 1024) : 0;
    if (column_blocks + row_blocks) {
        const Launch launch(column_blocks + row_blocks, 1024, 0, s);
        if (split > 1) launch(ln_backward_join_kernel<32>, dgamma, dbeta, p.part, p.groups, p.n, accumulate, column_blocks, rows);
        else launch(ln_backward_join_kernel<1>, dgamma, dbeta, p.part, p.groups, p.n, accumulate, column_blocks, rows);
        B200_LAUNCH_CHECK();
    }
    if (!w.one_pass) {
        Launch(dim3((unsigned)(w.pieces / (kLnSlice / 32)), (unsigned)w.groups), kLnSlice, 0, s)(ln_backward_apply_kernel<T, kLong>, p);
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
        const LnForward<T> p = {(T *)y, mean, rstd, codes, exponents, (const T *)x, gamma, beta, rows, n, x_pitch, y_pitch, eps,\
                                 wide_params(gamma, beta), 0, 0};                                                                                    \
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
    for (int v : {kLnLong<1>, kLnLong<4>}) {
        const LnPlan w = ln_plan(rows, n, v);
        const size_t bytes = row_bytes(w, rows) + sizeof(float) * 2 * n * (size_t)w.groups;
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
                                 x_pitch, dx_pitch, create_delta_weight != 0};                                             \
        return wide ? ln_backward_launch<T, kWide<T>>(p, dgamma, dbeta, accumulate, (char *)workspace, ST(stream))                                   \
                    : ln_backward_launch<T, 1>(p, dgamma, dbeta, accumulate, (char *)workspace, ST(stream));                                         \
    } while (0)
    if (type == B200_F32) B200_LN_BWD(float);
    if (type == B200_BF16) B200_LN_BWD(__nv_bfloat16);
    B200_LN_BWD(__half);
#undef B200_LN_BWD
}

}  // extern "C"
