// Weight and bias gradient of a Linear layer whose input was kept in 8 bits (ckpt8.cuh):
//   dweight[o][i] (+)= sum over rows of delta[row][o] * x[row][i],   dbias[o] (+)= sum over rows of delta[row][o]
#include "common.cuh"
#include "types.cuh"
#include "ckpt8.cuh"
#include "norm.h"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace b200 {

constexpr int kTile = 64, kDepth = 16;

// 64 x 64 outputs per block of 256 threads, 4 x 4 per thread, the checkpoint decoded while a slice of 16 rows is staged.  The blocks
// are numbered along the inputs first, in one dimension: the grid's second one ends at 65535, 4 194 240 outputs.
template <typename T>
__global__ void __launch_bounds__(256) ckpt8_wgrad_simt_kernel(float *dweight, float *dbias, const T *__restrict__ delta, const int8_t *__restrict__ codes,
                                                               const uint8_t *__restrict__ exponents, int rows, int out, size_t in, size_t pitch, size_t blocks,
                                                               int accumulate)
{
    __shared__ float a[kDepth][kTile], b[kDepth][kTile];
    grid_dependency_wait();
    const uint32_t tiles_in = (uint32_t)((in + kTile - 1) / kTile), tile_out = blockIdx.x / tiles_in;
    const size_t i0 = (size_t)(blockIdx.x - tile_out * tiles_in) * kTile;
    const int o0 = (int)tile_out * kTile;
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
        if (dbias && i0 == 0 && ti == 0) dbias[o] = accumulate ? dbias[o] + bias[x] : bias[x];
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const size_t i = i0 + ti * 4 + y;
            if (i >= in) break;
            float *w = dweight + (size_t)o * in + i;
            *w = accumulate ? *w + acc[x][y] : acc[x][y];
        }
    }
}

// ---- tensor-core form ---------------------------------------------------------------------------------------------------
//
// A CTA pair computes 256 x 256 outputs: 256 of delta's columns (128 per CTA) by 256 of the input's (128 decoded by each CTA and
// read by both), one 256-row MMA per 16 rows of the batch, accumulated in tensor memory.  Both operands are MN-major, so a
// row of delta or of the checkpoint becomes a row of the shared-memory tile as it lies in memory: no transposition anywhere.
//   * The kept values have 8 significant bits and are exact in bf16 with their scale.  delta is cut into PARTS pieces of 8 bits
//     (bf16 1, fp16 2, fp32 3, in either tensor-core mode), each exact, so every product is exact and the only roundings are
//     those of the fp32 accumulator.  The tensor core truncates its sums, a bias that grows with their number: after kChunk
//     stages the accumulator is added to the output (rounded to nearest) and starts again from zero.  8192 rows at a stretch
//     were off by 2.5e-6 of the result, chunks of 2048 are by 4e-7, for 22 of 264 us.
//   * One warp each brings the codes and delta in by TMA (bf16 straight into the operand tile); four groups of four warps decode
//     and split from shared memory into a ring of operand stages (five instructions for two values, once per pair and tile).
//     A group takes every fourth stage, so four stages are in work at a time: with all sixteen warps on each stage its chain of
//     waits, loads and stores was in series with the next one's.  Stages are as long as the rings allow (bf16 with 32 rows
//     in place of 64: 350 us for 264; fp16 with 16 for 32: 652 for 495), because a stage's waits, exponents and fences cost a
//     group some hundred instructions whatever its length.
//   * The grid is one pair per two SMs.  Whole tiles go round the pairs; what is left over (or everything, where there are
//     fewer tiles than pairs) is split along the batch into units that write partial tiles, joined by a second
//     kernel in the order of the units.  No atomics: the result does not depend on scheduling.
// Measured at 8192 rows, 4096 x 4096, a single pass with inputs from memory: bf16 272 us = 1.01 PFLOP/s (303 us after a second of
// nothing else, when the power limit holds the clock at 1.55 GHz; L2 prefetches ahead of the loads changed nothing), fp16 537, fp32
// 859; six passes in a row 269, 520 and 829 each.  The tensor pipe is active half the time in bf16, the converter warps issue in
// 58 % of the cycles, and without their stores (199 us of 264 at the time) or without the products (199 too) it is no faster than shared memory and
// the two together allow.
constexpr int kPairTile = 256;                     // outputs of a pair in both directions
constexpr int kEpilogueWarps = 4, kConverterWarps = 16, kGroupWarps = 4, kGroups = kConverterWarps / kGroupWarps;
constexpr int kConverters = kConverterWarps * 32;
constexpr int kTcThreads = (kEpilogueWarps + kConverterWarps + 3) * 32;
constexpr int kPitch = 36;                         // floats in a row of the epilogue's transposition buffer
constexpr size_t kUnitFloats = (size_t)kPairTile * kPairTile + kPairTile;      // a partial tile and its partial bias gradient

struct WgradParams {
    float *dweight, *dbias;
    const uint8_t *exponents;
    int rows, out, accumulate, vector_out;
    size_t in, blocks;
    int tiles_n, steps, chunk_steps, pairs, waves, first_tail, tail_units, splits;
    float *partial;
    unsigned *status;
    uint32_t idesc;
};

// One chunk of a tile: `first` starts its output, later ones add to it; `last` ends it.
struct WorkItem { int mt, nt, begin, steps, unit; bool first, last; };

// The work items of a pair in order: the chunks of its whole tiles, then those of its tail unit.
struct ItemCursor {
    WorkItem w;
    int turn, end;
    __device__ __forceinline__ bool open(const WgradParams &p, int pair)
    {
        int tile;
        w.begin = 0; end = p.steps; w.unit = -1;
        if (turn < p.waves) {
            tile = pair + turn * p.pairs;
        } else {
            if (turn > p.waves || pair >= p.tail_units) return false;
            const int split = pair % p.splits;
            tile = p.first_tail + pair / p.splits;
            w.begin = (int)((long long)p.steps * split / p.splits);
            end = (int)((long long)p.steps * (split + 1) / p.splits);
            if (p.splits > 1) w.unit = pair;
        }
        w.mt = tile / p.tiles_n;
        w.nt = tile - w.mt * p.tiles_n;
        w.first = true;
        return chunk(p);
    }
    __device__ __forceinline__ bool chunk(const WgradParams &p)
    {
        w.steps = min(p.chunk_steps, end - w.begin);
        w.last = w.begin + w.steps == end;
        return true;
    }
    __device__ __forceinline__ bool start(const WgradParams &p, int pair) { turn = 0; return open(p, pair); }
    __device__ __forceinline__ bool next(const WgradParams &p, int pair)
    {
        if (w.last) { turn++; return open(p, pair); }
        w.begin += w.steps;
        w.first = false;
        return chunk(p);
    }
};

// Eight codes with the scale of their block -> eight bf16 values.  The bytes 0x43, u form the bf16 bits of 128 + (u & 127) and
// of 128 + (u & 128); their difference is the signed code, exact, and so is its product with the power of two.
__device__ __forceinline__ uint4 decode8(uint2 codes, uint32_t exponent)
{
    const uint32_t f = __float_as_uint(ckpt8_unit(exponent) * 0.015625f);      // 2^(b-133), exact in bf16
    const uint32_t scale = __byte_perm(f, 0, 0x3232);
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t t = __byte_perm(i < 2 ? codes.x : codes.y, 0x43434343u, i & 1 ? 0x4342 : 0x4140);
        const uint32_t a = t & 0xff7fff7fu, b = t & 0xff80ff80u;
        __nv_bfloat162 q = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b));
        q = __hmul2(q, *reinterpret_cast<const __nv_bfloat162 *>(&scale));
        v[i] = *reinterpret_cast<uint32_t *>(&q);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// x = piece 0 + piece 1 + ..., each the upper 16 bits of what is left: exact.  An infinity has no remainder; a NaN stays one in
// the second piece.
__device__ __forceinline__ float remainder_of(float x, float &upper)
{
    upper = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    return fabsf(x) == INFINITY ? 0.f : x - upper;
}
__device__ __forceinline__ uint32_t upper_halves(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }

// eight values of delta from two (fp32) or one 16-byte vector
template <typename T> __device__ __forceinline__ void unpack8(uint4 lo, uint4 hi, float *f);
template <> __device__ __forceinline__ void unpack8<float>(uint4 lo, uint4 hi, float *f)
{
    const uint32_t u[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = __uint_as_float(u[i]);
}
template <> __device__ __forceinline__ void unpack8<__nv_bfloat16>(uint4 lo, uint4, float *f)
{
    const uint32_t u[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(u[i] << 16); f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
}
template <> __device__ __forceinline__ void unpack8<__half>(uint4 lo, uint4, float *f)
{
    const uint32_t u[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
        f[2 * i] = h.x; f[2 * i + 1] = h.y;
    }
}

// Rows of the batch in a stage, and the two rings: raw (codes as stored, and delta where it has to be split) and operands.  Both
// have a multiple of kGroups slots, so a slot always belongs to the same group: a group that waits for a phase has itself seen the
// one before, which the parity of a barrier cannot tell from it.
template <typename T, int PARTS> struct TcShape {
    static constexpr int kRows = PARTS == 1 ? 64 : PARTS == 2 ? 32 : 16;
    static constexpr uint32_t kOperand = kRows * 256u;                        // bytes of a 128-wide bf16 tile
    static constexpr uint32_t kStage = (PARTS + 1) * kOperand;
    static constexpr int kStages = PARTS == 3 ? 8 : 4;
    static constexpr uint32_t kCodes = kRows * 128u;
    static constexpr uint32_t kRaw = kCodes + (PARTS == 1 ? 0u : kRows * 128u * (uint32_t)sizeof(T));
    static constexpr int kRaws = PARTS == 3 ? 4 : 8;
    static constexpr uint32_t kRing = kStages * kStage;                       // bytes before the raw ring
    static constexpr int kCodePasses = kRows / 16, kDeltaPasses = kRows / 8;  // of a group's 128 threads over the stage
    static constexpr int kChunk = (PARTS == 1 ? 2048 : 1024) / kRows;         // stages after which the accumulator is emptied
};
constexpr int kAccumulators = 2;                                              // the epilogue of an item overlaps the products of the next
constexpr size_t kRingBytes = 200704;
constexpr size_t kTcSmem = 1024 + kRingBytes + kEpilogueWarps * 32 * kPitch * 4 + kConverterWarps * 128 * 4 + 512;

template <typename T, int PARTS>
__global__ void __launch_bounds__(kTcThreads, 1)
ckpt8_wgrad_tc_kernel(const __grid_constant__ CUtensorMap codes_map, const __grid_constant__ CUtensorMap delta_map, const __grid_constant__ WgradParams p)
{
    using S = TcShape<T, PARTS>;
    static_assert(S::kRing + S::kRaws * S::kRaw <= kRingBytes, "rings");
    static_assert(S::kStages % kGroups == 0 && S::kRaws % kGroups == 0, "a slot belongs to one group");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float *turn = reinterpret_cast<float *>(smem + kRingBytes);               // epilogue: 32 x 32 per warp
    float *bias_sums = turn + kEpilogueWarps * 32 * kPitch;                   // converters: [warp][128]
    uint64_t *bars = reinterpret_cast<uint64_t *>(bias_sums + kConverterWarps * 128);
    const uint32_t bar_base = ptx::smem_u32(bars);
    auto full_bar = [&](int s) { return bar_base + 8u * s; };                 // operand stage: a CTA's own converters (and its delta tile)
    auto empty_bar = [&](int s) { return bar_base + 8u * (S::kStages + s); };
    auto peer_bar = [&](int s) { return bar_base + 8u * (2 * S::kStages + s); };       // in the leader: the peer's stage is full
    auto raw_full_bar = [&](int s) { return bar_base + 8u * (3 * S::kStages + s); };
    auto raw_empty_bar = [&](int s) { return bar_base + 8u * (3 * S::kStages + S::kRaws + s); };
    auto tfull_bar = [&](int a) { return bar_base + 8u * (3 * S::kStages + 2 * S::kRaws + a); };
    auto tempty_bar = [&](int a) { return bar_base + 8u * (3 * S::kStages + 2 * S::kRaws + 2 + a); };
    constexpr int kBars = 3 * S::kStages + 2 * S::kRaws + 4;
    static_assert(kBars * 8 + 8 <= 512, "barriers");
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)ptx::cluster_ctarank(), pair = (int)(blockIdx.x >> 1);
    constexpr int kIssuer = kEpilogueWarps + kConverterWarps, kCodesLoader = kIssuer + 1, kDeltaLoader = kIssuer + 2;
    constexpr bool kDirect = PARTS == 1;                                      // delta goes straight into the operand stage

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; s++) {
            ptx::mbar_init(full_bar(s), kGroupWarps + (kDirect ? 1 : 0));
            ptx::mbar_init(empty_bar(s), 1 + (kDirect ? kGroupWarps : 0));
            ptx::mbar_init(peer_bar(s), 1);
        }
        for (int s = 0; s < S::kRaws; s++) { ptx::mbar_init(raw_full_bar(s), kDirect ? 1 : 2); ptx::mbar_init(raw_empty_bar(s), kGroupWarps); }
        for (int a = 0; a < 2; a++) { ptx::mbar_init(tfull_bar(a), 1); ptx::mbar_init(tempty_bar(a), 2 * kEpilogueWarps); }
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::prefetch_tensormap(&codes_map);
        ptx::prefetch_tensormap(&delta_map);
    }
    if (warp == kIssuer) { ptx::tmem_alloc_pair(ptx::smem_u32(tmem_slot), 512u); ptx::tmem_relinquish_pair(); }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    grid_dependency_wait();

    if (warp == kCodesLoader || warp == kDeltaLoader) {
        // ------------------------------------------------------------------ TMA loads (one thread each for the codes and for delta)
        if (lane == 0) {
            const bool codes = warp == kCodesLoader, direct = kDirect && !codes;
            const int slots = direct ? S::kStages : S::kRaws;
            const uint32_t base = ptx::smem_u32(smem) + (direct ? 0u : S::kRing + (codes ? 0u : S::kCodes)), pitch = direct ? S::kStage : S::kRaw;
            const uint32_t full = direct ? full_bar(0) : raw_full_bar(0), empty = direct ? empty_bar(0) : raw_empty_bar(0);
            const uint32_t bytes = codes ? S::kCodes : direct ? S::kOperand : S::kRaw - S::kCodes;
            const CUtensorMap *map = codes ? &codes_map : &delta_map;
            int slot = 0;
            uint32_t phase = 0;
            bool ok = true;
            ItemCursor at;
            for (bool more = at.start(p, pair); more && ok; more = at.next(p, pair)) {
                const int col = (codes ? at.w.nt : at.w.mt) * kPairTile + rank * 128, end = (at.w.begin + at.w.steps) * S::kRows;
                for (int row = at.w.begin * S::kRows; row < end; row += S::kRows) {
                    if (!(ok = wait_bar(empty + 8u * slot, phase ^ 1u, abort_flag, p.status, 0x100u + B200_E_TIMEOUT))) break;
                    const uint32_t dst = base + (uint32_t)slot * pitch, bar = full + 8u * slot;
                    ptx::mbar_arrive_expect_tx(bar, bytes);
                    ptx::tma_load_2d(dst, map, bar, col, row);
                    if (direct) ptx::tma_load_2d(dst + S::kOperand / 2, map, bar, col + 64, row);
                    if (++slot == slots) { slot = 0; phase ^= 1u; }
                }
            }
        }
    } else if (warp >= kEpilogueWarps && warp < kIssuer) {
        // ------------------------------------------------------------------ converters
        const int group = (warp - kEpilogueWarps) / kGroupWarps, t = (threadIdx.x - kEpilogueWarps * 32) & 127;
        const int r = t >> 3, c = t & 7;                                      // codes: row (of 16) and run of sixteen columns
        const int r8 = t >> 4, c8 = t & 15;                                   // delta: row (of 8) and group of eight columns

        // exponents of this thread's codes in the group's next stage, loaded while the current one is converted
        ItemCursor ahead;
        bool more_ahead = ahead.start(p, pair);
        int step_ahead = group, row_ahead = 0;
        const uint8_t *src_ahead = nullptr;
        uint32_t exps[S::kCodePasses];
        const size_t stride = (size_t)kGroups * S::kRows * p.blocks;
        auto fetch = [&](bool fresh) {
            while (more_ahead && step_ahead >= ahead.w.steps) {
                step_ahead -= ahead.w.steps;
                more_ahead = ahead.next(p, pair);
                fresh = true;
            }
            if (fresh) {
                const size_t i = (size_t)ahead.w.nt * kPairTile + rank * 128 + c * 16;
                row_ahead = (ahead.w.begin + step_ahead) * S::kRows + r;
                src_ahead = p.exponents + (size_t)row_ahead * p.blocks + i / kCkptBlock;
                if (!more_ahead || i >= p.blocks * kCkptBlock) row_ahead = p.rows;       // nothing to load
            }
#pragma unroll
            for (int k = 0; k < S::kCodePasses; k++) {
                exps[k] = 0;
                if (row_ahead + 16 * k < p.rows) exps[k] = __ldg(src_ahead + (size_t)(16 * k) * p.blocks);
            }
            if (row_ahead < p.rows) row_ahead += kGroups * S::kRows;
            src_ahead += stride;
            step_ahead += kGroups;
        };
        fetch(true);

        float sums[8] = {};
        // the end of a tile: its bias gradient
        auto finish = [&](const WorkItem &w) {
            // the thirty-two row slots (two a warp, joined by a shuffle), then one thread per column
#pragma unroll
            for (int x = 0; x < 8; x++) sums[x] += __shfl_xor_sync(0xffffffffu, sums[x], 16);
            if (lane < 16) {
#pragma unroll
                for (int x = 0; x < 8; x++) bias_sums[(warp - kEpilogueWarps) * 128 + c8 * 8 + x] = sums[x];
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kConverters) : "memory");
            if (group == 0) {
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < kConverterWarps; k++) s += bias_sums[k * 128 + t];
                const int o = w.mt * kPairTile + rank * 128 + t;
                if (w.unit >= 0) p.partial[(size_t)w.unit * kUnitFloats + kPairTile * kPairTile + rank * 128 + t] = s;
                else if (o < p.out) p.dbias[o] = p.accumulate ? p.dbias[o] + s : s;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kConverters) : "memory");
#pragma unroll
            for (int x = 0; x < 8; x++) sums[x] = 0.f;
        };

        ItemCursor at;
        bool more = at.start(p, pair), ok = true;
        int step = group, stage = group, rs = group;
        uint32_t phase = 0, rphase = 0;
        auto wrap = [&]() {
            if (rs >= S::kRaws) { rs -= S::kRaws; rphase ^= 1u; }
            if (stage >= S::kStages) { stage -= S::kStages; phase ^= 1u; }
        };
        while (true) {
            bool bias = p.dbias && at.w.nt == 0;
            while (more && step >= at.w.steps) {         // every group passes the end of every item, in the same order
                step -= at.w.steps;
                if (bias && at.w.last) finish(at.w);
                more = at.next(p, pair);
                bias = p.dbias && at.w.nt == 0;
            }
            if (!more) break;
            if (ok) {
                // All lanes wait: where one waits and the others stand by, the warp stays divided after it and does the stage's work
                // twice (fp32, 8192 x 4096 x 4096: 1320 us in place of 804; bf16 328 in place of 271).
                ok = wait_bar(raw_full_bar(rs), rphase, abort_flag, p.status, 0x800u + B200_E_TIMEOUT);
                ok = __all_sync(0xffffffffu, ok);
                const uint8_t *raw = smem + S::kRing + (uint32_t)rs * S::kRaw;
                // Chunks 2c and 2c + 1 of a row's sixteen.  The threads of the row's second half take theirs in the other order, so that
                // no two of a store meet in a bank.
                const int block = c >> 2, chunk = ((2 * c) & 7) + block;
                uint2 q[S::kCodePasses][2];
                if (ok) {
#pragma unroll
                    for (int k = 0; k < S::kCodePasses; k++) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(raw + k * 2048 + t * 16);
                        q[k][0] = block ? make_uint2(v.z, v.w) : make_uint2(v.x, v.y);
                        q[k][1] = block ? make_uint2(v.x, v.y) : make_uint2(v.z, v.w);
                    }
                    ok = wait_bar(empty_bar(stage), phase ^ 1u, abort_flag, p.status, 0x900u + B200_E_TIMEOUT);
                    ok = __all_sync(0xffffffffu, ok);
                }
                if (ok) {
                    uint8_t *tile = smem + (uint32_t)stage * S::kStage;
                    uint8_t *b = tile + PARTS * S::kOperand + block * (S::kRows * 128) + r * 128;
                    const uint32_t first = (uint32_t)((chunk ^ (r & 7)) << 4), second = (uint32_t)(((chunk + 1 - 2 * block) ^ (r & 7)) << 4);
#pragma unroll
                    for (int k = 0; k < S::kCodePasses; k++) {
                        *reinterpret_cast<uint4 *>(b + k * 2048 + first) = decode8(q[k][0], exps[k]);
                        *reinterpret_cast<uint4 *>(b + k * 2048 + second) = decode8(q[k][1], exps[k]);
                    }
                    if (!kDirect) {
                        uint8_t *a = tile + (c8 >> 3) * (S::kRows * 128) + r8 * 128 + (((c8 & 7) ^ (r8 & 7)) << 4);
                        const uint8_t *src = raw + S::kCodes + t * 8 * sizeof(T);
#pragma unroll
                        for (int k = 0; k < S::kDeltaPasses; k++) {
                            uint4 lo, hi = make_uint4(0, 0, 0, 0);
                            if (sizeof(T) == 4) {
                                // the upper four threads of eight take their halves in the other order
                                const int swap = (c8 >> 2) & 1;
                                const uint4 x = *reinterpret_cast<const uint4 *>(src + k * 1024 * sizeof(T) + swap * 16),
                                            y = *reinterpret_cast<const uint4 *>(src + k * 1024 * sizeof(T) + 16 - swap * 16);
                                lo = swap ? y : x;
                                hi = swap ? x : y;
                            } else {
                                lo = *reinterpret_cast<const uint4 *>(src + k * 1024 * sizeof(T));
                            }
                            float f[8];
                            unpack8<T>(lo, hi, f);
                            if (bias) {
#pragma unroll
                                for (int x = 0; x < 8; x++) sums[x] += f[x];
                            }
#pragma unroll
                            for (int part = 0; part < PARTS; part++) {
                                uint32_t h[4];
#pragma unroll
                                for (int x = 0; x < 4; x++) {
                                    float u0, u1;
                                    const float r0 = remainder_of(f[2 * x], u0), r1 = remainder_of(f[2 * x + 1], u1);
                                    h[x] = upper_halves(u0, u1);
                                    f[2 * x] = r0; f[2 * x + 1] = r1;
                                }
                                *reinterpret_cast<uint4 *>(a + part * S::kOperand + k * 1024) = make_uint4(h[0], h[1], h[2], h[3]);
                            }
                        }
                    }
                    // The fence stands between this thread's stores and the tensor core's reads, and between its loads and the copies that
                    // refill the raw slot.  (Released right after its loads had been issued, without a fence, the slot was refilled
                    // before some lanes had their codes: rows eight stages ahead in 0.4 % of the launches at 8192 rows, 2048 x
                    // 1024, bf16 with a bias gradient.)
                    ptx::fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::mbar_arrive(raw_empty_bar(rs));
                        ptx::mbar_arrive(full_bar(stage));
                    }
                    if (kDirect) {
                        // the bias gradient sums delta from the operand tile, which is not loaded again until every warp of the group has
                        // arrived here
                        if (bias) {
                            ok = wait_bar(full_bar(stage), phase, abort_flag, p.status, 0xa00u + B200_E_TIMEOUT);
                            ok = __all_sync(0xffffffffu, ok);
                            if (ok) {
#pragma unroll
                                for (int k = 0; k < S::kDeltaPasses; k++) {
                                    const uint4 lo = *reinterpret_cast<const uint4 *>(tile + (c8 >> 3) * (S::kRows * 128) + (k * 8 + r8) * 128 + (((c8 & 7) ^ r8) << 4));
                                    float f[8];
                                    unpack8<T>(lo, lo, f);
#pragma unroll
                                    for (int x = 0; x < 8; x++) sums[x] += f[x];
                                }
                            }
                            ptx::fence_proxy_async();                       // these loads, and the copy that follows the arrivals
                            __syncwarp();
                        }
                        if (lane == 0) ptx::mbar_arrive(empty_bar(stage));
                    }
                }
            }
            fetch(false);
            step += kGroups;
            rs += kGroups;
            stage += kGroups;
            wrap();
        }
    } else if (warp == kIssuer) {
        // ------------------------------------------------------------------ MMA issuer (one thread of the leader)
        // The peer's thread passes its full stages on, with an arrival of the default scope.  Each CTA's operands are read from its own
        // shared memory, where their writers have made them visible to the async proxy before they arrived on the CTA's own
        // barrier, and this thread has seen that barrier complete: nothing crosses over but the arrival.  That is an argument
        // about the machine; by the letter of the memory model the arrival would be a .release.cluster and the wait for it an
        // .acquire.cluster, a thousand cycles of latency on every stage: bf16 397 us for 269, fp32 1376 for 829 (8192 rows, 4096 x 4096);
        // with the stages dealt out to four threads 368 and 945.
        if (rank == 1 && lane == 0) {
            ItemCursor at;
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (bool more = at.start(p, pair); more && ok; more = at.next(p, pair)) {
                for (int step = 0; step < at.w.steps; step++) {
                    if (!(ok = wait_bar(full_bar(stage), phase, abort_flag, p.status, 0x500u + B200_E_TIMEOUT))) break;
                    ptx::mbar_arrive_remote(peer_bar(stage), 0);
                    if (++stage == S::kStages) { stage = 0; phase ^= 1u; }
                }
            }
        }
        if (rank == 0 && lane == 0) {
            const uint64_t desc = ptx::smem_desc(ptx::smem_u32(smem), S::kRows * 128u, 1024u, 2u);
            int stage = 0, n = 0;
            uint32_t phase = 0;
            bool ok = true;
            ItemCursor at;
            for (bool more = at.start(p, pair); ok && more; more = at.next(p, pair), n++) {
                const WorkItem w = at.w;
                const int acc = n % kAccumulators;
                if (!wait_bar(tempty_bar(acc), ((uint32_t)(n / kAccumulators) & 1u) ^ 1u, abort_flag, p.status, 0x200u + B200_E_TIMEOUT)) break;
                ptx::tc_fence_after();
                const uint32_t d = tmem + (uint32_t)acc * 256u;
                for (int step = 0; step < w.steps; step++) {
                    ok = wait_bar(full_bar(stage), phase, abort_flag, p.status, 0x300u + B200_E_TIMEOUT) &&
                         wait_bar(peer_bar(stage), phase, abort_flag, p.status, 0x600u + B200_E_TIMEOUT);
                    if (!ok) break;
                    ptx::tc_fence_after();
                    const uint64_t a = desc + (uint64_t)((uint32_t)stage * S::kStage >> 4), b = a + (PARTS * S::kOperand >> 4);
#pragma unroll
                    for (int k = 0; k < S::kRows / 16; k++) {
#pragma unroll
                        for (int part = PARTS - 1; part >= 0; part--)        // the small pieces first
                            ptx::mma_bf16_pair(d, a + (part * S::kOperand >> 4) + k * 128, b + k * 128, p.idesc, step > 0 || k > 0 || part < PARTS - 1);
                    }
                    ptx::mma_commit_pair(empty_bar(stage));
                    if (++stage == S::kStages) { stage = 0; phase ^= 1u; }
                }
                if (ok) ptx::mma_commit_pair(tfull_bar(acc));
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue (warps 0 to 3, 32 rows each)
        float *mine = turn + warp * 32 * kPitch;
        const int sub = lane >> 3, quad = (lane & 7) * 4;
        ItemCursor at;
        int n = 0;
        for (bool more = at.start(p, pair); more; more = at.next(p, pair), n++) {
            const WorkItem w = at.w;
            const bool add = !w.first || (w.unit < 0 && p.accumulate);
            const int acc = n % kAccumulators;
            const bool ok = wait_bar(tfull_bar(acc), (uint32_t)(n / kAccumulators) & 1u, abort_flag, p.status, 0x400u + B200_E_TIMEOUT);
            if (!__all_sync(0xffffffffu, ok)) break;
            ptx::tc_fence_after();
            const int row0 = rank * 128 + warp * 32, o0 = w.mt * kPairTile + row0;
            const size_t i0 = (size_t)w.nt * kPairTile;
            const uint32_t src = tmem + (uint32_t)acc * 256u + ((uint32_t)(warp * 32) << 16);
            // where nothing is ragged: 16 bytes a thread, eight threads on 128 bytes of a row, four rows at a time
            const size_t pitch = w.unit >= 0 ? (size_t)kPairTile : p.in;
            const bool even = w.unit >= 0 || (p.vector_out && o0 + 32 <= p.out && i0 + kPairTile <= p.in);
            float *corner = w.unit >= 0 ? p.partial + (size_t)w.unit * kUnitFloats + (size_t)row0 * kPairTile : p.dweight + (size_t)o0 * p.in + i0;
            corner += (size_t)sub * pitch + quad;
            for (int col = 0; col < kPairTile; col += 32) {
                uint32_t v[32];
                ptx::tmem_ld16_issue(src + col, v);
                ptx::tmem_ld16_issue(src + col + 16, v + 16);
                ptx::tmem_ld_wait(v);
                ptx::tmem_ld_wait(v + 16);
                if (col + 32 == kPairTile) {             // the accumulator is read: the next tile may have it
                    ptx::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive_remote(tempty_bar(acc), 0);
                }
                // each thread holds 32 columns of a row; turned around, eight threads write 128 bytes of a row together
#pragma unroll
                for (int k = 0; k < 32; k += 4) *reinterpret_cast<uint4 *>(mine + lane * kPitch + k) = make_uint4(v[k], v[k + 1], v[k + 2], v[k + 3]);
                __syncwarp();
                if (even) {
                    float4 x[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) x[k] = *reinterpret_cast<const float4 *>(mine + (4 * k + sub) * kPitch + quad);
                    float *dst = corner + col;
                    if (add) {
                        float4 old[8];
#pragma unroll
                        for (int k = 0; k < 8; k++) old[k] = *reinterpret_cast<const float4 *>(dst + (size_t)(4 * k) * pitch);
#pragma unroll
                        for (int k = 0; k < 8; k++) { x[k].x += old[k].x; x[k].y += old[k].y; x[k].z += old[k].z; x[k].w += old[k].w; }
                    }
#pragma unroll
                    for (int k = 0; k < 8; k++) *reinterpret_cast<float4 *>(dst + (size_t)(4 * k) * pitch) = x[k];
                } else {
                    const size_t i = i0 + col + quad;
                    for (int k = 0; k < 8; k++) {
                        const int rr = 4 * k + sub;
                        if (o0 + rr >= p.out) break;
                        const float4 x = *reinterpret_cast<const float4 *>(mine + rr * kPitch + quad);
                        const float y[4] = {x.x, x.y, x.z, x.w};
                        float *dst = corner + col + (size_t)(4 * k) * pitch;
#pragma unroll
                        for (int m = 0; m < 4; m++)
                            if (i + m < p.in) dst[m] = add ? dst[m] + y[m] : y[m];
                    }
                }
                __syncwarp();
            }
        }
    }

    if (*abort_flag) {            // MMAs still in flight get time to end before the shared memory is released
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) __nanosleep(200);
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();          // neither CTA leaves while its partner may still arrive on its barriers or read its shared memory
    if (warp == kIssuer) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem, 512u);
    }
}

// Sum of the units of each split tile, in their order, and of their bias gradients.
__global__ void __launch_bounds__(256) ckpt8_wgrad_join_kernel(const __grid_constant__ WgradParams p)
{
    grid_dependency_wait();
    const int tile_index = blockIdx.y, tile = p.first_tail + tile_index;
    const int mt = tile / p.tiles_n, nt = tile - mt * p.tiles_n;
    const float *first = p.partial + (size_t)tile_index * p.splits * kUnitFloats;
    const int at = (blockIdx.x * 256 + threadIdx.x) * 4;               // of the 256 x 256 outputs, then of the 256 sums
    if (at >= (int)kUnitFloats) return;
    float4 s = *reinterpret_cast<const float4 *>(first + at);
    for (int k = 1; k < p.splits; k++) {
        const float4 v = *reinterpret_cast<const float4 *>(first + (size_t)k * kUnitFloats + at);
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const float v[4] = {s.x, s.y, s.z, s.w};
    if (at >= kPairTile * kPairTile) {
        if (!p.dbias || nt) return;
#pragma unroll
        for (int m = 0; m < 4; m++) {
            const int o = mt * kPairTile + at - kPairTile * kPairTile + m;
            if (o < p.out) p.dbias[o] = p.accumulate ? p.dbias[o] + v[m] : v[m];
        }
        return;
    }
    const int o = mt * kPairTile + at / kPairTile;
    const size_t i = (size_t)nt * kPairTile + at % kPairTile;
    if (o >= p.out) return;
    float *dst = p.dweight + (size_t)o * p.in + i;
#pragma unroll
    for (int m = 0; m < 4; m++)
        if (i + m < p.in) dst[m] = p.accumulate ? dst[m] + v[m] : v[m];
}

// Division of the work: `pairs` CTA pairs, `waves` whole tiles each, then the tail in `tail_units` units.
struct WgradPlan { int tiles_m, tiles_n, steps, pairs, waves, first_tail, tail_units, splits, launch_pairs; };
static WgradPlan wgrad_plan(int parts, int rows, int out, size_t in)
{
    WgradPlan w;
    const int depth = parts == 3 ? TcShape<float, 3>::kRows : parts == 2 ? TcShape<__half, 2>::kRows : TcShape<__nv_bfloat16, 1>::kRows;
    w.tiles_m = ceil_div(out, kPairTile);
    w.tiles_n = (int)((in + kPairTile - 1) / kPairTile);
    w.steps = ceil_div(rows, depth);
    w.pairs = sm_count() / 2;
    const long long tiles = (long long)w.tiles_m * w.tiles_n;
    w.waves = (int)(tiles / w.pairs);
    w.first_tail = w.waves * w.pairs;
    const int rest = (int)(tiles - w.first_tail);
    // a unit has at least 128 rows: below that its partial tile costs more than the rows it saves
    w.splits = rest ? max(1, min(w.pairs / rest, rows / 128)) : 1;
    w.tail_units = rest * w.splits;
    w.launch_pairs = w.waves ? w.pairs : w.tail_units;
    return w;
}
static int wgrad_parts(int type) { return type == B200_BF16 ? 1 : type == B200_F16 ? 2 : 3; }

// delta with rows at 16-byte boundaries, for the tensor map
template <typename T>
__global__ void __launch_bounds__(256) ckpt8_wgrad_align_kernel(T *__restrict__ dst, const T *__restrict__ src, int rows, int out, size_t src_pitch, size_t dst_pitch)
{
    grid_dependency_wait();
    constexpr int kVector = 16 / sizeof(T);
    const size_t vectors = dst_pitch / kVector, total = (size_t)rows * vectors;
    for (size_t k = (size_t)blockIdx.x * 256 + threadIdx.x; k < total; k += (size_t)gridDim.x * 256) {
        const size_t row = k / vectors, col = (k - row * vectors) * kVector;
        T v[kVector];
#pragma unroll
        for (int x = 0; x < kVector; x++) v[x] = col + x < (size_t)out ? src[row * src_pitch + col + x] : from_float<T>(0.f);
        *reinterpret_cast<uint4 *>(dst + row * dst_pitch + col) = *reinterpret_cast<const uint4 *>(v);
    }
}

static bool delta_fits(const void *delta, int type, size_t pitch)
{
    return !(reinterpret_cast<uintptr_t>(delta) & 15) && !(pitch * type_size(type) & 15) && pitch * type_size(type) < ((size_t)1 << 40);
}
static size_t aligned_pitch(int type, int out) { return align_up((size_t)out, 16 / type_size(type)); }
static size_t partial_bytes(const WgradPlan &w) { return w.splits > 1 ? sizeof(float) * kUnitFloats * (size_t)w.tail_units : 0; }

template <typename T, int PARTS>
static int wgrad_tc_launch(WgradParams p, const WgradPlan &w, const void *delta, size_t delta_pitch, const int8_t *codes, int type, bool fits, cudaStream_t s)
{
    using S = TcShape<T, PARTS>;
    if (!fits) {
        T *copy = reinterpret_cast<T *>(reinterpret_cast<char *>(p.partial) + partial_bytes(w));
        const size_t pitch = aligned_pitch(type, p.out), vectors = (size_t)p.rows * pitch * sizeof(T) / 16;
        const size_t most = (size_t)sm_count() * 16;
        Launch((unsigned)min((vectors + 255) / 256, most), 256, 0, s)(ckpt8_wgrad_align_kernel<T>, copy, (const T *)delta, p.rows, p.out, delta_pitch, pitch);
        B200_LAUNCH_CHECK();
        delta = copy;
        delta_pitch = pitch;
    }
    CUtensorMap codes_map, delta_map;
    int r = tensor_map_2d(&codes_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, p.blocks * kCkptBlock, (size_t)p.rows, p.blocks * kCkptBlock, 128, S::kRows, false);
    if (r) return r;
    const CUtensorMapDataType kind = type == B200_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : type == B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    r = tensor_map_2d(&delta_map, kind, delta, (size_t)p.out, (size_t)p.rows, delta_pitch * sizeof(T), PARTS == 1 ? 64 : 128, S::kRows, PARTS == 1);
    if (r) return r;
    p.chunk_steps = S::kChunk;
    if ((r = allow_shared<ckpt8_wgrad_tc_kernel<T, PARTS>>((int)kTcSmem))) return r;
    Launch((unsigned)w.launch_pairs * 2, kTcThreads, kTcSmem, s).cluster(2)(ckpt8_wgrad_tc_kernel<T, PARTS>, codes_map, delta_map, p);
    B200_LAUNCH_CHECK();
    if (w.splits > 1) {
        Launch(dim3((unsigned)((kUnitFloats / 4 + 255) / 256), (unsigned)(w.tail_units / w.splits)), 256, 0, s)(ckpt8_wgrad_join_kernel, p);
        B200_LAUNCH_CHECK();
    }
    return B200_OK;
}

}  // namespace b200

using namespace b200;
#define ST(s) ((cudaStream_t)(s))

extern "C" {

size_t b200_ckpt8_wgrad_workspace(int type, int rows, int out, size_t in, const void *delta, size_t delta_pitch)
{
    if (!known_type(type) || check_rows(rows, in) || rows == 0 || out <= 0 || precision() == B200_FP32) return 0;
    const size_t copy = delta_fits(delta, type, delta_pitch) ? 0 : (size_t)rows * aligned_pitch(type, out) * type_size(type);
    return partial_bytes(wgrad_plan(wgrad_parts(type), rows, out, in)) + copy;
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
    if (precision() != B200_FP32) {
        const WgradPlan w = wgrad_plan(wgrad_parts(type), rows, out, in);
        const bool fits = delta_fits(delta, type, delta_pitch);
        const size_t need = partial_bytes(w) + (fits ? 0 : (size_t)rows * aligned_pitch(type, out) * type_size(type));
        if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15))) return fail(B200_E_ARG, "the workspace must be given, aligned to 16 bytes");
        if (workspace_bytes < need) return fail(B200_E_NOMEM, "the workspace has %zu bytes, %zu are needed", workspace_bytes, need);
        WgradParams p = {};
        p.dweight = dweight; p.dbias = dbias; p.exponents = exponents;
        p.rows = rows; p.out = out; p.accumulate = accumulate != 0;
        p.vector_out = !(reinterpret_cast<uintptr_t>(dweight) & 15) && !(in & 3);
        p.in = in; p.blocks = blocks;
        p.tiles_n = w.tiles_n; p.steps = w.steps; p.pairs = w.pairs; p.waves = w.waves; p.first_tail = w.first_tail;
        p.tail_units = w.tail_units; p.splits = w.splits;
        p.partial = (float *)workspace;
        p.idesc = make_idesc_bf16(kPairTile, 1, 1, kPairTile);
        if ((r = status_word(&p.status))) return r;
        set_path(B200_PATH_TCGEN05);
        if (type == B200_BF16) return wgrad_tc_launch<__nv_bfloat16, 1>(p, w, delta, delta_pitch, codes, type, fits, ST(stream));
        if (type == B200_F16) return wgrad_tc_launch<__half, 2>(p, w, delta, delta_pitch, codes, type, fits, ST(stream));
        return wgrad_tc_launch<float, 3>(p, w, delta, delta_pitch, codes, type, fits, ST(stream));
    }
    // B200_FP32: fp32 products on the CUDA cores, summed row by row
    const size_t tiles = ((in + kTile - 1) / kTile) * (((size_t)out + kTile - 1) / kTile);
    if (tiles > 0x7fffffffu) return fail(B200_E_SHAPE, "%zu tiles of the weight gradient are more than a grid has blocks", tiles);
    const Launch launch((unsigned)tiles, 256, 0, ST(stream));
    if (type == B200_F32) launch(ckpt8_wgrad_simt_kernel<float>, dweight, dbias, (const float *)delta, codes, exponents, rows, out, in, delta_pitch, blocks, accumulate);
    else if (type == B200_BF16) launch(ckpt8_wgrad_simt_kernel<__nv_bfloat16>, dweight, dbias, (const __nv_bfloat16 *)delta, codes, exponents, rows, out, in, delta_pitch, blocks, accumulate);
    else launch(ckpt8_wgrad_simt_kernel<__half>, dweight, dbias, (const __half *)delta, codes, exponents, rows, out, in, delta_pitch, blocks, accumulate);
    B200_LAUNCH_CHECK();
    set_path(B200_PATH_SIMT);
    return B200_OK;
}

}  // extern "C"
