// mx4_gemm.cu -- products of microscaled 4-bit operands on the block-scaled tensor-core instruction of sm_100a.
//
//     C[g][j][i] = sum_k P[g][i][k] Q[j][k]        values of 4-bit codes times a power of two for every 32 along k
//
// P are the lanes of the accumulator (weights: contiguous in C), Q its columns (tokens, the rows of C). Three walks over the groups g:
//     dense      one group, every row of Q
//     by rows    group g owns the rows [offsets[g], offsets[g + 1]) of Q and C and multiplies them by its own P[g]
//     along k    group g owns the k in [offsets[g], offsets[g + 1]) (multiples of 64); P and Q are shared, C[g] is its own
// The offsets live on the device. Accumulation is in FP32 in tensor memory, one rounding to the output type at the end.
//
// One kernel, warp-specialised, 128 rows of P by BN rows of Q to a tile, 256 values (128 bytes) of k to a stage:
//   warp 0     producer: one thread, TMA (128-byte swizzle) of both operands' codes into a ring of stages
//   warp 1     issuer: one thread; tcgen05.cp of the stage's scales into tensor memory, four tcgen05.mma kind::mxf4 (K = 64) on it
//   warps 2-3  scales: the row-major scale bytes of 128 + BN rows become the tiles of 128 rows x 4 blocks that the instruction
//              takes (row r of a tile at byte 16 (r % 32) + 4 (r / 32)): a lane reads 8 bytes of each of the rows l, l + 32,
//              l + 64, l + 96 and writes two 16-byte words, so the turn costs two conflict-free stores for 128 rows
//   warps 4-7  epilogue: tensor memory to registers to global memory, while the next tile accumulates
// The scales of a stage have tensor-memory columns of their own, so a stage's release covers them too.
// Rows of Q are few where latency counts, so BN is 16 to 192, chosen by the rows there are to a group, and with few tiles the k of
// a tile is split over a cluster of 2, 4 or 8 CTAs, whose partial tiles are added in a fixed order through distributed shared
// memory. Every wait is bounded: on expiry the CTA raises the status word, stops, frees its tensor memory and returns.
#include <type_traits>
#include "oz_async.cuh"
#include "oz_common.cuh"
#include "oz_kernels.h"
#include "oz_types.cuh"

namespace ozk {

namespace m4 {

constexpr int BP = 128;            // rows of P to a tile
constexpr int BK = 256, BKB = 128; // k of a stage, in values and in bytes
constexpr int UK = 64;             // k of one tcgen05.mma kind::mxf4
constexpr int THREADS = 256;
constexpr int MAX_GROUPS = 1024;

enum { DENSE = 0, BY_ROWS = 1, ALONG_K = 2 };

struct Params {
    int mode, groups;
    int rows_p, rows_q, K;          // rows of P (to a group), rows of Q, length along k
    int tiles_p, band;              // tiles of P, and how many of them are walked before the next tile of Q
    const int *offsets;             // [groups + 1] on the device (BY_ROWS, ALONG_K)
    const uint8_t *sp, *sq;         // scale bytes, row-major
    long long ldsp, ldsq;
    size_t plane_sp;                // bytes between the scales of two groups of P
    void *C;
    long long ldc;
    size_t plane_c;                 // elements between the results of two groups (ALONG_K)
    int *status;
};

template <int BN> struct Shape {
    static constexpr int Q_TILES = (BN + 127) / 128;               // scale tiles of 128 rows of Q
    static constexpr int P_BYTES = BP * BKB, Q_BYTES = BN * BKB;
    static constexpr int SP_BYTES = 2 * 512, SQ_BYTES = 2 * 512 * Q_TILES;
    static constexpr int STAGE = P_BYTES + Q_BYTES + SP_BYTES + SQ_BYTES;
    static constexpr int SCALE_COLS = 8 + 8 * Q_TILES;             // tensor-memory columns of a stage's scales
    static constexpr int STAGES = BN <= 32 ? 8 : BN <= 64 ? 7 : BN <= 128 ? 6 : 5;
    static constexpr int COLS = 2 * BN + STAGES * SCALE_COLS;      // two accumulators, and the scales
    static constexpr int TMEM_COLS = COLS <= 256 ? 256 : 512;
    static constexpr int BARS = 2 * STAGES + 4;
    static constexpr int SMEM = STAGES * STAGE + 1024 + 8 * BARS + 16 + 4 * (MAX_GROUPS + 1);
    static_assert(STAGE % 1024 == 0 && COLS <= 512 && SMEM <= 232448 - 64, "");
    static_assert(BN * BP * 4 <= STAGES * STAGE, "the partial tile of a split takes the place of the stages");
    // instruction descriptor: E2M1 x E2M1, both K-major, one power of two (UE8M0) for 32, N = BN, M = 128, K = 64
    static constexpr uint32_t IDESC = (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | (1u << 23) | (1u << 27);
};

__device__ __forceinline__ void mma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
// 512 bytes of scales (32 x 16) to four columns of tensor memory, the same in each quarter of the lanes
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
    const uint64_t desc = (uint64_t)((smem & 0x3FFFFu) >> 4) | (8ull << 32) | (1ull << 46);   // no swizzle, groups of 8 rows 128 bytes apart
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

// what a work item is
struct Tile {
    int group, tp, q0, q1;   // group, tile of P, rows [q0, q1) of Q (at most BN)
    int k0, k1;              // range along k
    int s0, s1;              // stages [s0, s1) of 256 that cover it (or this CTA's share of them)
};

// The range along k or of rows that `offsets` gives group g. Offsets that are out of order or out of range are cut to what is there.
__device__ __forceinline__ void segment(const Params &p, int g, int limit, int &lo, int &hi) {
    lo = min(max(__ldg(p.offsets + g), 0), limit);
    hi = min(max(__ldg(p.offsets + g + 1), lo), limit);
}

template <int BN> __device__ __forceinline__ int tiles_of(int rows) { return (rows + BN - 1) / BN; }

// item w -> tile; `cum` has the running number of tiles of Q (BY_ROWS). Bands of `band` tiles of P are walked tile of Q by tile of Q,
// so that the CTAs at work at one time share both operands' panels in L2.
template <int BN>
__device__ __forceinline__ Tile decode(const Params &p, const int *cum, int w) {
    Tile t;
    int tq, tiles_q, q_lo = 0, q_hi = p.rows_q, idx;
    t.k0 = 0;
    t.k1 = p.K;
    if (p.mode == BY_ROWS) {
        int lo = 0, hi = p.groups;   // the last group whose first item is not behind w
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (cum[mid] * p.tiles_p <= w) lo = mid; else hi = mid;
        }
        t.group = lo;
        idx = w - cum[lo] * p.tiles_p;
        tiles_q = cum[lo + 1] - cum[lo];
        segment(p, lo, p.rows_q, q_lo, q_hi);
    } else {
        tiles_q = tiles_of<BN>(p.rows_q);
        const int per_group = tiles_q * p.tiles_p;
        t.group = w / per_group;
        idx = w - t.group * per_group;
        if (p.mode == ALONG_K) {
            segment(p, t.group, p.K, t.k0, t.k1);
            t.k0 &= ~(UK - 1);
            t.k1 &= ~(UK - 1);
        }
    }
    const int span = p.band * tiles_q, b = idx / span, first = b * p.band, rows = min(p.band, p.tiles_p - first), within = idx - b * span;
    t.tp = first + within % rows;
    tq = within / rows;
    t.q0 = q_lo + tq * BN;
    t.q1 = min(q_hi, t.q0 + BN);
    t.s0 = t.k0 / BK;
    t.s1 = t.k1 > t.k0 ? (t.k1 + BK - 1) / BK : t.s0;
    return t;
}

// 32 columns of a tile: lane = row of P, v[c] = column c
template <class T>
__device__ __forceinline__ void store_columns(T *C, long long ldc, const uint32_t (&v)[32], int i, int rows_p, int j, int j1) {
    if (i >= rows_p) return;
    T *dst = C + (size_t)j * ldc + i;
#pragma unroll
    for (int c = 0; c < 32; c++)
        if (j + c < j1) dst[(size_t)c * ldc] = from_f32<T>(__uint_as_float(v[c]));
}

template <int BN, class T, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) mx4_gemm(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ,
                                                       const Params p) {
    using S = Shape<BN>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *const base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + S::STAGES * S::STAGE;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S::STAGES + s); };
    auto accfull_bar = [&](int a) { return bars + 8u * (2 * S::STAGES + a); };
    auto accempty_bar = [&](int a) { return bars + 8u * (2 * S::STAGES + 2 + a); };
    const uint32_t tmem_slot = bars + 8u * S::BARS;
    int *const cum = reinterpret_cast<int *>(base_ptr + S::STAGES * S::STAGE + 8 * S::BARS + 16);
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < S::STAGES; s++) { mbar_init(full_bar(s), 2); mbar_init(empty_bar(s), 1); }   // full: the TMA's bytes and a scale warp
        for (int a = 0; a < 2; a++) { mbar_init(accfull_bar(a), 1); mbar_init(accempty_bar(a), 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"((uint32_t)S::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 2 && p.mode == BY_ROWS) {   // running number of tiles of Q over the groups
        int run = 0;
        for (int g0 = 0; g0 < p.groups; g0 += 32) {
            int n = 0;
            if (g0 + lane < p.groups) {
                int lo, hi;
                segment(p, g0 + lane, p.rows_q, lo, hi);
                n = tiles_of<BN>(hi - lo);
            }
            int inc = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(~0u, inc, d);
                if (lane >= d) inc += o;
            }
            if (g0 + lane < p.groups) cum[g0 + lane] = run + inc - n;
            run += __shfl_sync(~0u, inc, 31);
        }
        if (lane == 0) cum[p.groups] = run;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    uint32_t tmem_base;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
    const uint32_t tmem_scales = tmem_base + 2 * BN;

    const int total = p.mode == BY_ROWS ? cum[p.groups] * p.tiles_p : tiles_of<BN>(p.rows_q) * p.tiles_p * (p.mode == ALONG_K ? p.groups : 1);
    uint32_t rank = 0, ranks = 1;
    int first = blockIdx.x, step = gridDim.x;
    if constexpr (SPLIT) {   // one tile to a cluster; this CTA takes its share of the stages
        rank = cluster_rank();
        asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
        first = blockIdx.x / ranks;
        step = 1 << 30;
    }
    auto tile_at = [&](int w) {
        Tile t = decode<BN>(p, cum, w);
        if constexpr (SPLIT) {
            const int n = t.s1 - t.s0, s0 = t.s0;
            t.s0 = s0 + (int)((long long)n * rank / ranks);
            t.s1 = s0 + (int)((long long)n * (rank + 1) / ranks);
        }
        return t;
    };
    volatile int *abortp = &abort_flag;
    uint32_t issued = 0;   // stages the producer has filled

    if (warp == 0) {
        if (lane == 0) {
            uint32_t it = 0;
            for (int w = first; w < total && !*abortp; w += step) {
                const Tile t = tile_at(w);
                for (int kb = t.s0; kb < t.s1; kb++, it++) {
                    const int s = it % S::STAGES;
                    if (!mbar_wait(empty_bar(s), ((it / S::STAGES) & 1u) ^ 1u, abortp, 0x110)) break;
                    mbar_expect_tx(full_bar(s), S::P_BYTES + S::Q_BYTES);
                    const uint32_t at = base + s * S::STAGE;
                    tma_load_3d(at, &mapP, kb * BKB, t.tp * BP, p.mode == BY_ROWS ? t.group : 0, full_bar(s));
                    tma_load_3d(at + S::P_BYTES, &mapQ, kb * BKB, t.q0, 0, full_bar(s));
                    issued = it + 1;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t it = 0, n = 0;
            for (int w = first; w < total && !*abortp; w += step, n++) {
                const Tile t = tile_at(w);
                const uint32_t acc = n & 1u;
                if (!mbar_wait(accempty_bar(acc), ((n >> 1) & 1u) ^ 1u, abortp, 0x120)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem_base + acc * BN;
                bool ok = true;
                uint32_t accumulate = 0;
                for (int kb = t.s0; kb < t.s1; kb++, it++) {
                    const int s = it % S::STAGES;
                    if (!mbar_wait(full_bar(s), (it / S::STAGES) & 1u, abortp, 0x130)) { ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = base + s * S::STAGE, sp = at + S::P_BYTES + S::Q_BYTES, sq = sp + S::SP_BYTES;
                    const uint32_t tp = tmem_scales + s * S::SCALE_COLS, tq = tp + 8;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        copy_scales(tp + 4 * h, sp + 512 * h);
#pragma unroll
                        for (int c = 0; c < S::Q_TILES; c++) copy_scales(tq + 4 * (h * S::Q_TILES + c), sq + 512 * (h * S::Q_TILES + c));
                    }
                    const uint64_t da = smem_desc(at), db = smem_desc(at + S::P_BYTES);
                    const int k_lo = (t.k0 - kb * BK) / UK, k_hi = (t.k1 - kb * BK + UK - 1) / UK;   // the instructions of this stage that are in range
#pragma unroll
                    for (int k = 0; k < BK / UK; k++) {
                        if (k < k_lo || k >= k_hi) continue;
                        const uint32_t id = S::IDESC | ((k & 1u) ? (2u << 4) | (2u << 29) : 0u);      // which two of a word's four scales
                        mma_mx4(d, da + 2u * k, db + 2u * k, id, tp + 4 * (k >> 1), tq + 4 * (k >> 1) * S::Q_TILES, accumulate);
                        accumulate = 1;
                    }
                    mma_commit(empty_bar(s));
                }
                if (!ok) break;
                mma_commit(accfull_bar(acc));
            }
        }
    } else if (warp < 4) {
        const uint32_t own = warp & 1u;   // this warp takes the stages of its parity
        const int blocks = (p.K + 31) / 32;
        uint32_t it = 0;
        for (int w = first; w < total && !*abortp; w += step) {
            const Tile t = tile_at(w);
            const uint8_t *rows_p = p.sp + (p.mode == BY_ROWS ? (size_t)t.group * p.plane_sp : 0);
            bool ok = true;
            for (int kb = t.s0; kb < t.s1; kb++, it++) {
                if ((it & 1u) != own) continue;
                const int s = it % S::STAGES;
                constexpr int TILES = 1 + S::Q_TILES;
                uint2 v[TILES][4];
                // scales behind the last block of a row, and of rows that are not there, become 1: their codes are zero or unused
                const int left = blocks - kb * 8;
#pragma unroll
                for (int c = 0; c < TILES; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = lane + 32 * i;
                        v[c][i] = make_uint2(0x7f7f7f7fu, 0x7f7f7f7fu);
                        if (c == 0) {
                            if (t.tp * BP + r < p.rows_p) v[c][i] = __ldg(reinterpret_cast<const uint2 *>(rows_p + (size_t)(t.tp * BP + r) * p.ldsp + (size_t)kb * 8));
                        } else {
                            const int q = t.q0 + (c - 1) * 128 + r;
                            if (q < t.q1) v[c][i] = __ldg(reinterpret_cast<const uint2 *>(p.sq + (size_t)q * p.ldsq + (size_t)kb * 8));
                        }
                    }
                if (left < 8) {
                    const uint32_t keep0 = left >= 4 ? ~0u : (1u << (8 * left)) - 1u, keep1 = left >= 4 ? (1u << (8 * (left - 4))) - 1u : 0u;
#pragma unroll
                    for (int c = 0; c < TILES; c++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            v[c][i].x = (v[c][i].x & keep0) | (0x7f7f7f7fu & ~keep0);
                            v[c][i].y = (v[c][i].y & keep1) | (0x7f7f7f7fu & ~keep1);
                        }
                }
                if (!__all_sync(~0u, mbar_wait(empty_bar(s), ((it / S::STAGES) & 1u) ^ 1u, abortp, 0x140))) { ok = false; break; }
                uint8_t *sp = base_ptr + s * S::STAGE + S::P_BYTES + S::Q_BYTES;
#pragma unroll
                for (int c = 0; c < TILES; c++) {
                    // tile of the first four blocks, then of the last four; Q's tiles of one half lie side by side
                    uint8_t *lo = c == 0 ? sp : sp + S::SP_BYTES + 512 * (c - 1), *hi = c == 0 ? sp + 512 : lo + 512 * S::Q_TILES;
                    *reinterpret_cast<uint4 *>(lo + 16 * lane) = make_uint4(v[c][0].x, v[c][1].x, v[c][2].x, v[c][3].x);
                    *reinterpret_cast<uint4 *>(hi + 16 * lane) = make_uint4(v[c][0].y, v[c][1].y, v[c][2].y, v[c][3].y);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the tensor core reads these through the async proxy
                __syncwarp();
                if (lane == 0) mbar_arrive(full_bar(s));
            }
            if (!ok) break;
        }
    } else {
        const int quarter = warp & 3;
        uint32_t n = 0;
        for (int w = first; w < total && !*abortp; w += step, n++) {
            const Tile t = tile_at(w);
            const uint32_t acc = n & 1u;
            if (!__all_sync(~0u, mbar_wait(accfull_bar(acc), (n >> 1) & 1u, abortp, 0x150))) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN;
            const bool some = t.s1 > t.s0;   // no stage: nothing was accumulated, the tile is zero
            const int i = t.tp * BP + quarter * 32 + lane;
            if constexpr (!SPLIT) {
                T *C = reinterpret_cast<T *>(p.C) + (p.mode == ALONG_K ? (size_t)t.group * p.plane_c : 0);
#pragma unroll 1
                for (int c = 0; c < BN; c += 32) {
                    if (t.q0 + c >= t.q1) break;
                    uint32_t v[32];
                    tmem_ld32(taddr + c, v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (!some) {
#pragma unroll
                        for (int e = 0; e < 32; e++) v[e] = 0;
                    }
                    store_columns<T>(C, p.ldc, v, i, p.rows_p, t.q0 + c, t.q1);
                }
            } else {   // the partial tile, [column][row of P], over the stages that this CTA has used up
                float *part = reinterpret_cast<float *>(base_ptr);
#pragma unroll 1
                for (int c = 0; c < BN; c += 32) {
                    uint32_t v[32];
                    tmem_ld32(taddr + c, v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        if (c + e < BN) part[(c + e) * BP + quarter * 32 + lane] = some ? __uint_as_float(v[e]) : 0.f;
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(accempty_bar(acc));
        }
    }

    __syncwarp();
    if constexpr (SPLIT) {
        // every CTA of the cluster adds its share of the columns over the ranks, in their order: the same sum on every run
        __syncthreads();
        cluster_sync_all();
        if (first < total) {
            const Tile t = decode<BN>(p, cum, first);
            T *C = reinterpret_cast<T *>(p.C) + (p.mode == ALONG_K ? (size_t)t.group * p.plane_c : 0);
            const int r = threadIdx.x & (BP - 1), i = t.tp * BP + r;
            const int n = t.q1 - t.q0, c0 = (int)((long long)n * rank / ranks), c1 = (int)((long long)n * (rank + 1) / ranks);
            for (int c = c0 + (threadIdx.x >> 7); c < c1; c += THREADS / BP) {
                float sum = 0.f;
                for (uint32_t q = 0; q < ranks; q++) {
                    float x;
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(map_to_cta(base + 4u * (c * BP + r), q)) : "memory");
                    sum += x;
                }
                if (i < p.rows_p) C[(size_t)(t.q0 + c) * p.ldc + i] = from_f32<T>(sum);
            }
        }
        cluster_sync_all();   // nobody leaves while a peer still reads its partial tile
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (abort_flag && warp == 0 && lane == 0) {   // copies in flight land before this CTA's shared memory is given back
        for (uint32_t it = issued > S::STAGES ? issued - S::STAGES : 0; it < issued; it++) {
            int ignore = 0;
            const unsigned long long until = now_ns() + 100000000ull;
            while (!mbar_try(full_bar(it % S::STAGES), (it / S::STAGES) & 1u) && !ignore) ignore = now_ns() > until;
        }
    }
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)S::TMEM_COLS) : "memory");
    if (threadIdx.x == 0 && abort_flag) {
        atomicCAS(p.status, 0, abort_flag);
        if (blockIdx.x < 63) p.status[1 + blockIdx.x] = abort_flag;
    }
}

// ---- host ----

// {bytes along k, row, plane}; 128 bytes of `box_rows` rows to a copy
cudaError_t make_map(CUtensorMap *map, const uint8_t *ptr, int K, int rows, int planes, long long ld, size_t plane, int box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {(cuuint64_t)((K + 31) / 32 * 16), (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)(planes > 1 ? plane : (size_t)ld * rows)};
    const cuuint32_t box[3] = {(cuuint32_t)BKB, (cuuint32_t)box_rows, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(ptr), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int BN, class T, bool SPLIT>
cudaError_t launch(const CUtensorMap &mapP, const CUtensorMap &mapQ, const Params &p, int grid, int split, cudaStream_t st) {
    static PerDevice pd;
    cudaError_t e = pd.once([] { return cudaFuncSetAttribute(mx4_gemm<BN, T, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<BN>::SMEM); });
    if (e) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Shape<BN>::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    if (SPLIT) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = split;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, mx4_gemm<BN, T, SPLIT>, mapP, mapQ, p);
}

}  // namespace m4

cudaError_t mx4_product(const Mx4Product &g, int *status, cudaStream_t st) {
    using namespace m4;
    Params p{};
    p.mode = g.mode;
    p.groups = g.groups;
    p.rows_p = g.rows_p;
    p.rows_q = g.rows_q;
    p.K = g.K;
    p.tiles_p = (g.rows_p + BP - 1) / BP;
    p.band = 16;
    p.offsets = g.offsets;
    p.sp = g.sp; p.ldsp = g.ldsp; p.plane_sp = g.plane_sp;
    p.sq = g.sq; p.ldsq = g.ldsq;
    p.C = g.C; p.ldc = g.ldc; p.plane_c = g.plane_c;
    p.status = status;
    int dev, sms;
    cudaError_t e = cudaGetDevice(&dev);
    if (!e) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e) return e;

    // the width of a tile: the rows of Q that a group has (on average, by rows), rounded up to what there is
    const int per_group = g.mode == BY_ROWS ? (g.rows_q + g.groups - 1) / g.groups : g.rows_q;
    const int bn = per_group <= 16 ? 16 : per_group <= 32 ? 32 : per_group <= 64 ? 64 : per_group <= 512 ? 128 : 192;
    // tiles of Q: exact, or (by rows) the most that there can be and the number to be expected of even segments
    long long most, expected;
    if (g.mode == BY_ROWS) {
        most = (long long)(g.groups < g.rows_q ? g.groups : g.rows_q) + g.rows_q / bn;
        expected = (long long)(g.groups < g.rows_q ? g.groups : g.rows_q) * ((per_group + bn - 1) / bn);
    } else {
        most = expected = (long long)((g.rows_q + bn - 1) / bn) * (g.mode == ALONG_K ? g.groups : 1);
    }
    most *= p.tiles_p;
    expected *= p.tiles_p;
    if (most > 0x3fffffffLL / 8) return cudaErrorInvalidValue;
    // few tiles: split k, while every CTA keeps at least four stages
    const int stages = (g.K + BK - 1) / BK;
    int split = 1;
    if (bn <= 128 && g.mode != ALONG_K)
        while (split < 8 && expected * split * 2 <= sms && stages / (split * 2) >= 4) split *= 2;

    CUtensorMap mapP, mapQ;
    if ((e = make_map(&mapP, g.p, g.K, g.rows_p, g.mode == BY_ROWS ? g.groups : 1, g.ldp, g.plane_p, BP))) return e;
    if ((e = make_map(&mapQ, g.q, g.K, g.rows_q, 1, g.ldq, 0, bn))) return e;
    const int grid = split > 1 ? (int)most * split : (int)(most < sms ? most : sms);
    e = cudaErrorInvalidValue;
    with_type(g.type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto width) {
            constexpr int BN = decltype(width)::value;
            if constexpr (BN <= 128) {
                if (split > 1) { e = launch<BN, T, true>(mapP, mapQ, p, grid, split, st); return; }
            }
            e = launch<BN, T, false>(mapP, mapQ, p, grid, 1, st);
        };
        switch (bn) {
        case 16: go(std::integral_constant<int, 16>()); break;
        case 32: go(std::integral_constant<int, 32>()); break;
        case 64: go(std::integral_constant<int, 64>()); break;
        case 128: go(std::integral_constant<int, 128>()); break;
        default: go(std::integral_constant<int, 192>()); break;
        }
    });
    return e;
}

}  // namespace ozk
