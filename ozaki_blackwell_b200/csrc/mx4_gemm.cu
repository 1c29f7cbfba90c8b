// mx4_gemm.cu -- products of microscaled 4-bit operands on the block-scaled tensor-core instruction of sm_100a.
//
//     Y[t][n] = sum_k X[t][k] W[n][k]        values of 4-bit codes times a power of two for every 32 along k
//
// X are the tokens, W the weights. Three walks over groups g:
//     dense      one group
//     by rows    group g owns the rows [offsets[g], offsets[g + 1]) of X and Y and multiplies them by its own W[g]
//     along k    group g owns the k in [offsets[g], offsets[g + 1]) (multiples of 64, or K for an end); X and W are shared, Y[g] is its
//                own. An instruction takes 64 of k: a segment that begins or ends inside them would take a neighbour's values or lose
//                some of its own, so its Y[g] is NaN and the status word is raised.
// The offsets live on the device. Accumulation is in FP32 in tensor memory, one rounding to the output type at the end.
//
// One kernel, warp-specialised: a tile is 128 rows of P, which are the lanes of the accumulator, by BN rows of Q, its columns; 256
// values (128 bytes) of k make a stage, 512 (16 scale bytes) a scale slot.
//   warp 0     producer: one thread, TMA of both operands' codes (128-byte swizzle) into a ring of stages. What lies outside a matrix
//              comes as zero codes.
//   warps 3, 8 .. 10  scales, in turns of one or two slots: a row's 16 bytes are four words, one to 128 values of k; the instruction wants, for a
//              word, 128 rows as 32 x 16 bytes (row r at 16 (r % 32) + 4 (r / 32)). A lane reads the rows l, l + 32, l + 64, l + 96
//              and writes the 4 x 4 words turned: four 16-byte loads and stores for 128 rows by 512 values, without bank conflicts.
//   warp 2     one thread; tcgen05.cp of a stage's turned scales into tensor memory, its completion counted by the stage's barrier
//   warp 1     issuer: one thread; four tcgen05.mma kind::mxf4 (K = 64) to a stage
//   warp 11    in a pair: tells the leader of the slots that the peer has turned
//   warps 4-7, 12-15  epilogue: tensor memory to registers to global memory, 32 columns at a time in turns, while the next tile
//              accumulates
// An instruction of tcgen05 takes 20 to 60 cycles to issue, whatever it does; with the four to six copies of a stage's scales in
// the thread that issues its four products the tensor pipe waited, so the copies have a thread of their own. Bringing the scale
// bytes by TMA was slower: boxes 16 bytes wide cost the TMA unit as much for a row as the 128 bytes of its codes (900 cycles a slot).
//
// Few tokens (NARROW): P = weights, Q = tokens, BN = 16 .. 128 by the tokens there are, Y's columns are the lanes, so that a warp stores
// contiguous columns of one token. With few tiles and a long k the k of a tile is split over a cluster of 2 or 4 CTAs (SPLIT), whose
// partial tiles are added in a fixed order through distributed shared memory. Many tokens (WIDE): P = tokens, Q = weights, BN = 192;
// two accumulators of 192 columns leave 128 columns of tensor memory for scales; tiles leave through shared memory and TMA. With
// enough tiles two CTAs (cta_group::2) share a tile of 256 tokens (PAIR): each loads its own 128 tokens and half of the weights' rows,
// and turns its own tokens' and all the weights' scales.
//
// What bounds it: for one token HBM (18432 x 7168 in 10.4 us, 6.7 TB/s with the weights partly in L2; 14.1 us from HBM); for many, what
// the L2 delivers. At 2048 x 18432 x 7168 (109 us, 4980 TFLOP/s, 0.75 of four times the measured burst rate of BF16, 0.88 of four times
// the sustained one) the CTAs fetch 1.2 GB of operands, 11 TB/s, and every other dense many-token shape comes to the same rate; the clock is
// then at 1.5 GHz under the power limit. WIDE fetches 40 KB to a stage of 128 x 192, PAIR 56 KB to one of 256 x 192.
// Every wait is bounded: on expiry the CTA raises the status word, stops, frees its tensor memory and returns.
#include <type_traits>
#include "oz_async.cuh"
#include "oz_common.cuh"
#include "oz_kernels.h"
#include "oz_launch.cuh"
#include "oz_types.cuh"

namespace ozk {

namespace m4 {

constexpr int BP = 128;            // rows of P to a CTA
constexpr int BK = 256, BKB = 128; // k of a stage, in values and in bytes
constexpr int UK = 64;             // k of one tcgen05.mma kind::mxf4
constexpr int THREADS = 512;       // warp 11 is idle but in a pair's peer: the epilogue's second four must be warps 0 .. 3 modulo 4
constexpr int MAX_GROUPS = 1024;
constexpr int AHEAD = 48;          // tiles of a CTA that are worked out before it starts

enum { DENSE = 0, BY_ROWS = 1, ALONG_K = 2 };
constexpr uint32_t NOT_A_NUMBER = 0x7fffffffu;
enum { NARROW = 0, SPLIT = 1, WIDE = 2, PAIR = 3 };

struct Params {
    int mode, groups;
    int tokens, weights, K;         // rows of X, rows of W (to a group), length along k
    int band;                       // tiles of P that are walked before the next tile of Q
    const int *offsets;             // [groups + 1] on the device (BY_ROWS, ALONG_K)
    const uint8_t *sp, *sq;         // scales of P and Q
    long long ldsp, ldsq;
    size_t plane_sp, plane_sq;      // bytes between two groups' (0: shared)
    void *Y;
    long long ldy;
    int whole_words;                // Y's rows start on 16 bytes: mapY is one of it
    size_t plane_y;                 // elements between the results of two groups (ALONG_K)
    int *status;
};

template <int FORM, int BN> struct Shape {
    static constexpr bool pair = FORM == PAIR, wide = FORM >= WIDE;
    static constexpr int P_TILE = pair ? 2 * BP : BP;              // rows of P to a tile
    static constexpr int TOKENS = wide ? P_TILE : BN, WEIGHTS = wide ? BN : P_TILE;
    static constexpr int Q_ROWS = pair ? BN / 2 : BN;              // rows of Q whose codes this CTA loads
    static constexpr int Q_TILES = (BN + 127) / 128;               // scale tiles of 128 rows of Q
    static constexpr int P_BYTES = BP * BKB, Q_BYTES = Q_ROWS * BKB, STAGE = P_BYTES + Q_BYTES;
    static constexpr int SLOT = 4 * 512 * (1 + Q_TILES);           // turned scales of 512 values of k: four words of P's tile, then of Q's
    static constexpr int SCALE_COLS = 8 + 8 * Q_TILES;             // tensor-memory columns of a stage's scales
    static constexpr int STAGES = pair ? 5 : BN <= 32 ? 8 : BN <= 64 ? 7 : BN <= 128 ? 5 : 4;
    // Scale slots, two to a turning warp: a slot is always the same warp's. (A warp that came to a slot before another had seen the slot's
    // last use would take the parity of the use before that for its own.) A warp turns HALVES slots at a time.
    static constexpr int TURNERS = FORM == WIDE ? 2 : 4, SLOTS = 2 * TURNERS, HALVES = wide ? 2 : 1, WINDOW = 2 * HALVES;   // WINDOW: stages of a turn
    static_assert(SLOT % 512 == 0, "the pieces behind the slots are swizzled");
    static constexpr int COLS = 2 * BN + STAGES * SCALE_COLS;      // two accumulators, and the scales
    static constexpr int TMEM_COLS = COLS <= 256 ? 256 : 512;
    static constexpr int BARS = 2 * STAGES + 2 * SLOTS + 4;
    static constexpr int TURN = wide ? 8 * 2 * 2048 : 0;            // two pieces of 32 rows x 64 bytes to each warp of the epilogue
    static constexpr int SMEM = STAGES * STAGE + SLOTS * SLOT + TURN + 1024 + 8 * BARS + 16 + 4 * (MAX_GROUPS + 4) + AHEAD * 32;
    static_assert(STAGE % 1024 == 0 && COLS <= 512 && SMEM <= 232448 - 64, "");
    static_assert(FORM != SPLIT || BN * BP * 4 <= STAGES * STAGE, "the partial tile of a split takes the place of the stages");
    // instruction descriptor: E2M1 x E2M1, both K-major, one power of two (UE8M0) for 32, N = BN, M = rows of P, K = 64
    static constexpr uint32_t IDESC = (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | (1u << 23) | ((uint32_t)(P_TILE >> 7) << 27);
};

template <bool PAIRED>
__device__ __forceinline__ void mma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
    if constexpr (PAIRED)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate) : "memory");
}
// 512 bytes of scales (32 x 16) to four columns of tensor memory, the same in each quarter of the lanes (in a pair: in both CTAs, each
// from its own shared memory)
template <bool PAIRED>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
    const uint64_t desc = (uint64_t)((smem & 0x3FFFFu) >> 4) | (8ull << 32) | (1ull << 46);   // no swizzle, groups of 8 rows 128 bytes apart
    if constexpr (PAIRED) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// everything issued so far, done: arrives on the barrier (in a pair: on the barriers of both CTAs at this offset)
template <bool PAIRED>
__device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (PAIRED)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
    else mma_commit(bar);
}

// The value of lane 0 in all lanes: the compiler then keeps it, and what is computed from it, in the registers that a warp shares,
// where tcgen05 and TMA instructions take their operands from.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(~0u, x, 0); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(~0u, x, 0); }

// the first n (0 < n < 16) bytes of v, zeros behind them
__device__ __forceinline__ uint4 first_bytes(uint4 v, int n) {
    auto keep = [&](uint32_t x, int from) { return n >= from + 4 ? x : n <= from ? 0u : x & ((1u << (8 * (n - from))) - 1u); };
    return make_uint4(keep(v.x, 0), keep(v.y, 4), keep(v.z, 8), keep(v.w, 12));
}

// what a work item is
struct Tile {
    int group;
    int p0, p1, q0, q1;      // rows of P and of Q: from the first, and where they end (this group's, not the tile's)
    int k0, k1;              // range along k; k1 = -1: it begins or ends inside an instruction's 64 and is refused
    int s0, s1;              // stages [s0, s1) of 256 that cover it (or this CTA's share of them)
};

// The range along k or of rows that `offsets` gives group g. Offsets that are out of order or out of range are cut to what is there.
__device__ __forceinline__ void segment(const Params &p, int g, int limit, int &lo, int &hi) {
    lo = min(max(p.offsets[g], 0), limit);
    hi = min(max(p.offsets[g + 1], lo), limit);
}

// item w -> tile; `cum` has the running number of token tiles (BY_ROWS). Bands of `band` tiles of P are walked tile of Q by tile of Q,
// so that the CTAs at work at one time share both operands' panels in L2.
template <class S>
__device__ __forceinline__ Tile decode(const Params &p, const int *cum, int w) {
    Tile t;
    const int nw = (p.weights + S::WEIGHTS - 1) / S::WEIGHTS;
    int nt, lo = 0, hi = p.tokens, idx;
    t.k0 = 0;
    t.k1 = p.K;
    if (p.mode == BY_ROWS) {
        int a = 0, b = p.groups;   // the last group whose first item is not behind w
        while (b - a > 1) {
            const int mid = (a + b) >> 1;
            if (cum[mid] * nw <= w) a = mid; else b = mid;
        }
        t.group = a;
        idx = w - cum[a] * nw;
        nt = cum[a + 1] - cum[a];
        segment(p, a, p.tokens, lo, hi);
    } else {
        nt = (p.tokens + S::TOKENS - 1) / S::TOKENS;
        const int per_group = nt * nw;
        t.group = w / per_group;
        idx = w - t.group * per_group;
        if (p.mode == ALONG_K) {
            segment(p, t.group, p.K, t.k0, t.k1);
            if (t.k1 > t.k0) t.k1 = t.k0 % UK || (t.k1 % UK && t.k1 != p.K) ? -1 : (t.k1 + UK - 1) & ~(UK - 1);   // what lies behind K is zero
        }
    }
    const int np = S::wide ? nt : nw, nq = S::wide ? nw : nt;
    const int span = p.band * nq, b = idx / span, first = b * p.band, rows = min(p.band, np - first), within = idx - b * span;
    const int tp = first + within % rows, tq = within / rows;
    t.p0 = (S::wide ? lo : 0) + tp * S::P_TILE;
    t.p1 = S::wide ? hi : p.weights;
    t.q0 = (S::wide ? 0 : lo) + tq * (S::wide ? S::WEIGHTS : S::TOKENS);
    t.q1 = S::wide ? p.weights : hi;
    return t;
}

// 32 columns of a tile, v[c] = column j + c of the lane's row. NARROW: Y's rows are the columns j, a warp stores 32 lanes side by side;
// 16-bit values change places with the neighbour lane's, so that one 4-byte store serves two rows of Y.
template <class T>
__device__ __forceinline__ void store_narrow(T *Y, long long ldy, const uint32_t (&v)[32], int i0, int lane, int i1, int j, int j1) {
    T *dst = Y + (size_t)j * ldy + i0 + lane;
    if constexpr (sizeof(T) == 2) {
        if (i0 + 32 <= i1 && !((reinterpret_cast<uintptr_t>(Y) & 3) | (ldy & 1))) {
            const bool odd = lane & 1;
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
                const uint32_t own = Vec16<T>::word(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), other = __shfl_xor_sync(~0u, own, 1);
                const uint32_t w = odd ? __byte_perm(other, own, 0x7632) : __byte_perm(own, other, 0x5410);   // row c of lanes l, l + 1; or row c + 1 of l - 1, l
                if (j + c + odd < j1) *reinterpret_cast<uint32_t *>(dst + (size_t)(c + odd) * ldy - odd) = w;
            }
            return;
        }
    }
    if (i0 + lane >= i1) return;
#pragma unroll
    for (int c = 0; c < 32; c++)
        if (j + c < j1) dst[(size_t)c * ldy] = from_f32<T>(__uint_as_float(v[c]));
}
// WIDE: Y's row is the lane's. Whole 64-byte pieces of 32 rows go to the warp's shared memory (16-byte words permuted by their row, as
// the TMA unit's 64-byte swizzle has them, so that no two lanes meet in a bank) and from there by TMA, which takes them while the warp
// goes on: with stores of its own the warp held its accumulator until the L2 had taken them (segments of 512 tokens: 39 us for 100
// MB). Where the group's rows end inside the piece, or Y's columns inside 16 bytes of it (the unit writes whole ones), four lanes store
// 64 contiguous bytes of each row that is there. Rows that do not start on 16 bytes leave the piece value by value, 64 contiguous bytes
// to a row (14 segments of 289 x 798 BF16: 14 us; from the lanes that have the rows, a sector to a value, about 60).
struct Piece {
    uint8_t *buffer;       // two of 2048 bytes
    uint32_t used;         // pieces so far
    uint64_t policy;       // Y is not read here: its lines are the first to leave the L2
};
template <class T>
__device__ __forceinline__ void store_wide(const CUtensorMap *map, bool whole_words, T *Y, long long ldy, const uint32_t (&v)[32], int i0, int lane, int i1, int j, int j1,
                                           int group, Piece &piece) {
    if (j >= j1 || i0 >= i1) return;
    constexpr int N = Vec16<T>::N, COLS = 4 * N;   // columns to 16 and to 64 bytes
#pragma unroll
    for (int h = 0; h < 32; h += COLS) {
        if (j + h >= j1) break;
        uint8_t *buf = piece.buffer + 2048 * (piece.used++ & 1);
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");   // the piece before the last has left its buffer
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; c++) {
            float f[N];
#pragma unroll
            for (int e = 0; e < N; e++) f[e] = __uint_as_float(v[h + c * N + e]);
            *reinterpret_cast<uint4 *>(buf + lane * 64 + 16 * (c ^ (lane >> 1 & 3))) = Vec16<T>::pack(f);
        }
        if (!whole_words) {   // COLS lanes to a row, value by value
            __syncwarp();
            const int c = lane % COLS, col = j + h + c;
#pragma unroll 8
            for (int r = lane / COLS; r < 32; r += 32 / COLS) {
                const T x = *reinterpret_cast<const T *>(buf + r * 64 + 16 * (c / N ^ (r >> 1 & 3)) + c % N * sizeof(T));
                if (i0 + r < i1 && col < j1) Y[(size_t)(i0 + r) * ldy + col] = x;
            }
            __syncwarp();
        } else if (i0 + 32 <= i1 && (j + h + COLS <= j1 || (j1 - j - h) % N == 0)) {   // columns behind the last are cut by the tensor map, 16 bytes at a time
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group.L2::cache_hint [%0, {%2, %3, %4}], [%1], %5;"
                             ::"l"(map), "r"(smem_u32(buf)), "r"((j + h) * (int)sizeof(T)), "r"(i0), "r"(group), "l"(piece.policy) : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        } else {
            __syncwarp();
#pragma unroll
            for (int r = 0; r < 32; r += 8) {
                const int row = r + (lane >> 2), c = lane & 3;
                const uint4 q = *reinterpret_cast<const uint4 *>(buf + row * 64 + 16 * (c ^ (row >> 1 & 3)));
                T *dst = Y + (size_t)(i0 + row) * ldy + j + h + c * N;
                if (i0 + row < i1) {
                    if (j + h + (c + 1) * N <= j1) __stcs(reinterpret_cast<uint4 *>(dst), q);
                    else {
                        float f[N];
                        Vec16<T>::unpack(q, f);
#pragma unroll
                        for (int e = 0; e < N; e++)
                            if (j + h + c * N + e < j1) dst[e] = from_f32<T>(f[e]);
                    }
                }
            }
            if (lane == 0) asm volatile("cp.async.bulk.commit_group;" ::: "memory");   // an empty one, to keep the count
            __syncwarp();
        }
    }
}

template <int FORM, int BN, class T>
__global__ void __launch_bounds__(THREADS, 1) mx4_gemm(const __grid_constant__ CUtensorMap mapP, const __grid_constant__ CUtensorMap mapQ,
                                                       const __grid_constant__ CUtensorMap mapY, const Params p) {
    using S = Shape<FORM, BN>;
    constexpr bool pair = S::pair;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *const base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t slots = base + S::STAGES * S::STAGE, bars = slots + S::SLOTS * S::SLOT + S::TURN;
    auto full_bar = [&](int s) { return bars + 8u * s; };                                        // codes are there, and the scales in tensor memory (in a pair: both CTAs', at the leader)
    auto empty_bar = [&](int s) { return bars + 8u * (S::STAGES + s); };                         // the stage has been used up
    auto turned_bar = [&](int s) { return bars + 8u * (2 * S::STAGES + s); };                    // a slot's scales are turned (at the leader of a pair: both CTAs')
    auto slot_bar = [&](int s) { return bars + 8u * (2 * S::STAGES + S::SLOTS + s); };           // the slot has been used up
    auto accfull_bar = [&](int a) { return bars + 8u * (2 * S::STAGES + 2 * S::SLOTS + a); };
    auto accempty_bar = [&](int a) { return bars + 8u * (2 * S::STAGES + 2 * S::SLOTS + 2 + a); };
    const uint32_t tmem_slot = bars + 8u * S::BARS;
    int *const cum = reinterpret_cast<int *>(base_ptr + S::STAGES * S::STAGE + S::SLOTS * S::SLOT + S::TURN + 8 * S::BARS + 16);
    int4 *const ahead = reinterpret_cast<int4 *>(cum + MAX_GROUPS + 4);   // [AHEAD][2]
    __shared__ int abort_flag;

    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    uint32_t rank = 0, ranks = 1;
    if constexpr (FORM == SPLIT || pair) {
        rank = uniform(cluster_rank());
        asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
    }
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < S::STAGES; s++) { mbar_init(full_bar(s), 2); mbar_init(empty_bar(s), 1); }
        for (int s = 0; s < S::SLOTS; s++) { mbar_init(turned_bar(s), pair && rank == 0 ? 2 : 1); mbar_init(slot_bar(s), 1); }
        for (int a = 0; a < 2; a++) { mbar_init(accfull_bar(a), 1); mbar_init(accempty_bar(a), pair ? 16 : 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (pair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"((uint32_t)S::TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"((uint32_t)S::TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    behind_predecessors();
    if (warp == 2 && p.mode == BY_ROWS) {   // running number of token tiles over the groups
        const int most = 0x3fffffff / ((p.weights + S::WEIGHTS - 1) / S::WEIGHTS);   // offsets out of order may name rows again and again
        int run = 0;
        for (int g0 = 0; g0 < p.groups; g0 += 32) {
            int n = 0;
            if (g0 + lane < p.groups) {
                int lo, hi;
                segment(p, g0 + lane, p.tokens, lo, hi);
                n = min((hi - lo + S::TOKENS - 1) / S::TOKENS, most / 32);
            }
            int inc = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(~0u, inc, d);
                if (lane >= d) inc += o;
            }
            if (g0 + lane < p.groups) cum[g0 + lane] = min(run + inc - n, most);
            run = min(run + __shfl_sync(~0u, inc, 31), most);
        }
        if (lane == 0) cum[p.groups] = run;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (pair) cluster_sync_all();   // the peer's barriers exist before anything arrives on them
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    uint32_t tmem_base;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
    tmem_base = uniform(tmem_base);
    const uint32_t tmem_scales = tmem_base + 2 * BN;

    const int nt = p.mode == BY_ROWS ? cum[p.groups] : (p.tokens + S::TOKENS - 1) / S::TOKENS * (p.mode == ALONG_K ? p.groups : 1);
    const int total = uniform(nt) * ((p.weights + S::WEIGHTS - 1) / S::WEIGHTS);
    int first = blockIdx.x, step = gridDim.x;
    if constexpr (FORM == SPLIT) {   // one tile to a cluster; this CTA takes its share of the stages
        first = blockIdx.x / ranks;
        step = 1 << 30;
    }
    if constexpr (pair) {
        first = blockIdx.x >> 1;
        step = gridDim.x >> 1;
    }
    // A tile takes divisions and looks at the offsets: 900 cycles, as much as a short tile's products. The first AHEAD tiles of this CTA
    // are worked out by a thread each; the roles then read them.
    for (int n = threadIdx.x; n < AHEAD && n * (long long)step + first < total; n += THREADS) {
        const Tile t = decode<S>(p, cum, first + n * step);
        ahead[2 * n] = make_int4(t.group, t.p0, t.p1, t.q0);
        ahead[2 * n + 1] = make_int4(t.q1, t.k0, t.k1, 0);
    }
    __syncthreads();
    auto tile_at = [&](int w, uint32_t n) {   // the n-th tile of this CTA, item w
        Tile t;
        if (n < AHEAD) {
            const int4 a = ahead[2 * n], b = ahead[2 * n + 1];
            t.group = a.x; t.p0 = a.y; t.p1 = a.z; t.q0 = a.w;
            t.q1 = b.x; t.k0 = b.y; t.k1 = b.z;
        } else t = decode<S>(p, cum, w);
        t.s0 = t.k0 / BK;
        t.s1 = t.k1 > t.k0 ? (t.k1 + BK - 1) / BK : t.s0;
        if constexpr (FORM == SPLIT) {
            const int n = t.s1 - t.s0, s0 = t.s0;
            t.s0 = s0 + (int)((long long)n * rank / ranks);
            t.s1 = s0 + (int)((long long)n * (rank + 1) / ranks);
        }
        t.group = uniform(t.group);
        t.p0 = uniform(t.p0); t.p1 = uniform(t.p1);
        t.q0 = uniform(t.q0); t.q1 = uniform(t.q1);
        t.k0 = uniform(t.k0); t.k1 = uniform(t.k1);
        t.s0 = uniform(t.s0); t.s1 = uniform(t.s1);
        return t;
    };
    volatile int *abortp = &abort_flag;
    uint32_t it = 0, sl = 0;   // running stage and slot (of the role that counts them)

    if (warp == 0) {
        uint32_t n = 0;
        for (int w = first; w < total && !__any_sync(~0u, *abortp); w += step, n++) {
            const Tile t = tile_at(w, n);
            const int zp = !S::wide && p.mode == BY_ROWS ? t.group : 0, zq = S::wide && p.mode == BY_ROWS ? t.group : 0;
            const int p0 = t.p0 + (pair ? (int)rank * BP : 0), q0 = t.q0 + (pair ? (int)rank * S::Q_ROWS : 0);
            for (int kb = t.s0; kb < t.s1; kb++, it++) {
                const int s = it % S::STAGES;
                if (!warp_wait(empty_bar(s), ((it / S::STAGES) & 1u) ^ 1u, abortp, 0x111)) break;
                const uint32_t at = base + s * S::STAGE;
                if (elect_one()) {
                    if constexpr (pair) {
                        const uint32_t lead = map_to_cta(full_bar(s), 0);
                        if (rank == 0) mbar_expect_tx(full_bar(s), 2 * S::STAGE);   // both CTAs' bytes arrive here
                        tma_load_3d_pair(at, &mapP, kb * BKB, p0, zp, lead);
                        tma_load_3d_pair(at + S::P_BYTES, &mapQ, kb * BKB, q0, zq, lead);
                    } else {
                        mbar_expect_tx(full_bar(s), S::STAGE);
                        tma_load_3d(at, &mapP, kb * BKB, p0, zp, full_bar(s));
                        tma_load_3d(at + S::P_BYTES, &mapQ, kb * BKB, q0, zq, full_bar(s));
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        if (!pair || rank == 0) {
            uint32_t n = 0;
            for (int w = first; w < total && !__any_sync(~0u, *abortp); w += step, n++) {
                const Tile t = tile_at(w, n);
                const uint32_t acc = n & 1u;
                if (!warp_wait(accempty_bar(acc), ((n >> 1) & 1u) ^ 1u, abortp, 0x120)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t d = tmem_base + acc * BN;
                bool ok = true;
                uint32_t accumulate = 0;
                // a stage's instructions [k_lo, k_hi) of four, and its release
                auto issue = [&](int s, int k_lo, int k_hi) {
                    const uint32_t at = base + s * S::STAGE, tp = tmem_scales + s * S::SCALE_COLS, tq = tp + 8;
                    const uint64_t da = smem_desc(at), db = smem_desc(at + S::P_BYTES);
#pragma unroll
                    for (int k = 0; k < BK / UK; k++) {
                        if (k < k_lo || k >= k_hi) continue;
                        const uint32_t id = S::IDESC | ((k & 1u) ? (2u << 4) | (2u << 29) : 0u);      // which two of a word's four scales
                        mma_mx4<pair>(d, da + 2u * k, db + 2u * k, id, tp + 4 * (k >> 1), tq + 4 * (k >> 1) * S::Q_TILES, accumulate);
                        accumulate = 1;
                    }
                    commit<pair>(empty_bar(s));
                };
                const int whole0 = (t.k0 + BK - 1) / BK, whole1 = t.k1 / BK;   // stages all of whose instructions are in range
                for (int kb = t.s0; kb < t.s1;) {
                    const int s = it % S::STAGES;
                    const uint32_t parity = (it / S::STAGES) & 1u;
                    if (kb >= whole0 && kb + 2 <= whole1 && kb + 2 <= t.s1) {   // two at a time: a wait costs as much as two instructions
                        const int s2 = (it + 1) % S::STAGES;
                        if (!(ok = warp_wait2(full_bar(s), parity, full_bar(s2), ((it + 1) / S::STAGES) & 1u, abortp, 0x130))) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (elect_one()) {
                            issue(s, 0, 4);
                            issue(s2, 0, 4);
                        }
                        accumulate = 1;
                        kb += 2;
                        it += 2;
                    } else {
                        if (!(ok = warp_wait(full_bar(s), parity, abortp, 0x130))) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (elect_one()) issue(s, max(0, (t.k0 - kb * BK) / UK), (t.k1 - kb * BK + UK - 1) / UK);
                        accumulate = 1;
                        kb++;
                        it++;
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (elect_one()) commit<pair>(accfull_bar(acc));
                __syncwarp();
            }
        }
    } else if (warp == 2) {
        if (!pair || rank == 0) {
            uint32_t n = 0;
            for (int w = first; w < total && !__any_sync(~0u, *abortp); w += step, n++) {
                const Tile t = tile_at(w, n);
                bool ok = true;
                for (int at = t.s0 & ~(S::WINDOW - 1); at < t.s1 && ok; at += S::WINDOW)
                    for (int half = 0; half < S::HALVES && ok; half++, sl++) {
                        const int r = sl % S::SLOTS, s = it % S::STAGES, s2 = (it + 1) % S::STAGES;
                        const int from = max(t.s0, at + 2 * half), count = min(t.s1, at + 2 * half + 2) - from;   // this slot's stages: two, one or none
                        const uint32_t parity = ((it / S::STAGES) & 1u) ^ 1u, parity2 = (((it + 1) / S::STAGES) & 1u) ^ 1u;
                        if constexpr (pair) ok = __all_sync(~0u, mbar_wait_acquire_cluster(turned_bar(r), (sl / S::SLOTS) & 1u, abortp, 0x131));
                        else ok = warp_wait(turned_bar(r), (sl / S::SLOTS) & 1u, abortp, 0x131);
                        if (ok && count > 1) ok = warp_wait2(empty_bar(s), parity, empty_bar(s2), parity2, abortp, 0x132);
                        else if (ok && count > 0) ok = warp_wait(empty_bar(s), parity, abortp, 0x132);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t words = slots + r * S::SLOT;
                        auto copy = [&](int s, int second) {   // the two words of a stage
                            const uint32_t tp = tmem_scales + s * S::SCALE_COLS, tq = tp + 8;
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                copy_scales<pair>(tp + 4 * h, words + 512 * (2 * second + h));
#pragma unroll
                                for (int c = 0; c < S::Q_TILES; c++) copy_scales<pair>(tq + 4 * (h * S::Q_TILES + c), words + 2048 + 512 * ((2 * second + h) * S::Q_TILES + c));
                            }
                            if constexpr (pair) mma_commit_pair(full_bar(s));
                            else mma_commit(full_bar(s));
                        };
                        if (elect_one()) {
                            if (count > 1) {
                                copy(s, 0);
                                copy(s2, 1);
                            } else if (count > 0) copy(s, from & 1);
                            commit<pair>(slot_bar(r));
                        }
                        __syncwarp();
                        it += max(count, 0);
                    }
                if (!ok) break;
            }
        }
    } else if (warp == 3 || (warp >= 8 && warp < 7 + S::TURNERS)) {
        // Of TURNERS warps, in turns of a window: while one waits for its window's bytes, the others do theirs. Where many tiles share the
        // L2 a window is two slots: a row's 32 bytes are one sector of the L2's and are asked for at once (slot by slot they were fetched
        // twice, 15 % of all that the CTAs fetched: 2048 x 18432 x 7168 under the power limit 133 us, 125 so). For few tokens it is one,
        // which is there sooner (64 x 4096 x 4096: 6.5 us, 7.3 with two).
        const uint32_t own = warp == 3 ? 0 : warp - 7;
        const int blocks = (p.K + 31) / 32;
        uint32_t n = 0;
        for (int w = first; w < total && !__any_sync(~0u, *abortp); w += step, n++) {
            const Tile t = tile_at(w, n);
            const int p0 = t.p0 + (pair ? (int)rank * BP : 0);
            bool ok = true;
            for (int at = t.s0 & ~(S::WINDOW - 1); at < t.s1; at += S::WINDOW, sl += S::HALVES) {
                if (sl / S::HALVES % S::TURNERS != own) continue;
                const int r = sl % S::SLOTS, byte = at * 8, left = blocks - byte;
                const uint32_t parity = ((sl / S::SLOTS) & 1u) ^ 1u;
                const uint8_t *sp = p.sp + (size_t)t.group * p.plane_sp + byte, *sq = p.sq + (size_t)t.group * p.plane_sq + byte;
                uint8_t *slot = base_ptr + S::STAGES * S::STAGE + r * S::SLOT + 16 * lane;
                using Words = uint4[S::HALVES][4];
                auto load = [&](Words &v, int c) {   // tile c: P's, then Q's
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int row = i * 32 + lane, q = (c - 1) * 128 + row;
                        const bool there = c == 0 ? p0 + row < t.p1 : q < BN && t.q0 + q < t.q1;
                        const uint8_t *from = c == 0 ? sp + (size_t)(p0 + row) * p.ldsp : sq + (size_t)(t.q0 + q) * p.ldsq;
#pragma unroll
                        for (int h = 0; h < S::HALVES; h++) {
                            v[h][i] = make_uint4(0, 0, 0, 0);   // 2^-127: rows that are not there, and words behind a row's last
                            if (there && left > 16 * h) v[h][i] = *reinterpret_cast<const uint4 *>(from + 16 * h);
                        }
                    }
                };
                auto turn = [&](Words &v, int c) {
                    const int pitch = c == 0 ? 512 : 512 * S::Q_TILES;   // to the tile of the next word
#pragma unroll
                    for (int h = 0; h < S::HALVES; h++) {
                        if (left < 16 * h + 16 && left > 16 * h) {   // bytes behind the last block may hold anything: their codes are zero, their scales become it
#pragma unroll
                            for (int i = 0; i < 4; i++) v[h][i] = first_bytes(v[h][i], left - 16 * h);
                        }
                        uint8_t *dst = slot + h * S::SLOT + (c == 0 ? 0 : 2048 + 512 * (c - 1));
                        *reinterpret_cast<uint4 *>(dst) = make_uint4(v[h][0].x, v[h][1].x, v[h][2].x, v[h][3].x);
                        *reinterpret_cast<uint4 *>(dst + pitch) = make_uint4(v[h][0].y, v[h][1].y, v[h][2].y, v[h][3].y);
                        *reinterpret_cast<uint4 *>(dst + 2 * pitch) = make_uint4(v[h][0].z, v[h][1].z, v[h][2].z, v[h][3].z);
                        *reinterpret_cast<uint4 *>(dst + 3 * pitch) = make_uint4(v[h][0].w, v[h][1].w, v[h][2].w, v[h][3].w);
                    }
                };
                Words a, b;   // a third tile takes the first one's registers
                load(a, 0);
                load(b, 1);
                ok = warp_wait(slot_bar(r), parity, abortp, 0x140);
                if (S::HALVES == 2 && ok) ok = warp_wait(slot_bar(r + 1), parity, abortp, 0x140);
                if (!ok) break;
                turn(a, 0);
                if constexpr (S::Q_TILES == 2) load(a, 2);
                turn(b, 1);
                if constexpr (S::Q_TILES == 2) turn(a, 2);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the tensor core reads these through the async proxy
                __syncwarp();
                if (lane < S::HALVES) mbar_arrive(turned_bar(r + lane));
            }
            if (!ok) break;
        }
    } else if (pair && warp == 11) {
        // The leader's thread starts the copies of both CTAs, so what the peer's warps turned must be ordered before it: their arrivals
        // here (at the scope of the CTA), then a release at the scope of the cluster at the leader, which acquires at that scope. The
        // release holds a warp for 1800 cycles, so the warps that turn leave it to this one, a window of 2300 at a time.
        if (rank == 1) {
            uint32_t n = 0;
            for (int w = first; w < total && !__any_sync(~0u, *abortp); w += step, n++) {
                const Tile t = tile_at(w, n);
                bool ok = true;
                for (int at = t.s0 & ~(S::WINDOW - 1); at < t.s1; at += S::WINDOW, sl += S::HALVES) {
                    const int r = sl % S::SLOTS;
                    const uint32_t parity = (sl / S::SLOTS) & 1u;
                    for (int h = 0; h < S::HALVES && ok; h++) ok = warp_wait(turned_bar(r + h), parity, abortp, 0x141);
                    if (!ok) break;
                    if (lane < S::HALVES) mbar_arrive_release_cluster(map_to_cta(turned_bar(r + lane), 0));
                    __syncwarp();
                }
                if (!ok) break;
            }
        }
    } else if ((warp >= 4 && warp < 8) || warp >= 12) {
        const int quarter = warp & 3, half = warp >= 12;   // lanes 32 quarter .. +31, every other 32 columns
        Piece piece = {base_ptr + S::STAGES * S::STAGE + S::SLOTS * S::SLOT + (quarter + 4 * half) * 4096, 0, 0};
        asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(piece.policy));
        uint32_t n = 0;
        for (int w = first; w < total && !__any_sync(~0u, *abortp); w += step, n++) {
            const Tile t = tile_at(w, n);
            const uint32_t acc = n & 1u;
            if (!warp_wait(accfull_bar(acc), (n >> 1) & 1u, abortp, 0x150)) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * BN;
            const bool some = t.s1 > t.s0;   // no stage: nothing was accumulated, the tile is zero (or refused)
            const uint32_t nothing = t.k1 < 0 ? NOT_A_NUMBER : 0u;
            if (nothing && quarter == 0 && !half && lane == 0) atomicCAS(p.status, 0, STATUS_OFFSETS);
            const int i0 = t.p0 + (pair ? (int)rank * BP : 0) + quarter * 32;   // the warp's first row of P
            if constexpr (FORM != SPLIT) {
                T *Y = reinterpret_cast<T *>(p.Y) + (p.mode == ALONG_K ? (size_t)t.group * p.plane_y : 0);
#pragma unroll 1
                for (int c = 32 * half; c < BN; c += 64) {
                    if (t.q0 + c >= t.q1) break;
                    uint32_t v[32];
                    tmem_ld32(taddr + c, v);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (!some) {
#pragma unroll
                        for (int e = 0; e < 32; e++) v[e] = nothing;
                    }
                    const int j1 = min(t.q1, t.q0 + BN);   // a tile of 16 columns: the other 16 are not its own
                    if constexpr (S::wide) store_wide<T>(&mapY, p.whole_words, Y, p.ldy, v, i0, lane, t.p1, t.q0 + c, j1, p.mode == ALONG_K ? t.group : 0, piece);
                    else store_narrow<T>(Y, p.ldy, v, i0, lane, t.p1, t.q0 + c, j1);
                }
            } else {   // the partial tile, [column][row of P], over the stages that this CTA has used up
                float *part = reinterpret_cast<float *>(base_ptr);
#pragma unroll 1
                for (int c = 32 * half; c < BN; c += 64) {
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
            if (lane == 0) {
                if constexpr (pair) mbar_arrive_cluster(map_to_cta(accempty_bar(acc), 0));   // hands over no data: what was read is in registers
                else mbar_arrive(accempty_bar(acc));
            }
        }
        if (S::wide && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // every piece is in Y
    }

    __syncwarp();
    if constexpr (FORM == SPLIT) {
        // every CTA of the cluster adds its share of the columns over the ranks, in their order: the same sum on every run
        __syncthreads();
        cluster_sync_all();
        if (first < total) {
            const Tile t = decode<S>(p, cum, first);
            T *Y = reinterpret_cast<T *>(p.Y) + (p.mode == ALONG_K ? (size_t)t.group * p.plane_y : 0);
            const int r = threadIdx.x & (BP - 1), i = t.p0 + r;
            const int n = min(BN, t.q1 - t.q0), c0 = (int)((long long)n * rank / ranks), c1 = (int)((long long)n * (rank + 1) / ranks);
            for (int c = c0 + (threadIdx.x >> 7); c < c1; c += THREADS / BP) {
                float x[4], sum = 0.f;
#pragma unroll
                for (uint32_t q = 0; q < 4; q++)   // all in flight; ranks beyond the cluster's read this CTA's and are not added
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[q]) : "r"(map_to_cta(base + 4u * (c * BP + r), q < ranks ? q : rank)));
#pragma unroll
                for (uint32_t q = 0; q < 4; q++)
                    if (q < ranks) sum += x[q];
                if (i < t.p1) Y[(size_t)(t.q0 + c) * p.ldy + i] = from_f32<T>(sum);
            }
        }
        cluster_sync_all();   // nobody leaves while a peer still reads its partial tile
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (abort_flag && warp == 0 && lane == 0) {   // copies in flight land before this CTA's shared memory is given back
        const unsigned long long until = now_ns() + 200000000ull;
        for (uint32_t k = it > S::STAGES ? it - S::STAGES : 0; k < it && !pair; k++)
            while (!mbar_try(full_bar(k % S::STAGES), (k / S::STAGES) & 1u) && now_ns() < until) {}
        while (now_ns() < until) {}
    }
    __syncthreads();
    if constexpr (pair) cluster_sync_all();   // nobody leaves while the peer can still signal into its shared memory
    if (warp == 1) {
        if constexpr (pair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)S::TMEM_COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)S::TMEM_COLS) : "memory");
    }
    if (threadIdx.x == 0 && abort_flag) {
        atomicCAS(p.status, 0, abort_flag);
        if (blockIdx.x < 63) p.status[1 + blockIdx.x] = abort_flag;
    }
}

// ---- host ----

// {bytes along k, row, plane} of codes, in boxes of 128 bytes (256 values) by `box_rows` rows, swizzled
cudaError_t make_map(CUtensorMap *map, const uint8_t *ptr, int K, int rows, int planes, long long ld, size_t plane, int box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {(cuuint64_t)(((long long)K + 31) / 32 * 16), (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)(planes > 1 ? plane : (size_t)ld)};
    const cuuint32_t box[3] = {(cuuint32_t)BKB, (cuuint32_t)box_rows, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// what a form of the kernel does with a product: how many tiles, in how many CTAs
struct Work { long long most, expected; };   // token tiles times weight tiles: at most, and with even segments
Work work_of(const Mx4Product &g, int tokens, int weights) {
    const long long nw = (g.weights + weights - 1) / weights;
    if (g.mode != BY_ROWS) {
        const long long n = (long long)((g.tokens + tokens - 1) / tokens) * (g.mode == ALONG_K ? g.groups : 1) * nw;
        return {n, n};
    }
    const long long some = g.groups < g.tokens ? g.groups : g.tokens, each = (g.tokens + g.groups - 1) / g.groups;   // groups with rows, rows of one
    return {(some + g.tokens / tokens) * nw, some * ((each + tokens - 1) / tokens) * nw};
}

// {bytes of a row, row, group} of Y, in boxes of 64 bytes by 32 rows
cudaError_t make_map_y(CUtensorMap *map, void *y, long long bytes, int rows, int groups, long long ld, size_t plane) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {(cuuint64_t)bytes, (cuuint64_t)rows, (cuuint64_t)groups};
    const cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)(groups > 1 ? plane : (size_t)ld)};
    const cuuint32_t box[3] = {64, 32, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, y, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                           CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// how many clusters of `per` CTAs of the kernel the device holds at once
template <int FORM, int BN, class T>
int room_for(int per, int sms) {
    static int known[64][5] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return sms / per;
    int &n = known[dev & 63][per];
    if (!n) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(sms / per * per));
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = Shape<FORM, BN>::SMEM;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = per;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int found = 0;
        if (cudaOccupancyMaxActiveClusters(&found, mx4_gemm<FORM, BN, T>, &cfg) != cudaSuccess || found <= 0) { cudaGetLastError(); found = sms / per / 2; }
        n = found;
    }
    return n;
}

template <int FORM, int BN, class T>
cudaError_t launch(const Mx4Product &g, Params p, int sms, int split, cudaStream_t st) {
    using S = Shape<FORM, BN>;
    static PerDevice pd;
    cudaError_t e = pd.once([] { return cudaFuncSetAttribute(mx4_gemm<FORM, BN, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); });
    if (e) return e;
    const Work w = work_of(g, S::TOKENS, S::WEIGHTS);
    if (w.most > 0x0fffffffLL) return cudaErrorInvalidValue;
    const int planes = g.mode == BY_ROWS ? g.groups : 1;
    CUtensorMap x, w4;
    if ((e = make_map(&x, g.x, g.K, g.tokens, 1, g.ldx, 0, S::wide ? BP : S::Q_ROWS))) return e;
    if ((e = make_map(&w4, g.w, g.K, g.weights, planes, g.ldw, g.plane_w, S::wide ? S::Q_ROWS : BP))) return e;
    CUtensorMap y = x;
    const int results = g.mode == ALONG_K ? g.groups : 1;
    p.whole_words = S::wide && !(reinterpret_cast<uintptr_t>(g.y) & 15) && !(g.ldy * sizeof(T) & 15) && !(results > 1 && (g.plane_y * sizeof(T) & 15));
    if (p.whole_words && (e = make_map_y(&y, g.y, (long long)g.weights * sizeof(T), g.tokens, results, g.ldy * sizeof(T), g.plane_y * sizeof(T)))) return e;
    const size_t plane = planes > 1 ? g.plane_ws : 0;
    p.sp = S::wide ? g.xs : g.ws; p.ldsp = S::wide ? g.ldxs : g.ldws; p.plane_sp = S::wide ? 0 : plane;
    p.sq = S::wide ? g.ws : g.xs; p.ldsq = S::wide ? g.ldws : g.ldxs; p.plane_sq = S::wide ? plane : 0;
    // CTAs to a cluster, and clusters. A grid that is not resident as a whole takes twice its time: a pair that started behind another
    // would find its share of the tiles still to do. Not every SM has free neighbours, so the device is asked how many clusters there
    // can be (16 clusters of 8 were too many, for one).
    int per = 1;
    long long clusters = w.most < sms ? w.most : sms;
    if constexpr (FORM == PAIR) {
        per = 2;
        long long room = room_for<FORM, BN, T>(2, sms);
        clusters = w.most < room ? w.most : room;
    } else if constexpr (FORM == SPLIT) {
        for (per = split; per > 1 && w.expected > room_for<FORM, BN, T>(per, sms); per /= 2) {}
        clusters = w.most;
        if (per == 1) return launch<NARROW, BN, T>(g, p, sms, 1, st);
    }
    return launch_behind(mx4_gemm<FORM, BN, T>, (int)(clusters * per), THREADS, S::SMEM, per, st, S::wide ? x : w4, S::wide ? w4 : x, y, p);
}

}  // namespace m4

cudaError_t mx4_product(const Mx4Product &g, int *status, cudaStream_t st) {
    using namespace m4;
    Params p{};
    p.mode = g.mode;
    p.groups = g.groups;
    p.tokens = g.tokens;
    p.weights = g.weights;
    p.K = g.K;
    // 2048 x 18432 x 7168 in us with 4 : 8 : 16 : 32 : 64: 115 : 109 : 109 : 110 : 121; 8192^3, under the power limit, and 1024 x 8192 x 8192 the
    // same from 8 on
    p.band = 16;
    p.offsets = g.offsets;
    p.Y = g.y; p.ldy = g.ldy; p.plane_y = g.plane_y;
    p.status = status;
    int dev, sms;
    cudaError_t e = cudaGetDevice(&dev);
    if (!e) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e) return e;

    const int each = g.mode == BY_ROWS ? (g.tokens + g.groups - 1) / g.groups : g.tokens;   // tokens of a group
    const int stages = (g.K + BK - 1) / BK;
    auto run = [&](auto form, auto width, int split) {
        with_type(g.type, [&](auto t) { e = launch<decltype(form)::value, decltype(width)::value, decltype(t)>(g, p, sms, split, st); });
    };
#define M4_FORM(F) std::integral_constant<int, F>()
    // Many tokens to a group: tokens as lanes, in pairs of CTAs where there are tiles for all of them (groups of fewer than 512 tokens
    // fill too little of a pair's 256: 16 experts of 580, 21.6 us alone and 20.5 in pairs; 32 of 256, 50.5 and 53.4). Where 128 x 128
    // tiles are one to an SM or fewer they are better: 256 x 8192 x 8192 15.8 us with tokens as lanes, 13.4 without.
    if (each > 128 && work_of(g, 2 * BP, 192).expected >= sms / 2 && (g.mode != BY_ROWS || each >= 512)) run(M4_FORM(PAIR), M4_FORM(192), 1);
    else if (each > 128 && work_of(g, 128, BP).expected > sms) run(M4_FORM(WIDE), M4_FORM(192), 1);
    else {
        // Few tokens, or few tiles: weights as lanes; narrower tiles if that fills more SMs (333 x 1030 x 2085: 10.8 us at 128, 5.4 at 32).
        int bn = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128;
        while (bn > 32 && work_of(g, bn, BP).expected * 2 <= sms) bn /= 2;
        // Still few, and a long k: in two or four. The partial tiles cost about 2 us, 16 stages 3 (40 x 1024 x 8192: 8.8 us whole, 7.6 in
        // four; 32 x 2048 x 2048: 4.9 whole, 6.9 in two).
        const long long tiles = work_of(g, bn, BP).expected;
        int split = 1;
        if (bn <= 32 && g.mode != ALONG_K && stages >= 32)
            while (split < 4 && tiles * split * 2 <= sms && stages / (split * 2) >= 8) split *= 2;
        if (bn == 16 && split > 1) run(M4_FORM(SPLIT), M4_FORM(16), split);
        else if (bn == 32 && split > 1) run(M4_FORM(SPLIT), M4_FORM(32), split);
        else if (bn == 16) run(M4_FORM(NARROW), M4_FORM(16), 1);
        else if (bn == 32) run(M4_FORM(NARROW), M4_FORM(32), 1);
        else if (bn == 64) run(M4_FORM(NARROW), M4_FORM(64), 1);
        else run(M4_FORM(NARROW), M4_FORM(128), 1);
    }
#undef M4_FORM
    return e;
}

}  // namespace ozk
