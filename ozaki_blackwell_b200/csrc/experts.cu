// experts.cu -- tokens in the order of their experts and back.
//
// A token t of T goes to `top` experts; slot s = t * top + j is its j-th choice, ids[s] the expert (any number outside 0 .. E-1: the
// slot is dropped). sort puts the slots in the order of their experts, stable, each expert's segment padded to a multiple of
// `align` rows: row_of[s] and its inverse slot_of[r] (-1: none). With them
//     gather        xs[row_of[t, j]] = x[t]                          (zeros where there is no slot)
//     combine       y[t] = sum_j w[t, j] z[row_of[t, j]]             (in FP32, in the order of j)
//     its gradient  dz[r] = w[s] dy[s / top],  dw[s] = <dy[s / top], z[row_of[s]]>
// and the gradient of gather is combine without weights. An index that is out of range counts as none: nothing is read or
// written outside the arrays, whatever they hold.
#include <type_traits>
#include "oz_common.cuh"
#include "oz_kernels.h"
#include "oz_launch.cuh"
#include "oz_types.cuh"

namespace ozk {

namespace {

constexpr int MAX_EXPERTS = 1024;
// Up to here every block adds up all chunks' counts itself, behind it sort_scan comes between. Both sides in us, added : scanned: 64 experts
// 12.0 : 13.5 at 128 chunks, 15.3 : 14.6 at 256, 27.6 : 19.7 at 512; 8 experts 14.1 : 14.9 at 512. The counts matter more than the chunks:
// 1024 experts 11.6 : 12.9 at 32 chunks, 20.1 : 15.0 at 64, 65 : 18.2 at 256.
constexpr int FEW_CHUNKS = 256;
constexpr int CHUNK = 1024, SORT_THREADS = 256, SORT_WARPS = 8, PER_WARP = CHUNK / SORT_WARPS, ROUNDS = PER_WARP / 32, PLACE_THREADS = 1024;

// the expert of slot s, or `experts` for a dropped one
__device__ __forceinline__ int key_of(const void *ids, int id_bytes, int experts, int s) {
    const long long id = id_bytes == 8 ? *(reinterpret_cast<const long long *>(ids) + s) : (long long)*(reinterpret_cast<const int *>(ids) + s);
    return id >= 0 && id < experts ? (int)id : experts;
}

struct SortShared {
    int count[SORT_WARPS][MAX_EXPERTS];
    int total[MAX_EXPERTS], before[MAX_EXPERTS];
    int warp_sum[32];
};

// Ranks of a chunk's slots among its slots of the same expert, in their order. A warp owns PER_WARP consecutive slots and takes them 32
// at a time: lanes with the same expert find each other by a vote, the last of them adds their number to the warp's count, and a
// lane's rank is the count before plus the peers below it; then the counts of the warps before are added. total[e]: the chunk's.
__device__ __forceinline__ void rank_slots(SortShared &sh, const void *ids, int id_bytes, int experts, int slots, int first, int (&key)[ROUNDS], int (&rank)[ROUNDS]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int w = 0; w < SORT_WARPS; w++)
        for (int e = threadIdx.x; e < experts; e += SORT_THREADS) sh.count[w][e] = 0;
    first += warp * PER_WARP;
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int s = first + i * 32 + lane;
        key[i] = s < slots ? key_of(ids, id_bytes, experts, s) : experts;
        rank[i] = 0;
    }
    __syncthreads();
    int *count = sh.count[warp];
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        if (first + i * 32 >= slots) break;   // the same for the whole warp
        const uint32_t peers = __match_any_sync(~0u, key[i]);
        const int before = key[i] < experts ? count[key[i]] : 0;
        rank[i] = before + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
        if (key[i] < experts && (peers >> lane) == 1u) count[key[i]] = before + __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += SORT_THREADS) {
        int n = 0;
#pragma unroll
        for (int w = 0; w < SORT_WARPS; w++) {
            const int c = sh.count[w][e];
            sh.count[w][e] = n;
            n += c;
        }
        sh.total[e] = n;
        sh.before[e] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROUNDS; i++)
        if (key[i] < experts) rank[i] += count[key[i]];
}

// Where each segment begins, from the padded totals: total[e] becomes it, `offsets` is written if it is not null.
template <int THREADS>
__device__ __forceinline__ void place_segments(SortShared &sh, int experts, int align, int *offsets) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = (experts + THREADS - 1) / THREADS;   // consecutive experts to a thread
    int sum = 0;
    for (int i = 0; i < per; i++) {
        const int e = threadIdx.x * per + i;
        if (e < experts) sum += (sh.total[e] + align - 1) / align * align;
    }
    int inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(~0u, inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 31) sh.warp_sum[warp] = inc;
    __syncthreads();
    int at = inc - sum;
    for (int w = 0; w < warp; w++) at += sh.warp_sum[w];
    for (int i = 0; i < per; i++) {
        const int e = threadIdx.x * per + i;
        if (e >= experts) break;
        const int n = (sh.total[e] + align - 1) / align * align;
        sh.total[e] = at;
        if (offsets) offsets[e] = at;
        at += n;
        if (offsets && e == experts - 1) offsets[experts] = at;
    }
    __syncthreads();
}

// Up to CHUNK slots: one block does it all. More: sort_count ranks the slots of each chunk (row_of holds the ranks meanwhile), counts
// them by expert and clears slot_of; sort_place adds up the counts -- of all chunks for the segments' lengths, of the chunks before its
// own for where its slots go -- and writes both maps. With more than FEW_CHUNKS that would be the square of their number, so sort_scan
// comes between, which turns the counts into running sums over the chunks. All counts are whole numbers: the order is the same on
// every run.
__global__ void __launch_bounds__(SORT_THREADS) sort_one(const void *ids, int id_bytes, int experts, int slots, int align, int R, int *offsets, int *row_of, int *slot_of) {
    behind_predecessors();
    __shared__ SortShared sh;
    for (int r = threadIdx.x; r < R; r += SORT_THREADS) slot_of[r] = -1;
    int key[ROUNDS], rank[ROUNDS];
    rank_slots(sh, ids, id_bytes, experts, slots, 0, key, rank);
    place_segments<SORT_THREADS>(sh, experts, align, offsets);
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int s = (threadIdx.x >> 5) * PER_WARP + i * 32 + (threadIdx.x & 31);
        if (s >= slots) continue;
        const int row = key[i] < experts ? sh.total[key[i]] + rank[i] : -1;
        if (row >= 0) slot_of[row] = s;
        row_of[s] = row;
    }
}

__global__ void __launch_bounds__(SORT_THREADS) sort_count(const void *ids, int id_bytes, int experts, int slots, int R, int *row_of, int *slot_of, int *counts) {
    behind_predecessors();
    __shared__ SortShared sh;
    for (long long r = (long long)blockIdx.x * SORT_THREADS + threadIdx.x; r < R; r += (long long)gridDim.x * SORT_THREADS) slot_of[r] = -1;
    int key[ROUNDS], rank[ROUNDS];
    rank_slots(sh, ids, id_bytes, experts, slots, blockIdx.x * CHUNK, key, rank);
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int s = blockIdx.x * CHUNK + (threadIdx.x >> 5) * PER_WARP + i * 32 + (threadIdx.x & 31);
        if (s < slots) row_of[s] = rank[i];
    }
    for (int e = threadIdx.x; e < experts; e += SORT_THREADS) counts[(size_t)blockIdx.x * experts + e] = sh.total[e];
}

// total[e] = all chunks' counts, before[e] = those of the chunks before this block's; eight loads in flight to a thread (of 1024: with 256 the 16384 counts of
// 128 chunks by 128 experts took 8 us)
__device__ __forceinline__ void add_counts(SortShared &sh, const int *counts, int experts) {
    for (int e = threadIdx.x; e < experts; e += PLACE_THREADS) sh.total[e] = sh.before[e] = 0;
    __syncthreads();
    const int n = gridDim.x * experts, own = blockIdx.x * experts, step = PLACE_THREADS % experts;
    int e = threadIdx.x % experts;
    for (int i0 = threadIdx.x; i0 < n; i0 += 8 * PLACE_THREADS) {
        int c[8];
#pragma unroll
        for (int k = 0; k < 8; k++) c[k] = i0 + k * PLACE_THREADS < n ? counts[i0 + k * PLACE_THREADS] : 0;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (c[k]) {
                atomicAdd(&sh.total[e], c[k]);
                if (i0 + k * PLACE_THREADS < own) atomicAdd(&sh.before[e], c[k]);
            }
            e += step;
            if (e >= experts) e -= experts;
        }
    }
    __syncthreads();
}

// counts[chunk][e] -> the sum over the chunks before it; totals[e]. A block has 32 experts, a warp a range of the chunks.
__global__ void __launch_bounds__(1024) sort_scan(int *counts, int *totals, int chunks, int experts) {
    behind_predecessors();
    __shared__ int sums[32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    const int b0 = (int)((long long)chunks * warp / 32), b1 = (int)((long long)chunks * (warp + 1) / 32);
    int sum = 0;
    if (e < experts)
#pragma unroll 8
        for (int b = b0; b < b1; b++) sum += counts[(size_t)b * experts + e];
    sums[warp][lane] = sum;
    __syncthreads();
    int run = 0;
    for (int w = 0; w < warp; w++) run += sums[w][lane];
    if (e >= experts) return;
    if (warp == 31) totals[e] = run + sum;
    for (int b = b0; b < b1; b++) {
        const int n = counts[(size_t)b * experts + e];
        counts[(size_t)b * experts + e] = run;
        run += n;
    }
}

__global__ void __launch_bounds__(PLACE_THREADS) sort_place(const void *ids, int id_bytes, int experts, int slots, int align, int R, int *offsets,
                                                           int *row_of, int *slot_of, const int *counts, const int *totals) {
    behind_predecessors();
    __shared__ SortShared sh;
    int rank[CHUNK / PLACE_THREADS], key[CHUNK / PLACE_THREADS];
#pragma unroll
    for (int i = 0; i < CHUNK / PLACE_THREADS; i++) {
        const int s = blockIdx.x * CHUNK + i * PLACE_THREADS + threadIdx.x;
        key[i] = s < slots ? key_of(ids, id_bytes, experts, s) : experts;
        rank[i] = s < slots ? row_of[s] : 0;
    }
    if (totals) {   // the counts are running sums
        for (int e = threadIdx.x; e < experts; e += PLACE_THREADS) {
            sh.total[e] = totals[e];
            sh.before[e] = counts[(size_t)blockIdx.x * experts + e];
        }
        __syncthreads();
    } else add_counts(sh, counts, experts);
    place_segments<PLACE_THREADS>(sh, experts, align, blockIdx.x == 0 ? offsets : nullptr);
#pragma unroll
    for (int i = 0; i < CHUNK / PLACE_THREADS; i++) {
        const int s = blockIdx.x * CHUNK + i * PLACE_THREADS + threadIdx.x;
        if (s >= slots) continue;
        const int row = key[i] < experts ? sh.total[key[i]] + sh.before[key[i]] + rank[i] : -1;
        if (row >= 0) slot_of[row] = s;
        row_of[s] = row;
    }
}

// A warp reads a piece of a token's row once and writes it to the rows of all its slots; then it looks through 32 rows at a time for those
// without a slot and clears them. Rows move as they are: 16 bytes to a lane and load, four loads in flight, or single elements where
// rows do not start on 16 bytes. (Row by row, the tokens were read again from HBM for most of their slots: 824 MB for 605 at
// 16384 x 8 rows of 4 KB.)
template <class E>
__global__ void __launch_bounds__(256) gather_rows(const E *X, long long pitch_x, const int *row_of, const int *slot_of, int top, int T, int R, int n, E *Y,
                                                   long long pitch_y) {
    behind_predecessors();
    constexpr int DEPTH = 4, PIECE = 32 * DEPTH;
    const int lane = threadIdx.x & 31, pieces = (n + PIECE - 1) / PIECE;
    const long long warp = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), warps = (long long)gridDim.x * 8, slots = (long long)T * top;
    auto write = [&](long long r, int c0, const E (&v)[DEPTH]) {
#pragma unroll
        for (int i = 0; i < DEPTH; i++)
            if (c0 + 32 * i < n) __stcs(Y + r * pitch_y + c0 + 32 * i, v[i]);
    };
    for (long long w = warp; w < (long long)T * pieces; w += warps) {
        const long long t = w / pieces;
        const int c0 = (int)(w - t * pieces) * PIECE + lane;
        E v[DEPTH];
#pragma unroll
        for (int i = 0; i < DEPTH; i++) v[i] = X[t * pitch_x + min(c0 + 32 * i, n - 1)];
        for (int j = 0; j < top; j++) {
            const int r = row_of[t * top + j];
            if (r >= 0 && r < R) write(r, c0, v);
        }
    }
    for (long long r0 = warp * 32; r0 < R; r0 += warps * 32) {
        const int s = r0 + lane < R ? slot_of[r0 + lane] : 0;
        uint32_t none = __ballot_sync(~0u, s < 0 || s >= slots);
        const E zero[DEPTH] = {};
        while (none) {
            const int i = __ffs(none) - 1;
            none &= none - 1;
            for (int c0 = lane; c0 < n; c0 += PIECE) write(r0 + i, c0, zero);
        }
    }
}

// lanes that combine_rows gives to a token
template <bool VEC, int N> __host__ __device__ int combine_lanes(int H) { return VEC ? (H + N - 1) / N : (H + 32 * N - 1) / (32 * N) * 32; }

// A lane holds 16 bytes' worth of columns of one token and adds the token's rows in the order of j, U at a time: U loads are in flight,
// made whether the slot has a row or not (from row 0 if not), since loads under a condition each would wait for one another. Where rows
// do not start on 16 bytes its columns are 32 apart instead, so that a warp's loads and stores are side by side (4096 x 4 rows of 2047
// FP32: 34 us, 40 with neighbouring columns to a lane and conditions).
template <class T, bool VEC, int U>
__global__ void __launch_bounds__(256) combine_rows(const T *Z, long long ldz, int R, const int *row_of, const float *weights, int tokens, int top, int H,
                                                    T *Y, long long ldy) {
    behind_predecessors();
    constexpr int N = VEC ? Vec16<T>::N : 4, STEP = VEC ? 1 : 32;
    const int cols = combine_lanes<VEC, N>(H);
    const long long total = (long long)tokens * cols;
    for (long long w = (long long)blockIdx.x * 256 + threadIdx.x; w < total; w += (long long)gridDim.x * 256) {
        const int t = (int)(w / cols), l = (int)(w - (long long)t * cols), c = VEC ? l * N : (l & ~31) * N + (l & 31);
        float sum[N] = {};
        for (int j0 = 0; j0 < top; j0 += U) {
            int r[U];
            float f[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const long long s = (long long)t * top + min(j0 + u, top - 1);
                r[u] = j0 + u < top ? row_of[s] : -1;
                f[u] = weights ? weights[s] : 1.f;
                if (r[u] >= R) r[u] = -1;
            }
            if constexpr (VEC) {
                if (c + N <= H) {
                    uint4 q[U];
#pragma unroll
                    for (int u = 0; u < U; u++) q[u] = __ldcs(reinterpret_cast<const uint4 *>(Z + (size_t)max(r[u], 0) * ldz + c));
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        float v[N];
                        Vec16<T>::unpack(q[u], v);
                        if (r[u] >= 0)
#pragma unroll
                            for (int i = 0; i < N; i++) sum[i] = fmaf(f[u], v[i], sum[i]);
                    }
                } else {   // the last columns of a row that ends inside 16 bytes
#pragma unroll
                    for (int u = 0; u < U; u++)
                        if (r[u] >= 0)
#pragma unroll
                            for (int i = 0; i < N; i++)
                                if (c + i < H) sum[i] = fmaf(f[u], to_f32<T>(Z[(size_t)r[u] * ldz + c + i]), sum[i]);
                }
            } else {
                T v[U][N];
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int i = 0; i < N; i++) v[u][i] = Z[(size_t)max(r[u], 0) * ldz + min(c + i * STEP, H - 1)];
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (r[u] >= 0)
#pragma unroll
                        for (int i = 0; i < N; i++) sum[i] = fmaf(f[u], to_f32<T>(v[u][i]), sum[i]);
            }
        }
        T *y = Y + (size_t)t * ldy + c;
        if constexpr (VEC) {
            if (c + N <= H) {
                *reinterpret_cast<uint4 *>(y) = Vec16<T>::pack(sum);
                continue;
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++)
            if (c + i * STEP < H) y[i * STEP] = from_f32<T>(sum[i]);
    }
}

// A warp takes a row: dz from its token's dy, and the product of the two rows summed by lanes and then across them (a fixed order).
template <class T, bool VEC>
__global__ void __launch_bounds__(256) combine_grad_rows(const T *dY, long long lddy, const T *Z, long long ldz, int R, const int *row_of, const int *slot_of,
                                                         const float *weights, int slots, int top, int H, T *dZ, long long lddz, float *dW) {
    behind_predecessors();
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 31;
    for (long long s = (long long)blockIdx.x * 256 + threadIdx.x; s < slots; s += (long long)gridDim.x * 256) {
        const int r = row_of[s];
        if (r < 0 || r >= R) dW[s] = 0.f;   // a dropped slot
    }
    for (long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < R; r += (long long)gridDim.x * 8) {
        const int s = slot_of[r];
        T *dz = dZ + (size_t)r * lddz;
        constexpr int U = 4;   // pieces of both rows in flight
        if (s < 0 || s >= slots) {
            for (int c = lane * N; c < H; c += 32 * N) {
                if (VEC && c + N <= H) *reinterpret_cast<uint4 *>(dz + c) = make_uint4(0, 0, 0, 0);
                else
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (c + i < H) dz[c + i] = from_f32<T>(0.f);
            }
            continue;
        }
        const float f = weights ? weights[s] : 1.f;
        const T *dy = dY + (size_t)(s / top) * lddy, *z = Z + (size_t)r * ldz;
        float dot = 0.f;
        auto use = [&](float (&a)[N], const float (&b)[N]) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                dot = fmaf(a[i], b[i], dot);
                a[i] *= f;
            }
        };
        int c0 = 0;
        if constexpr (VEC) {
            for (; H - c0 >= U * 32 * N; c0 += U * 32 * N) {   // (a sum may pass 31 bits behind the last piece of the widest rows)
                uint4 qa[U], qb[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    qa[u] = *reinterpret_cast<const uint4 *>(dy + c0 + (u * 32 + lane) * N);
                    qb[u] = __ldcs(reinterpret_cast<const uint4 *>(z + c0 + (u * 32 + lane) * N));
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    float a[N], b[N];
                    Vec16<T>::unpack(qa[u], a);
                    Vec16<T>::unpack(qb[u], b);
                    use(a, b);
                    __stcs(reinterpret_cast<uint4 *>(dz + c0 + (u * 32 + lane) * N), Vec16<T>::pack(a));
                }
            }
        }
        if constexpr (VEC) {
            for (; H - c0 >= 32 * N; c0 += 32 * N) {
                float a[N], b[N];
                Vec16<T>::unpack(*reinterpret_cast<const uint4 *>(dy + c0 + lane * N), a);
                Vec16<T>::unpack(__ldcs(reinterpret_cast<const uint4 *>(z + c0 + lane * N)), b);
                use(a, b);
                __stcs(reinterpret_cast<uint4 *>(dz + c0 + lane * N), Vec16<T>::pack(a));
            }
        }
        constexpr int S = 8;
        // what is left, or rows that do not start on 16 bytes: single columns, S in flight (4096 x 4 rows of 2047 BF16: 42 us, 63 one by
        // one, behind each other's stores)
        for (int c = c0 + lane; c < H; c += 32 * S) {
            T a[S], b[S];
#pragma unroll
            for (int u = 0; u < S; u++) {
                a[u] = dy[min(c + 32 * u, H - 1)];
                b[u] = z[min(c + 32 * u, H - 1)];
            }
#pragma unroll
            for (int u = 0; u < S; u++) {
                if (c + 32 * u >= H) break;
                dot = fmaf(to_f32<T>(a[u]), to_f32<T>(b[u]), dot);
                dz[c + 32 * u] = from_f32<T>(f * to_f32<T>(a[u]));
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(~0u, dot, d);
        if (lane == 0) dW[s] = dot;
    }
}

int grid_of(long long blocks) { return (int)(blocks < (1 << 20) ? blocks : (1 << 20)); }
bool aligned(const void *p, long long ld, int size) { return !(reinterpret_cast<uintptr_t>(p) & 15) && !(ld * size & 15); }

}  // namespace

size_t expert_sort_scratch(int slots, int experts) {
    const size_t chunks = (slots + CHUNK - 1) / CHUNK;
    return chunks > 1 ? (chunks + (chunks > FEW_CHUNKS)) * experts * sizeof(int) : 0;
}

cudaError_t expert_sort(int slots, int experts, const void *ids, int id_bytes, int align, int R, int *offsets, int *rows, int *slot_of, void *scratch,
                        cudaStream_t st) {
    const int chunks = (slots + CHUNK - 1) / CHUNK;
    if (chunks == 1) {
        return launch_behind(sort_one, 1, SORT_THREADS, 0, 1, st, ids, id_bytes, experts, slots, align, R, offsets, rows, slot_of);
    }
    int *counts = static_cast<int *>(scratch);
    if (cudaError_t e = launch_behind(sort_count, chunks, SORT_THREADS, 0, 1, st, ids, id_bytes, experts, slots, R, rows, slot_of, counts)) return e;
    int *totals = nullptr;
    if (chunks > FEW_CHUNKS) {
        totals = counts + (size_t)chunks * experts;
        if (cudaError_t e = launch_behind(sort_scan, (experts + 31) / 32, 1024, 0, 1, st, counts, totals, chunks, experts)) return e;
    }
    return launch_behind(sort_place, chunks, PLACE_THREADS, 0, 1, st, ids, id_bytes, experts, slots, align, R, offsets, rows, slot_of, counts, totals);
}

cudaError_t expert_gather(int T, int top, int H, const void *X, int type, long long ldx, int R, const int *rows, const int *slots, void *Y,
                          long long ldy, cudaStream_t st) {
    const int size = type_size(type);
    auto grid = [&](int n) { return grid_of(((long long)T * ((n + 127) / 128) + R / 32 + 7) / 8); };
    if (aligned(X, ldx, size) && aligned(Y, ldy, size) && !((long long)H * size & 15)) {
        const int n = H * size / 16;
        return launch_behind(gather_rows<uint4>, grid(n), 256, 0, 1, st, (const uint4 *)X, ldx * size / 16, rows, slots, top, T, R, n, (uint4 *)Y, ldy * size / 16);
    }
    if (size == 4)
        return launch_behind(gather_rows<uint32_t>, grid(H), 256, 0, 1, st, (const uint32_t *)X, ldx, rows, slots, top, T, R, H, (uint32_t *)Y, ldy);
    return launch_behind(gather_rows<uint16_t>, grid(H), 256, 0, 1, st, (const uint16_t *)X, ldx, rows, slots, top, T, R, H, (uint16_t *)Y, ldy);
}

cudaError_t expert_combine(int T, int top, int H, const void *Z, int type, int R, long long ldz, const int *rows, const float *weights, void *Y,
                           long long ldy, cudaStream_t st) {
    cudaError_t e = cudaErrorInvalidValue;
    const int size = type_size(type);
    const bool vec = aligned(Z, ldz, size) && aligned(Y, ldy, size);
    const int lanes = !vec ? combine_lanes<false, 4>(H) : size == 4 ? combine_lanes<true, 4>(H) : combine_lanes<true, 8>(H);
    const int grid = grid_of(((long long)T * lanes + 255) / 256);
    with_type(type, [&](auto t) {
        using E = decltype(t);
        auto go = [&](auto many) {
            constexpr int U = decltype(many)::value;
            e = launch_behind(vec ? combine_rows<E, true, U> : combine_rows<E, false, U>, grid, 256, 0, 1, st, (const E *)Z, ldz, R, rows, weights, T, top, H, (E *)Y, ldy);
        };
        // Loads behind `top` are made for nothing, loads not in flight are waited for. With 2 : 4 : 8 of them, BF16 in us: 8192 x 2 rows of
        // 2048 19.0 : 23.0 : 36.0, x 4 29.8 : 27.6 : 38.8, x 6 40.5 : 40.9 : 43.5, x 8 50.8 : 46.2 : 48.4; 16 x 8 rows 2.75 : 2.35 : 2.13; 4096 x 6
        // rows of 2047 55.8 : 53.7 : 47.2, x 8 70.0 : 54.5 : 49.0.
        if (top <= 2) go(std::integral_constant<int, 2>());
        else if (top <= 4) go(std::integral_constant<int, 4>());
        else go(std::integral_constant<int, 8>());
    });
    return e;
}

cudaError_t expert_combine_grad(int T, int top, int H, const void *dY, int type, long long lddy, const void *Z, long long ldz, int R, const int *rows,
                                const int *slots, const float *weights, void *dZ, long long lddz, float *dweights, cudaStream_t st) {
    cudaError_t e = cudaErrorInvalidValue;
    const int size = type_size(type);
    const bool vec = aligned(dY, lddy, size) && aligned(Z, ldz, size) && aligned(dZ, lddz, size);
    const int grid = grid_of(((long long)R + 7) / 8);
    with_type(type, [&](auto t) {
        using E = decltype(t);
        e = launch_behind(vec ? combine_grad_rows<E, true> : combine_grad_rows<E, false>, grid, 256, 0, 1, st, (const E *)dY, lddy, (const E *)Z, ldz, R, rows, slots, weights, T * top, top, H, (E *)dZ, lddz, dweights);
    });
    return e;
}

}  // namespace ozk
