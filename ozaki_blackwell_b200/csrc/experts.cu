// experts.cu -- tokens in the order of their experts and back.
//
// A token t of T goes to `top` experts; slot s = t * top + j is its j-th choice, ids[s] the expert (any number outside 0 .. E-1: the
// slot is dropped). sort puts the slots in the order of their experts, stable, each expert's segment padded to a multiple of
// `align` rows: row_of[s] and its inverse slot_of[r] (-1: none). With them
//     gather        xs[r] = x[slot_of[r] / top]                      (zeros where there is no slot)
//     combine       y[t] = sum_j w[t, j] z[row_of[t, j]]             (in FP32, in the order of j)
//     its gradient  dz[r] = w[s] dy[s / top],  dw[s] = <dy[s / top], z[row_of[s]]>
// and the gradient of gather is combine without weights. An index that is out of range counts as none: nothing is read or
// written outside the arrays, whatever they hold.
#include "oz_common.cuh"
#include "oz_kernels.h"
#include "oz_types.cuh"

namespace ozk {

namespace {

constexpr int MAX_EXPERTS = 1024;
constexpr int CHUNK = 2048, SORT_THREADS = 256, SORT_WARPS = 8, PER_WARP = CHUNK / SORT_WARPS, ROUNDS = PER_WARP / 32;

// the expert of slot s, or `experts` for a dropped one
__device__ __forceinline__ int key_of(const void *ids, int id_bytes, int experts, int s) {
    const long long id = id_bytes == 8 ? __ldg(reinterpret_cast<const long long *>(ids) + s) : (long long)__ldg(reinterpret_cast<const int *>(ids) + s);
    return id >= 0 && id < experts ? (int)id : experts;
}

// A warp owns PER_WARP consecutive slots of the chunk and takes them 32 at a time in their order: lanes with the same expert find each
// other by a vote, the first of them adds their number to the warp's count, and a lane's rank is the count before plus the peers
// below it. rank[i]: the rank of the i-th round's slot among the warp's slots of its expert; count[e]: the warp's total.
__device__ __forceinline__ void rank_slots(const void *ids, int id_bytes, int experts, int slots, int first, int *count, int (&key)[ROUNDS], int (&rank)[ROUNDS]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int s = first + i * 32 + lane;
        key[i] = s < slots ? key_of(ids, id_bytes, experts, s) : experts;
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        if (first + i * 32 >= slots) break;   // the same for the whole warp
        const uint32_t peers = __match_any_sync(~0u, key[i]);
        const int before = key[i] < experts ? count[key[i]] : 0;
        rank[i] = before + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
        if (key[i] < experts && (peers >> lane) == 1u) count[key[i]] = before + __popc(peers);   // the highest of the peers
        __syncwarp();
    }
}

// Two kernels where there is more than one chunk: the first counts each chunk's slots by expert (and clears slot_of), the second
// adds up the counts of all chunks -- of every chunk for the segments' lengths, of the chunks before its own for where its slots
// go -- and writes both maps. With one chunk the second does it all. Every count is an integer sum: the order is exact and the same
// on every run.
__global__ void __launch_bounds__(SORT_THREADS) sort_count(const void *ids, int id_bytes, int experts, int slots, int R, int *slot_of, int *counts) {
    __shared__ int count[SORT_WARPS][MAX_EXPERTS];
    const int warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < experts * SORT_WARPS; e += SORT_THREADS) count[e / experts][e % experts] = 0;
    for (long long r = (long long)blockIdx.x * SORT_THREADS + threadIdx.x; r < R; r += (long long)gridDim.x * SORT_THREADS) slot_of[r] = -1;
    __syncthreads();
    int key[ROUNDS], rank[ROUNDS];
    rank_slots(ids, id_bytes, experts, slots, blockIdx.x * CHUNK + warp * PER_WARP, count[warp], key, rank);
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += SORT_THREADS) {
        int n = 0;
#pragma unroll
        for (int w = 0; w < SORT_WARPS; w++) n += count[w][e];
        counts[(size_t)blockIdx.x * experts + e] = n;
    }
}

__global__ void __launch_bounds__(SORT_THREADS) sort_place(const void *ids, int id_bytes, int experts, int slots, int align, int R, int *offsets,
                                                           int *row_of, int *slot_of, const int *counts) {
    __shared__ int count[SORT_WARPS][MAX_EXPERTS];   // where the next slot of a warp for an expert goes, in the end
    __shared__ int warp_sum[SORT_WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool alone = counts == nullptr;
    for (int e = threadIdx.x; e < experts * SORT_WARPS; e += SORT_THREADS) count[e / experts][e % experts] = 0;
    if (alone) for (int r = threadIdx.x; r < R; r += SORT_THREADS) slot_of[r] = -1;
    __syncthreads();
    const int first = blockIdx.x * CHUNK + warp * PER_WARP;
    int key[ROUNDS], rank[ROUNDS];
    rank_slots(ids, id_bytes, experts, slots, first, count[warp], key, rank);
    __syncthreads();
    // a thread takes up to four consecutive experts
    constexpr int PER = MAX_EXPERTS / SORT_THREADS;
    int before[PER], length[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = threadIdx.x * PER + i;
        before[i] = length[i] = 0;
        if (e >= experts) continue;
        if (alone) {
#pragma unroll
            for (int w = 0; w < SORT_WARPS; w++) length[i] += count[w][e];
        } else {
            for (int b = 0; b < (int)gridDim.x; b++) {
                const int n = __ldg(counts + (size_t)b * experts + e);
                if (b < (int)blockIdx.x) before[i] += n;
                length[i] += n;
            }
        }
        length[i] = (length[i] + align - 1) / align * align;
        sum += length[i];
    }
    int inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(~0u, inc, d);
        if (lane >= d) inc += o;
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    int at = inc - sum;
    for (int w = 0; w < warp; w++) at += warp_sum[w];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = threadIdx.x * PER + i;
        if (e >= experts) continue;
        if (blockIdx.x == 0) offsets[e] = at;
        int next = at + before[i];
#pragma unroll
        for (int w = 0; w < SORT_WARPS; w++) {
            const int n = count[w][e];
            count[w][e] = next;
            next += n;
        }
        at += length[i];
        if (blockIdx.x == 0 && e == experts - 1) offsets[experts] = at;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int s = first + i * 32 + lane;
        if (s >= slots) continue;
        int row = -1;
        if (key[i] < experts) {
            row = count[warp][key[i]] + rank[i];
            if (row < R) slot_of[row] = s;   // always: the caller's R holds every padded segment
        }
        row_of[s] = row;
    }
}

// Rows move as they are: 16 bytes to a lane and load, four loads in flight, or single elements where rows do not start on 16 bytes.
template <class E>
__global__ void __launch_bounds__(256) gather_rows(const E *X, long long pitch_x, const int *slot_of, int top, int T, int R, int n, E *Y, long long pitch_y) {
    constexpr int DEPTH = 4;
    const int lane = threadIdx.x & 31, pieces = (n + 32 * DEPTH - 1) / (32 * DEPTH);
    const long long total = (long long)R * pieces;
    for (long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); w < total; w += (long long)gridDim.x * 8) {
        const int r = (int)(w / pieces), c0 = (int)(w - (long long)r * pieces) * 32 * DEPTH + lane;
        const int s = __ldg(slot_of + r), t = s >= 0 ? s / top : -1;
        E v[DEPTH];
#pragma unroll
        for (int i = 0; i < DEPTH; i++) {
            v[i] = E();
            if (t >= 0 && t < T && c0 + 32 * i < n) v[i] = __ldg(X + (size_t)t * pitch_x + c0 + 32 * i);
        }
#pragma unroll
        for (int i = 0; i < DEPTH; i++)
            if (c0 + 32 * i < n) Y[(size_t)r * pitch_y + c0 + 32 * i] = v[i];
    }
}

// A lane holds 16 bytes' worth of columns of one token and adds the token's rows in the order of j.
template <class T, bool VEC>
__global__ void __launch_bounds__(256) combine_rows(const T *Z, long long ldz, int R, const int *row_of, const float *weights, int tokens, int top, int H,
                                                    T *Y, long long ldy) {
    constexpr int N = Vec16<T>::N;
    const int cols = (H + N - 1) / N;
    const long long total = (long long)tokens * cols;
    for (long long w = (long long)blockIdx.x * 256 + threadIdx.x; w < total; w += (long long)gridDim.x * 256) {
        const int t = (int)(w / cols), c = (int)(w - (long long)t * cols) * N;
        float sum[N] = {};
#pragma unroll 4
        for (int j = 0; j < top; j++) {
            const long long s = (long long)t * top + j;
            const int r = __ldg(row_of + s);
            if (r < 0 || r >= R) continue;
            const float f = weights ? __ldg(weights + s) : 1.f;
            const T *z = Z + (size_t)r * ldz + c;
            float v[N];
            if (VEC && c + N <= H) Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(z)), v);
            else
#pragma unroll
                for (int i = 0; i < N; i++) v[i] = c + i < H ? to_f32<T>(z[i]) : 0.f;
#pragma unroll
            for (int i = 0; i < N; i++) sum[i] = fmaf(f, v[i], sum[i]);
        }
        T *y = Y + (size_t)t * ldy + c;
        if (VEC && c + N <= H) *reinterpret_cast<uint4 *>(y) = Vec16<T>::pack(sum);
        else
#pragma unroll
            for (int i = 0; i < N; i++)
                if (c + i < H) y[i] = from_f32<T>(sum[i]);
    }
}

// A warp takes a row: dz from its token's dy, and the product of the two rows summed by lanes and then across them (a fixed order).
template <class T, bool VEC>
__global__ void __launch_bounds__(256) combine_grad_rows(const T *dY, long long lddy, const T *Z, long long ldz, int R, const int *row_of, const int *slot_of,
                                                         const float *weights, int slots, int top, int H, T *dZ, long long lddz, float *dW) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 31;
    for (long long s = (long long)blockIdx.x * 256 + threadIdx.x; s < slots; s += (long long)gridDim.x * 256) {
        const int r = __ldg(row_of + s);
        if (r < 0 || r >= R) dW[s] = 0.f;   // a dropped slot
    }
    for (long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); r < R; r += (long long)gridDim.x * 8) {
        const int s = __ldg(slot_of + r);
        const bool there = s >= 0 && s < slots;
        const float f = !there ? 0.f : weights ? __ldg(weights + s) : 1.f;
        const T *dy = dY + (size_t)(there ? s / top : 0) * lddy, *z = Z + (size_t)r * ldz;
        T *dz = dZ + (size_t)r * lddz;
        float dot = 0.f;
#pragma unroll 2
        for (int c = lane * N; c < H; c += 32 * N) {
            float a[N] = {}, b[N] = {};
            if (VEC && c + N <= H) {
                if (there) {
                    Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(dy + c)), a);
                    Vec16<T>::unpack(__ldg(reinterpret_cast<const uint4 *>(z + c)), b);
                }
            } else if (there) {
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (c + i < H) { a[i] = to_f32<T>(dy[c + i]); b[i] = to_f32<T>(z[c + i]); }
            }
#pragma unroll
            for (int i = 0; i < N; i++) {
                dot = fmaf(a[i], b[i], dot);
                a[i] = there ? f * a[i] : 0.f;
            }
            if (VEC && c + N <= H) *reinterpret_cast<uint4 *>(dz + c) = Vec16<T>::pack(a);
            else
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (c + i < H) dz[c + i] = from_f32<T>(a[i]);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(~0u, dot, d);
        if (lane == 0 && there) dW[s] = dot;
    }
}

int grid_of(long long blocks) { return (int)(blocks < (1 << 20) ? blocks : (1 << 20)); }
bool aligned(const void *p, long long ld, int size) { return !(reinterpret_cast<uintptr_t>(p) & 15) && !(ld * size & 15); }

}  // namespace

size_t expert_sort_scratch(int slots, int experts) {
    return slots > CHUNK ? (size_t)((slots + CHUNK - 1) / CHUNK) * experts * sizeof(int) : 0;
}

cudaError_t expert_sort(int slots, int experts, const void *ids, int id_bytes, int align, int R, int *offsets, int *rows, int *slot_of, void *scratch,
                        cudaStream_t st) {
    const int chunks = (slots + CHUNK - 1) / CHUNK;
    int *counts = chunks > 1 ? static_cast<int *>(scratch) : nullptr;
    if (counts) sort_count<<<chunks, SORT_THREADS, 0, st>>>(ids, id_bytes, experts, slots, R, slot_of, counts);
    sort_place<<<chunks, SORT_THREADS, 0, st>>>(ids, id_bytes, experts, slots, align, R, offsets, rows, slot_of, counts);
    return cudaGetLastError();
}

cudaError_t expert_gather(int R, int H, const void *X, int type, long long ldx, int T, const int *slots, int top, void *Y, long long ldy,
                          cudaStream_t st) {
    const int size = type_size(type);
    auto grid = [&](int n) { return grid_of(((long long)R * ((n + 127) / 128) + 7) / 8); };
    if (aligned(X, ldx, size) && aligned(Y, ldy, size) && !((long long)H * size & 15)) {
        const int n = H * size / 16;
        gather_rows<uint4><<<grid(n), 256, 0, st>>>((const uint4 *)X, ldx * size / 16, slots, top, T, R, n, (uint4 *)Y, ldy * size / 16);
    } else if (size == 4) {
        gather_rows<uint32_t><<<grid(H), 256, 0, st>>>((const uint32_t *)X, ldx, slots, top, T, R, H, (uint32_t *)Y, ldy);
    } else {
        gather_rows<uint16_t><<<grid(H), 256, 0, st>>>((const uint16_t *)X, ldx, slots, top, T, R, H, (uint16_t *)Y, ldy);
    }
    return cudaGetLastError();
}

cudaError_t expert_combine(int T, int top, int H, const void *Z, int type, int R, long long ldz, const int *rows, const float *weights, void *Y,
                           long long ldy, cudaStream_t st) {
    const int size = type_size(type), n = 16 / size;
    const bool vec = aligned(Z, ldz, size) && aligned(Y, ldy, size);
    const int grid = grid_of(((long long)T * ((H + n - 1) / n) + 255) / 256);
    with_type(type, [&](auto t) {
        using E = decltype(t);
        if (vec) combine_rows<E, true><<<grid, 256, 0, st>>>((const E *)Z, ldz, R, rows, weights, T, top, H, (E *)Y, ldy);
        else combine_rows<E, false><<<grid, 256, 0, st>>>((const E *)Z, ldz, R, rows, weights, T, top, H, (E *)Y, ldy);
    });
    return cudaGetLastError();
}

cudaError_t expert_combine_grad(int T, int top, int H, const void *dY, int type, long long lddy, const void *Z, long long ldz, int R, const int *rows,
                                const int *slots, const float *weights, void *dZ, long long lddz, float *dweights, cudaStream_t st) {
    const int size = type_size(type);
    const bool vec = aligned(dY, lddy, size) && aligned(Z, ldz, size) && aligned(dZ, lddz, size);
    const int grid = grid_of(((long long)R + 7) / 8);
    with_type(type, [&](auto t) {
        using E = decltype(t);
        if (vec) combine_grad_rows<E, true><<<grid, 256, 0, st>>>((const E *)dY, lddy, (const E *)Z, ldz, R, rows, slots, weights, T * top, top, H, (E *)dZ, lddz, dweights);
        else combine_grad_rows<E, false><<<grid, 256, 0, st>>>((const E *)dY, lddy, (const E *)Z, ldz, R, rows, slots, weights, T * top, top, H, (E *)dZ, lddz, dweights);
    });
    return cudaGetLastError();
}

}  // namespace ozk
