// mx4.cu -- the microscaled 4-bit format: rounding to it by rows and by columns, and back.
//
// A vector is cut into blocks of 32. With amax the largest magnitude of a block, its scale is 2^e, |e| <= 127, and a value x is
// the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to |x| 2^-e (ties to the even code), with its sign:
//     rule 0:  e = floor(log2 amax) - 2          (the largest value lands in [4, 8) and saturates at 6)
//     rule 1:  e = ceil(log2(amax / 6))          (nothing saturates)
// With amax = 1.f 2^p both are integer arithmetic on the bits of amax: p - 2, plus one under rule 1 if 1.f > 1.5. The scale is
// stored as the byte e + 127, clamped at 0 (an empty block, or values below 2^-125); 255 marks a block that holds an infinity or a
// NaN. x 2^-e is exact: it is below 8, and what falls below 2^-126 is rounded to the code of 0 either way. The rounding itself is
// the hardware's conversion (cvt.rn.satfinite.e2m1x2.f32).
#include <type_traits>
#include "oz_common.cuh"
#include "oz_kernels.h"
#include "oz_launch.cuh"
#include "oz_types.cuh"

namespace ozk {

namespace {

// eight values -> eight codes, the first in the lowest four bits
__device__ __forceinline__ uint32_t codes_of(const float *v) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
__device__ __forceinline__ uint32_t codes_of4(const float *v) {   // four
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, z;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.u8.u32 z, 0;\n\t"
        "mov.b32 %0, {b0, b1, z, z};\n\t}"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
    return r;
}
// two codes (a byte) -> two values
__device__ __forceinline__ float2 pair_of(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 b;\n\t"
        "cvt.u8.u32 b, %1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b;\n\t}"
        : "=r"(h) : "r"(byte));
    __half2 p;
    memcpy(&p, &h, 4);
    return __half22float2(p);
}
// N codes -> N values
template <int N> __device__ __forceinline__ void values_of(uint32_t c, float *v) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const float2 f = pair_of(c >> (4 * i) & 0xffu);
        v[i] = f.x;
        v[i + 1] = f.y;
    }
}
// the block's scale byte from the bits of its largest magnitude (0 .. 255)
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits, int rule) {
    if (amax_bits >= 0x7f800000u) return 255;
    const int field = (int)((amax_bits + (rule ? 0x3fffffu : 0u)) >> 23);   // mantissa above 1.5: the next power of two
    return field > 2 ? (uint32_t)(field - 2) : 0u;
}
// 2^-e for the byte e + 127, which is at most 253 (e of the largest number is 126). For 255, a block that is not a number, it
// is minus infinity, and the codes that come of it are cleared.
__device__ __forceinline__ float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float scale_of(uint32_t byte) {
    return __uint_as_float(byte == 255 ? 0x7fffffffu : byte ? byte << 23 : 0x00400000u);
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// the row of X that vector or element r takes its values from; -1: none (zeros)
__device__ __forceinline__ long long source_row(const int *slots, int per, int sources, int r) {
    if (!slots) return r;
    const int s = slots[r];
    if (s < 0) return -1;
    const int row = s / per;
    return row < sources ? row : -1;
}

// The largest magnitude of the values in a 16-byte word, as the bits of a float: two 16-bit values at a time (a magnitude's bits order
// like the number, infinities and NaN above all).
template <class T> __device__ __forceinline__ uint32_t magnitude_of(const uint4 &q) {
    if constexpr (sizeof(T) == 4) return max(max(q.x & 0x7fffffffu, q.y & 0x7fffffffu), max(q.z & 0x7fffffffu, q.w & 0x7fffffffu));
    else {
        constexpr uint32_t M = 0x7fff7fffu;
        uint32_t m = __vmaxu2(__vmaxu2(q.x & M, q.y & M), __vmaxu2(q.z & M, q.w & M));
        m = max(m & 0xffffu, m >> 16);
        T t;
        memcpy(&t, &m, sizeof t);
        return magnitude(to_f32<T>(t));
    }
}

// Blocks along the rows of X. A lane holds 16 bytes of values, 4 or 8 lanes a block; a warp's load is 512 contiguous bytes and UNITS of
// them are in flight. Bound by HBM, and near the limit of instruction issue, so magnitudes are compared and values scaled two at a
// time. (With 32 or 64 contiguous bytes to a lane the loads touched two or four times the lines: 81 us for 16384 x 7168 BF16.)
// ROUTED: the warp's row is a token, rounded once and written to the rows of all its slots; then rows without a slot are looked for,
// 32 at a time, and become zeros.
constexpr int UNITS = 4;
template <class T, bool VEC, bool ROUTED, int U>
__global__ void __launch_bounds__(256) mx4_rows(const T *X, int nvec, int len, long long ldx, size_t plane_x, int planes, int rule,
                                                const int *row_of, const int *slot_of, int top, int tokens, uint8_t *codes, long long ldq,
                                                size_t plane_q, uint8_t *scales, long long lds, size_t plane_s) {
    behind_predecessors();
    constexpr int N = Vec16<T>::N, LOAD = 32 * N, SHARE = 32 / N;   // values of a lane, of a load of the warp; lanes of a block
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t units = (len + LOAD * U - 1) / (LOAD * U);
    const long long total = (long long)(ROUTED ? tokens : (long long)planes * nvec) * units;
    for (long long w = (long long)blockIdx.x * 8 + warp; w < total; w += (long long)gridDim.x * 8) {
        const long long vec = total < 0x80000000ll ? (long long)((uint32_t)w / units) : w / units;
        const long long z = planes > 1 ? vec / nvec : 0, r = vec - z * nvec;
        const int at = (int)(w - vec * units) * LOAD * U + lane * N;   // the lane's first value
        const T *x = X + z * plane_x + r * ldx;
        uint4 q[U];
        int mine = -1;   // ROUTED: 32 of the token's rows, a lane each
        if constexpr (VEC) {   // rows start on 16 bytes and end on them; loads behind the end are made at the end, and cleared
#pragma unroll
            for (int u = 0; u < U; u++) q[u] = *reinterpret_cast<const uint4 *>(x + min(at + u * LOAD, len - N));
#pragma unroll
            for (int u = 0; u < U; u++)
                if (at + u * LOAD >= len) q[u] = make_uint4(0, 0, 0, 0);
        } else {   // value by value, zeros behind the last
#pragma unroll
            for (int u = 0; u < U; u++) {
                T v[N];
#pragma unroll
                for (int i = 0; i < N; i++) v[i] = x[min(at + u * LOAD + i, len - 1)];
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (at + u * LOAD + i >= len) v[i] = from_f32<T>(0.f);
                memcpy(&q[u], v, 16);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int e = at + u * LOAD;
            if (e - lane * N >= len) break;   // the same for the whole warp
            uint32_t m = magnitude_of<T>(q[u]);
#pragma unroll
            for (int d = 1; d < SHARE; d <<= 1) m = max(m, __shfl_xor_sync(~0u, m, d));
            const uint32_t byte = scale_byte(m, rule);
            const float2 inv = make_float2(inverse_scale(byte), inverse_scale(byte));
            float v[8] = {};
            Vec16<T>::unpack(q[u], v);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float2 f = __fmul2_rn(make_float2(v[i], v[i + 1]), inv);
                v[i] = f.x;
                v[i + 1] = f.y;
            }
            const uint32_t c = byte == 255 ? 0u : N == 8 ? codes_of(v) : codes_of4(v);
            auto write = [&](uint8_t *codes_row, uint8_t *scales_row) {   // a block is written whole, zeros behind the last value
                if ((e & ~31) >= len) return;
                if constexpr (N == 8) *reinterpret_cast<uint32_t *>(codes_row + (e >> 1)) = c;
                else *reinterpret_cast<uint16_t *>(codes_row + (e >> 1)) = (uint16_t)c;
                if (lane % SHARE == 0) scales_row[e >> 5] = (uint8_t)byte;
            };
            if constexpr (ROUTED) {
                for (int j = 0; j < top; j++) {
                    if (j % 32 == 0) mine = j + lane < top ? row_of[r * top + j + lane] : -1;
                    const int row = __shfl_sync(~0u, mine, j % 32);
                    if (row >= 0 && row < nvec) write(codes + (size_t)row * ldq, scales + (size_t)row * lds);
                }
            } else write(codes + z * plane_q + r * ldq, scales + z * plane_s + r * lds);
        }
    }
    if constexpr (ROUTED) {
        const long long slots = (long long)tokens * top;
        const int blocks = (len + 31) / 32;
        for (long long r0 = ((long long)blockIdx.x * 8 + warp) * 32; r0 < nvec; r0 += (long long)gridDim.x * 256) {
            const int s = r0 + lane < nvec ? slot_of[r0 + lane] : 0;
            uint32_t none = __ballot_sync(~0u, s < 0 || s >= slots);
            while (none) {
                const long long r = r0 + __ffs(none) - 1;
                none &= none - 1;
                for (int b = lane; b < blocks; b += 32) {
                    *reinterpret_cast<uint4 *>(codes + r * ldq + b * 16) = make_uint4(0, 0, 0, 0);
                    scales[r * lds + b] = 0;
                }
            }
        }
    }
}

// Blocks down the columns of a row-major X (len x nvec): vector c is column c, and comes out as a row. A block of threads takes 256
// rows of 64 (FP32) or 128 columns: warp w holds rows 32w .. 32w+31, 8 bytes of columns to a lane (single columns are loaded one by
// one where groups are not aligned, two to a lane), in registers, so that a lane has a whole block of each of its columns and 32
// loads of 256 contiguous bytes are in flight to a warp (with 4 bytes to a lane 16-bit matrices came at 4.0 TB/s where FP32 ones
// reached 6.5). The codes turn through shared memory into 128 contiguous bytes for each column.
constexpr int CT_ROWS = 256, CT_PITCH = 128 + 16;
template <class T, bool VEC> struct Columns { static constexpr int LANE = VEC ? 8 / (int)sizeof(T) : 2, TILE = 32 * LANE; };
template <class T, bool VEC>
__global__ void __launch_bounds__(256) mx4_cols(const T *X, int nvec, int len, long long ldx, size_t plane_x, int rule, const int *slots,
                                                int top, int tokens, uint8_t *codes, long long ldq, size_t plane_q, uint8_t *scales,
                                                long long lds, size_t plane_s, int col_tiles, int row_tiles) {
    behind_predecessors();
    constexpr int L = Columns<T, VEC>::LANE, TILE = Columns<T, VEC>::TILE;
    __shared__ __align__(16) uint8_t tile[TILE * CT_PITCH];
    __shared__ __align__(8) uint8_t stile[TILE * 8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long b = blockIdx.x;
    const int ct = (int)(b % col_tiles);
    b /= col_tiles;
    const int rt = (int)(b % row_tiles), z = (int)(b / row_tiles);
    const int c = ct * TILE + L * lane, k0 = rt * CT_ROWS + warp * 32;
    X += (size_t)z * plane_x;
    codes += (size_t)z * plane_q;
    scales += (size_t)z * plane_s;
    struct alignas(L * sizeof(T)) Group { T t[L]; };
    Group v[32];
    // Every load is made, from a place that exists, and what was not there is cleared behind them: under a condition each they would
    // wait for one another (a tile took the latency of 32 loads, 40 us where 8 are enough).
    const long long mine = k0 + lane < len ? source_row(slots, top, tokens, k0 + lane) : -1;
#pragma unroll
    for (int i = 0; i < 32; i++) {
        const T *x = X + (size_t)max(__shfl_sync(~0u, mine, i), 0ll) * ldx;
        if constexpr (VEC) v[i] = *reinterpret_cast<const Group *>(x + (c < nvec ? c : 0));   // whole groups of columns
        else
#pragma unroll
            for (int g = 0; g < L; g++) v[i].t[g] = x[min(c + g, nvec - 1)];
    }
    const uint32_t rows = __ballot_sync(~0u, mine >= 0);
#pragma unroll
    for (int g = 0; g < L; g++) {
        float f[32];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; i++) {
            f[i] = rows >> i & 1 ? to_f32<T>(v[i].t[g]) : 0.f;
            m = max(m, magnitude(f[i]));
        }
        const uint32_t byte = scale_byte(m, rule), number = byte == 255 ? 0u : ~0u;
        const float inv = inverse_scale(byte);
#pragma unroll
        for (int i = 0; i < 32; i++) f[i] *= inv;
        *reinterpret_cast<uint4 *>(tile + (L * lane + g) * CT_PITCH + warp * 16) =
            make_uint4(codes_of(f) & number, codes_of(f + 8) & number, codes_of(f + 16) & number, codes_of(f + 24) & number);
        stile[(L * lane + g) * 8 + warp] = (uint8_t)byte;
    }
    __syncthreads();
    const int blocks = (len + 31) / 32, kb = rt * 8;   // blocks of a column, and this tile's first
#pragma unroll
    for (int i = 0; i < TILE * 8 / 256; i++) {
        const int col = i * 32 + (threadIdx.x >> 3), blk = threadIdx.x & 7, g = ct * TILE + col;
        if (g < nvec && kb + blk < blocks)
            *reinterpret_cast<uint4 *>(codes + (size_t)g * ldq + (size_t)(kb + blk) * 16) = *reinterpret_cast<const uint4 *>(tile + col * CT_PITCH + blk * 16);
    }
    if (threadIdx.x < TILE && ct * TILE + (int)threadIdx.x < nvec) {
        uint8_t *dst = scales + (size_t)(ct * TILE + threadIdx.x) * lds + kb;
        if (kb + 8 <= blocks) *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(stile + threadIdx.x * 8);
        else for (int i = 0; kb + i < blocks; i++) dst[i] = stile[threadIdx.x * 8 + i];
    }
}

// Codes and scales back to values. Every product of a code's value and a power of two is exact in FP32 (or an infinity); T rounds it
// once (FP16 may overflow or lose small values, BF16 does not lose any). Where rows start and end on 16 bytes a lane stores 16 bytes
// beside its neighbours', four of them from loads in flight together; else a warp turns 512 values through shared memory, so that
// single values are stored side by side.
template <class T, bool VEC>
__global__ void __launch_bounds__(256) mx4_values(const uint8_t *codes, long long ldq, const uint8_t *scales, long long lds, int nvec, int len,
                                                  T *Y, long long ldy) {
    behind_predecessors();
    __shared__ float turn[VEC ? 1 : 8][32 * 17];
    constexpr int N = Vec16<T>::N, LOAD = VEC ? 32 * N : 512, PIECE = VEC ? LOAD * UNITS : LOAD;
    const int lane = threadIdx.x & 31;
    const uint32_t pieces = (len + PIECE - 1) / PIECE;
    const long long total = (long long)nvec * pieces;
    for (long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); w < total; w += (long long)gridDim.x * 8) {
        const long long r = total < 0x80000000ll ? (long long)((uint32_t)w / pieces) : w / pieces;
        const int at = (int)(w - r * pieces) * PIECE;
        T *y = Y + r * ldy;
        const uint8_t *c = codes + r * ldq, *s = scales + r * lds;
        if constexpr (VEC) {
            uint32_t q[UNITS];
            uint8_t b[UNITS];
#pragma unroll
            for (int u = 0; u < UNITS; u++) {
                const int e = min(at + u * LOAD + lane * N, len - N);
                // four codes: the half of an aligned word that holds them
                q[u] = *reinterpret_cast<const uint32_t *>(c + ((e >> 1) & ~3)) >> (N == 8 ? 0 : 4 * (e & 4));
                b[u] = s[e >> 5];
            }
#pragma unroll
            for (int u = 0; u < UNITS; u++) {
                const int e = at + u * LOAD + lane * N;
                float v[N];
                values_of<N>(q[u], v);
#pragma unroll
                for (int i = 0; i < N; i++) v[i] *= scale_of(b[u]);
                if (e < len) *reinterpret_cast<uint4 *>(y + e) = Vec16<T>::pack(v);
            }
        } else {
            const int i0 = at + lane * 16;
            float v[16];
            if (i0 < len) {
                const uint2 q = *reinterpret_cast<const uint2 *>(c + (i0 >> 1));
                const float scale = scale_of(s[i0 >> 5]);
                values_of<8>(q.x, v);
                values_of<8>(q.y, v + 8);
#pragma unroll
                for (int i = 0; i < 16; i++) v[i] *= scale;
            }
            float *mine = turn[threadIdx.x >> 5];
#pragma unroll
            for (int i = 0; i < 16; i++) mine[lane * 17 + i] = v[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int e = i * 32 + lane;
                if (at + e < len) y[at + e] = from_f32<T>(mine[e + (e >> 4)]);
            }
            __syncwarp();
        }
    }
}

int warp_grid(long long warps) {   // eight warps to a block, at most 2^20 blocks (the kernels stride)
    const long long blocks = (warps + 7) / 8;
    return (int)(blocks < (1 << 20) ? blocks : (1 << 20));
}

}  // namespace

cudaError_t mx4_quantize_rows(const void *X, int type, int nvec, int len, long long ldx, size_t plane_x, int planes, int rule, const int *rows,
                              const int *slots, int top, int tokens, uint8_t *codes, long long ldq, size_t plane_q, uint8_t *scales, long long lds,
                              size_t plane_s, cudaStream_t st) {
    const int size = type_size(type);
    const bool vec = !(reinterpret_cast<uintptr_t>(X) & 15) && !(ldx * size & 15) && !(plane_x * size & 15) && !((long long)len * size & 15);
    const long long vectors = slots ? tokens : (long long)planes * nvec;
    const int load = 512 / size;   // values that a warp loads at a time
    const bool few = vectors * ((len + load - 1) / load) < 16LL * multiprocessors();   // loads in all
    const int unit = few ? load : load * UNITS;
    const int grid = warp_grid(vectors * ((len + unit - 1) / unit) + (slots ? nvec / 32 : 0));
    cudaError_t e = cudaErrorInvalidValue;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto vec_, auto routed_) {
            constexpr bool v = decltype(vec_)::value, r = decltype(routed_)::value;
            // Four loads in flight to a warp, or one where there are few. BF16 in us, four : one: (16, 4096) 2.1 : 1.4, (128, 4096) 2.15 : 1.7,
            // (1024, 4096) 4.0 : 4.2, (2048, 7168) 8.5 : 11.3; between 16 and 64 loads to an SM, where it is four, one would be the shorter:
            // (512, 4096) 3.4 : 2.7.
            e = few ? launch_behind(mx4_rows<T, v, r, 1>, grid, 256, 0, 1, st, (const T *)X, nvec, len, ldx, plane_x, planes, rule, rows, slots, top, tokens, codes, ldq,
                                    plane_q, scales, lds, plane_s)
                    : launch_behind(mx4_rows<T, v, r, UNITS>, grid, 256, 0, 1, st, (const T *)X, nvec, len, ldx, plane_x, planes, rule, rows, slots, top, tokens, codes,
                                    ldq, plane_q, scales, lds, plane_s);
        };
        if (vec && slots) go(std::true_type(), std::true_type());
        else if (vec) go(std::true_type(), std::false_type());
        else if (slots) go(std::false_type(), std::true_type());
        else go(std::false_type(), std::false_type());
    });
    return e;
}

cudaError_t mx4_quantize_cols(const void *X, int type, int nvec, int len, long long ldx, size_t plane_x, int planes, int rule, const int *,
                              const int *slots, int top, int tokens, uint8_t *codes, long long ldq, size_t plane_q, uint8_t *scales, long long lds,
                              size_t plane_s, cudaStream_t st) {
    const int size = type_size(type);
    const int group = 8 / size;
    const bool vec = !(reinterpret_cast<uintptr_t>(X) & 7) && !((ldx | nvec) % group) && !(plane_x % group);
    const int tile = 32 * (vec ? group : 2);   // columns of a block
    const int col_tiles = (nvec + tile - 1) / tile, row_tiles = (len + CT_ROWS - 1) / CT_ROWS;
    const long long grid = (long long)col_tiles * row_tiles * planes;
    if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
    cudaError_t e = cudaErrorInvalidValue;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        e = launch_behind(vec ? mx4_cols<T, true> : mx4_cols<T, false>, (int)grid, 256, 0, 1, st, (const T *)X, nvec, len, ldx, plane_x, rule, slots, top, tokens, codes, ldq,
                          plane_q, scales, lds, plane_s, col_tiles, row_tiles);
    });
    return e;
}

cudaError_t mx4_dequantize(const uint8_t *codes, long long ldq, const uint8_t *scales, long long lds, int nvec, int len, void *Y, int type,
                           long long ldy, cudaStream_t st) {
    const int size = type_size(type);
    const bool vec = !(reinterpret_cast<uintptr_t>(Y) & 15) && !(ldy * size & 15) && !((long long)len * size & 15);
    cudaError_t e = cudaErrorInvalidValue;
    const int piece = vec ? 512 / size * UNITS : 512;   // values that a warp takes at a time
    const int grid = warp_grid((long long)nvec * ((len + piece - 1) / piece));
    with_type(type, [&](auto t) {
        using T = decltype(t);
        e = launch_behind(vec ? mx4_values<T, true> : mx4_values<T, false>, grid, 256, 0, 1, st, codes, ldq, scales, lds, nvec, len, (T *)Y, ldy);
    });
    return e;
}

}  // namespace ozk
