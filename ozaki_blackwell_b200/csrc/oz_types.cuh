// oz_types.cuh -- the element types of the low-bit and expert operators (OZB_F32, OZB_BF16, OZB_F16 of ozb.h) on the device.
#pragma once
#include <cstdint>
#include <cstring>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace ozk {

template <class T> struct IsHalf { static constexpr bool value = false; };
template <> struct IsHalf<__half> { static constexpr bool value = true; };

template <class T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

template <class T> __device__ __forceinline__ T from_f32(float x);   // round to nearest even
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// 16 bytes of T as floats and back. The 16-bit types go two at a time: a conversion of one value runs at a quarter of the rate of the
// packed instruction.
template <class T> struct Vec16 {
    static constexpr int N = 16 / (int)sizeof(T);
    static __device__ __forceinline__ float2 two(uint32_t w) {
        if constexpr (sizeof(T) == 2 && !IsHalf<T>::value) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        else {
            __half2 p;
            memcpy(&p, &w, 4);
            return __half22float2(p);
        }
    }
    static __device__ __forceinline__ uint32_t word(float a, float b) {
        uint32_t w;
        if constexpr (IsHalf<T>::value) {
            const __half2 p = __floats2half2_rn(a, b);
            memcpy(&w, &p, 4);
        } else {
            const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
            memcpy(&w, &p, 4);
        }
        return w;
    }
    static __device__ __forceinline__ void unpack(const uint4 &q, float *f) {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) f[i] = __uint_as_float(w[i]);
            else {
                const float2 v = two(w[i]);
                f[2 * i] = v.x;
                f[2 * i + 1] = v.y;
            }
        }
    }
    static __device__ __forceinline__ uint4 pack(const float *f) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
            else w[i] = word(f[2 * i], f[2 * i + 1]);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// runs f with a value of the element type that `type` names; false if it names none
template <class F> bool with_type(int type, F &&f) {
    switch (type) {
    case 0: f(float()); return true;
    case 1: f(__nv_bfloat16()); return true;
    case 2: f(__half()); return true;
    default: return false;
    }
}
inline int type_size(int type) { return type == 0 ? 4 : 2; }

}  // namespace ozk
