// oz_types.cuh -- the element types of the low-bit and expert operators (OZB_F32, OZB_BF16, OZB_F16 of ozb.h) on the device.
#pragma once
#include <cstdint>
#include <cstring>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace ozk {

template <class T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

template <class T> __device__ __forceinline__ T from_f32(float x);   // round to nearest even
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// 16 bytes of T as floats and back
template <class T> struct Vec16 {
    static constexpr int N = 16 / (int)sizeof(T);
    static __device__ __forceinline__ void unpack(const uint4 &q, float *f) {
        T t[N];
        memcpy(t, &q, 16);
#pragma unroll
        for (int i = 0; i < N; i++) f[i] = to_f32<T>(t[i]);
    }
    static __device__ __forceinline__ uint4 pack(const float *f) {
        T t[N];
#pragma unroll
        for (int i = 0; i < N; i++) t[i] = from_f32<T>(f[i]);
        uint4 q;
        memcpy(&q, t, 16);
        return q;
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
