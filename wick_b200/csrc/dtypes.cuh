// Element types of the operators that take more than f32 (ggml type ids, wick/src/gguf.rs:36-46).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace wick {

constexpr int DT_F32 = 0, DT_F16 = 1, DT_BF16 = 30;

__host__ __device__ inline int dtype_bytes(int dtype) { return dtype == DT_F32 ? 4 : dtype == DT_F16 || dtype == DT_BF16 ? 2 : 0; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The elements of one 16-byte load, as f32.
__device__ __forceinline__ void unpack16(uint4 w, float (&x)[4], const float*) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void unpack16(uint4 w, float (&x)[8], const __half*) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack16(uint4 w, float (&x)[8], const __nv_bfloat16*) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) x[2 * i] = __uint_as_float(u[i] << 16), x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
}

}  // namespace wick
