// Rows of fp16, bf16 or fp32 as fp32 numbers, eight at a time.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace tcb {
namespace io {

template <typename T> constexpr bool kIsHalf = false;
template <> constexpr bool kIsHalf<__half> = true;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }

// Eight elements as they lie in memory.
template <typename T> struct Pack8 { uint4 w[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ Pack8<T> load8(const T* p) {
    Pack8<T> r;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Pack8<T>& r) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}
template <typename T> __device__ __forceinline__ void unpack8(const Pack8<T>& r, float (&f)[8]) {
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f<T>(e[i]);
}
template <typename T> __device__ __forceinline__ Pack8<T> pack8(const float (&f)[8]) {
    Pack8<T> r;
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f<T>(f[i]);
    return r;
}

}  // namespace io
}  // namespace tcb
