// Element types of the operators that take float32, float16 and bfloat16
// alike: 16-byte vector loads and stores with arithmetic in float32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace rdvb {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// Two float32 operations in one packed instruction (sm_100): (a0, a1) op
// (b0, b1) into the first pair, and a b + c.
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y));
    return p;
}
__device__ __forceinline__ void add2(float& a0, float& a1, float b0, float b1) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_of(a0, a1)), "l"(pair_of(b0, b1)));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(d));
}
__device__ __forceinline__ void mul2(float& a0, float& a1, float b0, float b1) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_of(a0, a1)), "l"(pair_of(b0, b1)));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(d));
}
__device__ __forceinline__ void fma2(float& a0, float& a1, float b0, float b1, float c0, float c1) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair_of(a0, a1)), "l"(pair_of(b0, b1)), "l"(pair_of(c0, c1)));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(d));
}

// N consecutive elements moved as one access (N * sizeof(T) is 1 to 16 bytes
// and the address a multiple of it).
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_f32(const T* p, float (&out)[N]) {
    const Vec<T, N> a = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = to_f32<T>(a.v[i]);
}

template <typename T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&in)[N]) {
    Vec<T, N> a;
#pragma unroll
    for (int i = 0; i < N; ++i) a.v[i] = from_f32<T>(in[i]);
    *reinterpret_cast<Vec<T, N>*>(p) = a;
}

}  // namespace rdvb
