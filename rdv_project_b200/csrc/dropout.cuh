// Dropout whose mask comes from a counter and is never stored: element i is
// kept iff word i % 4 of the Philox 4x32 block with ten rounds at counter
// offset + i / 4 and key seed is at least round(p 2^32) (Salmon, Moraes,
// Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011). The
// same call on an output gradient is the backward pass.
//
// One pass over the data, 16 bytes a thread and access. Nothing is full: of the
// issue slots 65 % are taken, and of the pipe of wide integer products 67 %
// (19 32 x 32 -> 64-bit multiplications and 20 three-way xors a block of four
// elements, the latter on a pipe 55 % busy; the rounds' keys come from the
// host), of DRAM's rate 26 %. 33.5 M bfloat16 elements take 46 us with a
// residual (memory 31) and 40 us without (21).
#pragma once
#include <cstdint>

#include "types.cuh"

namespace rdvb {
namespace dropout {

constexpr int kThreads = 256;

__device__ __forceinline__ uint4 philox(uint64_t counter, const uint2 (&key)[10]) {
    uint4 c = make_uint4(static_cast<uint32_t>(counter), static_cast<uint32_t>(counter >> 32), 0u, 0u);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = static_cast<uint64_t>(c.x) * 0xD2511F53u;
        const uint64_t b = static_cast<uint64_t>(c.z) * 0xCD9E8D57u;
        c = make_uint4(static_cast<uint32_t>(b >> 32) ^ c.y ^ key[r].x, static_cast<uint32_t>(b),
                       static_cast<uint32_t>(a >> 32) ^ c.w ^ key[r].y, static_cast<uint32_t>(a));
    }
    return c;
}

struct Params {
    const void* x;
    const void* residual;  // may be null
    void* y;
    int64_t n;
    uint64_t offset;
    uint2 key[10];       // of each round
    uint32_t threshold;  // kept iff word >= threshold
    float scale;         // 1 / (1 - p)
};

// kWide: x, residual and y are 16-byte aligned. A thread owns the elements
// of one 16-byte vector: one block of the generator for float32, two for the
// 16-bit types. A dropped element is selected to 0, so an infinite or NaN x
// does not pass the mask. The product and the residual's addition are in
// float32 and rounded once.
template <typename T, bool kWide, bool kResidual>
__global__ void __launch_bounds__(kThreads) dropout_kernel(const Params p) {
    constexpr int kVec = 16 / sizeof(T);
    const int64_t i0 = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kVec;
    if (i0 >= p.n) return;
    const T* from = static_cast<const T*>(p.x) + i0;
    const T* add = static_cast<const T*>(p.residual) + i0;
    T* to = static_cast<T*>(p.y) + i0;
    const bool whole = kWide && i0 + kVec <= p.n;
    Vec<T, kVec> x, res, y;
    if (whole) {
        x = *reinterpret_cast<const Vec<T, kVec>*>(from);
        if (kResidual) res = *reinterpret_cast<const Vec<T, kVec>*>(add);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (i0 + i < p.n) {
                x.v[i] = from[i];
                if (kResidual) res.v[i] = add[i];
            }
    }
#pragma unroll
    for (int b = 0; b < kVec / 4; ++b) {
        const uint4 w = philox(p.offset + static_cast<uint64_t>(i0 / 4 + b), p.key);
        const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float kept = word[i] >= p.threshold ? to_f32<T>(x.v[4 * b + i]) * p.scale : 0.0f;
            y.v[4 * b + i] = from_f32<T>(kResidual ? kept + to_f32<T>(res.v[4 * b + i]) : kept);
        }
    }
    if (whole) {
        *reinterpret_cast<Vec<T, kVec>*>(to) = y;
    } else {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (i0 + i < p.n) to[i] = y.v[i];
    }
}

}  // namespace dropout
}  // namespace rdvb
