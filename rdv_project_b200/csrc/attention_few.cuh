// Attention of a few query rows (attention.cuh has the mathematics): at most
// eight rows share a key head (positions times query heads a key head), as
// when a position at a time is served. Every element type.
//
// Bound: memory up to two rows (5.8 TB/s); at four the conversions, sums and
// exchanges of a key's rows in three warps a scheduler (4.4 TB/s: 0.63 of the
// issue slots, 57 % of DRAM). A key's dimensions lie along a group of lanes, 16
// bytes each; a warp's step is kUnroll keys a group, K and V at once, copied to
// shared memory by the lanes that read them, kStages steps in flight beside the
// sums of the oldest; no lane reads what another copied, so there is no barrier.
// Partial products of kUnroll keys are summed over the lanes in one exchange
// that leaves each lane one key's score. Every group of lanes keeps its own
// maximum, sum and output row; groups are joined at the end in order, blocks
// (splits of the keys) by join_forward_kernel.
#pragma once
#include <cstdint>

#include "attention.cuh"
#include "attention_tc.cuh"

namespace rdvb {
namespace attn {

constexpr int kFewThreads = 128, kFewWarps = kFewThreads / 32, kFewRows = 8;

// (c0, c1) += (a0 b0, a1 b1) in one packed instruction.
__device__ __forceinline__ void fma_f32x2_acc(float& c0, float& c1, float a0, float a1, float b0, float b1) {
    fma2(a0, a1, b0, b1, c0, c1);
    c0 = a0;
    c1 = a1;
}

template <typename T, int kLanes, int kRows>
struct Few {
    static constexpr int kVec = 16 / sizeof(T);            // dimensions a lane
    static constexpr int kUnroll = kRows > 4 ? 4 : 8;      // keys of a group's step
    static constexpr int kGroups = 32 / kLanes;            // groups of a warp
    static constexpr int kBlock = kGroups * kUnroll;       // keys of a warp's step
    static constexpr int kStages = kRows > 4 ? 4 : 2;      // steps of a warp in flight
    static constexpr int kStage = 2 * kUnroll * 32;        // pieces of 16 bytes: a lane's of each key, then value
    static constexpr int kBytes = kFewWarps * kStages * kStage * 16;
};

// 16 bytes to shared memory while the thread goes on; zeros, and nothing read, where !ok.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool ok) {
    const int bytes = ok ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// Registers and stages for three blocks a processor up to four rows (100003
// states, 4 samples, 16 heads of 128 over 4, float16, with the join: 188 us over
// inputs in turn. Over one input again, whose end is still in L2: 171 us; two
// blocks with three stages 185 us, steps of four keys in three blocks with four
// stages 191 us, in four with three 195 us; loads straight to registers, which
// wait for the sums, 211 us).
template <typename T, int kLanes, int kRows>
__global__ void __launch_bounds__(kFewThreads, kRows > 4 ? 2 : 3) few_kernel(const Params p) {
    using F = Few<T, kLanes, kRows>;
    constexpr int kVec = F::kVec, kU = F::kUnroll;
    static_assert(kLanes >= kU, "a score a lane");
    uint32_t id = blockIdx.x;
    const int split = id % p.splits;
    id /= p.splits;
    const int hk = id % p.kv_heads, b = id / p.kv_heads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane % kLanes, group = lane / kLanes;
    const int rows = static_cast<int>(p.q_len) * p.group;
    const bool in = sub * kVec < p.dim;
    const int64_t len = length_of(p, b);
    const int64_t begin = split * p.split_len, end = min(len, begin + p.split_len);
    const float c = p.scale * kLog2e;

    // queries, scaled so that scores are powers of two's exponents
    float q[kRows][kVec], acc[kRows][kVec] = {}, top[kRows], total[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        top[r] = -INFINITY;
        total[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < kVec; ++i) q[r][i] = 0.0f;
        if (in && r < rows) {
            const int64_t at = b * p.qs.batch + (r / p.group) * p.qs.pos + (hk * p.group + r % p.group) * p.qs.head;
            load_f32<T, kVec>(static_cast<const T*>(p.q) + at + sub * kVec, q[r]);
#pragma unroll
            for (int i = 0; i < kVec; ++i) q[r][i] *= c;
        }
    }
    const T* k_base = static_cast<const T*>(p.k) + b * p.ks.batch + hk * p.ks.head + sub * kVec;
    const T* v_base = static_cast<const T*>(p.v) + b * p.vs.batch + hk * p.vs.head + sub * kVec;
    const uint8_t* mask = p.mask ? p.mask + b * p.mask_stride : nullptr;
    // The key whose score this lane holds after the exchange: its group's
    // `mine`-th. Bit i of it is lane bit log2(kLanes) - 1 - i.
    int mine = 0;
#pragma unroll
    for (int i = 0, half = kLanes / 2; (1 << i) < kU; ++i, half /= 2) mine |= (sub & half ? 1 : 0) << i;
    bool any = false;

    // A lane reads only the pieces that it copied, so its own waits are all that the stages need.
    extern __shared__ uint4 few_stages[];
    uint4* const stages = few_stages + warp * F::kStages * F::kStage + lane;
    const uint32_t stages_at = static_cast<uint32_t>(__cvta_generic_to_shared(stages));
    constexpr int64_t kStep = kFewWarps * F::kBlock;
    // Which of the keys of the step from k0 this group may read.
    auto allowed = [&](int64_t k0) -> uint32_t {
        uint32_t on = 0;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int64_t key = k0 + u * F::kGroups + group;
            on |= static_cast<uint32_t>(key < end && (!mask || mask[key] != 0)) << u;
        }
        return on;
    };
    // A key that is not allowed is not read: zeros stand for it.
    auto fetch = [&](int64_t k0, uint32_t on, int stage) {
        if (k0 < end) {
            const int64_t key = k0 + group;
            const T *k = k_base + key * p.ks.pos, *v = v_base + key * p.vs.pos;
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const bool ok = in && (on >> u & 1u);
                const uint32_t to = stages_at + (stage * F::kStage + u * 32) * 16;
                copy16(to, ok ? k + u * F::kGroups * p.ks.pos : k_base, ok);
                copy16(to + kU * 512, ok ? v + u * F::kGroups * p.vs.pos : v_base, ok);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int64_t k0 = begin + warp * F::kBlock;
    uint32_t queue = 0;  // the allowed keys of the steps in flight, the oldest lowest
#pragma unroll
    for (int i = 0; i < F::kStages; ++i) {
        const uint32_t on = allowed(k0 + i * kStep);
        fetch(k0 + i * kStep, on, i);
        queue |= on << i * kU;
    }
    for (int stage = 0; k0 < end; k0 += kStep, stage = stage + 1 == F::kStages ? 0 : stage + 1) {
        const uint32_t on = queue & ((1u << kU) - 1), later = allowed(k0 + F::kStages * kStep);
        queue = queue >> kU | later << (F::kStages - 1) * kU;
        asm volatile("cp.async.wait_group %0;" ::"n"(F::kStages - 1) : "memory");
        if (!__any_sync(0xffffffffu, on != 0)) {
            fetch(k0 + F::kStages * kStep, later, stage);
            continue;
        }
        any |= on != 0;
        const uint4* at = stages + stage * F::kStage;
        float s[kU][kRows];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float x[kVec];
            load_f32<T, kVec>(reinterpret_cast<const T*>(at + u * 32), x);
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                float s0 = q[r][0] * x[0], s1 = q[r][1] * x[1];
#pragma unroll
                for (int i = 2; i < kVec; i += 2) fma_f32x2_acc(s0, s1, q[r][i], q[r][i + 1], x[i], x[i + 1]);
                s[u][r] = s0 + s1;
            }
        }
        // sum over the group's lanes: each exchange halves the keys a lane holds
#pragma unroll
        for (int half = kLanes / 2, step = 1; half > 0; half /= 2, step *= 2) {
            if (step < kU) {
                const bool upper = (sub & half) != 0;
#pragma unroll
                for (int u = 0; u < kU; u += 2 * step)
#pragma unroll
                    for (int r = 0; r < kRows; ++r) {
                        const float give = upper ? s[u][r] : s[u + step][r], keep = upper ? s[u + step][r] : s[u][r];
                        s[u][r] = keep + __shfl_xor_sync(0xffffffffu, give, half);
                    }
            } else {
#pragma unroll
                for (int r = 0; r < kRows; ++r) s[0][r] += __shfl_xor_sync(0xffffffffu, s[0][r], half);
            }
        }
        const bool here = on >> mine & 1u;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            // the group's maximum over its keys: across the lanes that tell keys apart
            float m = here ? s[0][r] : -INFINITY;
#pragma unroll
            for (int half = kLanes / 2, step = 1; step < kU; half /= 2, step *= 2)
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, half));
            m = fmaxf(m, top[r]);
            const float base = m == -INFINITY ? 0.0f : m;
            const float old = exp2f(top[r] - base);
            const float e = here ? exp2f(s[0][r] - base) : 0.0f;
            top[r] = m;
            total[r] *= old;
#pragma unroll
            for (int i = 0; i < kVec; ++i) acc[r][i] *= old;
            s[0][r] = e;
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float x[kVec];
            load_f32<T, kVec>(reinterpret_cast<const T*>(at + (kU + u) * 32), x);
            // the lane of this group that holds key u
            int from = 0;
#pragma unroll
            for (int i = 0, half = kLanes / 2; (1 << i) < kU; ++i, half /= 2) from |= (u >> i & 1) * half;
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const float e = __shfl_sync(0xffffffffu, s[0][r], group * kLanes + from);
                total[r] += e;
#pragma unroll
                for (int i = 0; i < kVec; i += 2) fma_f32x2_acc(acc[r][i], acc[r][i + 1], e, e, x[i], x[i + 1]);
            }
        }
        fetch(k0 + F::kStages * kStep, later, stage);
    }

    // Joins the block's groups, in order.
    constexpr int kParts = kFewWarps * F::kGroups;
    __shared__ float s_acc[kParts][kLanes * kVec + 1];
    __shared__ float s_top[kParts][kRows], s_total[kParts][kRows];
    const bool seen = __syncthreads_or(any);
    const int part = warp * F::kGroups + group;
    if (sub == 0) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) s_top[part][r] = top[r], s_total[part][r] = total[r];
    }
    const int64_t all_rows = static_cast<int64_t>(p.batch) * p.q_len * p.heads;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (r >= rows) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kVec; ++i) s_acc[part][sub * kVec + i] = acc[r][i];
        __syncthreads();
        float m = -INFINITY, l = 0.0f;
        for (int i = 0; i < kParts; ++i) m = fmaxf(m, s_top[i][r]);
        const float base = m == -INFINITY ? 0.0f : m;
        for (int i = 0; i < kParts; ++i) l = fmaf(s_total[i][r], exp2f(s_top[i][r] - base), l);
        const int64_t pos = r / p.group, h = hk * p.group + r % p.group;
        const int64_t row = (b * p.q_len + pos) * p.heads + h;
        for (int d = threadIdx.x; d < p.dim; d += kFewThreads) {
            float o = 0.0f;
            for (int i = 0; i < kParts; ++i) o = fmaf(s_acc[i][d], exp2f(s_top[i][r] - base), o);
            if (p.splits > 1)
                p.part[(split * all_rows + row) * p.dim + d] = seen ? o : 0.0f;
            else
                static_cast<T*>(p.o)[row * p.dim + d] = from_f32<T>(seen ? o / l : 0.0f);
        }
        if (threadIdx.x == 0) {
            if (p.splits > 1) {
                p.part_stat[2 * (split * all_rows + row)] = m;
                p.part_stat[2 * (split * all_rows + row) + 1] = seen ? l : -1.0f;
            } else if (p.lse) {
                p.lse[(static_cast<int64_t>(b) * p.heads + h) * p.q_len + pos] =
                    seen ? (base + log2f(l)) * kLn2 : -INFINITY;
            }
        }
    }
}

}  // namespace attn
}  // namespace rdvb
