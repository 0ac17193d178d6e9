// Gradients of attention on the tensor cores (attention.cuh has the
// mathematics, attention_tc.cuh the tile formats and the conditions).
//
// Two kernels recompute S and dP = dO V^T, so that dQ, dK and dV each have
// one owner and a fixed order of summation: seven products a pair of tiles
// instead of the five of one kernel that adds dQ up in memory, and no
// atomics. Measured (bfloat16): 16384 x 4096, 2 samples of 16 heads of 64, dQ 1294
// and dK, dV 1360 us; 16384 x 4099, 16 heads of 128 over 4, 1478 and 2176 us. Bound:
// a tile's chain of products and exponentials; the tensor pipe is 28 to 51 %
// busy. One block a processor, 512 TMEM columns. Warps 0-7: probabilities
// and score gradients, a thread a row (a lane of TMEM) and half the columns.
// Warp 8: loads. Warp 9: the products S and dP. Warp 11: the products that
// take P and dS. Warp 10: zeroes rows of K whose keys are not allowed (dQ). A
// barrier that its producer could complete twice before a slow reader looked
// (the readers tell phases apart by parity) comes in two, for even and odd
// tiles.
//
// P and dS are rounded to the inputs' type, as the tensor cores take them
// (bfloat16 gradients are 2.4e-3 of their size off, 1.7e-3 of it by their own
// rounding).
// float16 has few exponents: P is held times 2^15 (P <= 1), dS times 2^E with
// the largest E that keeps 2 max|dO| max|V| 2^E <= 2^15, a bound of |dS|, so
// that gradients keep their digits whatever the loss was scaled by.
#pragma once
#include <cstdint>
#include <type_traits>

#include "attention_tc.cuh"

namespace rdvb {
namespace attn {

constexpr int kGradThreads = 12 * 32;
constexpr int kPrepBlocks = 592;
constexpr int kGradPoly = 1;  // of four pairs of exponentials, those taken by the polynomial

struct GradParams {
    Params a;
    uint32_t* status;
    float* neg_lse;    // [batch, heads, q_pad]: -lse log2 e; -inf past q_len
    float* neg_delta;  // [batch, heads, q_pad]: -rowsum(dO O); 0 past q_len
    float2* norms;     // [kPrepBlocks]: largest |dO|^2 and |V|^2 of a row (float16)
    float* slips;      // [splits of dQ, batch, heads, q_pad]: a split's sum of dS; splits > 1
    int64_t q_pad;     // q_len rounded up to whole tiles
    uint32_t k_steps, n_pv;
    int guarded;
};

// neg_lse, neg_delta and norms: kLanes lanes a row of 16 bytes each, four
// rows of dO and O in flight a thread. A warp takes consecutive positions of
// one head, so that what it writes lies together. Bound: memory.
template <int kLanes, bool kBf16>
__global__ void __launch_bounds__(kThreads) tc_prep_kernel(const GradParams p) {
    constexpr int kFlight = 4, kGroups = 32 / kLanes, kChunk = kFlight * kGroups;  // rows of a warp's step
    const Params& a = p.a;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, group = lane / kLanes;
    auto load8 = [&](const void* src, int64_t at, float (&v)[8]) {
        if (kBf16)
            load_f32<__nv_bfloat16, 8>(static_cast<const __nv_bfloat16*>(src) + at, v);
        else
            load_f32<__half, 8>(static_cast<const __half*>(src) + at, v);
    };
    const bool in = sub * 8 < a.dim;
    const uint32_t per_head = static_cast<uint32_t>(p.q_pad / kChunk);
    const int64_t chunks = static_cast<int64_t>(a.batch) * a.heads * per_head;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
    float most_do = 0.0f, most_v = 0.0f;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads / 32) + threadIdx.x / 32; i < chunks; i += warps) {
        const int64_t head = i / per_head, q0 = (i - head * per_head) * kChunk + group;  // of all samples' heads
        const int64_t b = head / a.heads, h = head - b * a.heads;
        uint4 raw_o[kFlight], raw_g[kFlight];
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            const int64_t q = q0 + j * kGroups;
            const int64_t at = ((b * a.q_len + q) * a.heads + h) * a.dim + sub * 8;
            raw_o[j] = raw_g[j] = make_uint4(0, 0, 0, 0);
            if (q < a.q_len && in) {
                raw_o[j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.out) + at));
                raw_g[j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.dout) + at));
            }
        }
#pragma unroll
        for (int j = 0; j < kFlight; ++j) {
            float o[8], g[8], dot = 0.0f, norm = 0.0f;
            load8(&raw_o[j], 0, o);
            load8(&raw_g[j], 0, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                dot = fmaf(o[e], g[e], dot);
                norm = fmaf(g[e], g[e], norm);
            }
#pragma unroll
            for (int e = kLanes / 2; e > 0; e >>= 1) {
                dot += __shfl_xor_sync(0xffffffffu, dot, e);
                if (!kBf16) norm += __shfl_xor_sync(0xffffffffu, norm, e);
            }
            const int64_t q = q0 + j * kGroups;
            if (sub == 0) {
                p.neg_delta[head * p.q_pad + q] = -dot;  // 0 past the end
                p.neg_lse[head * p.q_pad + q] = q < a.q_len ? -a.lse[head * a.q_len + q] * kLog2e : -INFINITY;
            }
            if (!kBf16) most_do = fmaxf(most_do, norm);
        }
    }
    if (kBf16) return;
    const int64_t first = (blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x) / kLanes;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kThreads / kLanes);
    const int64_t v_rows = static_cast<int64_t>(a.batch) * a.kv_len * a.kv_heads;
    const int64_t v_rounds = (v_rows + step - 1) / step;
    for (int64_t i = 0; i < v_rounds; ++i) {
        const int64_t row = first + i * step;
        const int64_t h = row % a.kv_heads, key = row / a.kv_heads % a.kv_len, b = row / a.kv_heads / a.kv_len;
        float norm = 0.0f;
        if (row < v_rows && in && allowed(a, static_cast<int>(b), key, length_of(a, static_cast<int>(b)))) {
            float v[8];
            load8(a.v, b * a.vs.batch + key * a.vs.pos + h * a.vs.head + sub * 8, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) norm = fmaf(v[j], v[j], norm);
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) norm += __shfl_xor_sync(0xffffffffu, norm, o);
        most_v = fmaxf(most_v, norm);
    }
    __shared__ float s_most[2][kThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        most_do = fmaxf(most_do, __shfl_xor_sync(0xffffffffu, most_do, o));
        most_v = fmaxf(most_v, __shfl_xor_sync(0xffffffffu, most_v, o));
    }
    if (threadIdx.x % 32 == 0) {
        s_most[0][threadIdx.x / 32] = most_do;
        s_most[1][threadIdx.x / 32] = most_v;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kThreads / 32; ++i) {
            most_do = fmaxf(most_do, s_most[0][i]);
            most_v = fmaxf(most_v, s_most[1][i]);
        }
        p.norms[blockIdx.x] = make_float2(most_do, most_v);
    }
}

// E of dS's factor 2^E; 0 for bfloat16. The same in every thread of a warp.
template <bool kBf16>
__device__ __forceinline__ float grad_exponent(const GradParams& p) {
    if (kBf16) return 0.0f;
    float x = 0.0f, y = 0.0f;
    for (int i = threadIdx.x & 31; i < kPrepBlocks; i += 32) {
        const float2 n = p.norms[i];
        x = fmaxf(x, n.x);
        y = fmaxf(y, n.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, o));
    }
    const float bound = 2.0f * sqrtf(x) * sqrtf(y);
    if (!(bound > 0.0f && bound < INFINITY)) return 0.0f;
    return fminf(fmaxf(floorf(15.0f - log2f(bound)), -100.0f), 100.0f);
}

__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// D += A B with A in TMEM in two halves 64 columns apart (P, dS), B a tile
// of 128 rows taken along them.
__device__ __forceinline__ void product_columns(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool first) {
#pragma unroll
    for (uint32_t j = 0; j < kTcTile / 16; ++j)
        umma_ts(d, a + (j >> 2) * 64 + (j & 3) * 8, b + j * 128, idesc, !first || j > 0);
}

// Stores 16 columns of a gradient row from accumulators: 16-bit, or float32
// parts.
template <bool kBf16>
__device__ __forceinline__ void store_columns(const Params& a, void* out, float* part, int64_t at, int d,
                                              const uint32_t (&r)[16], float f, bool on) {
#pragma unroll
    for (int e = 0; e < 16; e += 8) {
        if (d + e >= a.dim) return;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = on ? __uint_as_float(r[e + k]) * f : 0.0f;
        if (part) {
            *reinterpret_cast<float4*>(part + at + d + e) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(part + at + d + e + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                w[k] = kBf16 ? pack_bf16x2(v[2 * k], v[2 * k + 1]) : pack_f16x2(v[2 * k], v[2 * k + 1]);
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at + d + e) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// ------------------------------------------------------------------------ dQ
//
// An item: 128 query rows of one head over the keys of one split. S has two
// buffers (dS(i) replaces S(i)), dP one: S(i + 1) and dP(i + 1) run beside the
// exponentials of i and dQ(i). A block stays and takes item after item, with
// counters that run on from one to the next; up to 64 dimensions Q, dO and dQ
// have two buffers, so that short key sequences do not wait between items.
//
// delta = rowsum(dO O) comes from the rounded O, which shows where few keys
// matter: dP - delta is then a small difference (of one key: 0). Its exact
// value is sum P dP. Where a sample's keys are one tile, dS is made with that;
// where they are several, the sum of dS, which should be 0, is what delta was
// off by, and the kernel of dK and dV after this one gets delta with it (where
// the keys are split, from tc_slips_kernel, which adds the splits' sums up).
template <int DP>
struct TcDq {
    static constexpr int kAtoms = DP / 64, kKStages = 3, kVStages = 2, kItems = DP == 64 ? 2 : 1;
    static constexpr uint32_t kTileBytes = kTcTile * DP * 2;
    static constexpr uint32_t kOffK = 2 * kItems * kTileBytes, kOffV = kOffK + kKStages * kTileBytes,
                              kOffBar = kOffV + kVStages * kTileBytes;
    static constexpr uint32_t kOffRow = kOffBar + 512;  // a float a half row: sums exchanged by a row's two threads
    static constexpr uint32_t kBytes = kOffRow + 1024 + 1024;
    static constexpr uint32_t kColS = 0, kColDp = 256, kColDq = 384;
};

template <int DP, bool kBf16>
__global__ void __launch_bounds__(kGradThreads, 1)
    tc_dq_kernel(const GradParams p, const uint32_t items, const __grid_constant__ TcMap map_q,
                 const __grid_constant__ TcMap map_k, const __grid_constant__ TcMap map_v,
                 const __grid_constant__ TcMap map_do) {
    using F = TcDq<DP>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t s_q = base, s_k = base + F::kOffK, s_v = base + F::kOffV, bars = base + F::kOffBar;
    // by item (even and odd where there are two buffers), by key tile, by stage
    const uint32_t q_full = bars, q_empty = bars + 16, dq_full = bars + 32, dq_read = bars + 48, dp_full = bars + 64,
                   drain = bars + 72, s_full = bars + 80, ds_full = bars + 96, dq_done = bars + 112,
                   k_tma = bars + 128, k_ok = bars + 152, k_empty = bars + 176, v_full = bars + 200,
                   v_empty = bars + 216;
    const uint32_t tmem_slot = bars + 232, row_pair = bars + 240;
    volatile uint32_t* abort_flag =
        reinterpret_cast<volatile uint32_t*>(smem_raw + (bars - smem_addr(smem_raw)) + 236);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Params& a = p.a;

    if (threadIdx.x == 0) {
        *abort_flag = 0u;
        for (int i = 0; i < 4; ++i) mbar_init(row_pair + 8 * i, 2);
        mbar_init(dp_full, 1);
        mbar_init(drain, 2);  // an arrival an issuing warp
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + 8 * i, 2);  // Q and dO
            mbar_init(q_empty + 8 * i, 1);
            mbar_init(dq_full + 8 * i, 1);
            mbar_init(dq_read + 8 * i, 8);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(ds_full + 8 * i, 8);
            mbar_init(dq_done + 8 * i, 1);
            mbar_init(v_full + 8 * i, 1);
            mbar_init(v_empty + 8 * i, 1);
        }
        for (int i = 0; i < F::kKStages; ++i) {
            mbar_init(k_tma + 8 * i, 1);
            mbar_init(k_ok + 8 * i, 1);
            mbar_init(k_empty + 8 * i, 1);
        }
        fence_mbarrier_init();
    }
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

    if (warp == 8) {
        if (lane == 0) {
            uint32_t n = 0, m = 0, k_sent = 0, v_sent = 0, id = blockIdx.x;  // n: key tiles, m: items so far
            TcItem t;
            bool ok = true;
            for (; ok && next_item<1>(a, items, id, t); id += gridDim.x) {
                const uint32_t slot = m % F::kItems;
                if (!mbar_wait(q_empty + 8 * slot, ((m / F::kItems) & 1) ^ 1, abort_flag, p.status, kStatusTimeoutWEmpty))
                    break;
                ++m;
                tc_load<F::kAtoms>(s_q + 2 * slot * F::kTileBytes, map_q, t.h, t.q0, t.b, q_full + 8 * slot);
                tc_load<F::kAtoms>(s_q + (2 * slot + 1) * F::kTileBytes, map_do, t.h, t.q0, t.b, q_full + 8 * slot);
                for (int i = 0; i < t.tiles; ++i, ++n) {
                    const uint32_t sk = n % F::kKStages, sv = n % F::kVStages;
                    const int64_t k0 = t.begin + static_cast<int64_t>(i) * kTcTile;
                    ok = mbar_wait(k_empty + 8 * sk, ((n / F::kKStages) & 1) ^ 1, abort_flag, p.status, kStatusTimeoutXEmpty);
                    if (!ok) break;
                    tc_load<F::kAtoms>(s_k + sk * F::kTileBytes, map_k, t.hk, k0, t.b, k_tma + 8 * sk);
                    ++k_sent;
                    ok = mbar_wait(v_empty + 8 * sv, ((n / F::kVStages) & 1) ^ 1, abort_flag, p.status, kStatusTimeoutXEmpty);
                    if (!ok) break;
                    tc_load<F::kAtoms>(s_v + sv * F::kTileBytes, map_v, t.hk, k0, t.b, v_full + 8 * sv);
                    ++v_sent;
                }
            }
            // no copy may be in flight when the block ends
            for (uint32_t s = 0; s < F::kItems; ++s)
                if (m > s) drain_wait(q_full + 8 * s, ((m - 1 - s) / F::kItems) & 1, p.status);
            for (uint32_t s = 0; s < F::kKStages; ++s)
                if (k_sent > s) drain_wait(k_tma + 8 * s, ((k_sent - 1 - s) / F::kKStages) & 1, p.status);
            for (uint32_t s = 0; s < F::kVStages; ++s)
                if (v_sent > s) drain_wait(v_full + 8 * s, ((v_sent - 1 - s) / F::kVStages) & 1, p.status);
        }
    } else if (warp == 9) {
        if (lane == 0) {
            const uint32_t idesc = umma_idesc_f16(kTcTile, kBf16);
            const uint32_t k_ready = p.guarded ? k_ok : k_tma;
            const uint32_t q_desc = desc_k_major(s_q), k_desc = desc_k_major(s_k), v_desc = desc_k_major(s_v);
            constexpr uint32_t kTile = F::kTileBytes / 16;
            auto score = [&](uint32_t n, uint32_t m, bool first) {  // S(n) of item m, over dS(n - 2)
                const uint32_t s = n % F::kKStages, half = n & 1, slot = m % F::kItems;
                if (first &&
                    !mbar_wait(q_full + 8 * slot, (m / F::kItems) & 1, abort_flag, p.status, kStatusTimeoutWFull))
                    return false;
                if (n >= 2 &&
                    !mbar_wait(dq_done + 8 * half, (n / 2 - 1) & 1, abort_flag, p.status, kStatusTimeoutAccFull))
                    return false;
                if (!mbar_wait(k_ready + 8 * s, (n / F::kKStages) & 1, abort_flag, p.status, kStatusTimeoutXFull))
                    return false;
                tc_fence_after();
                product_rows<DP / 16>(tmem + F::kColS + half * 128, q_desc + 2 * slot * kTile, k_desc + s * kTile,
                                      p.k_steps, idesc);
                umma_commit(s_full + 8 * half);
                return true;
            };
            auto reach = [&](uint32_t n, uint32_t m, bool last) {  // dP(n), over dP(n - 1), which dS(n - 1) was made of
                const uint32_t s = n % F::kVStages, slot = m % F::kItems;
                if (n >= 1 && !mbar_wait(ds_full + 8 * ((n - 1) & 1), ((n - 1) / 2) & 1, abort_flag, p.status,
                                         kStatusTimeoutAFull))
                    return false;
                if (!mbar_wait(v_full + 8 * s, (n / F::kVStages) & 1, abort_flag, p.status, kStatusTimeoutXFull))
                    return false;
                tc_fence_after();
                product_rows<DP / 16>(tmem + F::kColDp, q_desc + (2 * slot + 1) * kTile, v_desc + s * kTile, p.k_steps,
                                      idesc);
                umma_commit(v_empty + 8 * s);
                umma_commit(dp_full);
                if (last) umma_commit(q_empty + 8 * slot);
                return true;
            };
            uint32_t id = blockIdx.x, n = 0;
            TcItem t;
            bool ok = true, have = next_item<1>(a, items, id, t);
            if (have) ok = score(0, 0, true);
            for (uint32_t m = 0; ok && have; ++m) {
                const int tiles = t.tiles;
                id += gridDim.x;
                have = next_item<1>(a, items, id, t);
                for (int i = 0; ok && i < tiles; ++i, ++n) {
                    const bool last = i + 1 == tiles;
                    ok = reach(n, m, last);
                    if (ok && (!last || have)) ok = score(n + 1, last ? m + 1 : m, last);
                }
            }
            umma_commit(drain);
            drain_wait(drain, 0, p.status);
        }
    } else if (warp == 11) {
        if (lane == 0) {
            const uint32_t idesc = umma_idesc_f16(p.n_pv, kBf16) | kIdescBTransposed;
            const uint32_t k_desc = desc_mn_major(s_k);
            uint32_t id = blockIdx.x, n = 0;
            TcItem t;
            bool ok = true;
            for (uint32_t m = 0; ok && next_item<1>(a, items, id, t); id += gridDim.x, ++m) {
                const uint32_t slot = m % F::kItems;
                if (m >= F::kItems && !mbar_wait(dq_read + 8 * slot, (m / F::kItems - 1) & 1, abort_flag, p.status,
                                                 kStatusTimeoutDrain))
                    break;
                for (int i = 0; i < t.tiles; ++i, ++n) {
                    const uint32_t s = n % F::kKStages, half = n & 1;
                    ok = mbar_wait(ds_full + 8 * half, (n / 2) & 1, abort_flag, p.status, kStatusTimeoutAFull);
                    if (!ok) break;
                    tc_fence_after();
                    product_columns(tmem + F::kColDq + slot * DP, tmem + F::kColS + half * 128,
                                    k_desc + s * (F::kTileBytes / 16), idesc, i == 0);
                    umma_commit(k_empty + 8 * s);
                    umma_commit(dq_done + 8 * half);
                }
                if (ok) umma_commit(dq_full + 8 * slot);
            }
            umma_commit(drain);
            drain_wait(drain, 0, p.status);
        }
    } else if (warp == 10) {
        if (p.guarded) {
            uint32_t n = 0, id = blockIdx.x;
            TcItem t;
            bool ok = true;
            for (; ok && next_item<1>(a, items, id, t); id += gridDim.x) {
                KeyLoad keys = key_load(a, t.b, t.begin, t.end);
                for (int i = 0; i < t.tiles; ++i, ++n) {
                    const uint32_t s = n % F::kKStages;
                    const KeyBits bits = key_bits(a, keys);
                    keys = key_load(a, t.b, t.begin + (i + 1ll) * kTcTile, t.end);
                    ok = mbar_wait_warp(k_tma + 8 * s, (n / F::kKStages) & 1, abort_flag, p.status, kStatusTimeoutXFull);
                    if (!ok) break;
                    if (!bits.all()) {
                        zero_rows<F::kAtoms>(s_k + s * F::kTileBytes, bits);
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                    if (lane == 0) mbar_arrive(k_ok + 8 * s);
                }
            }
        }
    } else {
        const int half = warp >> 2;
        const uint32_t row_base = tmem + (static_cast<uint32_t>(warp & 3) << 21);
        const float c = a.scale * kLog2e;
        const float e2 = grad_exponent<kBf16>(p);
        const float to_p = exp2f(-e2), f = a.scale * to_p;
        const int64_t rows = static_cast<int64_t>(a.batch) * a.q_len * a.heads;
        uint32_t n = 0, m = 0, pair_phase = 0;
        bool ok = true;
        // v summed over the two threads of a row (warps w and w + 4); false when the wait ran out
        const uint32_t pair = row_pair + 8 * (warp & 3), cell = base + F::kOffRow + ((warp & 3) * 32 + lane) * 4;
        auto row_sum = [&](float& v) {
            asm volatile("st.shared.f32 [%0], %1;" ::"r"(cell + half * 512), "f"(v) : "memory");
            for (int step = 0; step < 2; ++step) {  // written by both; read by both
                __syncwarp();
                if (lane == 0) mbar_arrive(pair);
                if (!mbar_wait_warp(pair, pair_phase++ & 1, abort_flag, p.status, kStatusTimeoutOther)) return false;
                if (step == 0) {
                    float other;
                    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(other) : "r"(cell + (half ^ 1) * 512) : "memory");
                    v = half ? other + v : v + other;
                }
            }
            return true;
        };
        for (uint32_t id = blockIdx.x; ok && id < items; id += gridDim.x) {
            const TcItem t = tc_item<1>(a, id);
            const bool one = t.tiles == 1 && length_of(a, t.b) <= kTcTile;
            float slip0 = 0.0f, slip1 = 0.0f;  // sum of dS
            const int64_t q = t.q0 + (warp & 3) * 32 + lane;
            const int64_t stat = (static_cast<int64_t>(t.b) * a.heads + t.h) * p.q_pad + q;
            const float minus = p.neg_lse[stat] + e2;
            float neg_delta = p.neg_delta[stat];
            bool any = false;
            KeyLoad keys = key_load(a, t.b, t.begin, t.end);
            for (int i = 0; i < t.tiles; ++i, ++n) {
                const KeyBits bits = key_bits(a, keys);
                keys = key_load(a, t.b, t.begin + (i + 1ll) * kTcTile, t.end);
                const bool whole = bits.all();
                any |= !bits.none();
                const uint32_t s_col = row_base + F::kColS + (n & 1) * 128 + half * 64;
                ok = mbar_wait_warp(s_full + 8 * (n & 1), (n / 2) & 1, abort_flag, p.status, kStatusTimeoutAccFull);
                if (!ok) break;
                tc_fence_after();
                uint32_t r[2][32];
                tmem_ld32(s_col, r[0]);
                tmem_ld32(s_col + 32, r[1]);
                tmem_wait_ld32(r[0]);
                reg_barrier32(r[1]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float x = __uint_as_float(r[j][e]), y = __uint_as_float(r[j][e + 1]);
                        fma2(x, y, c, c, minus, minus);
                        exp2_pair<kGradPoly>(x, y, e / 2);
                        r[j][e] = __float_as_uint(x);
                        r[j][e + 1] = __float_as_uint(y);
                    }
                ok = mbar_wait_warp(dp_full, n & 1, abort_flag, p.status, kStatusTimeoutAccFull);
                if (!ok) break;
                tc_fence_after();
                uint32_t d[2][32];
                tmem_ld32(row_base + F::kColDp + half * 64, d[0]);
                tmem_ld32(row_base + F::kColDp + half * 64 + 32, d[1]);
                tmem_wait_ld32(d[0]);
                reg_barrier32(d[1]);
                // Two copies of the arithmetic: selecting what is not allowed away costs a tenth where all are.
                auto finish = [&](auto masked) {
                    constexpr bool kMasked = decltype(masked)::value;
                    auto keep = [&](float& x, float& y, uint32_t word, int e) {
                        if (kMasked) {  // whatever stood where the key is not allowed
                            x = word >> e & 1u ? x : 0.0f;
                            y = word >> (e + 1) & 1u ? y : 0.0f;
                        }
                    };
                    if (one) {
                        float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t word = half ? bits.w[2 + j] : bits.w[j];
#pragma unroll
                            for (int e = 0; e < 32; e += 2) {
                                float x = __uint_as_float(r[j][e]), y = __uint_as_float(r[j][e + 1]);
                                mul2(x, y, __uint_as_float(d[j][e]), __uint_as_float(d[j][e + 1]));
                                keep(x, y, word, e);
                                add2(s0, s1, x, y);
                            }
                        }
                        s0 += s1;
                        if (!row_sum(s0)) return false;
                        neg_delta = -s0 * to_p;
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint32_t packed[16];
                        const uint32_t word = half ? bits.w[2 + j] : bits.w[j];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float x = __uint_as_float(d[j][e]), y = __uint_as_float(d[j][e + 1]);
                            add2(x, y, neg_delta, neg_delta);
                            mul2(x, y, __uint_as_float(r[j][e]), __uint_as_float(r[j][e + 1]));
                            keep(x, y, word, e);
                            add2(slip0, slip1, x, y);
                            packed[e / 2] = kBf16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
                        }
                        tmem_st16(s_col + 16 * j, packed);
                    }
                    return true;
                };
                ok = whole ? finish(std::false_type{}) : finish(std::true_type{});
                if (!ok) break;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(ds_full + 8 * (n & 1));
            }
            if (t.tiles > 0 && ok) {
                if (!one) {
                    slip0 += slip1;
                    ok = row_sum(slip0);
                }
                if (ok && half == 0) {
                    if (!one && a.splits > 1)
                        p.slips[t.split * (static_cast<int64_t>(a.batch) * a.heads * p.q_pad) + stat] = slip0 * to_p;
                    else if (any && q < a.q_len)
                        p.neg_delta[stat] = one ? neg_delta : neg_delta - slip0 * to_p;
                }
            }
            const uint32_t slot = m % F::kItems;
            if (t.tiles > 0 && ok)
                ok = mbar_wait_warp(dq_full + 8 * slot, (m / F::kItems) & 1, abort_flag, p.status, kStatusTimeoutAccFull);
            if (!ok) break;
            tc_fence_after();
            const int64_t row = (t.b * a.q_len + q) * a.heads + t.h;
            float* part = a.splits > 1 ? a.part + t.split * rows * a.dim : nullptr;
#pragma unroll 1
            for (int d = half * (DP / 2); d < (half + 1) * (DP / 2); d += 16) {
                if (d >= a.dim) break;
                uint32_t r[16] = {};
                __syncwarp();  // the load takes the whole warp; lanes past q_len skipped the last store
                if (t.tiles > 0) {
                    tmem_ld16(row_base + F::kColDq + slot * DP + d, r);
                    tmem_wait_ld(r);
                }
                if (q < a.q_len) store_columns<kBf16>(a, a.dq, part, row * a.dim, d, r, f, any);
            }
            if (t.tiles > 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(dq_read + 8 * slot);
                ++m;
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (warp == 9) {
        tmem_relinquish();
        tmem_dealloc(tmem, 512);
    }
}

// delta of rows whose keys are several tiles in several splits: the splits'
// sums of dS in order, a thread a row. Splits past a sample's length have none.
// Bound: its launch (2.4 us at 600 to 4096 rows and 4 to 16 splits).
__global__ void __launch_bounds__(kThreads) tc_slips_kernel(const GradParams p) {
    const Params& a = p.a;
    const int64_t rows = static_cast<int64_t>(a.batch) * a.heads * p.q_pad;
    const int64_t row = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
    if (row >= rows) return;
    const int64_t len = length_of(a, static_cast<int>(row / p.q_pad / a.heads));
    if (len <= kTcTile) return;
    float sum = 0.0f;
    for (int64_t s = 0; s * a.split_len < len; ++s) sum += p.slips[s * rows + row];
    p.neg_delta[row] -= sum;
}

// ------------------------------------------------------------------- dK, dV
//
// A block: 128 keys of one key head over the (query head, query tile) pairs
// of one split, with keys as TMEM lanes: S^T = K Q^T, dP^T = V dO^T, dV += P^T
// dO, dK += dS^T Q. P(i) and dS(i) go where S(i) was (a half row each). Up to
// 64 dimensions S has two buffers and dP one, so S(i + 1) is ready when dS(i)
// is; at 128, where O's columns leave two in all, S(i + 1) takes dP(i)'s as
// soon as that has been read, and dP(i + 1) S(i)'s once dK(i) has.
template <int DP>
struct TcDkv {
    static constexpr int kAtoms = DP / 64, kStages = DP == 64 ? 3 : 2;
    static constexpr bool kSwap = DP == 128;
    static constexpr uint32_t kTileBytes = kTcTile * DP * 2;
    static constexpr uint32_t kOffV = kTileBytes, kOffQ = 2 * kTileBytes, kOffDo = kOffQ + kStages * kTileBytes,
                              kOffStat = kOffDo + kStages * kTileBytes;  // [stage][-lse, -delta][128]
    static constexpr uint32_t kOffBar = kOffStat + kStages * 1024;
    static constexpr uint32_t kBytes = kOffBar + 512 + 1024;
    static constexpr uint32_t kColDv = kSwap ? 256 : 384, kColDk = kSwap ? 384 : 448;
    static __device__ __forceinline__ uint32_t col_s(int i) { return (i & 1) * 128; }
    static __device__ __forceinline__ uint32_t col_dp(int i) { return kSwap ? (~i & 1) * 128 : 256; }
};

template <int DP, bool kBf16>
__global__ void __launch_bounds__(kGradThreads, 1)
    tc_dkv_kernel(const GradParams p, const __grid_constant__ TcMap map_q, const __grid_constant__ TcMap map_k,
                  const __grid_constant__ TcMap map_v, const __grid_constant__ TcMap map_do) {
    using F = TcDkv<DP>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t s_k = base, s_v = base + F::kOffV, s_q = base + F::kOffQ, s_do = base + F::kOffDo,
                   s_stat = base + F::kOffStat, bars = base + F::kOffBar;
    const uint32_t kv_full = bars, dp_full = bars + 8, dp_read = bars + 16, drain = bars + 24, s_full = bars + 32,
                   p_full = bars + 48, ds_full = bars + 64, dk_done = bars + 80, q_full = bars + 96,
                   q_empty = bars + 120, do_full = bars + 144, do_empty = bars + 168;
    const uint32_t tmem_slot = bars + 192;
    volatile uint32_t* abort_flag =
        reinterpret_cast<volatile uint32_t*>(smem_raw + (bars - smem_addr(smem_raw)) + 196);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Params& a = p.a;
    const uint32_t k_tiles = static_cast<uint32_t>((a.kv_len + kTcTile - 1) / kTcTile);
    const int q_tiles = static_cast<int>(p.q_pad / kTcTile);
    uint32_t id = blockIdx.x;
    const int64_t k0 = static_cast<int64_t>(id % k_tiles) * kTcTile;
    id /= k_tiles;
    const int hk = id % a.kv_heads;
    id /= a.kv_heads;
    const int b = id % a.batch, split = id / a.batch;
    const KeyBits bits = key_bits(a, key_load(a, b, k0, length_of(a, b)));
    const int first = static_cast<int>(split * a.split_len);
    const int last = min(q_tiles * a.group, static_cast<int>(first + a.split_len));
    const int items = bits.none() ? 0 : last - first;

    if (threadIdx.x == 0) {
        *abort_flag = 0u;
        mbar_init(kv_full, 2);
        mbar_init(dp_full, 1);
        mbar_init(dp_read, 8);
        mbar_init(drain, 2);  // an arrival an issuing warp
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 8);
            mbar_init(ds_full + 8 * i, 8);
            mbar_init(dk_done + 8 * i, 1);
        }
        for (int i = 0; i < F::kStages; ++i) {
            mbar_init(q_full + 8 * i, 2);  // the tile and its -lse
            mbar_init(q_empty + 8 * i, 1);
            mbar_init(do_full + 8 * i, 2);  // the tile and its -delta
            mbar_init(do_empty + 8 * i, 1);
        }
        fence_mbarrier_init();
    }
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

    if (warp == 8) {
        if (lane == 0 && items > 0) {
            int q_sent = 0, do_sent = 0;
            tc_load<F::kAtoms>(s_k, map_k, hk, k0, b, kv_full);
            tc_load<F::kAtoms>(s_v, map_v, hk, k0, b, kv_full);
            for (int i = 0; i < items; ++i) {
                const int s = i % F::kStages;
                const uint32_t parity = ((i / F::kStages) & 1) ^ 1;
                const int h = hk * a.group + (first + i) / q_tiles;
                const int64_t q0 = static_cast<int64_t>((first + i) % q_tiles) * kTcTile;
                const int64_t stat = (static_cast<int64_t>(b) * a.heads + h) * p.q_pad + q0;
                if (!mbar_wait(q_empty + 8 * s, parity, abort_flag, p.status, kStatusTimeoutXEmpty)) break;
                tc_load<F::kAtoms>(s_q + s * F::kTileBytes, map_q, h, q0, b, q_full + 8 * s);
                mbar_arrive_expect_tx(q_full + 8 * s, 512);
                bulk_g2s(s_stat + s * 1024, p.neg_lse + stat, 512, q_full + 8 * s);
                ++q_sent;
                if (!mbar_wait(do_empty + 8 * s, parity, abort_flag, p.status, kStatusTimeoutXEmpty)) break;
                tc_load<F::kAtoms>(s_do + s * F::kTileBytes, map_do, h, q0, b, do_full + 8 * s);
                mbar_arrive_expect_tx(do_full + 8 * s, 512);
                bulk_g2s(s_stat + s * 1024 + 512, p.neg_delta + stat, 512, do_full + 8 * s);
                ++do_sent;
            }
            drain_wait(kv_full, 0, p.status);
            for (int s = 0; s < F::kStages; ++s) {
                if (q_sent > s) drain_wait(q_full + 8 * s, ((q_sent - 1 - s) / F::kStages) & 1, p.status);
                if (do_sent > s) drain_wait(do_full + 8 * s, ((do_sent - 1 - s) / F::kStages) & 1, p.status);
            }
        }
    } else if (warp == 9) {
        if (lane == 0 && items > 0) {
            const uint32_t idesc = umma_idesc_f16(kTcTile, kBf16);
            const uint32_t k_desc = desc_k_major(s_k), v_desc = desc_k_major(s_v), q_desc = desc_k_major(s_q),
                           do_desc = desc_k_major(s_do);
            // the (i / 2)-th phase of a barrier of even and odd tiles
            auto wait2 = [&](uint32_t bar, int i, uint32_t code) {
                return mbar_wait(bar + 8 * (i & 1), (i / 2) & 1, abort_flag, p.status, code);
            };
            auto score = [&](int i) {
                const uint32_t s = i % F::kStages;
                if (F::kSwap ? i >= 1 && !mbar_wait(dp_read, (i - 1) & 1, abort_flag, p.status, kStatusTimeoutAFull)
                             : i >= 2 && !wait2(dk_done, i - 2, kStatusTimeoutAccFull))
                    return false;
                if (!mbar_wait(q_full + 8 * s, (i / F::kStages) & 1, abort_flag, p.status, kStatusTimeoutXFull))
                    return false;
                tc_fence_after();
                product_rows<DP / 16>(tmem + F::col_s(i), k_desc, q_desc + s * (F::kTileBytes / 16), p.k_steps, idesc);
                umma_commit(s_full + 8 * (i & 1));
                return true;
            };
            auto reach = [&](int i) {
                const uint32_t s = i % F::kStages;
                if (i >= 1 && !wait2(F::kSwap ? dk_done : ds_full, i - 1, kStatusTimeoutAccFull)) return false;
                if (!mbar_wait(do_full + 8 * s, (i / F::kStages) & 1, abort_flag, p.status, kStatusTimeoutXFull))
                    return false;
                tc_fence_after();
                product_rows<DP / 16>(tmem + F::col_dp(i), v_desc, do_desc + s * (F::kTileBytes / 16), p.k_steps, idesc);
                umma_commit(dp_full);
                return true;
            };
            bool ok = mbar_wait(kv_full, 0, abort_flag, p.status, kStatusTimeoutWFull) && score(0);
            for (int i = 0; ok && i < items; ++i) {
                ok = reach(i);
                if (ok && i + 1 < items) ok = score(i + 1);
            }
            umma_commit(drain);
            drain_wait(drain, 0, p.status);
        }
    } else if (warp == 11) {
        if (lane == 0 && items > 0) {
            const uint32_t idesc = umma_idesc_f16(p.n_pv, kBf16) | kIdescBTransposed;
            const uint32_t q_desc = desc_mn_major(s_q), do_desc = desc_mn_major(s_do);
            for (int i = 0; i < items; ++i) {
                const uint32_t s = i % F::kStages, half = i & 1, at = s * (F::kTileBytes / 16);
                if (!mbar_wait(p_full + 8 * half, (i / 2) & 1, abort_flag, p.status, kStatusTimeoutAFull)) break;
                // P(i) says that Q(i) has come, not that dO(i) has
                if (!mbar_wait(do_full + 8 * s, (i / F::kStages) & 1, abort_flag, p.status, kStatusTimeoutXFull)) break;
                tc_fence_after();
                product_columns(tmem + F::kColDv, tmem + F::col_s(i), do_desc + at, idesc, i == 0);
                if (!mbar_wait(ds_full + 8 * half, (i / 2) & 1, abort_flag, p.status, kStatusTimeoutAFull)) break;
                tc_fence_after();
                product_columns(tmem + F::kColDk, tmem + F::col_s(i) + 32, q_desc + at, idesc, i == 0);
                umma_commit(do_empty + 8 * s);  // dS(i) took dP(i), so nothing reads dO(i) any more either
                umma_commit(q_empty + 8 * s);
                umma_commit(dk_done + 8 * half);
            }
            umma_commit(drain);
            drain_wait(drain, 0, p.status);
        }
    } else if (warp < 8) {
        const int half = warp >> 2;
        const uint32_t row_base = tmem + (static_cast<uint32_t>(warp & 3) << 21);
        const int64_t key = k0 + (warp & 3) * 32 + lane;
        const uint32_t low = warp & 1 ? bits.w[1] : bits.w[0], high = warp & 1 ? bits.w[3] : bits.w[2];
        const bool on = (warp & 2 ? high : low) >> lane & 1u;
        const float c = a.scale * kLog2e;
        const float e2 = grad_exponent<kBf16>(p);
        constexpr float kP = kBf16 ? 0.0f : 15.0f;  // P is held times 2^kP
        const float to_ds = kBf16 ? 1.0f : exp2f(e2 - kP);
        bool ok = true;
        for (int i = 0; i < items; ++i) {
            const uint32_t stat = s_stat + (i % F::kStages) * 1024 + half * 256;
            if (!(ok = mbar_wait_warp(s_full + 8 * (i & 1), (i / 2) & 1, abort_flag, p.status, kStatusTimeoutAccFull)))
                break;
            // the copy of -lse completed with the tile that S(i) was made of; this orders it for this thread
            if (!(ok = mbar_wait_warp(q_full + 8 * (i % F::kStages), (i / F::kStages) & 1, abort_flag, p.status,
                                      kStatusTimeoutXFull)))
                break;
            tc_fence_after();
            const uint32_t col = row_base + F::col_s(i) + half * 64;  // P in its first 32 columns, dS in the others
            uint32_t r[2][32];
            tmem_ld32(col, r[0]);
            tmem_ld32(col + 32, r[1]);
            tmem_wait_ld32(r[0]);
            reg_barrier32(r[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t packed[16];
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    float4 l = ld_shared_f4(stat + (32 * j + e) * 4);
                    if (!kBf16) l.x += kP, l.y += kP, l.z += kP, l.w += kP;
                    float x[4] = {__uint_as_float(r[j][e]), __uint_as_float(r[j][e + 1]), __uint_as_float(r[j][e + 2]),
                                  __uint_as_float(r[j][e + 3])};
                    fma2(x[0], x[1], c, c, l.x, l.y);
                    fma2(x[2], x[3], c, c, l.z, l.w);
                    exp2_pair<kGradPoly>(x[0], x[1], e / 2);
                    exp2_pair<kGradPoly>(x[2], x[3], e / 2 + 1);
                    packed[e / 2] = kBf16 ? pack_bf16x2(x[0], x[1]) : pack_f16x2(x[0], x[1]);
                    packed[e / 2 + 1] = kBf16 ? pack_bf16x2(x[2], x[3]) : pack_f16x2(x[2], x[3]);
                    if (!kBf16) {
                        mul2(x[0], x[1], to_ds, to_ds);
                        mul2(x[2], x[3], to_ds, to_ds);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) r[j][e + k] = __float_as_uint(x[k]);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) packed[e] = on ? packed[e] : 0u;
                tmem_st16(col + 16 * j, packed);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * (i & 1));
            if (!(ok = mbar_wait_warp(dp_full, i & 1, abort_flag, p.status, kStatusTimeoutAccFull))) break;
            if (!(ok = mbar_wait_warp(do_full + 8 * (i % F::kStages), (i / F::kStages) & 1, abort_flag, p.status,
                                      kStatusTimeoutXFull)))
                break;
            tc_fence_after();
            uint32_t d[2][32];
            tmem_ld32(row_base + F::col_dp(i) + half * 64, d[0]);
            tmem_ld32(row_base + F::col_dp(i) + half * 64 + 32, d[1]);
            tmem_wait_ld32(d[0]);
            reg_barrier32(d[1]);
            if (F::kSwap) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(dp_read);
                __syncwarp();  // the stores below take the whole warp
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t packed[16];
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const float4 n = ld_shared_f4(stat + 512 + (32 * j + e) * 4);
                    float x[4] = {__uint_as_float(d[j][e]), __uint_as_float(d[j][e + 1]), __uint_as_float(d[j][e + 2]),
                                  __uint_as_float(d[j][e + 3])};
                    add2(x[0], x[1], n.x, n.y);
                    add2(x[2], x[3], n.z, n.w);
                    mul2(x[0], x[1], __uint_as_float(r[j][e]), __uint_as_float(r[j][e + 1]));
                    mul2(x[2], x[3], __uint_as_float(r[j][e + 2]), __uint_as_float(r[j][e + 3]));
                    packed[e / 2] = kBf16 ? pack_bf16x2(x[0], x[1]) : pack_f16x2(x[0], x[1]);
                    packed[e / 2 + 1] = kBf16 ? pack_bf16x2(x[2], x[3]) : pack_f16x2(x[2], x[3]);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) packed[e] = on ? packed[e] : 0u;
                tmem_st16(col + 32 + 16 * j, packed);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ds_full + 8 * (i & 1));
        }
        if (items > 0 && ok) ok = mbar_wait_warp(drain, 0, abort_flag, p.status, kStatusTimeoutAccFull);
        tc_fence_after();
        // WG 0 writes dV, WG 1 dK
        const int64_t rows = static_cast<int64_t>(a.batch) * a.kv_len * a.kv_heads;
        const int64_t row = (b * a.kv_len + key) * a.kv_heads + hk;
        float* part = a.splits > 1 ? a.part_kv + (2 * split + (half ? 0 : 1)) * rows * a.dim : nullptr;
        const float f = half ? a.scale * exp2f(-e2) : exp2f(-kP);
#pragma unroll 1
        for (int d = 0; d < DP; d += 16) {
            if (d >= a.dim) break;
            uint32_t r[16] = {};
            __syncwarp();  // the load takes the whole warp; lanes past kv_len skipped the last store
            if (items > 0) {
                tmem_ld16(row_base + (half ? F::kColDk : F::kColDv) + d, r);
                tmem_wait_ld(r);
            }
            if (ok && key < a.kv_len)
                store_columns<kBf16>(a, half ? a.dk : a.dv, part, row * a.dim, d, r, f, on && items > 0);
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (warp == 9) {
        tmem_relinquish();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace attn
}  // namespace rdvb
