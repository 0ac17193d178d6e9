// Attention (attention.cuh has the mathematics) on the tensor cores, for
// float16 and bfloat16 with head dimensions up to 128, multiples of 8.
//
// A block owns 128 query rows of one head and walks over the keys 128 at a
// time: S = Q K^T into TMEM (one row a lane), a thread a row takes the
// running maximum and the exponentials and leaves P, 16 bits an element, in
// TMEM, and O += P V takes it from there. Q, K and V come by TMA into
// 128-byte-swizzled tiles; V is the MN-major operand of the second product,
// so nothing is transposed. Two blocks a processor: while one's warps are in
// the exponentials the other's products run. Warps 0-3: softmax. Warp 4:
// loads. Warp 5: products. Warp 6: zeroes the rows of V whose keys are not
// allowed (their P is 0, but 0 times NaN is not).
//
// S, the row sums and O are float32; P is rounded to the inputs' type, as the
// tensor cores take it. O is rescaled only when a row's maximum has grown by
// more than 2^8 since the last time: P stays below 2^8, well inside both types.
// The scale is above 0, so that the largest score is the scaled largest
// product and a score of -inf stays one.
#pragma once
#include <cuda.h>

#include <cstdint>

#include "attention.cuh"
#include "ptx.cuh"

namespace rdvb {
namespace attn {

constexpr int kTcTile = 128;       // query rows and keys of a tile
constexpr int kTcThreads = 8 * 32;  // one warp is idle: registers are shared out by groups of four
// Registers of a thread at launch (two blocks fill a processor's 65,536), and
// after the softmax warps have taken some of the others' (208 + 48 = 2 x 128).
constexpr int kTcRegisters = 128, kSoftmaxRegisters = 208, kOtherRegisters = 48;
constexpr float kGrowth = 8.0f;    // log2 of the growth of a row's maximum that O is rescaled at

struct TcParams {
    Params a;
    uint32_t* status;
    uint32_t k_steps;  // ceil(dim / 16)
    uint32_t n_pv;     // dim rounded up to 16
    int guarded;       // lengths or a mask: warp 6 takes part
};

// The tensor map of q, k or v, and whether its head and sample axes are walked
// (0: broadcast).
struct TcMap {
    CUtensorMap map;
    int head_step, batch_step;
};
// Loads 128 rows of one head, kAtoms x 64 dimensions; x is a multiple of 128
// bytes.
template <int kAtoms>
__device__ __forceinline__ void tc_load(uint32_t dst, const TcMap& m, int head, int64_t row, int sample, uint32_t bar) {
    mbar_arrive_expect_tx(bar, kAtoms * 128 * 128);
#pragma unroll
    for (int i = 0; i < kAtoms; ++i)
        tma_load_4d(dst + i * 128 * 128, &m.map, 64 * i, head * m.head_step, static_cast<int>(row),
                    sample * m.batch_step, bar);
}

// The 128-byte-swizzled MN-major operand of 16-bit elements: rows of 64 n
// elements (128 bytes) per k, 8-k groups 1024 bytes apart, the next 64 n
// elements `lbo` bytes on. 16 k are 2048 bytes.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t saddr, uint32_t lbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}
constexpr uint32_t kIdescBTransposed = 1u << 16;

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// Waits for this thread's TMEM loads; redefines the registers so that no use
// of them moves above the wait.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void reg_barrier32(uint32_t (&r)[32]) {
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// (a0 b + c, a1 b + c) in one packed instruction.
__device__ __forceinline__ void fma_f32x2(float& a0, float& a1, float b, float c) {
    uint64_t pa, pb, pc, pd;
    asm("mov.b64 %0, {%1, %2};" : "=l"(pa) : "f"(a0), "f"(a1));
    asm("mov.b64 %0, {%1, %1};" : "=l"(pb) : "f"(b));
    asm("mov.b64 %0, {%1, %1};" : "=l"(pc) : "f"(c));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(pd) : "l"(pa), "l"(pb), "l"(pc));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(pd));
}

// Which of the 128 keys from k0 on are allowed, as four words; the same in
// every lane of a warp. Call with all 32 lanes.
struct KeyBits {
    uint32_t w[4];
    __device__ __forceinline__ bool all() const { return (w[0] & w[1] & w[2] & w[3]) == 0xffffffffu; }
    __device__ __forceinline__ bool none() const { return (w[0] | w[1] | w[2] | w[3]) == 0u; }
};
__device__ __forceinline__ KeyBits key_bits(const Params& p, int b, int64_t k0, int64_t end) {
    KeyBits bits;
    const int64_t left = end - k0;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t n = left - 32 * i;
        uint32_t w = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
        if (p.mask) {
            const bool in = 32 * i + lane < left;
            w = __ballot_sync(0xffffffffu, in && p.mask[b * p.mask_stride + k0 + 32 * i + lane] != 0);
        }
        bits.w[i] = w;
    }
    return bits;
}

// Zeroes the rows of a 128-row tile (atoms of 64 elements, kAtoms of them)
// whose bit is not set. Call with all 32 lanes of one warp, then fence.
template <int kAtoms>
__device__ __forceinline__ void zero_rows(uint32_t tile, const KeyBits& bits) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        for (uint32_t off = ~bits.w[i]; off; off &= off - 1) {
            const uint32_t row = 32 * i + __ffs(off) - 1;
            if (lane < 8 * kAtoms)
                st_shared_v4(tile + (lane >> 3) * (kTcTile * 128) + row * 128 + (lane & 7) * 16, 0, 0, 0, 0);
        }
}

// A block's place in the forward pass and dQ: query tile, head, sample,
// split.
struct TcPlace {
    int64_t q0, begin, end;
    int h, hk, b, split, tiles;
};
__device__ __forceinline__ TcPlace tc_place(const Params& p) {
    TcPlace t;
    const uint32_t q_tiles = static_cast<uint32_t>((p.q_len + kTcTile - 1) / kTcTile);
    uint32_t id = blockIdx.x;
    t.q0 = static_cast<int64_t>(id % q_tiles) * kTcTile;
    id /= q_tiles;
    t.h = id % p.heads;
    id /= p.heads;
    t.b = id % p.batch;
    t.split = id / p.batch;
    t.hk = t.h / p.group;
    const int64_t len = length_of(p, t.b);
    t.begin = t.split * p.split_len;
    t.end = min(len, t.begin + p.split_len);
    t.tiles = t.end > t.begin ? static_cast<int>((t.end - t.begin + kTcTile - 1) / kTcTile) : 0;
    return t;
}

template <int DP>
struct TcForward {
    static constexpr int kAtoms = DP / 64;
    static constexpr uint32_t kTileBytes = kTcTile * DP * 2;
    static constexpr int kStages = DP == 64 ? 2 : 1;  // K and V tiles in flight; 96 KB either way
    // TMEM columns: S, O and, where there is room, P beside S instead of over it
    static constexpr bool kOwnP = DP == 64;
    static constexpr uint32_t kColS = 0, kColO = 128, kColP = kOwnP ? 192 : 0, kCols = 256;
    static constexpr uint32_t kOffK = kTileBytes, kOffV = kOffK + kStages * kTileBytes,
                              kOffBar = kOffV + kStages * kTileBytes;
    static constexpr uint32_t kBytes = kOffBar + 256 + 1024;  // barriers; slack for the 1024-byte alignment
};

template <int DP, bool kBf16>
__global__ void __launch_bounds__(kTcThreads, 2)
    tc_forward_kernel(const TcParams p, const __grid_constant__ TcMap map_q,
                      const __grid_constant__ TcMap map_k, const __grid_constant__ TcMap map_v) {
    using F = TcForward<DP>;
    constexpr int kStages = F::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t s_q = base, s_k = base + F::kOffK, s_v = base + F::kOffV, bars = base + F::kOffBar;
    const uint32_t q_full = bars, s_full = bars + 8, s_read = bars + 16, p_full = bars + 24, o_full = bars + 32,
                   drain = bars + 40, k_full = bars + 48, k_empty = bars + 64, v_tma = bars + 80, v_full = bars + 96,
                   v_empty = bars + 112;
    const uint32_t tmem_slot = bars + 128;
    volatile uint32_t* abort_flag =
        reinterpret_cast<volatile uint32_t*>(smem_raw + (bars - smem_addr(smem_raw)) + 132);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Params& a = p.a;
    const TcPlace t = tc_place(a);

    if (threadIdx.x == 0) {
        *abort_flag = 0u;
        mbar_init(q_full, 1);
        mbar_init(s_full, 1);
        mbar_init(s_read, 4);
        mbar_init(p_full, 4);
        mbar_init(o_full, 1);
        mbar_init(drain, 1);
        for (int i = 0; i < kStages; ++i) {
            mbar_init(k_full + 8 * i, 1);
            mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_tma + 8 * i, 1);
            mbar_init(v_full + 8 * i, 1);
            mbar_init(v_empty + 8 * i, 1);
        }
        fence_mbarrier_init();
    }
    if (warp == 5) tmem_alloc(tmem_slot, F::kCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

    if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == 4) {
        if (lane == 0 && t.tiles > 0) {
            int k_sent = 0, v_sent = 0;
            tc_load<F::kAtoms>(s_q, map_q, t.h, t.q0, t.b, q_full);
            for (int i = 0; i < t.tiles; ++i) {
                const int s = i % kStages;
                const uint32_t parity = ((i / kStages) & 1) ^ 1;
                const int64_t k0 = t.begin + static_cast<int64_t>(i) * kTcTile;
                if (!mbar_wait(k_empty + 8 * s, parity, abort_flag, p.status, kStatusTimeoutXEmpty)) break;
                tc_load<F::kAtoms>(s_k + s * F::kTileBytes, map_k, t.hk, k0, t.b, k_full + 8 * s);
                ++k_sent;
                if (!mbar_wait(v_empty + 8 * s, parity, abort_flag, p.status, kStatusTimeoutXEmpty)) break;
                tc_load<F::kAtoms>(s_v + s * F::kTileBytes, map_v, t.hk, k0, t.b, v_tma + 8 * s);
                ++v_sent;
            }
            // no copy may be in flight when the block ends
            drain_wait(q_full, 0, p.status);
            for (int s = 0; s < kStages; ++s) {
                if (k_sent > s) drain_wait(k_full + 8 * s, ((k_sent - 1 - s) / kStages) & 1, p.status);
                if (v_sent > s) drain_wait(v_tma + 8 * s, ((v_sent - 1 - s) / kStages) & 1, p.status);
            }
        }
    } else if (warp == 5) {
        if (lane == 0 && t.tiles > 0) {
            const uint32_t idesc_s = umma_idesc_f16(kTcTile, kBf16);
            const uint32_t idesc_o = umma_idesc_f16(p.n_pv, kBf16) | kIdescBTransposed;
            const uint32_t v_ready = p.guarded ? v_full : v_tma;
            auto score = [&](int i) {  // S(i) = Q K(i)^T
                const int s = i % kStages;
                if (!mbar_wait(k_full + 8 * s, (i / kStages) & 1, abort_flag, p.status, kStatusTimeoutXFull)) return false;
                tc_fence_after();
                for (uint32_t j = 0; j < p.k_steps; ++j) {
                    const uint32_t at = (j >> 2) * (kTcTile * 128) + (j & 3) * 32;
                    umma_f16(tmem + F::kColS, umma_desc_sw128(s_q + at),
                             umma_desc_sw128(s_k + s * F::kTileBytes + at), idesc_s, j > 0);
                }
                umma_commit(k_empty + 8 * s);
                umma_commit(s_full);
                return true;
            };
            auto mix = [&](int i) {  // O += P(i) V(i)
                const int s = i % kStages;
                if (!mbar_wait(v_ready + 8 * s, (i / kStages) & 1, abort_flag, p.status, kStatusTimeoutXFull)) return false;
                if (!mbar_wait(p_full, i & 1, abort_flag, p.status, kStatusTimeoutAFull)) return false;
                tc_fence_after();
#pragma unroll
                for (uint32_t j = 0; j < kTcTile / 16; ++j)
                    umma_f16_ts(tmem + F::kColO, tmem + F::kColP + 8 * j,
                                umma_desc_mn_sw128(s_v + s * F::kTileBytes + j * 2048, kTcTile * 128), idesc_o,
                                i > 0 || j > 0);
                umma_commit(v_empty + 8 * s);
                umma_commit(o_full);
                return true;
            };
            bool ok = mbar_wait(q_full, 0, abort_flag, p.status, kStatusTimeoutWFull) && score(0);
            for (int i = 0; ok && i < t.tiles; ++i) {
                if (F::kOwnP) {
                    // the next scores may start when the softmax has read these
                    if (i + 1 < t.tiles)
                        ok = mbar_wait(s_read, i & 1, abort_flag, p.status, kStatusTimeoutAccFull) && score(i + 1);
                    ok = ok && mix(i);
                } else {
                    ok = mix(i);
                    // P(i) lies where S(i + 1) goes
                    if (ok && i + 1 < t.tiles)
                        ok = mbar_wait(o_full, i & 1, abort_flag, p.status, kStatusTimeoutAccFull) && score(i + 1);
                }
            }
            umma_commit(drain);
            drain_wait(drain, 0, p.status);
        }
    } else if (warp == 6) {
        if (p.guarded) {
            for (int i = 0; i < t.tiles; ++i) {
                const int s = i % kStages;
                const KeyBits bits = key_bits(a, t.b, t.begin + static_cast<int64_t>(i) * kTcTile, t.end);
                if (!mbar_wait_warp(v_tma + 8 * s, (i / kStages) & 1, abort_flag, p.status, kStatusTimeoutXFull)) break;
                if (!bits.all()) {
                    zero_rows<F::kAtoms>(s_v + s * F::kTileBytes, bits);
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                if (lane == 0) mbar_arrive(v_full + 8 * s);
            }
        }
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
        const uint32_t row_base = tmem + (static_cast<uint32_t>(warp) << 21);  // lane 32 * warp of TMEM
        const float c = a.scale * kLog2e;
        float top = -INFINITY, total = 0.0f;
        bool any = false, ok = true;
        for (int i = 0; i < t.tiles; ++i) {
            const KeyBits bits = key_bits(a, t.b, t.begin + static_cast<int64_t>(i) * kTcTile, t.end);
            const bool whole = bits.all();
            any |= !bits.none();
            if (!(ok = mbar_wait_warp(s_full, i & 1, abort_flag, p.status, kStatusTimeoutAccFull))) break;
            tc_fence_after();
            uint32_t r[8][16];
#pragma unroll
            for (int j = 0; j < 8; ++j) tmem_ld16(row_base + F::kColS + 16 * j, r[j]);
            tmem_wait_ld(r[0]);
#pragma unroll
            for (int j = 1; j < 8; ++j) reg_barrier(r[j]);
            if (F::kOwnP) {  // S has been read
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_read);
            }
            if (!whole) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        r[j][e] = bits.w[j / 2] >> (j % 2 * 16 + e) & 1u ? r[j][e] : 0xff800000u;
            }
            float high[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 16; e += 2)
                    high[j & 3] = fmaxf(fmaxf(high[j & 3], __uint_as_float(r[j][e])), __uint_as_float(r[j][e + 1]));
            const float m = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3])) * c;
            const bool grows = m > top + kGrowth || (top == -INFINITY && m > -INFINITY);
            if (i > 0 && !mbar_wait_warp(o_full, (i - 1) & 1, abort_flag, p.status, kStatusTimeoutAccFull)) {
                ok = false;
                break;
            }
            if (__any_sync(0xffffffffu, grows)) {
                const float fresh = grows ? m : top;
                const float f = fresh == -INFINITY ? 1.0f : exp2_approx(top - fresh);
                total *= f;
                top = fresh;
                if (i > 0) {
                    tc_fence_after();
#pragma unroll 1
                    for (uint32_t j = 0; j < p.n_pv; j += 16) {
                        uint32_t o[16];
                        tmem_ld16(row_base + F::kColO + j, o);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st16(row_base + F::kColO + j, o);
                    }
                }
            }
            const float minus = top == -INFINITY ? 0.0f : -top;
            float sum[4] = {};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t packed[8];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    float x = __uint_as_float(r[j][e]), y = __uint_as_float(r[j][e + 1]);
                    fma_f32x2(x, y, c, minus);
                    x = exp2_approx(x);
                    y = exp2_approx(y);
                    add_f32x2(sum[e & 2], sum[(e & 2) + 1], x, y);
                    packed[e / 2] = kBf16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
                }
                tmem_st8(row_base + F::kColP + 8 * j, packed);
            }
            total += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full);
        }
        if (t.tiles > 0 && ok)
            ok = mbar_wait_warp(o_full, (t.tiles - 1) & 1, abort_flag, p.status, kStatusTimeoutAccFull);
        tc_fence_after();
        const int64_t q = t.q0 + threadIdx.x;
        const bool mine = q < a.q_len && ok;
        const int64_t row = (t.b * a.q_len + q) * a.heads + t.h;
        const int64_t rows = static_cast<int64_t>(a.batch) * a.q_len * a.heads;
        const float inv = any ? 1.0f / total : 0.0f;
#pragma unroll 1
        for (int j = 0; j < DP / 32; ++j) {
            if (32 * j >= a.dim) break;
            uint32_t r[32];
            if (t.tiles > 0) {
                tmem_ld32(row_base + F::kColO + 32 * j, r);
                tmem_wait_ld32(r);
            }
            if (!any) {
#pragma unroll
                for (int e = 0; e < 32; ++e) r[e] = 0u;
            }
            if (!mine) continue;
            if (a.splits > 1) {
                float* dst = a.part + (t.split * rows + row) * a.dim + 32 * j;
#pragma unroll
                for (int e = 0; e < 32; e += 4)
                    if (32 * j + e < a.dim)
                        *reinterpret_cast<uint4*>(dst + e) = make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]);
            } else {
                uint16_t* dst = static_cast<uint16_t*>(a.o) + row * a.dim + 32 * j;
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float x = __uint_as_float(r[e + 2 * k]) * inv, y = __uint_as_float(r[e + 2 * k + 1]) * inv;
                        w[k] = kBf16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
                    }
                    if (32 * j + e < a.dim) *reinterpret_cast<uint4*>(dst + e) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        if (mine) {
            if (a.splits > 1) {
                a.part_stat[2 * (t.split * rows + row)] = top;
                a.part_stat[2 * (t.split * rows + row) + 1] = any ? total : -1.0f;
            } else if (a.lse) {
                a.lse[(static_cast<int64_t>(t.b) * a.heads + t.h) * a.q_len + q] =
                    any ? (top + log2f(total)) * kLn2 : -INFINITY;
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (warp == 5) {
        tmem_relinquish();
        tmem_dealloc(tmem, F::kCols);
    }
}

}  // namespace attn
}  // namespace rdvb
