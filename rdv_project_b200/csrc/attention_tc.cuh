// Attention (attention.cuh has the mathematics) on the tensor cores, for
// float16 and bfloat16 with head dimensions up to 128, multiples of 8.
//
// A block owns two tiles of 128 query rows of one head and walks over the
// keys 128 at a time: S = Q K^T into TMEM (one row a lane), a thread a row
// takes the running maximum and the exponentials and leaves P, 16 bits an
// element, in TMEM, and O += P V takes it from there. Q, K and V come by TMA
// into 128-byte-swizzled tiles; V is the MN-major operand of the second
// product, so nothing is transposed. The two tiles take turns: while one's
// warps are in the exponentials the other's products run, and both read the
// same K and V. The hardware keeps one block with TMEM on a processor, so a
// block stays and takes one (head, query tiles) item after another: the next
// item's first products and loads run beside this one's last rows. Warps 0-3
// and 4-7: softmax of a tile each. Warp 8: loads. Warps 9 and 11: products of
// a tile each up to 64 dimensions (one thread issues a product in 60 to 110
// cycles; with two, the first case below went from 1000 to 869 us, before masks were
// read a tile ahead, which costs it 41), at 128 warp 9 for both
// (two: 1169 to 1620 us, their products delaying each other's). Warp 10: zeroes the
// rows of V whose keys are not allowed (their P is 0, but 0 times NaN is not).
//
// S, the row sums and O are float32; P is rounded to the inputs' type, as the
// tensor cores take it (P in float32 as two 16-bit parts would take half as many
// products again): where the rounding of O alone leaves 2.1e-4 of the result in
// float16, it is 2.5e-4 with it. O is rescaled only when a row's maximum has grown by
// more than 2^8 since the last time: P stays below 2^8. float16 has few exponents:
// it holds P times 2^7, so that a probability keeps its digits down to 2^-21 of
// its row's largest (and is 0 below 2^-32).
// The scale is above 0, so that the largest score is the scaled largest
// product and a score of -inf stays one.
//
// Measured (bfloat16): 16384 x 4096, 2 samples of 16 heads of 64, 910 us, 604
// TFLOP/s; 16384 x 4099, 16 heads of 128 over 4, 1176 us, 935 TFLOP/s. Bound: the
// chain of a tile -- scores, about 1,100 cycles of exponentials, the product
// that takes them -- of which two tiles overlap; the tensor pipe is 23 and 36 %
// busy, the exponential unit 42 %.
#pragma once
#include <cuda.h>

#include <cstdint>

#include "attention.cuh"
#include "ptx.cuh"

namespace rdvb {
namespace attn {

constexpr int kTcTile = 128;       // query rows and keys of a tile
constexpr int kTcThreads = 12 * 32;
// Registers of a thread at launch, and after the softmax warps have taken
// some of the others' (2 x 208 + 88 = 3 x 168).
constexpr int kSoftmaxRegisters = 208, kOtherRegisters = 88;
constexpr float kGrowth = 8.0f;    // log2 of the growth of a row's maximum that O is rescaled at

struct TcParams {
    Params a;
    uint32_t* status;
    uint32_t k_steps;  // ceil(dim / 16)
    uint32_t n_pv;     // dim rounded up to 16
    int guarded;       // lengths or a mask: warp 10 takes part
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

// Shared-memory operands of a product in two words: the low one holds the
// address (16-byte units, 14 bits), so that a step along K is an addition.
// K-major, 128-byte swizzle: rows of 64 elements, 8-row groups 1024 bytes
// apart; 16 k are 32 bytes. MN-major, 128-byte swizzle: rows of 64 n elements
// per k, 8-k groups 1024 bytes apart, the next 64 n elements a tile (16 KB)
// on; 16 k are 2048 bytes.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k_major(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn_major(uint32_t saddr) {
    return (saddr >> 4) | ((kTcTile * 128u >> 4) << 16);
}
constexpr uint32_t kIdescBTransposed = 1u << 16;

// D (+)= A B^T with both operands in shared memory, one K step of 16.
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 x, {%1, %3};\n\t"
        "mov.b64 y, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "n"(kDescHigh), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// The same with A in TMEM.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 y, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "n"(kDescHigh), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// D = A B^T, both K-major tiles of 128 rows (descriptors of their starts),
// `steps` of at most kMost steps of 16.
template <int kMost>
__device__ __forceinline__ void product_rows(uint32_t d, uint32_t a, uint32_t b, uint32_t steps, uint32_t idesc) {
#pragma unroll
    for (uint32_t j = 0; j < kMost; ++j) {
        const uint32_t at = (j >> 2) * (kTcTile * 128 / 16) + (j & 3) * 2;
        if (j < steps) umma_ss(d, a + at, b + at, idesc, j > 0);
    }
}

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
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Which of the 128 keys from k0 on are allowed, as four words; the same in
// every lane of a warp. key_load reads the mask's bytes (a lane's four), so
// that a loop can have them on their way for its next step; key_bits votes.
// Call both with all 32 lanes.
struct KeyBits {
    uint32_t w[4];
    __device__ __forceinline__ bool all() const { return (w[0] & w[1] & w[2] & w[3]) == 0xffffffffu; }
    __device__ __forceinline__ bool none() const { return (w[0] | w[1] | w[2] | w[3]) == 0u; }
};
struct KeyLoad {
    int left;  // keys from k0 to the end, at most 128
    uint8_t m[4];
};
__device__ __forceinline__ KeyLoad key_load(const Params& p, int b, int64_t k0, int64_t end) {
    KeyLoad l;
    const int64_t left = end - k0;
    l.left = left < 0 ? 0 : left < 128 ? static_cast<int>(left) : 128;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        l.m[i] = p.mask && 32 * i + lane < l.left ? p.mask[b * p.mask_stride + k0 + 32 * i + lane] : 0;
    return l;
}
// The first `left` keys.
__device__ __forceinline__ KeyBits key_range(int left) {
    KeyBits bits;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = left - 32 * i;
        bits.w[i] = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
    }
    return bits;
}
__device__ __forceinline__ KeyBits key_bits(const Params& p, const KeyLoad& l) {
    if (!p.mask) return key_range(l.left);
    KeyBits bits;
#pragma unroll
    for (int i = 0; i < 4; ++i) bits.w[i] = __ballot_sync(0xffffffffu, l.m[i] != 0);
    return bits;
}

// Zeroes the rows of a 128-row tile (atoms of 64 elements, kAtoms of them)
// whose bit is not set: a lane a row, 16 bytes a store, its columns turned so
// that the lanes' banks differ. Call with all 32 lanes of one warp, then fence.
template <int kAtoms>
__device__ __forceinline__ void zero_rows(uint32_t tile, const KeyBits& bits) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (bits.w[i] == 0xffffffffu) continue;
        if (bits.w[i] >> lane & 1u) continue;
        const uint32_t row = tile + (32 * i + lane) * 128;
#pragma unroll
        for (int j = 0; j < 8 * kAtoms; ++j)
            st_shared_v4(row + (j >> 3) * (kTcTile * 128) + ((j + lane) & 7) * 16, 0, 0, 0, 0);
    }
}

// An item of the forward pass (two tiles of query rows of one head over the
// keys of one split) or of dQ (one tile).
struct TcItem {
    int q0, begin, end;  // positions fit 31 bits
    int h, hk, b, split, tiles;
    bool both;  // the second tile has rows
};
template <int kTiles>
__device__ __forceinline__ TcItem tc_item(const Params& p, uint32_t id) {
    TcItem t;
    const uint32_t q_items = static_cast<uint32_t>((p.q_len + kTiles * kTcTile - 1) / (kTiles * kTcTile));
    t.q0 = static_cast<int>(id % q_items) * (kTiles * kTcTile);
    id /= q_items;
    t.h = id % p.heads;
    id /= p.heads;
    t.b = id % p.batch;
    t.split = id / p.batch;
    t.hk = t.h / p.group;
    t.both = kTiles == 2 && t.q0 + kTcTile < p.q_len;
    const int64_t len = length_of(p, t.b), begin = t.split * p.split_len, end = min(len, begin + p.split_len);
    t.begin = static_cast<int>(begin);
    t.end = static_cast<int>(end);
    t.tiles = end > begin ? static_cast<int>((end - begin + kTcTile - 1) / kTcTile) : 0;
    return t;
}

// The next item of this block with keys, from `id` on; false past the last.
template <int kTiles>
__device__ __forceinline__ bool next_item(const Params& p, uint32_t items, uint32_t& id, TcItem& t) {
    for (; id < items; id += gridDim.x) {
        t = tc_item<kTiles>(p, id);
        if (t.tiles > 0) return true;
    }
    return false;
}

// 2^x for x <= 128: x = n + f, |f| <= 1/2, times a polynomial of degree 4 in
// f with the least largest relative error (2.6e-6, a hundredth of what P is
// rounded by). Below 2^-126 it is 0, a NaN stays one. It runs on the FMA
// pipe, beside the exponential unit that ex2 takes.
__device__ __forceinline__ void exp2_poly2(float& x, float& y) {
    constexpr float kRound = 12582912.0f + 127.0f;  // adding it leaves n + 127 in the low bits
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(x));  // -127
    asm("max.NaN.f32 %0, %0, 0fC2FE0000;" : "+f"(y));
    float n0 = x, n1 = y;
    add2(n0, n1, kRound, kRound);
    const float s0 = __uint_as_float(__float_as_uint(n0) << 23), s1 = __uint_as_float(__float_as_uint(n1) << 23);
    add2(n0, n1, -kRound, -kRound);
    float f0 = n0, f1 = n1;
    fma2(f0, f1, -1.0f, -1.0f, x, y);
    float p0 = f0, p1 = f1;
    fma2(p0, p1, 0.009570101908f, 0.009570101908f, 0.05591786032f, 0.05591786032f);
    fma2(p0, p1, f0, f1, 0.2402474483f, 0.2402474483f);
    fma2(p0, p1, f0, f1, 0.6931218147f, 0.6931218147f);
    fma2(p0, p1, f0, f1, 0.9999992614f, 0.9999992614f);
    mul2(p0, p1, s0, s1);
    x = p0;
    y = p1;
}
// 2^x and 2^y: `poly` of every four pairs by the polynomial.
template <int kPoly>
__device__ __forceinline__ void exp2_pair(float& x, float& y, int pair) {
    if (pair % 4 >= 4 - kPoly) {
        exp2_poly2(x, y);
    } else {
        x = exp2_approx(x);
        y = exp2_approx(y);
    }
}

template <int DP>
struct TcForward {
    static constexpr int kAtoms = DP / 64;
    static constexpr uint32_t kTileBytes = kTcTile * DP * 2;
    static constexpr int kStages = DP == 64 ? 3 : 2;  // K and V tiles in flight
    // TMEM columns: S and O of the two tiles and, where there is room, P beside S instead of over it
    static constexpr bool kOwnP = DP == 64;
    static constexpr int kIssuers = DP == 64 ? 2 : 1;
    static constexpr uint32_t kColS = 0, kColO = 256, kColP = kOwnP ? 384 : 0, kStepP = kOwnP ? 64 : 128;
    static constexpr uint32_t kOffK = 2 * kTileBytes, kOffV = kOffK + kStages * kTileBytes,
                              kOffBar = kOffV + kStages * kTileBytes;
    static constexpr uint32_t kBytes = kOffBar + 256 + 1024;  // barriers; slack for the 1024-byte alignment
    // Of four pairs of exponentials, those taken by the polynomial: at 64
    // dimensions the exponential unit is what the products wait for.
    static constexpr int kPoly = DP == 64 ? 1 : 0;
};

template <int DP, bool kBf16>
__global__ void __launch_bounds__(kTcThreads, 1)
    tc_forward_kernel(const TcParams p, const uint32_t items, const __grid_constant__ TcMap map_q,
                      const __grid_constant__ TcMap map_k, const __grid_constant__ TcMap map_v) {
    using F = TcForward<DP>;
    constexpr int kStages = F::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t s_q = base, s_k = base + F::kOffK, s_v = base + F::kOffV, bars = base + F::kOffBar;
    const uint32_t q_full = bars, q_empty = bars + 8, drain = bars + 16, s_full = bars + 24, s_read = bars + 40,
                   p_full = bars + 56, o_full = bars + 72, o_read = bars + 88, k_full = bars + 104,
                   k_empty = bars + 128, v_tma = bars + 152, v_full = bars + 176, v_empty = bars + 200;
    const uint32_t tmem_slot = bars + 224;
    volatile uint32_t* abort_flag =
        reinterpret_cast<volatile uint32_t*>(smem_raw + (bars - smem_addr(smem_raw)) + 228);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Params& a = p.a;

    if (threadIdx.x == 0) {
        *abort_flag = 0u;
        mbar_init(q_full, 2);  // an arrival a tile
        mbar_init(q_empty, 2);  // the empty barriers: an arrival a query tile
        mbar_init(drain, F::kIssuers);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + 8 * i, 1);
            mbar_init(s_read + 8 * i, 4);
            mbar_init(p_full + 8 * i, 4);
            mbar_init(o_full + 8 * i, 1);
            mbar_init(o_read + 8 * i, 4);
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(k_full + 8 * i, 1);
            mbar_init(k_empty + 8 * i, 2);
            mbar_init(v_tma + 8 * i, 1);
            mbar_init(v_full + 8 * i, 1);
            mbar_init(v_empty + 8 * i, 2);
        }
        fence_mbarrier_init();
    }
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
        if (warp == 8) {
            if (lane == 0) {
                uint32_t n = 0, k_sent = 0, v_sent = 0, q_sent = 0, id = blockIdx.x;  // n: key tiles so far
                TcItem t;
                bool ok = true;
                for (; ok && next_item<2>(a, items, id, t); id += gridDim.x) {
                    if (!mbar_wait(q_empty, (q_sent & 1) ^ 1, abort_flag, p.status, kStatusTimeoutWEmpty)) break;
                    ++q_sent;
                    tc_load<F::kAtoms>(s_q, map_q, t.h, t.q0, t.b, q_full);
                    if (t.both)
                        tc_load<F::kAtoms>(s_q + F::kTileBytes, map_q, t.h, t.q0 + kTcTile, t.b, q_full);
                    else
                        mbar_arrive(q_full);
                    for (int i = 0; i < t.tiles; ++i, ++n) {
                        const uint32_t s = n % kStages, parity = ((n / kStages) & 1) ^ 1;
                        const int64_t k0 = t.begin + static_cast<int64_t>(i) * kTcTile;
                        ok = mbar_wait(k_empty + 8 * s, parity, abort_flag, p.status, kStatusTimeoutXEmpty);
                        if (!ok) break;
                        tc_load<F::kAtoms>(s_k + s * F::kTileBytes, map_k, t.hk, k0, t.b, k_full + 8 * s);
                        ++k_sent;
                        ok = mbar_wait(v_empty + 8 * s, parity, abort_flag, p.status, kStatusTimeoutXEmpty);
                        if (!ok) break;
                        tc_load<F::kAtoms>(s_v + s * F::kTileBytes, map_v, t.hk, k0, t.b, v_tma + 8 * s);
                        ++v_sent;
                    }
                }
                // no copy may be in flight when the block ends
                if (q_sent > 0) drain_wait(q_full, (q_sent - 1) & 1, p.status);
                for (uint32_t s = 0; s < kStages; ++s) {
                    if (k_sent > s) drain_wait(k_full + 8 * s, ((k_sent - 1 - s) / kStages) & 1, p.status);
                    if (v_sent > s) drain_wait(v_tma + 8 * s, ((v_sent - 1 - s) / kStages) & 1, p.status);
                }
            }
        } else if (warp == 9 || (warp == 11 && F::kIssuers == 2)) {
            if (lane == 0) {
                // Products of query tile w: of both, or of this warp's own. A barrier that is told apart by parity
                // must not move on by two phases behind a warp that waits on it. So the second tile's own issuer
                // goes through every item: where one has no second tile it waits for what it would have read and
                // releases that at once, and no phase ends without it. A single issuer's releases count twice there.
                const int w0 = F::kIssuers == 2 && warp == 11 ? 1 : 0;
                constexpr int kMine = F::kIssuers == 2 ? 1 : 2;
                const uint32_t idesc_s = umma_idesc_f16(kTcTile, kBf16);
                const uint32_t idesc_o = umma_idesc_f16(p.n_pv, kBf16) | kIdescBTransposed;
                const uint32_t v_ready = p.guarded ? v_full : v_tma;
                const uint32_t q_desc = desc_k_major(s_q), k_desc = desc_k_major(s_k), v_desc = desc_mn_major(s_v);
                uint32_t scores[kMine] = {}, begun[kMine] = {};  // S issued (P V: one less or as many), O begun
                auto wait = [&](uint32_t bar, uint32_t parity, uint32_t code) {
                    return mbar_wait(bar, parity & 1, abort_flag, p.status, code);
                };
                auto release = [&](uint32_t bar, bool both) {
                    umma_commit(bar);
                    if (F::kIssuers == 1 && !both) umma_commit(bar);
                };
                // Whether item v has this warp's m-th tile. With an issuer a tile, the functions below are called for
                // every item; with one, for the tiles that there are.
                auto has = [&](int m, const TcItem& v) { return w0 + m == 0 || v.both; };
                auto takes = [&](int m, const TcItem& v) { return F::kIssuers == 2 || has(m, v); };
                // S of key tile i (the block's n-th) of item v, its query_item-th
                auto score = [&](int m, const TcItem& v, int i, uint32_t n, uint32_t query_item) {
                    const uint32_t s = n % kStages, w = w0 + m;
                    if (i == 0 && m == 0 && !wait(q_full, query_item, kStatusTimeoutWFull)) return false;
                    if (m == 0 && !wait(k_full + 8 * s, n / kStages, kStatusTimeoutXFull)) return false;
                    if (!has(m, v)) {
                        mbar_arrive(k_empty + 8 * s);
                        if (i == v.tiles - 1) mbar_arrive(q_empty);
                        return true;
                    }
                    // the softmax has read the last scores, and P does not lie over them or was taken
                    if (scores[m] > 0 &&
                        !wait((F::kOwnP ? s_read : o_full) + 8 * w, scores[m] - 1, kStatusTimeoutAccFull))
                        return false;
                    tc_fence_after();
                    product_rows<DP / 16>(tmem + F::kColS + 128 * w, q_desc + w * (F::kTileBytes / 16),
                                          k_desc + s * (F::kTileBytes / 16), p.k_steps, idesc_s);
                    umma_commit(s_full + 8 * w);
                    ++scores[m];
                    release(k_empty + 8 * s, v.both);
                    if (i == v.tiles - 1) release(q_empty, v.both);
                    return true;
                };
                // O += P V with the block's n-th key tile; `mixes` before it
                auto mix = [&](int m, const TcItem& v, int i, uint32_t n, uint32_t mixes) {
                    const uint32_t s = n % kStages, w = w0 + m;
                    if (m == 0 && !wait(v_ready + 8 * s, n / kStages, kStatusTimeoutXFull)) return false;
                    if (!has(m, v)) {
                        mbar_arrive(v_empty + 8 * s);
                        return true;
                    }
                    if (i == 0 && begun[m]++ > 0 && !wait(o_read + 8 * w, begun[m] - 2, kStatusTimeoutDrain))
                        return false;
                    if (!wait(p_full + 8 * w, mixes, kStatusTimeoutAFull)) return false;
                    tc_fence_after();
#pragma unroll
                    for (uint32_t j = 0; j < kTcTile / 16; ++j)
                        umma_ts(tmem + F::kColO + DP * w, tmem + F::kColP + F::kStepP * w + 8 * j,
                                v_desc + s * (F::kTileBytes / 16) + 128 * j, idesc_o, i > 0 || j > 0);
                    umma_commit(o_full + 8 * w);
                    release(v_empty + 8 * s, v.both);
                    return true;
                };
                uint32_t id = blockIdx.x, n = 0, query_items = 0;
                TcItem t, u;
                bool ok = true, have = next_item<2>(a, items, id, t);
#pragma unroll
                for (int m = 0; m < kMine; ++m)
                    if (ok && have && takes(m, t)) ok = score(m, t, 0, 0, 0);
                while (ok && have) {
                    uint32_t next = id + gridDim.x;  // u: the item after t
                    const bool more = next_item<2>(a, items, next, u);
                    ++query_items;
                    for (int i = 0; ok && i < t.tiles; ++i, ++n) {
                        const bool within = i + 1 < t.tiles;
#pragma unroll
                        for (int m = 0; m < kMine; ++m) {
                            const bool here = takes(m, t);
                            const bool ahead = within ? here : more && takes(m, u);
                            const uint32_t mixes = scores[m] - 1;
                            if (F::kOwnP && ok && ahead)
                                ok = within ? score(m, t, i + 1, n + 1, query_items - 1)
                                            : score(m, u, 0, n + 1, query_items);
                            if (ok && here) ok = mix(m, t, i, n, mixes);
                            if (!F::kOwnP && ok && ahead)
                                ok = within ? score(m, t, i + 1, n + 1, query_items - 1)
                                            : score(m, u, 0, n + 1, query_items);
                        }
                    }
                    have = more;
                    t = u;
                    id = next;
                }
                umma_commit(drain);
                drain_wait(drain, 0, p.status);
            }
        } else if (warp == 10) {
            if (p.guarded) {
                uint32_t n = 0, id = blockIdx.x;
                TcItem t;
                bool ok = true;
                for (; ok && next_item<2>(a, items, id, t); id += gridDim.x) {
                    KeyLoad keys = key_load(a, t.b, t.begin, t.end);
                    for (int i = 0; i < t.tiles; ++i, ++n) {
                        const uint32_t s = n % kStages;
                        const KeyBits bits = key_bits(a, keys);
                        keys = key_load(a, t.b, t.begin + (i + 1ll) * kTcTile, t.end);
                        ok = mbar_wait_warp(v_tma + 8 * s, (n / kStages) & 1, abort_flag, p.status, kStatusTimeoutXFull);
                        if (!ok) break;
                        if (!bits.all()) {
                            zero_rows<F::kAtoms>(s_v + s * F::kTileBytes, bits);
                            fence_proxy_async_smem();
                            __syncwarp();
                        }
                        if (lane == 0) mbar_arrive(v_full + 8 * s);
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
        const int w = warp >> 2;
        const uint32_t row_base = tmem + (static_cast<uint32_t>(warp & 3) << 21);  // lane 32 (warp % 4) of TMEM
        const uint32_t col_s = row_base + F::kColS + 128 * w, col_o = row_base + F::kColO + DP * w,
                       col_p = row_base + F::kColP + F::kStepP * w;
        const float c = a.scale * kLog2e;
        constexpr float kHeld = kBf16 ? 0.0f : 7.0f;  // P, its sum and O are held times 2^kHeld
        uint32_t n = 0;                               // key tiles of this query tile so far
        bool ok = true;
        for (uint32_t id = blockIdx.x; ok && id < items; id += gridDim.x) {
            const TcItem t = tc_item<2>(a, id);
            if (w && !t.both) continue;
            float top = -INFINITY, total = 0.0f;
            bool any = false;
            KeyLoad keys = key_load(a, t.b, t.begin, t.end);
            for (int i = 0; i < t.tiles; ++i, ++n) {
                KeyBits bits;
                bool whole;
                if (a.mask) {
                    bits = key_bits(a, keys);
                    keys = key_load(a, t.b, t.begin + (i + 1ll) * kTcTile, t.end);
                    whole = bits.all();
                    any |= !bits.none();
                } else {
                    bits = key_range(t.end - t.begin - i * kTcTile);
                    whole = i + 1 < t.tiles || (t.end - t.begin) % kTcTile == 0;
                    any = true;
                }
                if (!(ok = mbar_wait_warp(s_full + 8 * w, n & 1, abort_flag, p.status, kStatusTimeoutAccFull))) break;
                tc_fence_after();
                uint32_t r[8][16];
#pragma unroll
                for (int j = 0; j < 8; ++j) tmem_ld16(col_s + 16 * j, r[j]);
                tmem_wait_ld(r[0]);
#pragma unroll
                for (int j = 1; j < 8; ++j) reg_barrier(r[j]);
                if (F::kOwnP) {  // S has been read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_read + 8 * w);
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
                // the last product has read P and written O
                if (i > 0 && !mbar_wait_warp(o_full + 8 * w, (n - 1) & 1, abort_flag, p.status, kStatusTimeoutAccFull)) {
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
                            tmem_ld16(col_o + j, o);
                            tmem_wait_ld(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st8(col_o + j, *reinterpret_cast<uint32_t(*)[8]>(&o[0]));
                            tmem_st8(col_o + j + 8, *reinterpret_cast<uint32_t(*)[8]>(&o[8]));
                        }
                    }
                }
                const float minus = top == -INFINITY ? 0.0f : kHeld - top;
                float sum[4] = {};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t packed[8];
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        float x = __uint_as_float(r[j][e]), y = __uint_as_float(r[j][e + 1]);
                        fma2(x, y, c, c, minus, minus);
                        exp2_pair<F::kPoly>(x, y, e / 2);
                        add2(sum[e & 2], sum[(e & 2) + 1], x, y);
                        packed[e / 2] = kBf16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
                    }
                    tmem_st8(col_p + 8 * j, packed);
                }
                total += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * w);
            }
            if (t.tiles > 0 && ok)
                ok = mbar_wait_warp(o_full + 8 * w, (n - 1) & 1, abort_flag, p.status, kStatusTimeoutAccFull);
            if (!ok) break;
            tc_fence_after();
            const int64_t q = t.q0 + static_cast<int>(threadIdx.x);  // 128 rows a tile: warps 4-7 are its second half
            const bool mine = q < a.q_len;
            const int64_t row = (t.b * a.q_len + q) * a.heads + t.h;
            const int64_t rows = static_cast<int64_t>(a.batch) * a.q_len * a.heads;
            const float inv = any ? 1.0f / total : 0.0f;
#pragma unroll 1
            for (int j = 0; j < a.dim; j += 16) {
                uint32_t r[16] = {};
                __syncwarp();  // the load takes the whole warp; lanes past q_len skipped the last store
                if (t.tiles > 0) {
                    tmem_ld16(col_o + j, r);
                    tmem_wait_ld(r);
                }
                if (!mine) continue;
                if (a.splits > 1) {
                    float* dst = a.part + (t.split * rows + row) * a.dim + j;
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        if (j + e < a.dim)
                            *reinterpret_cast<uint4*>(dst + e) =
                                any ? make_uint4(r[e], r[e + 1], r[e + 2], r[e + 3]) : make_uint4(0, 0, 0, 0);
                } else {
                    uint16_t* dst = static_cast<uint16_t*>(a.o) + row * a.dim + j;
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        uint32_t v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float x = __uint_as_float(r[e + 2 * k]) * inv,
                                        y = __uint_as_float(r[e + 2 * k + 1]) * inv;
                            v[k] = !any ? 0u : kBf16 ? pack_bf16x2(x, y) : pack_f16x2(x, y);
                        }
                        if (j + e < a.dim) *reinterpret_cast<uint4*>(dst + e) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
            }
            if (t.tiles > 0) {  // the next item may begin its O
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_read + 8 * w);
            }
            if (mine) {
                if (a.splits > 1) {
                    a.part_stat[2 * (t.split * rows + row)] = top - kHeld;
                    a.part_stat[2 * (t.split * rows + row) + 1] = any ? total : -1.0f;
                } else if (a.lse) {
                    a.lse[(static_cast<int64_t>(t.b) * a.heads + t.h) * a.q_len + q] =
                        any ? (top - kHeld + log2f(total)) * kLn2 : -INFINITY;
                }
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

}  // namespace attn
}  // namespace rdvb
