// Attention of query positions to a sequence of another length, forward and
// backward, for every element type, head dimension up to 256 and stride:
//   S = scale Q K^T,  P = softmax of S over the allowed keys,  O = P V,
//   lse = log sum exp S,  delta = rowsum(dO O),  dS = P (dO V^T - delta),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,
// dK and dV summed over the query heads that share the key head. A key is
// allowed below its sample's length and where the mask is true; a row with
// no allowed key is 0 and gives no gradient. What lies at a key that is not
// allowed is never read, so NaN and infinities there stay there.
//
// CUDA cores, float32 throughout: the exact path of float32 inputs, and the
// path of 16-bit inputs that the tensor-core kernels do not take. Tiles of
// 64 queries x 64 keys (32 x 32 above 128 dimensions) in shared memory, a
// 4 x 4 piece of S a thread, one pass over the keys with the running maximum
// and sum. Bound: the FMA pipe (half busy), and the shared-memory reads that
// feed it; 2048 x 2048, 4 samples of 8 heads of 64: forward 1330 us, 26 TFLOP/s,
// backward 3580 us, 24 TFLOP/s of the formula's work.
// Gradients take two kernels, one by query tile (dQ) and one by key tile (dK,
// dV), so that every sum has one owner and a fixed order: no atomics. Where
// a call has few tiles, the long axis is split and the parts are joined in
// order by a second launch.
#pragma once
#include <cstdint>

#include "types.cuh"

namespace rdvb {
namespace attn {

constexpr int kThreads = 256;

struct Strides {
    int64_t batch, pos, head;
};

struct Params {
    const void *q, *k, *v;
    const void *out, *dout;  // backward: dense
    void *o, *dq, *dk, *dv;  // dense
    float* lse;              // [batch, heads, q_len]
    float* delta;            // [batch, heads, q_len]
    float* part;             // partial results of splits: rows of the forward pass, dQ
    float* part_kv;          // of dK and dV
    float* part_stat;
    const int32_t* lengths;  // may be null
    const uint8_t* mask;     // may be null
    int64_t mask_stride;
    Strides qs, ks, vs;
    int64_t q_len, kv_len;
    int dtype, batch, heads, kv_heads, group, dim;
    int splits;
    int64_t split_len;  // keys (forward, dQ) or query tiles of the group's heads (dK, dV) of a split
    int wide;           // rows of q, k, v, out, dout can be read four elements at a time
    float scale;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float load1(const void* p, int dtype, int64_t i) {
    if (dtype == 0) return static_cast<const float*>(p)[i];
    if (dtype == 1) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store1(void* p, int dtype, int64_t i, float v) {
    if (dtype == 0)
        static_cast<float*>(p)[i] = v;
    else if (dtype == 1)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float4 load4(const void* p, int dtype, int64_t i, int count, int wide) {
    float v[4] = {};
    if (wide && count >= 4) {
        if (dtype == 0)
            load_f32<float, 4>(static_cast<const float*>(p) + i, v);
        else if (dtype == 1)
            load_f32<__half, 4>(static_cast<const __half*>(p) + i, v);
        else
            load_f32<__nv_bfloat16, 4>(static_cast<const __nv_bfloat16*>(p) + i, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < count) v[j] = load1(p, dtype, i + j);
    }
    return make_float4(v[0], v[1], v[2], v[3]);
}

// Keys of a sample below its length.
__device__ __forceinline__ int64_t length_of(const Params& p, int b) {
    if (!p.lengths) return p.kv_len;
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : (n < p.kv_len ? n : p.kv_len);
}
__device__ __forceinline__ bool allowed(const Params& p, int b, int64_t key, int64_t len) {
    return key < len && (!p.mask || p.mask[b * p.mask_stride + key] != 0);
}

template <int DP>
struct Shape {
    static constexpr int kTile = DP > 128 ? 32 : 64;  // queries and keys of a tile
    static constexpr int kPer = kTile / 16;           // rows and columns of S a thread
    static constexpr int kRow = DP + 4;               // floats of a tile row in shared memory
    static constexpr int kPRow = kTile + 4;
    static constexpr int kCols = DP / 16;  // dimensions of an output row a thread
    static constexpr int kTileFloats = kTile * kRow;
    static constexpr int kPFloats = kTile * kPRow;
    static constexpr int kForwardBytes = (3 * kTileFloats + kPFloats + kTile) * 4;
    static constexpr int kBackwardBytes = (4 * kTileFloats + 2 * kPFloats + 3 * kTile) * 4;
};

// Dimension of a thread's j-th output element: chunks of up to four
// consecutive ones, 16 threads side by side.
template <int DP>
__device__ __forceinline__ int out_dim(int tx, int j) {
    constexpr int kChunk = DP >= 64 ? 4 : 2;
    return (j / kChunk) * 16 * kChunk + tx * kChunk + j % kChunk;
}

// Rows [row0, row0 + tile) of one head into shared memory; rows past the end
// or not in s_ok (when given), and dimensions past dim, are 0.
template <int DP>
__device__ __forceinline__ void load_tile(const Params& p, const void* src, int64_t head_base, int64_t stride,
                                          int64_t row0, int64_t row_end, const float* s_ok, float* dst) {
    constexpr int kTile = Shape<DP>::kTile, kQuads = DP / 4;
    for (int e = threadIdx.x; e < kTile * kQuads; e += kThreads) {
        const int r = e / kQuads, d = (e % kQuads) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (row0 + r < row_end && d < p.dim && (!s_ok || s_ok[r] != 0.0f))
            v = load4(src, p.dtype, head_base + (row0 + r) * stride + d, p.dim - d, p.wide);
        *reinterpret_cast<float4*>(dst + r * Shape<DP>::kRow + d) = v;
    }
}

// s[i][j] = a[ty + 16 i] . b[tx + 16 j] over the DP dimensions.
template <int DP>
__device__ __forceinline__ void tile_dot(const float* a, const float* b, int ty, int tx,
                                         float (&s)[Shape<DP>::kPer][Shape<DP>::kPer]) {
    constexpr int kPer = Shape<DP>::kPer, kRow = Shape<DP>::kRow;
    // even and odd dimensions' sums side by side: one packed instruction for two products
    float odd[kPer][kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int j = 0; j < kPer; ++j) s[i][j] = odd[i][j] = 0.0f;
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
        float4 x[kPer], y[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = *reinterpret_cast<const float4*>(a + (ty + 16 * i) * kRow + d);
#pragma unroll
        for (int j = 0; j < kPer; ++j) y[j] = *reinterpret_cast<const float4*>(b + (tx + 16 * j) * kRow + d);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                float p0 = x[i].x, p1 = x[i].y;
                fma2(p0, p1, y[j].x, y[j].y, s[i][j], odd[i][j]);
                s[i][j] = x[i].z, odd[i][j] = x[i].w;
                fma2(s[i][j], odd[i][j], y[j].z, y[j].w, p0, p1);
            }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int j = 0; j < kPer; ++j) s[i][j] += odd[i][j];
}

// acc[i][j] += sum over n of w[ty + 16 i][n] x[n][out_dim(tx, j)].
template <int DP>
__device__ __forceinline__ void tile_mac(const float* w, const float* x, int ty, int tx,
                                         float (&acc)[Shape<DP>::kPer][Shape<DP>::kCols]) {
    constexpr int kPer = Shape<DP>::kPer, kRow = Shape<DP>::kRow, kPRow = Shape<DP>::kPRow, kCols = Shape<DP>::kCols;
#pragma unroll 2
    for (int n = 0; n < Shape<DP>::kTile; n += 4) {
        float a[kPer][4];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(w + (ty + 16 * i) * kPRow + n);
            a[i][0] = v.x, a[i][1] = v.y, a[i][2] = v.z, a[i][3] = v.w;
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            float b[kCols];
            constexpr int kChunk = DP >= 64 ? 4 : 2;
#pragma unroll
            for (int j = 0; j < kCols; j += kChunk) {
                const auto v = *reinterpret_cast<const Vec<float, kChunk>*>(x + (n + m) * kRow + out_dim<DP>(tx, j));
#pragma unroll
                for (int i = 0; i < kChunk; ++i) b[j + i] = v.v[i];
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i)
#pragma unroll
                for (int j = 0; j < kCols; j += 2) {
                    float p0 = b[j], p1 = b[j + 1];
                    fma2(p0, p1, a[i][m], a[i][m], acc[i][j], acc[i][j + 1]);
                    acc[i][j] = p0, acc[i][j + 1] = p1;
                }
        }
    }
}

__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Forward. A block: one query tile of one head, over the keys of one split.
// With splits > 1 it leaves its unnormalised rows in part, and the maximum
// and sum (-1 where it saw no allowed key) in part_stat.
template <int DP>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Params p) {
    using Sh = Shape<DP>;
    constexpr int kTile = Sh::kTile, kPer = Sh::kPer;
    extern __shared__ float smem[];
    float *s_q = smem, *s_k = s_q + Sh::kTileFloats, *s_v = s_k + Sh::kTileFloats, *s_p = s_v + Sh::kTileFloats;
    float* s_ok = s_p + Sh::kPFloats;
    const int64_t q_tiles = (p.q_len + kTile - 1) / kTile;
    int64_t id = blockIdx.x;
    const int64_t q0 = id % q_tiles * kTile;
    id /= q_tiles;
    const int h = static_cast<int>(id % p.heads);
    id /= p.heads;
    const int b = static_cast<int>(id % p.batch), split = static_cast<int>(id / p.batch);
    const int hk = h / p.group;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int64_t len = length_of(p, b);
    const int64_t begin = split * p.split_len, end = min(len, begin + p.split_len);
    const float c = p.scale * kLog2e;
    float top[kPer], total[kPer], acc[kPer][Sh::kCols] = {};
    bool any = false;
#pragma unroll
    for (int i = 0; i < kPer; ++i) top[i] = -INFINITY, total[i] = 0.0f;
    load_tile<DP>(p, p.q, b * p.qs.batch + h * p.qs.head, p.qs.pos, q0, p.q_len, nullptr, s_q);
    for (int64_t k0 = begin; k0 < end; k0 += kTile) {
        __syncthreads();
        bool mine = false;
        if (threadIdx.x < kTile) {
            mine = k0 + threadIdx.x < end && allowed(p, b, k0 + threadIdx.x, len);
            s_ok[threadIdx.x] = mine ? 1.0f : 0.0f;
        }
        if (!__syncthreads_or(mine)) continue;
        any = true;
        load_tile<DP>(p, p.k, b * p.ks.batch + hk * p.ks.head, p.ks.pos, k0, end, s_ok, s_k);
        load_tile<DP>(p, p.v, b * p.vs.batch + hk * p.vs.head, p.vs.pos, k0, end, s_ok, s_v);
        __syncthreads();
        float s[kPer][kPer];
        tile_dot<DP>(s_q, s_k, ty, tx, s);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            float m = -INFINITY;
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (s_ok[tx + 16 * j] != 0.0f) m = fmaxf(m, s[i][j] * c);
            m = fmaxf(top[i], half_warp_max(m));
            const float base = m == -INFINITY ? 0.0f : m;  // every score so far is -inf
            const float old = exp2f(top[i] - base);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const float e = s_ok[tx + 16 * j] != 0.0f ? exp2f(fmaf(s[i][j], c, -base)) : 0.0f;
                s_p[(ty + 16 * i) * Sh::kPRow + tx + 16 * j] = e;
                sum += e;
            }
            total[i] = fmaf(total[i], old, half_warp_sum(sum));
            top[i] = m;
#pragma unroll
            for (int j = 0; j < Sh::kCols; ++j) acc[i][j] *= old;
        }
        __syncthreads();
        tile_mac<DP>(s_p, s_v, ty, tx, acc);
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int64_t q = q0 + ty + 16 * i;
        if (q >= p.q_len) continue;
        const int64_t row = (b * p.q_len + q) * p.heads + h;
        if (p.splits > 1) {
            const int64_t rows = static_cast<int64_t>(p.batch) * p.q_len * p.heads;
            float* dst = p.part + (split * rows + row) * p.dim;
#pragma unroll
            for (int j = 0; j < Sh::kCols; ++j)
                if (out_dim<DP>(tx, j) < p.dim) dst[out_dim<DP>(tx, j)] = acc[i][j];
            if (tx == 0) {
                p.part_stat[2 * (split * rows + row)] = top[i];
                p.part_stat[2 * (split * rows + row) + 1] = any ? total[i] : -1.0f;
            }
            continue;
        }
        const float inv = any ? 1.0f / total[i] : 0.0f;
#pragma unroll
        for (int j = 0; j < Sh::kCols; ++j)
            if (out_dim<DP>(tx, j) < p.dim)
                store1(p.o, p.dtype, row * p.dim + out_dim<DP>(tx, j), any ? acc[i][j] * inv : 0.0f);
        if (tx == 0 && p.lse)
            p.lse[(static_cast<int64_t>(b) * p.heads + h) * p.q_len + q] =
                any ? (top[i] + log2f(total[i])) * kLn2 : -INFINITY;
    }
}

constexpr int kMaxSplits = 128;

// Joins the splits of the forward pass in split order: a warp a row's 32
// dimensions, a lane up to four splits' weights.
__global__ void __launch_bounds__(kThreads) join_forward_kernel(const Params p) {
    const int64_t rows = static_cast<int64_t>(p.batch) * p.q_len * p.heads;
    const int chunks = (p.dim + 31) / 32;
    const int64_t id = blockIdx.x * static_cast<int64_t>(kThreads / 32) + threadIdx.x / 32;
    const int64_t row = id / chunks;
    if (row >= rows) return;
    const int lane = threadIdx.x % 32, d = static_cast<int>(id % chunks) * 32 + lane;
    constexpr int kMine = kMaxSplits / 32;
    float top = -INFINITY, tops[kMine], totals[kMine];
    bool any = false;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int s = 32 * i + lane;
        tops[i] = -INFINITY;
        totals[i] = 0.0f;
        if (s < p.splits) {
            const float2 v = reinterpret_cast<const float2*>(p.part_stat)[s * rows + row];
            if (v.y != -1.0f) {
                any = true;
                tops[i] = v.x;
                totals[i] = v.y;
            }
        }
        top = fmaxf(top, tops[i]);
    }
    any = __any_sync(0xffffffffu, any);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.0f : top;
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        tops[i] = exp2f(tops[i] - base);  // the split's weight
        total = fmaf(totals[i], tops[i], total);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    float acc = 0.0f;
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int n = min(32, p.splits - 32 * i);
#pragma unroll 16
        for (int s = 0; s < n; ++s) {
            const float f = __shfl_sync(0xffffffffu, tops[i], s);
            // a split without an allowed key has weight 0 and wrote zeros
            if (d < p.dim) acc = fmaf(p.part[((32 * i + s) * rows + row) * p.dim + d], f, acc);
        }
    }
    if (d < p.dim) store1(p.o, p.dtype, row * p.dim + d, any ? acc / total : 0.0f);
    if (d == 0 && p.lse) {
        const int64_t h = row % p.heads, q = row / p.heads % p.q_len, b = row / p.heads / p.q_len;
        p.lse[(b * p.heads + h) * p.q_len + q] = any ? (base + log2f(total)) * kLn2 : -INFINITY;
    }
}

// delta = rowsum(dO O): a warp a row.
__global__ void __launch_bounds__(kThreads) delta_kernel(const Params p) {
    const int64_t rows = static_cast<int64_t>(p.batch) * p.q_len * p.heads;
    const int64_t row = blockIdx.x * static_cast<int64_t>(kThreads / 32) + threadIdx.x / 32;
    if (row >= rows) return;
    float sum = 0.0f;
    for (int d = (threadIdx.x % 32) * 4; d < p.dim; d += 128) {
        const float4 a = load4(p.out, p.dtype, row * p.dim + d, p.dim - d, p.wide);
        const float4 g = load4(p.dout, p.dtype, row * p.dim + d, p.dim - d, p.wide);
        sum += a.x * g.x + a.y * g.y + a.z * g.z + a.w * g.w;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x % 32 == 0) {
        const int64_t h = row % p.heads, q = row / p.heads % p.q_len, b = row / p.heads / p.q_len;
        p.delta[(b * p.heads + h) * p.q_len + q] = sum;
    }
}

// P and dS of one tile: s and t hold q . k and dO . v on entry, P and dS
// after. A pair that is not allowed is selected to 0.
template <int DP>
__device__ __forceinline__ void gradient_tile(const Params& p, const float* s_ok, const float* s_lse,
                                              const float* s_delta, int64_t q_left, int ty, int tx,
                                              float (&s)[Shape<DP>::kPer][Shape<DP>::kPer],
                                              float (&t)[Shape<DP>::kPer][Shape<DP>::kPer]) {
    constexpr int kPer = Shape<DP>::kPer;
    const float c = p.scale * kLog2e;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int r = ty + 16 * i;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const bool on = s_ok[tx + 16 * j] != 0.0f && r < q_left;
            s[i][j] = on ? exp2f(fmaf(s[i][j], c, -s_lse[r])) : 0.0f;
            t[i][j] = on ? s[i][j] * (t[i][j] - s_delta[r]) : 0.0f;
        }
    }
}

template <int DP>
__device__ __forceinline__ void load_stats(const Params& p, int64_t base, int64_t q0, float* s_lse, float* s_delta) {
    if (threadIdx.x < Shape<DP>::kTile) {
        const bool in = q0 + threadIdx.x < p.q_len;
        s_lse[threadIdx.x] = in ? p.lse[base + q0 + threadIdx.x] * kLog2e : 0.0f;
        s_delta[threadIdx.x] = in ? p.delta[base + q0 + threadIdx.x] : 0.0f;
    }
}

// dQ. A block: one query tile of one head, over the keys of one split.
template <int DP>
__global__ void __launch_bounds__(kThreads) dq_kernel(const Params p) {
    using Sh = Shape<DP>;
    constexpr int kTile = Sh::kTile, kPer = Sh::kPer;
    extern __shared__ float smem[];
    float *s_q = smem, *s_do = s_q + Sh::kTileFloats, *s_k = s_do + Sh::kTileFloats, *s_v = s_k + Sh::kTileFloats;
    float *s_ds = s_v + Sh::kTileFloats, *s_ok = s_ds + 2 * Sh::kPFloats, *s_lse = s_ok + kTile,
          *s_delta = s_lse + kTile;
    const int64_t q_tiles = (p.q_len + kTile - 1) / kTile;
    int64_t id = blockIdx.x;
    const int64_t q0 = id % q_tiles * kTile;
    id /= q_tiles;
    const int h = static_cast<int>(id % p.heads);
    id /= p.heads;
    const int b = static_cast<int>(id % p.batch), split = static_cast<int>(id / p.batch);
    const int hk = h / p.group;
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int64_t len = length_of(p, b);
    const int64_t begin = split * p.split_len, end = min(len, begin + p.split_len);
    float acc[kPer][Sh::kCols] = {};
    load_tile<DP>(p, p.q, b * p.qs.batch + h * p.qs.head, p.qs.pos, q0, p.q_len, nullptr, s_q);
    load_tile<DP>(p, p.dout, (b * p.q_len * p.heads + h) * p.dim, static_cast<int64_t>(p.heads) * p.dim, q0, p.q_len,
                  nullptr, s_do);
    load_stats<DP>(p, (static_cast<int64_t>(b) * p.heads + h) * p.q_len, q0, s_lse, s_delta);
    for (int64_t k0 = begin; k0 < end; k0 += kTile) {
        __syncthreads();
        bool mine = false;
        if (threadIdx.x < kTile) {
            mine = k0 + threadIdx.x < end && allowed(p, b, k0 + threadIdx.x, len);
            s_ok[threadIdx.x] = mine ? 1.0f : 0.0f;
        }
        if (!__syncthreads_or(mine)) continue;
        load_tile<DP>(p, p.k, b * p.ks.batch + hk * p.ks.head, p.ks.pos, k0, end, s_ok, s_k);
        load_tile<DP>(p, p.v, b * p.vs.batch + hk * p.vs.head, p.vs.pos, k0, end, s_ok, s_v);
        __syncthreads();
        float s[kPer][kPer], t[kPer][kPer];
        tile_dot<DP>(s_q, s_k, ty, tx, s);
        tile_dot<DP>(s_do, s_v, ty, tx, t);
        gradient_tile<DP>(p, s_ok, s_lse, s_delta, p.q_len - q0, ty, tx, s, t);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int j = 0; j < kPer; ++j) s_ds[(ty + 16 * i) * Sh::kPRow + tx + 16 * j] = t[i][j];
        __syncthreads();
        tile_mac<DP>(s_ds, s_k, ty, tx, acc);
    }
    const int64_t rows = static_cast<int64_t>(p.batch) * p.q_len * p.heads;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int64_t q = q0 + ty + 16 * i;
        if (q >= p.q_len) continue;
        const int64_t row = (b * p.q_len + q) * p.heads + h;
#pragma unroll
        for (int j = 0; j < Sh::kCols; ++j) {
            const int d = out_dim<DP>(tx, j);
            if (d >= p.dim) continue;
            if (p.splits > 1)
                p.part[(split * rows + row) * p.dim + d] = acc[i][j] * p.scale;
            else
                store1(p.dq, p.dtype, row * p.dim + d, acc[i][j] * p.scale);
        }
    }
}

// dK and dV. A block: one key tile of one key head, over the (query head,
// query tile) pairs of one split of the head's group.
template <int DP>
__global__ void __launch_bounds__(kThreads) dkv_kernel(const Params p) {
    using Sh = Shape<DP>;
    constexpr int kTile = Sh::kTile, kPer = Sh::kPer;
    extern __shared__ float smem[];
    float *s_k = smem, *s_v = s_k + Sh::kTileFloats, *s_q = s_v + Sh::kTileFloats, *s_do = s_q + Sh::kTileFloats;
    float *s_p = s_do + Sh::kTileFloats, *s_ds = s_p + Sh::kPFloats, *s_ok = s_ds + Sh::kPFloats,
          *s_lse = s_ok + kTile, *s_delta = s_lse + kTile;
    const int64_t k_tiles = (p.kv_len + kTile - 1) / kTile, q_tiles = (p.q_len + kTile - 1) / kTile;
    int64_t id = blockIdx.x;
    const int64_t k0 = id % k_tiles * kTile;
    id /= k_tiles;
    const int hk = static_cast<int>(id % p.kv_heads);
    id /= p.kv_heads;
    const int b = static_cast<int>(id % p.batch), split = static_cast<int>(id / p.batch);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const int64_t len = length_of(p, b);
    bool mine = false;
    if (threadIdx.x < kTile) {
        mine = k0 + threadIdx.x < p.kv_len && allowed(p, b, k0 + threadIdx.x, len);
        s_ok[threadIdx.x] = mine ? 1.0f : 0.0f;
    }
    const bool any = __syncthreads_or(mine);
    float dk[kPer][Sh::kCols] = {}, dv[kPer][Sh::kCols] = {};
    const int64_t items = q_tiles * p.group;
    const int64_t begin = split * p.split_len, end = any ? min(items, begin + p.split_len) : begin;
    if (any) {
        load_tile<DP>(p, p.k, b * p.ks.batch + hk * p.ks.head, p.ks.pos, k0, p.kv_len, s_ok, s_k);
        load_tile<DP>(p, p.v, b * p.vs.batch + hk * p.vs.head, p.vs.pos, k0, p.kv_len, s_ok, s_v);
    }
    for (int64_t it = begin; it < end; ++it) {
        const int h = hk * p.group + static_cast<int>(it / q_tiles);
        const int64_t q0 = it % q_tiles * kTile;
        __syncthreads();
        load_tile<DP>(p, p.q, b * p.qs.batch + h * p.qs.head, p.qs.pos, q0, p.q_len, nullptr, s_q);
        load_tile<DP>(p, p.dout, (b * p.q_len * p.heads + h) * p.dim, static_cast<int64_t>(p.heads) * p.dim, q0,
                      p.q_len, nullptr, s_do);
        load_stats<DP>(p, (static_cast<int64_t>(b) * p.heads + h) * p.q_len, q0, s_lse, s_delta);
        __syncthreads();
        float s[kPer][kPer], t[kPer][kPer];
        tile_dot<DP>(s_q, s_k, ty, tx, s);
        tile_dot<DP>(s_do, s_v, ty, tx, t);
        gradient_tile<DP>(p, s_ok, s_lse, s_delta, p.q_len - q0, ty, tx, s, t);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                s_p[(tx + 16 * j) * Sh::kPRow + ty + 16 * i] = s[i][j];
                s_ds[(tx + 16 * j) * Sh::kPRow + ty + 16 * i] = t[i][j];
            }
        __syncthreads();
        tile_mac<DP>(s_p, s_do, ty, tx, dv);
        tile_mac<DP>(s_ds, s_q, ty, tx, dk);
    }
    const int64_t rows = static_cast<int64_t>(p.batch) * p.kv_len * p.kv_heads;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int64_t key = k0 + ty + 16 * i;
        if (key >= p.kv_len) continue;
        const int64_t row = (b * p.kv_len + key) * p.kv_heads + hk;
        // a NaN in a query row of P = 0 would survive the product
        const bool on = s_ok[ty + 16 * i] != 0.0f;
#pragma unroll
        for (int j = 0; j < Sh::kCols; ++j) {
            const int d = out_dim<DP>(tx, j);
            if (d >= p.dim) continue;
            const float gk = on ? dk[i][j] * p.scale : 0.0f, gv = on ? dv[i][j] : 0.0f;
            if (p.splits > 1) {
                p.part_kv[(2 * split * rows + row) * p.dim + d] = gk;
                p.part_kv[((2 * split + 1) * rows + row) * p.dim + d] = gv;
            } else {
                store1(p.dk, p.dtype, row * p.dim + d, gk);
                store1(p.dv, p.dtype, row * p.dim + d, gv);
            }
        }
    }
}

// One gradient's parts: `splits` of n floats each, `pitch` apart; 0 splits:
// nothing to join.
struct Join {
    const float* part;
    void* out;
    int64_t n, pitch;
    int splits;
};
struct Joins {
    Join g[3];  // dQ, dK, dV
    int dtype;
    int wide;  // every n and pitch a multiple of 4: four elements a thread
};
// Sums the parts in split order. Block y: which gradient. A thread has four
// places (of four elements each where `wide`) in flight.
__global__ void __launch_bounds__(kThreads) join_kernel(const Joins p) {
    constexpr int kFlight = 4;
    const Join& g = p.g[blockIdx.y];
    if (g.splits == 0) return;
    const int width = p.wide ? 4 : 1;
    const int64_t first = (blockIdx.x * static_cast<int64_t>(kThreads) * kFlight + threadIdx.x) * width;
    float sum[kFlight][4] = {};
    for (int s = 0; s < g.splits; ++s) {
#pragma unroll
        for (int f = 0; f < kFlight; ++f) {
            const int64_t i = first + static_cast<int64_t>(f) * kThreads * width;
            if (i >= g.n) break;
            if (p.wide) {
                const float4 v = __ldcs(reinterpret_cast<const float4*>(g.part + s * g.pitch + i));
                sum[f][0] += v.x, sum[f][1] += v.y, sum[f][2] += v.z, sum[f][3] += v.w;
            } else {
                sum[f][0] += g.part[s * g.pitch + i];
            }
        }
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
        const int64_t i = first + static_cast<int64_t>(f) * kThreads * width;
        if (i >= g.n) break;
        if (!p.wide)
            store1(g.out, p.dtype, i, sum[f][0]);
        else if (p.dtype == 0)
            store_f32<float, 4>(static_cast<float*>(g.out) + i, sum[f]);
        else if (p.dtype == 1)
            store_f32<__half, 4>(static_cast<__half*>(g.out) + i, sum[f]);
        else
            store_f32<__nv_bfloat16, 4>(static_cast<__nv_bfloat16*>(g.out) + i, sum[f]);
    }
}

}  // namespace attn
}  // namespace rdvb
