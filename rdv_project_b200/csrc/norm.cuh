// Group norm with an activation over channels-last maps x [n, rows, c]:
//   xhat = (x - mu) rstd,  z = w_c xhat + b_c,  y = act(z)
// with mu and rstd = 1 / sqrt(var + eps) over the rows and the c / groups
// channels of a sample's group, and its gradients: with dz = dy act'(z),
//   db_c = sum dz,  dw_c = sum dz xhat,
//   dx = rstd (w dz - mean(w dz) - xhat mean(w dz xhat)).
//
// Bound: memory; ~10 (forward) and ~25 (backward) float32 operations an
// element, two of them of the exponential unit for silu. A pass over the data
// takes sums of a slab of rows (a block a slab; threads lie along the
// channels, up to 16 bytes each, so a warp reads whole lines whatever the
// group's width), a second pass joins the slabs' sums in slab order -- no
// atomics, so results repeat bit for bit -- and normalises. The second pass
// finds what fits in L2 there. (One launch that kept the slabs in shared
// memory and waited for the sample's other blocks read less, but the waits and
// the joins by every block cost more: 125 us for 8 x 256 x 256 x 64 float16.)
// A sample that fits one block's shared memory takes one launch
// (small_kernel).
//
// Measured: 8 x 256 x 256 x 64 float16 with silu, 19 us for the sums and 36 us for
// the result (3.5 and 3.7 TB/s); 16 x 64 x 64 x 512 bfloat16, 22 + 40 us forward and
// 49 + 49 us backward.
//
// A thread sums its elements' distances from its first one in float32, so a
// mean far from zero costs no digits; parts are joined by their means, in 64
// bits (a few thousand additions a block), and squared deviations, not by
// sums of squares. The mean used is the exact one rounded to float32.
#pragma once
#include <cstdint>

#define RDVB_STATUS_ELSEWHERE
#include "ptx.cuh"
#include "types.cuh"

namespace rdvb {
namespace norm {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxGroups = 2048;
constexpr int kMaxSlabs = 128;
constexpr int kRuntime = -1;  // a kernel's activation is Params::act

enum Activation { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

struct Params {
    const void* x;
    const void* dy;
    void* out;           // y or dx
    const void* weight;  // may be null (1)
    const void* bias;    // may be null (0)
    float* stats;        // [n, groups, 2] mean, rstd; may be null in the forward pass
    float* dweight;      // [c]
    float* dbias;
    double2* mean_part;  // forward: [n, slabs, groups]: (mean, squared deviations)
    float2* group_part;  // backward: [n, slabs, groups]: (sum w dz, sum w dz xhat)
    float2* chan_part;   // [n, slabs, c]: (sum dz, sum dz xhat)
    int64_t rows;        // positions of a sample
    int64_t slab_rows;
    int n, c, groups, per, slabs;
    int param_type;  // RDVB_* code of weight and bias
    int act;
    float eps;
};

__device__ __forceinline__ float param_at(const void* p, int type, int i, float none) {
    if (!p) return none;
    if (type == 0) return static_cast<const float*>(p)[i];
    if (type == 1) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Two exponential-unit instructions, each within 2 units in the last place
// (and the product's rounding in the exponent), as the bound of the forward
// and backward passes is close to that unit: 1 / (1 + 2^(-z log2 e)).
__device__ __forceinline__ void sigmoid2(float& x, float& y) {
    constexpr float kNegLog2e = -1.4426950408889634f;
    mul2(x, y, kNegLog2e, kNegLog2e);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(y));
    add2(x, y, 1.0f, 1.0f);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(y));
}

// z to act(z), two at a time.
__device__ __forceinline__ void activate2(float& x, float& y, int act) {
    if (act == kRelu) {
        x = x < 0.0f ? 0.0f : x;  // keeps a NaN
        y = y < 0.0f ? 0.0f : y;
    } else if (act == kSilu) {
        float s0 = x, s1 = y;
        sigmoid2(s0, s1);
        mul2(x, y, s0, s1);
    } else if (act == kGelu) {
        x *= 0.5f * (1.0f + erff(x * 0.70710678118654752f));
        y *= 0.5f * (1.0f + erff(y * 0.70710678118654752f));
    }
}

// z to act'(z), two at a time.
__device__ __forceinline__ void slope2(float& x, float& y, int act) {
    if (act == kRelu) {
        x = x > 0.0f ? 1.0f : 0.0f;
        y = y > 0.0f ? 1.0f : 0.0f;
    } else if (act == kSilu) {  // s (1 + z (1 - s))
        float s0 = x, s1 = y;
        sigmoid2(s0, s1);
        float t0 = s0, t1 = s1;
        fma2(t0, t1, -1.0f, -1.0f, 1.0f, 1.0f);
        fma2(x, y, t0, t1, 1.0f, 1.0f);
        mul2(x, y, s0, s1);
    } else if (act == kGelu) {
        auto one = [](float z) {
            return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
        };
        x = one(x);
        y = one(y);
    } else {
        x = y = 1.0f;
    }
}

// f(v0, v1, i, j) over a vector's elements in pairs; a single element has
// itself as its partner's index and a partner that nothing reads.
template <int kVec, typename F>
__device__ __forceinline__ void in_pairs(float (&v)[kVec], F&& f) {
    if constexpr (kVec == 1) {
        float none = 0.0f;
        f(v[0], none, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < kVec; i += 2) f(v[i], v[i + 1], i, i + 1);
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}


__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <int kAct>
__device__ __forceinline__ int act_of(const Params& p) {
    return kAct == kRuntime ? p.act : kAct;
}

// A block's sample and slab.
struct Place {
    int sample, slab, rows;
    int64_t start;  // its first element
};
__device__ __forceinline__ Place place(const Params& p) {
    Place a;
    a.sample = blockIdx.x / p.slabs;
    a.slab = blockIdx.x % p.slabs;
    const int64_t row0 = a.slab * p.slab_rows, left = p.rows - row0;
    a.rows = static_cast<int>(left < p.slab_rows ? left : p.slab_rows);
    a.start = (a.sample * p.rows + row0) * p.c;
    return a;
}

// e / d of small whole numbers from the float32 reciprocal of d.
__device__ __forceinline__ int quotient(int e, float inv) { return static_cast<int>((e + 0.5f) * inv); }

// kOne: a thread's vector lies in one group, so its statistics are one
// number; otherwise each of its channels has its own.

// Slab sums of the forward pass: mean_part[sample][slab][group]. Dynamic
// shared memory: a double and a float a group.
template <typename T, int kVec, bool kOne>
__global__ void __launch_bounds__(kThreads) sums_kernel(const Params p) {
    constexpr int kStat = kOne ? 1 : kVec;
    __shared__ double s_mean[kStat * kThreads];
    __shared__ float s_dev[kStat * kThreads];
    extern __shared__ double s_join[];  // means, then (float) squared deviations
    float* s_join_dev = reinterpret_cast<float*>(s_join + p.groups);
    const Place a = place(p);
    const int cols = p.c / kVec, cells = kOne ? p.per / kVec : p.per;  // cells of a group in a row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int col0 = 0; col0 < cols; col0 += kThreads) {
        const int tile = min(cols - col0, kThreads);
        const int lanes = kThreads / tile;
        const int tx = threadIdx.x % tile, ty = threadIdx.x / tile;
        const int mine = ty < lanes && ty < a.rows ? (a.rows - ty + lanes - 1) / lanes : 0;
        float first[kStat] = {}, s1[kStat] = {}, s2[kStat] = {};
        if (mine > 0) {
            const T* at = static_cast<const T*>(p.x) + a.start + static_cast<int64_t>(ty) * p.c + (col0 + tx) * kVec;
            const int64_t step = static_cast<int64_t>(lanes) * p.c;
            {
                float v[kVec];
                load_f32<T, kVec>(at, v);
#pragma unroll
                for (int i = 0; i < kStat; ++i) first[i] = v[i];
            }
#pragma unroll 8
            for (int r = 0; r < mine; ++r, at += step) {
                float v[kVec];
                load_f32<T, kVec>(at, v);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const int k = kOne ? 0 : i;
                    const float d = v[i] - first[k];
                    s1[k] += d;
                    s2[k] = fmaf(d, d, s2[k]);
                }
            }
        }
        const float inv = mine > 0 ? 1.0f / static_cast<float>(mine * (kVec / kStat)) : 0.0f;
#pragma unroll
        for (int i = 0; i < kStat; ++i) {
            s_mean[i * kThreads + threadIdx.x] = static_cast<double>(first[i]) + s1[i] * inv;
            s_dev[i * kThreads + threadIdx.x] = fmaxf(s2[i] - s1[i] * s1[i] * inv, 0.0f) + 0.0f * s2[i];
        }
        __syncthreads();
        // a warp a group: its cells inside this tile, over the thread rows
        const int c0 = col0 * kStat, c1 = c0 + tile * kStat;
        const int used = min(a.rows, lanes);
        for (int g = c0 / cells + warp; g < p.groups && g * cells < c1; g += kWarps) {
            const int lo = max(g * cells, c0), width = min((g + 1) * cells, c1) - lo;
            const float inv_width = 1.0f / static_cast<float>(width);
            double total = 0.0;
            for (int e = lane; e < width * used; e += 32) {
                const int row = quotient(e, inv_width), cell = lo - c0 + e - row * width;
                total += static_cast<double>((a.rows - row + lanes - 1) / lanes) *
                         s_mean[(cell % kStat) * kThreads + row * tile + cell / kStat];
            }
            const double cell_rows = static_cast<double>(a.rows) * width;
            const double mean = warp_sum(total) / cell_rows;
            float dev = 0.0f;
            for (int e = lane; e < width * used; e += 32) {
                const int row = quotient(e, inv_width), cell = lo - c0 + e - row * width;
                const int at = (cell % kStat) * kThreads + row * tile + cell / kStat;
                const float m = static_cast<float>((a.rows - row + lanes - 1) / lanes * (kVec / kStat));
                const float d = static_cast<float>(s_mean[at] - mean);
                dev += s_dev[at] + m * d * d;
            }
            dev = warp_sum(dev);
            if (lane == 0) {
                // with the cells of this group that an earlier tile has summed
                const double count = cell_rows * (kVec / kStat);
                const double before = static_cast<double>(a.rows) * (lo - g * cells) * (kVec / kStat);
                if (before == 0.0) {
                    s_join[g] = mean;
                    s_join_dev[g] = dev;
                } else {
                    const double d = mean - s_join[g], f = count / (before + count);
                    s_join_dev[g] += dev + static_cast<float>(d * d * before * f);
                    s_join[g] += d * f;
                }
            }
        }
        __syncthreads();
    }
    double2* out = p.mean_part + static_cast<int64_t>(blockIdx.x) * p.groups;
    for (int g = threadIdx.x; g < p.groups; g += kThreads) out[g] = make_double2(s_join[g], s_join_dev[g]);
}

// Joins the slabs of this block's sample into s_group: means, then rstds.
__device__ __forceinline__ void join_slabs(const Params& p, int sample, float* s_group) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const double2* part = p.mean_part + static_cast<int64_t>(sample) * p.slabs * p.groups;
    const double last = static_cast<double>(p.rows - (p.slabs - 1) * p.slab_rows);
    const double each = static_cast<double>(p.slab_rows), all = static_cast<double>(p.rows);
    for (int g = warp; g < p.groups; g += kWarps) {
        double total = 0.0;
        for (int s = lane; s < p.slabs; s += 32)
            total += (s == p.slabs - 1 ? last : each) * part[static_cast<int64_t>(s) * p.groups + g].x;
        const double mean = warp_sum(total) / all;
        double dev = 0.0;
        for (int s = lane; s < p.slabs; s += 32) {
            const double2 v = part[static_cast<int64_t>(s) * p.groups + g];
            const double d = v.x - mean;
            dev += v.y + (s == p.slabs - 1 ? last : each) * p.per * d * d;
        }
        dev = warp_sum(dev);
        if (lane == 0) {
            s_group[g] = static_cast<float>(mean);
            s_group[p.groups + g] = static_cast<float>(1.0 / sqrt(dev / (all * p.per) + p.eps));
        }
    }
}

// Second pass of the forward pass. Dynamic shared memory: 2 groups floats.
template <typename T, int kVec, bool kOne, int kAct>
__global__ void __launch_bounds__(kThreads) apply_kernel(const Params p) {
    constexpr int kStat = kOne ? 1 : kVec;
    extern __shared__ float s_group[];
    const Place a = place(p);
    join_slabs(p, a.sample, s_group);
    __syncthreads();
    if (p.stats && a.slab == 0) {
        float* out = p.stats + static_cast<int64_t>(a.sample) * p.groups * 2;
        for (int g = threadIdx.x; g < p.groups; g += kThreads) {
            out[2 * g] = s_group[g];
            out[2 * g + 1] = s_group[p.groups + g];
        }
    }
    const int cols = p.c / kVec;
    for (int col0 = 0; col0 < cols; col0 += kThreads) {
        const int tile = min(cols - col0, kThreads);
        const int lanes = kThreads / tile;
        const int tx = threadIdx.x % tile, ty = threadIdx.x / tile;
        if (ty >= lanes) continue;
        const int c0 = (col0 + tx) * kVec;
        float mean[kStat], gain[kVec], bias[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int g = (c0 + i) / p.per;
            if (i < kStat) mean[i] = s_group[g];
            gain[i] = s_group[p.groups + g] * param_at(p.weight, p.param_type, c0 + i, 1.0f);
            bias[i] = param_at(p.bias, p.param_type, c0 + i, 0.0f);
        }
        const int64_t first = a.start + static_cast<int64_t>(ty) * p.c + c0, step = static_cast<int64_t>(lanes) * p.c;
        const T* in = static_cast<const T*>(p.x) + first;
        T* out = static_cast<T*>(p.out) + first;
#pragma unroll 4
        for (int r = ty; r < a.rows; r += lanes, in += step, out += step) {
            float v[kVec];
            load_f32<T, kVec>(in, v);
            in_pairs<kVec>(v, [&](float& x, float& y, int i, int j) {
                add2(x, y, -mean[kOne ? 0 : i], -mean[kOne ? 0 : j]);
                fma2(x, y, gain[i], gain[j], bias[i], bias[j]);
                activate2(x, y, act_of<kAct>(p));
            });
            store_f32<T, kVec>(out, v);
        }
    }
}

// A thread's channels of a backward pass: their group's statistics and their
// own parameters.
template <int kVec, bool kOne>
struct Channels {
    static constexpr int kStat = kOne ? 1 : kVec;
    float mean[kStat], rstd[kStat], w[kVec], bias[kVec];
    __device__ __forceinline__ void load(const Params& p, int sample, int c0) {
        const float* stats = p.stats + static_cast<int64_t>(sample) * p.groups * 2;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            if (i < kStat) {
                const int g = (c0 + i) / p.per;
                mean[i] = stats[2 * g];
                rstd[i] = stats[2 * g + 1];
            }
            w[i] = param_at(p.weight, p.param_type, c0 + i, 1.0f);
            bias[i] = param_at(p.bias, p.param_type, c0 + i, 0.0f);
        }
    }
    // x to xhat and dy to dz of channels i and j
    template <int kAct>
    __device__ __forceinline__ void at(const Params& p, int i, int j, float& x0, float& x1, float& d0, float& d1) const {
        const int k = kOne ? 0 : i, l = kOne ? 0 : j;
        add2(x0, x1, -mean[k], -mean[l]);
        mul2(x0, x1, rstd[k], rstd[l]);
        float z0 = x0, z1 = x1;
        fma2(z0, z1, w[i], w[j], bias[i], bias[j]);
        slope2(z0, z1, act_of<kAct>(p));
        mul2(d0, d1, z0, z1);
    }
};

// Slab sums of the backward pass: chan_part[sample][slab][channel] and
// group_part[sample][slab][group].
template <typename T, int kVec, bool kOne, int kAct>
__global__ void __launch_bounds__(kThreads) grad_sums_kernel(const Params p) {
    __shared__ float s_dz[kVec * kThreads], s_dzx[kVec * kThreads];
    const Place a = place(p);
    const int cols = p.c / kVec;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float2* chan = p.chan_part + static_cast<int64_t>(blockIdx.x) * p.c;
    for (int col0 = 0; col0 < cols; col0 += kThreads) {
        const int tile = min(cols - col0, kThreads);
        const int lanes = kThreads / tile;
        const int tx = threadIdx.x % tile, ty = threadIdx.x / tile;
        float sdz[kVec] = {}, sdzx[kVec] = {};
        if (ty < lanes) {
            const int c0 = (col0 + tx) * kVec;
            Channels<kVec, kOne> ch;
            ch.load(p, a.sample, c0);
            const int64_t first = a.start + static_cast<int64_t>(ty) * p.c + c0, step = static_cast<int64_t>(lanes) * p.c;
            const T* x = static_cast<const T*>(p.x) + first;
            const T* dy = static_cast<const T*>(p.dy) + first;
#pragma unroll 2
            for (int r = ty; r < a.rows; r += lanes, x += step, dy += step) {
                float v[kVec], d[kVec];
                load_f32<T, kVec>(x, v);
                load_f32<T, kVec>(dy, d);
                in_pairs<kVec>(v, [&](float& x0, float& x1, int i, int j) {
                    float d0 = d[i], d1 = d[j];
                    ch.template at<kAct>(p, i, j, x0, x1, d0, d1);
                    if constexpr (kVec == 1) {
                        sdz[0] += d0;
                        sdzx[0] = fmaf(d0, x0, sdzx[0]);
                    } else {
                        fma2(x0, x1, d0, d1, sdzx[i], sdzx[j]);
                        sdzx[i] = x0, sdzx[j] = x1;
                        add2(sdz[i], sdz[j], d0, d1);
                    }
                });
            }
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            s_dz[i * kThreads + threadIdx.x] = sdz[i];
            s_dzx[i * kThreads + threadIdx.x] = sdzx[i];
        }
        __syncthreads();
        // a channel's thread rows, four threads a channel; the sums end in the first
        const int width = tile * kVec;
        for (int e0 = 0; e0 < width * 4; e0 += kThreads) {
            const int e = e0 + threadIdx.x, ch = e >> 2;
            float sum = 0.0f, sumx = 0.0f;
            if (ch < width)
                for (int r = e & 3; r < lanes; r += 4) {
                    const int at = (ch % kVec) * kThreads + r * tile + ch / kVec;
                    sum += s_dz[at];
                    sumx += s_dzx[at];
                }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                sum += __shfl_xor_sync(0xffffffffu, sum, o);
                sumx += __shfl_xor_sync(0xffffffffu, sumx, o);
            }
            if (ch < width && (e & 3) == 0) chan[col0 * kVec + ch] = make_float2(sum, sumx);
        }
        __syncthreads();  // also makes this block's chan entries readable below
    }
    for (int g = warp; g < p.groups; g += kWarps) {
        float sum = 0.0f, sumx = 0.0f;
        for (int i = lane; i < p.per; i += 32) {
            const float2 v = chan[g * p.per + i];
            const float w = param_at(p.weight, p.param_type, g * p.per + i, 1.0f);
            sum = fmaf(w, v.x, sum);
            sumx = fmaf(w, v.y, sumx);
        }
        sum = warp_sum(sum);
        sumx = warp_sum(sumx);
        if (lane == 0)
            p.group_part[static_cast<int64_t>(blockIdx.x) * p.groups + g] = make_float2(sum, sumx);
    }
}

// The channel gradients of 32 channels from `parts` rows of chan_part, in
// order: warps over the parts, then over the warps.
__device__ __forceinline__ void join_channels(const Params& p, int64_t parts, int ch0) {
    __shared__ float2 s_part[kWarps][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int ch = ch0 + lane;
    float sum = 0.0f, sumx = 0.0f;
    if (ch < p.c) {
#pragma unroll 4
        for (int64_t i = warp; i < parts; i += kWarps) {
            const float2 v = p.chan_part[i * p.c + ch];
            sum += v.x;
            sumx += v.y;
        }
    }
    s_part[warp][lane] = make_float2(sum, sumx);
    __syncthreads();
    if (warp == 0 && ch < p.c) {
        for (int i = 1; i < kWarps; ++i) {
            sum += s_part[i][lane].x;
            sumx += s_part[i][lane].y;
        }
        if (p.dbias) p.dbias[ch] = sum;
        if (p.dweight) p.dweight[ch] = sumx;
    }
}

// Second pass of the backward pass: dx, and in the blocks past n * slabs the
// channel gradients.
template <typename T, int kVec, bool kOne, int kAct>
__global__ void __launch_bounds__(kThreads) grad_apply_kernel(const Params p) {
    constexpr int kStat = kOne ? 1 : kVec;
    extern __shared__ float s_group[];  // means of w dz, then of w dz xhat
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t parts = static_cast<int64_t>(p.n) * p.slabs;
    if (blockIdx.x >= parts) {
        join_channels(p, parts, static_cast<int>(blockIdx.x - parts) * 32);
        return;
    }
    const Place a = place(p);
    {
        const float2* part = p.group_part + static_cast<int64_t>(a.sample) * p.slabs * p.groups;
        const float inv = 1.0f / (static_cast<float>(p.rows) * static_cast<float>(p.per));
        for (int g = warp; g < p.groups; g += kWarps) {
            float sum = 0.0f, sumx = 0.0f;
            for (int s = lane; s < p.slabs; s += 32) {
                const float2 v = part[static_cast<int64_t>(s) * p.groups + g];
                sum += v.x;
                sumx += v.y;
            }
            sum = warp_sum(sum);
            sumx = warp_sum(sumx);
            if (lane == 0) {
                s_group[g] = sum * inv;
                s_group[p.groups + g] = sumx * inv;
            }
        }
    }
    __syncthreads();
    const int cols = p.c / kVec;
    for (int col0 = 0; col0 < cols; col0 += kThreads) {
        const int tile = min(cols - col0, kThreads);
        const int lanes = kThreads / tile;
        const int tx = threadIdx.x % tile, ty = threadIdx.x / tile;
        if (ty >= lanes) continue;
        const int c0 = (col0 + tx) * kVec;
        Channels<kVec, kOne> ch;
        ch.load(p, a.sample, c0);
        float m1[kStat], m2[kStat];
#pragma unroll
        for (int i = 0; i < kStat; ++i) {
            m1[i] = s_group[(c0 + i) / p.per];
            m2[i] = s_group[p.groups + (c0 + i) / p.per];
        }
        const int64_t first = a.start + static_cast<int64_t>(ty) * p.c + c0, step = static_cast<int64_t>(lanes) * p.c;
        const T* x = static_cast<const T*>(p.x) + first;
        const T* dy = static_cast<const T*>(p.dy) + first;
        T* out = static_cast<T*>(p.out) + first;
#pragma unroll 2
        for (int r = ty; r < a.rows; r += lanes, x += step, dy += step, out += step) {
            float v[kVec], d[kVec];
            load_f32<T, kVec>(x, v);
            load_f32<T, kVec>(dy, d);
            in_pairs<kVec>(v, [&](float& x0, float& x1, int i, int j) {
                const int k = kOne ? 0 : i, l = kOne ? 0 : j;
                float d0 = d[i], d1 = d[j];
                ch.template at<kAct>(p, i, j, x0, x1, d0, d1);
                fma2(d0, d1, ch.w[i], ch.w[j], -m1[k], -m1[l]);
                fma2(x0, x1, -m2[k], -m2[l], d0, d1);
                mul2(x0, x1, ch.rstd[k], ch.rstd[l]);
            });
            store_f32<T, kVec>(out, v);
        }
    }
}

// ------------------------------------------------- samples of one block each

// A block a sample whose slab fits shared memory: one copy in, two sums over
// it (the mean, then the squared distances from it), one result out.
constexpr int kSmallBytes = 65536;

// Sums v over the threads of each group (whole vectors); every thread of the
// group gets its sum. s: a float a thread and a group.
__device__ __forceinline__ float group_sum(float v, float* s, int cols, int lanes, int width, int groups, int group) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    s[threadIdx.x] = v;
    __syncthreads();
    const float inv = 1.0f / static_cast<float>(width);
    for (int g = warp; g < groups; g += kWarps) {
        float x = 0.0f;
        for (int e = lane; e < width * lanes; e += 32) {
            const int row = quotient(e, inv);
            x += s[row * cols + g * width + e - row * width];
        }
        x = warp_sum(x);
        if (lane == 0) s[kThreads + g] = x;
    }
    __syncthreads();
    return group < groups ? s[kThreads + group] : 0.0f;
}

template <typename T, int kVec, int kAct>
__global__ void __launch_bounds__(kThreads) small_kernel(const Params p, uint32_t* status) {
    extern __shared__ __align__(16) uint8_t smem[];  // the sample
    __shared__ float s_sum[kThreads + kThreads];
    __shared__ __align__(8) uint64_t s_full;
    const int cols = p.c / kVec, lanes = kThreads / cols, width = p.per / kVec, rows = static_cast<int>(p.rows);
    const int tx = threadIdx.x % cols, ty = threadIdx.x / cols;
    const int group = ty < lanes ? tx / width : p.groups, c0 = tx * kVec;
    const int64_t start = static_cast<int64_t>(blockIdx.x) * rows * p.c;
    if (threadIdx.x == 0) {
        const uint32_t bytes = static_cast<uint32_t>(rows) * p.c * sizeof(T), bar = smem_addr(&s_full);
        mbar_init(bar, 1);
        fence_mbarrier_init();
        mbar_arrive_expect_tx(bar, bytes);
        bulk_g2s(smem_addr(smem), static_cast<const T*>(p.x) + start, bytes, bar);
    }
    float gain[kVec], bias[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        gain[i] = ty < lanes ? param_at(p.weight, p.param_type, c0 + i, 1.0f) : 0.0f;
        bias[i] = ty < lanes ? param_at(p.bias, p.param_type, c0 + i, 0.0f) : 0.0f;
    }
    __syncthreads();
    uint32_t none = 0;
    if (!mbar_wait(smem_addr(&s_full), 0, &none, status, kStatusTimeoutXFull)) return;
    const T* x = reinterpret_cast<const T*>(smem) + c0;
    const int end = ty < lanes ? rows : 0;
    // distances from the group's first element keep a far mean's digits
    const float shift = ty < lanes ? to_f32<T>(reinterpret_cast<const T*>(smem)[group * p.per]) : 0.0f;
    const float inv = 1.0f / (static_cast<float>(rows) * static_cast<float>(p.per));
    float sum = 0.0f;
#pragma unroll 4
    for (int r = ty; r < end; r += lanes) {
        float v[kVec];
        load_f32<T, kVec>(x + r * p.c, v);
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum += v[i] - shift;
    }
    const float mean = shift + group_sum(sum, s_sum, cols, lanes, width, p.groups, group) * inv;
    sum = 0.0f;
#pragma unroll 4
    for (int r = ty; r < end; r += lanes) {
        float v[kVec];
        load_f32<T, kVec>(x + r * p.c, v);
#pragma unroll
        for (int i = 0; i < kVec; ++i) sum = fmaf(v[i] - mean, v[i] - mean, sum);
    }
    const float rstd = 1.0f / sqrtf(group_sum(sum, s_sum, cols, lanes, width, p.groups, group) * inv + p.eps);
    if (p.stats && ty == 0 && tx % width == 0) {
        float* out = p.stats + (static_cast<int64_t>(blockIdx.x) * p.groups + group) * 2;
        out[0] = mean;
        out[1] = rstd;
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) gain[i] *= rstd;
    T* y = static_cast<T*>(p.out) + start + c0;
#pragma unroll 2
    for (int r = ty; r < end; r += lanes) {
        float v[kVec];
        load_f32<T, kVec>(x + r * p.c, v);
        in_pairs<kVec>(v, [&](float& x, float& y, int i, int j) {
            add2(x, y, -mean, -mean);
            fma2(x, y, gain[i], gain[j], bias[i], bias[j]);
            activate2(x, y, act_of<kAct>(p));
        });
        store_f32<T, kVec>(y + static_cast<int64_t>(r) * p.c, v);
    }
}

}  // namespace norm
}  // namespace rdvb
