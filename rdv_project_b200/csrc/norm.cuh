// Group norm with an activation over channels-last maps x [n, rows, c]:
//   xhat = (x - mu) rstd,  z = w_c xhat + b_c,  y = act(z)
// with mu and rstd = 1 / sqrt(var + eps) over the rows and the c / groups
// channels of a sample's group, and its gradients: with dz = dy act'(z),
//   db_c = sum dz,  dw_c = sum dz xhat,
//   dx = rstd (w dz - mean(w dz) - xhat mean(w dz xhat)).
//
// Bound: memory; ~10 (forward) and ~25 (backward) float32 operations an
// element. A pass over the data takes sums of a slab of rows (a block a
// slab; threads lie along the channels, 16 bytes each, so a warp reads whole
// lines whatever the group's width), a second pass joins the slabs' sums
// in slab order -- no atomics, so results repeat bit for bit -- and
// normalises. The second pass finds what fits in L2 there.
//
// A thread sums its elements' distances from its first one in float32, so a
// mean far from zero costs no digits; parts are joined by their means, in 64
// bits (a few thousand additions a block), and squared deviations, not by
// sums of squares. The mean used is the exact one rounded to float32.
#pragma once
#include <cstdint>

#include "types.cuh"

namespace rdvb {
namespace norm {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxGroups = 2048;
constexpr int kMaxSlabs = 128;

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

__device__ __forceinline__ float sigmoid(float z) { return 1.0f / (1.0f + __expf(-z)); }

__device__ __forceinline__ float activate(float z, int act) {
    if (act == kRelu) return z < 0.0f ? 0.0f : z;  // keeps a NaN
    if (act == kSilu) return z * sigmoid(z);
    if (act == kGelu) return z * (0.5f * (1.0f + erff(z * 0.70710678118654752f)));
    return z;
}

__device__ __forceinline__ float slope(float z, int act) {
    if (act == kRelu) return z > 0.0f ? 1.0f : 0.0f;
    if (act == kSilu) {
        const float s = sigmoid(z);
        return s * (1.0f + z * (1.0f - s));
    }
    if (act == kGelu)
        return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
    return 1.0f;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A block's place: sample, slab, and how its threads lie over `tile` of the
// channel vectors (cols of them) and `lanes` rows at a time.
struct Place {
    int sample, slab;
    int64_t row0, rows;
};

__device__ __forceinline__ Place place(const Params& p) {
    Place a;
    a.sample = blockIdx.x / p.slabs;
    a.slab = blockIdx.x % p.slabs;
    a.row0 = a.slab * p.slab_rows;
    const int64_t left = p.rows - a.row0;
    a.rows = left < p.slab_rows ? left : p.slab_rows;
    return a;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Slab sums of the forward pass: mean_part[sample][slab][group]. Dynamic
// shared memory: a double and a float a group.
template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) sums_kernel(const Params p) {
    __shared__ double s_mean[kVec * kThreads];
    __shared__ float s_dev[kVec * kThreads];
    extern __shared__ double s_join[];  // means, then (float) squared deviations
    float* s_join_dev = reinterpret_cast<float*>(s_join + p.groups);
    const Place a = place(p);
    const int cols = p.c / kVec;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* base = static_cast<const T*>(p.x) + (a.sample * p.rows + a.row0) * p.c;
    for (int col0 = 0; col0 < cols; col0 += kThreads) {
        const int tile = min(cols - col0, kThreads);
        const int lanes = kThreads / tile;
        const int tx = threadIdx.x % tile, ty = threadIdx.x / tile;
        const int64_t mine = ty < lanes && ty < a.rows ? (a.rows - ty + lanes - 1) / lanes : 0;
        float first[kVec], s1[kVec] = {}, s2[kVec] = {};
        if (mine > 0) {
            const T* at = base + static_cast<int64_t>(ty) * p.c + static_cast<int64_t>(col0 + tx) * kVec;
            const int64_t step = static_cast<int64_t>(lanes) * p.c;
            load_f32<T, kVec>(at, first);
#pragma unroll 4
            for (int64_t r = 1; r < mine; ++r) {
                float v[kVec];
                load_f32<T, kVec>(at + r * step, v);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const float d = v[i] - first[i];
                    s1[i] += d;
                    s2[i] = fmaf(d, d, s2[i]);
                }
            }
        }
        const float inv = mine > 0 ? 1.0f / static_cast<float>(mine) : 0.0f;
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            s_mean[i * kThreads + threadIdx.x] = mine > 0 ? static_cast<double>(first[i]) + s1[i] * inv : 0.0;
            s_dev[i * kThreads + threadIdx.x] = fmaxf(s2[i] - s1[i] * s1[i] * inv, 0.0f) + 0.0f * s2[i];
        }
        __syncthreads();
        // a warp a group: its channels inside this tile, over the thread rows
        const int c0 = col0 * kVec, c1 = c0 + tile * kVec;
        const int used = a.rows < lanes ? static_cast<int>(a.rows) : lanes;
        for (int g = c0 / p.per + warp; g < p.groups && g * p.per < c1; g += kWarps) {
            const int lo = max(g * p.per, c0), width = min((g + 1) * p.per, c1) - lo;
            double total = 0.0;
            for (int e = lane; e < width * used; e += 32) {
                const int ch = lo - c0 + e % width, row = e / width;
                const double m = static_cast<double>((a.rows - row + lanes - 1) / lanes);
                total += m * s_mean[(ch % kVec) * kThreads + row * tile + ch / kVec];
            }
            const double count = static_cast<double>(a.rows) * width;
            const double mean = warp_sum(total) / count;
            float dev = 0.0f;
            for (int e = lane; e < width * used; e += 32) {
                const int ch = lo - c0 + e % width, row = e / width;
                const float m = static_cast<float>((a.rows - row + lanes - 1) / lanes);
                const int at = (ch % kVec) * kThreads + row * tile + ch / kVec;
                const float d = static_cast<float>(s_mean[at] - mean);
                dev += s_dev[at] + m * d * d;
            }
            dev = warp_sum(dev);
            if (lane == 0) {
                // with the channels of this group that an earlier tile has summed
                const double before = static_cast<double>(a.rows) * (lo - g * p.per);
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
template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) apply_kernel(const Params p) {
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
    const int64_t start = (a.sample * p.rows + a.row0) * p.c;
    for (int col0 = 0; col0 < cols; col0 += kThreads) {
        const int tile = min(cols - col0, kThreads);
        const int lanes = kThreads / tile;
        const int tx = threadIdx.x % tile, ty = threadIdx.x / tile;
        if (ty >= lanes) continue;
        const int c0 = (col0 + tx) * kVec;
        float mean[kVec], gain[kVec], bias[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int g = (c0 + i) / p.per;
            mean[i] = s_group[g];
            gain[i] = s_group[p.groups + g] * param_at(p.weight, p.param_type, c0 + i, 1.0f);
            bias[i] = param_at(p.bias, p.param_type, c0 + i, 0.0f);
        }
        const T* in = static_cast<const T*>(p.x) + start + c0;
        T* out = static_cast<T*>(p.out) + start + c0;
#pragma unroll 4
        for (int64_t r = ty; r < a.rows; r += lanes) {
            float v[kVec];
            load_f32<T, kVec>(in + r * p.c, v);
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[i] = activate(fmaf(v[i] - mean[i], gain[i], bias[i]), p.act);
            store_f32<T, kVec>(out + r * p.c, v);
        }
    }
}

// Slab sums of the backward pass: chan_part[sample][slab][channel] and
// group_part[sample][slab][group].
template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) grad_sums_kernel(const Params p) {
    __shared__ float s_dz[kVec * kThreads], s_dzx[kVec * kThreads];
    extern __shared__ float s_group[];  // sums of w dz, then of w dz xhat
    const Place a = place(p);
    const int cols = p.c / kVec;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t start = (a.sample * p.rows + a.row0) * p.c;
    const float* stats = p.stats + static_cast<int64_t>(a.sample) * p.groups * 2;
    float2* chan = p.chan_part + static_cast<int64_t>(blockIdx.x) * p.c;
    for (int col0 = 0; col0 < cols; col0 += kThreads) {
        const int tile = min(cols - col0, kThreads);
        const int lanes = kThreads / tile;
        const int tx = threadIdx.x % tile, ty = threadIdx.x / tile;
        float sdz[kVec] = {}, sdzx[kVec] = {};
        if (ty < lanes) {
            const int c0 = (col0 + tx) * kVec;
            float mean[kVec], rstd[kVec], w[kVec], bias[kVec];
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const int g = (c0 + i) / p.per;
                mean[i] = stats[2 * g];
                rstd[i] = stats[2 * g + 1];
                w[i] = param_at(p.weight, p.param_type, c0 + i, 1.0f);
                bias[i] = param_at(p.bias, p.param_type, c0 + i, 0.0f);
            }
            const T* x = static_cast<const T*>(p.x) + start + c0;
            const T* dy = static_cast<const T*>(p.dy) + start + c0;
#pragma unroll 2
            for (int64_t r = ty; r < a.rows; r += lanes) {
                float v[kVec], d[kVec];
                load_f32<T, kVec>(x + r * p.c, v);
                load_f32<T, kVec>(dy + r * p.c, d);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const float xhat = (v[i] - mean[i]) * rstd[i];
                    const float dz = d[i] * slope(fmaf(xhat, w[i], bias[i]), p.act);
                    sdz[i] += dz;
                    sdzx[i] = fmaf(dz, xhat, sdzx[i]);
                }
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
            __syncwarp();
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

// Second pass of the backward pass: dx, and in the blocks past n * slabs the
// channel gradients (32 channels a block, its warps over the slabs).
template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) grad_apply_kernel(const Params p) {
    extern __shared__ float s_group[];  // means of w dz, then of w dz xhat
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t parts = static_cast<int64_t>(p.n) * p.slabs;
    if (blockIdx.x >= parts) {
        __shared__ float2 s_part[kWarps][32];
        const int ch = static_cast<int>(blockIdx.x - parts) * 32 + lane;
        float sum = 0.0f, sumx = 0.0f;
        if (ch < p.c)
            for (int64_t i = warp; i < parts; i += kWarps) {
                const float2 v = p.chan_part[i * p.c + ch];
                sum += v.x;
                sumx += v.y;
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
    const int64_t start = (a.sample * p.rows + a.row0) * p.c;
    const float* stats = p.stats + static_cast<int64_t>(a.sample) * p.groups * 2;
    for (int col0 = 0; col0 < cols; col0 += kThreads) {
        const int tile = min(cols - col0, kThreads);
        const int lanes = kThreads / tile;
        const int tx = threadIdx.x % tile, ty = threadIdx.x / tile;
        if (ty >= lanes) continue;
        const int c0 = (col0 + tx) * kVec;
        float mean[kVec], rstd[kVec], w[kVec], bias[kVec], m1[kVec], m2[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int g = (c0 + i) / p.per;
            mean[i] = stats[2 * g];
            rstd[i] = stats[2 * g + 1];
            w[i] = param_at(p.weight, p.param_type, c0 + i, 1.0f);
            bias[i] = param_at(p.bias, p.param_type, c0 + i, 0.0f);
            m1[i] = s_group[g];
            m2[i] = s_group[p.groups + g];
        }
        const T* x = static_cast<const T*>(p.x) + start + c0;
        const T* dy = static_cast<const T*>(p.dy) + start + c0;
        T* out = static_cast<T*>(p.out) + start + c0;
#pragma unroll 2
        for (int64_t r = ty; r < a.rows; r += lanes) {
            float v[kVec], d[kVec];
            load_f32<T, kVec>(x + r * p.c, v);
            load_f32<T, kVec>(dy + r * p.c, d);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const float xhat = (v[i] - mean[i]) * rstd[i];
                const float dz = d[i] * slope(fmaf(xhat, w[i], bias[i]), p.act);
                v[i] = rstd[i] * (fmaf(w[i], dz, -m1[i]) - xhat * m2[i]);
            }
            store_f32<T, kVec>(out + r * p.c, v);
        }
    }
}

}  // namespace norm
}  // namespace rdvb
