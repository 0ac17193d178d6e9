// rdvb_group_norm_* (include/rdvb.h).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "host.h"
#include "norm.cuh"

using rdvb_host::aligned;
using rdvb_host::fail;

namespace {
using namespace rdvb::norm;

struct Plan {
    int slabs;
    int64_t slab_rows;
    int64_t part_bytes, bytes;
};

// Slabs of a sample: about eight blocks a processor over the batch, but at
// least 16 rows each, so that the join of the slabs stays small beside them.
Plan plan(int64_t n, int64_t rows, int c, int groups, int backward) {
    Plan a;
    const int64_t want = std::max<int64_t>(1, 1184 / std::max<int64_t>(n, 1));
    const int64_t most = std::min<int64_t>({want, static_cast<int64_t>(kMaxSlabs), (rows + 15) / 16});
    a.slab_rows = (rows + most - 1) / std::max<int64_t>(most, 1);
    a.slabs = static_cast<int>((rows + a.slab_rows - 1) / std::max<int64_t>(a.slab_rows, 1));
    a.part_bytes = (n * a.slabs * groups * (backward ? 8 : 16) + 15) / 16 * 16;
    a.bytes = a.part_bytes + (backward ? n * a.slabs * c * 8 : 0);
    return a;
}

int check_shape(int dtype, int64_t n, int64_t rows, int c, int groups, int param_type, int act, float eps) {
    if (dtype != RDVB_F32 && dtype != RDVB_F16 && dtype != RDVB_BF16)
        return fail(RDVB_ERR_INVALID_ARG, "dtype %d is not RDVB_F32/F16/BF16", dtype);
    if (param_type != RDVB_F32 && param_type != RDVB_F16 && param_type != RDVB_BF16)
        return fail(RDVB_ERR_INVALID_ARG, "param_dtype %d is not RDVB_F32/F16/BF16", param_type);
    if (n < 0 || rows < 0) return fail(RDVB_ERR_INVALID_ARG, "n and rows must be >= 0");
    if (c < 1 || groups < 1 || c % groups)
        return fail(RDVB_ERR_INVALID_ARG, "groups (%d) must divide the channels (%d)", groups, c);
    if (groups > kMaxGroups)
        return fail(RDVB_ERR_UNSUPPORTED, "at most %d groups, got %d", kMaxGroups, groups);
    if (act < kNone || act > kGelu) return fail(RDVB_ERR_INVALID_ARG, "activation %d is not RDVB_ACT_*", act);
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(RDVB_ERR_INVALID_ARG, "eps must be finite and >= 0");
    if (rows > 0 && n > 0x7fffffffLL / kMaxSlabs) return fail(RDVB_ERR_UNSUPPORTED, "n = %lld is too large",
                                                              static_cast<long long>(n));
    return RDVB_OK;
}

// Elements of one access: the most that divide the channels and that every
// pointer is aligned to, at most 16 bytes.
int vector_width(int dtype, int c, std::initializer_list<const void*> ptrs) {
    const int size = dtype == RDVB_F32 ? 4 : 2;
    int w = 16 / size;
    while (w > 1 && c % w) w /= 2;
    for (const void* q : ptrs)
        while (w > 1 && !aligned(q, static_cast<uintptr_t>(w) * size)) w /= 2;
    return w;
}

template <typename F>
void each_type(int dtype, int vec, F&& f) {
    if (dtype == RDVB_F32)
        vec == 4 ? f(float{}, std::integral_constant<int, 4>{})
                 : vec == 2 ? f(float{}, std::integral_constant<int, 2>{}) : f(float{}, std::integral_constant<int, 1>{});
    else if (dtype == RDVB_F16)
        vec == 8 ? f(__half{}, std::integral_constant<int, 8>{})
        : vec == 4 ? f(__half{}, std::integral_constant<int, 4>{})
        : vec == 2 ? f(__half{}, std::integral_constant<int, 2>{})
                   : f(__half{}, std::integral_constant<int, 1>{});
    else
        vec == 8 ? f(__nv_bfloat16{}, std::integral_constant<int, 8>{})
        : vec == 4 ? f(__nv_bfloat16{}, std::integral_constant<int, 4>{})
        : vec == 2 ? f(__nv_bfloat16{}, std::integral_constant<int, 2>{})
                   : f(__nv_bfloat16{}, std::integral_constant<int, 1>{});
}

void fill(Params& p, const void* x, int64_t n, int64_t rows, int c, int groups, const void* weight, const void* bias,
          int param_type, int act, float eps, const Plan& a, void* workspace) {
    memset(&p, 0, sizeof(p));
    p.x = x;
    p.weight = weight;
    p.bias = bias;
    p.mean_part = static_cast<double2*>(workspace);
    p.group_part = static_cast<float2*>(workspace);
    p.chan_part = reinterpret_cast<float2*>(static_cast<char*>(workspace) + a.part_bytes);
    p.rows = rows;
    p.slab_rows = a.slab_rows;
    p.n = static_cast<int>(n);
    p.c = c;
    p.groups = groups;
    p.per = c / groups;
    p.slabs = a.slabs;
    p.param_type = param_type;
    p.act = act;
    p.eps = eps;
}

}  // namespace

extern "C" {

int64_t rdvb_group_norm_workspace_bytes(int64_t n, int64_t rows, int c, int groups, int backward) {
    if (n < 1 || rows < 1 || c < 1 || groups < 1) return 0;
    return plan(n, rows, c, groups, backward).bytes;
}

int rdvb_group_norm(const void* x, int dtype, int64_t n, int64_t rows, int c, int groups, const void* weight,
                    const void* bias, int param_dtype, int activation, float eps, void* y, float* stats,
                    void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check_shape(dtype, n, rows, c, groups, param_dtype, activation, eps)) return rc;
    if (n == 0 || rows == 0) return RDVB_OK;
    if (!x || !y || !workspace) return fail(RDVB_ERR_INVALID_ARG, "x, y and workspace must not be NULL");
    const uintptr_t size = dtype == RDVB_F32 ? 4 : 2, psize = param_dtype == RDVB_F32 ? 4 : 2;
    if (!aligned(x, size) || !aligned(y, size) || !aligned(weight, psize) || !aligned(bias, psize) ||
        !aligned(stats, 4) || !aligned(workspace, 16))
        return fail(RDVB_ERR_INVALID_ARG, "a pointer is not aligned (workspace: 16 bytes, others: their element)");
    const Plan a = plan(n, rows, c, groups, 0);
    if (workspace_bytes < static_cast<size_t>(a.bytes))
        return fail(RDVB_ERR_INVALID_ARG, "workspace holds %zu bytes; %lld are needed", workspace_bytes,
                    static_cast<long long>(a.bytes));
    rdvb_host::Device dev;
    if (int rc = rdvb_host::device(&dev)) return rc;
    Params p;
    fill(p, x, n, rows, c, groups, weight, bias, param_dtype, activation, eps, a, workspace);
    p.out = y;
    p.stats = stats;
    const unsigned grid = static_cast<unsigned>(n * a.slabs);
    const size_t smem = static_cast<size_t>(groups) * 8;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int rc = RDVB_OK;
    each_type(dtype, vector_width(dtype, c, {x, y}), [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int kVec = decltype(v)::value;
        sums_kernel<T, kVec><<<grid, kThreads, groups * 12, st>>>(p);
        if ((rc = rdvb_host::launched("group_norm sums_kernel"))) return;
        apply_kernel<T, kVec><<<grid, kThreads, smem, st>>>(p);
        rc = rdvb_host::launched("group_norm apply_kernel");
    });
    return rc;
}

int rdvb_group_norm_backward(const void* dy, const void* x, const float* stats, int dtype, int64_t n, int64_t rows,
                             int c, int groups, const void* weight, const void* bias, int param_dtype, int activation,
                             void* dx, float* dweight, float* dbias, void* workspace, size_t workspace_bytes,
                             void* stream) {
    if (int rc = check_shape(dtype, n, rows, c, groups, param_dtype, activation, 0.0f)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uintptr_t size = dtype == RDVB_F32 ? 4 : 2, psize = param_dtype == RDVB_F32 ? 4 : 2;
    if (!aligned(dweight, 4) || !aligned(dbias, 4))
        return fail(RDVB_ERR_INVALID_ARG, "dweight and dbias must be 4-byte aligned");
    if (n == 0 || rows == 0) {  // sums over nothing
        rdvb_host::Device dev;
        if (int rc = rdvb_host::device(&dev)) return rc;
        for (float* q : {dweight, dbias}) {
            cudaError_t e = q ? cudaMemsetAsync(q, 0, static_cast<size_t>(c) * 4, st) : cudaSuccess;
            if (e != cudaSuccess) return fail(RDVB_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
        }
        return RDVB_OK;
    }
    if (!dy || !x || !stats || !dx || !workspace)
        return fail(RDVB_ERR_INVALID_ARG, "dy, x, stats, dx and workspace must not be NULL");
    if (!aligned(x, size) || !aligned(dy, size) || !aligned(dx, size) || !aligned(weight, psize) ||
        !aligned(bias, psize) || !aligned(stats, 4) || !aligned(workspace, 16))
        return fail(RDVB_ERR_INVALID_ARG, "a pointer is not aligned (workspace: 16 bytes, others: their element)");
    const Plan a = plan(n, rows, c, groups, 1);
    if (workspace_bytes < static_cast<size_t>(a.bytes))
        return fail(RDVB_ERR_INVALID_ARG, "workspace holds %zu bytes; %lld are needed", workspace_bytes,
                    static_cast<long long>(a.bytes));
    rdvb_host::Device dev;
    if (int rc = rdvb_host::device(&dev)) return rc;
    Params p;
    fill(p, x, n, rows, c, groups, weight, bias, param_dtype, activation, 0.0f, a, workspace);
    p.dy = dy;
    p.out = dx;
    p.stats = const_cast<float*>(stats);
    p.dweight = dweight;
    p.dbias = dbias;
    const unsigned grid = static_cast<unsigned>(n * a.slabs);
    const unsigned more = dweight || dbias ? (c + 31) / 32 : 0;
    const size_t smem = static_cast<size_t>(groups) * 8;
    int rc = RDVB_OK;
    each_type(dtype, vector_width(dtype, c, {x, dy, dx}), [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int kVec = decltype(v)::value;
        grad_sums_kernel<T, kVec><<<grid, kThreads, 0, st>>>(p);
        if ((rc = rdvb_host::launched("group_norm grad_sums_kernel"))) return;
        grad_apply_kernel<T, kVec><<<grid + more, kThreads, smem, st>>>(p);
        rc = rdvb_host::launched("group_norm grad_apply_kernel");
    });
    return rc;
}

}  // extern "C"
