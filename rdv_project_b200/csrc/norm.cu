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

// Slabs of a sample: four blocks a processor over the batch, so that one round
// of blocks does it, but at least 16 rows each and at most kMaxSlabs a sample
// (of up to four samples, fewer blocks than that).
Plan plan(int64_t n, int64_t rows, int c, int groups, int backward) {
    Plan a;
    const int64_t want = std::max<int64_t>(1, 592 / std::max<int64_t>(n, 1));
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

// How a call's threads lie: elements of one access, and whether each access
// lies in one group. The most (up to 16 bytes) that divide a group's channels
// and that every pointer is aligned to, where that is four bytes or more;
// otherwise the most that divide the row, across groups.
struct Access {
    int vec;
    bool one;
};
Access access(int dtype, int c, int groups, std::initializer_list<const void*> ptrs) {
    const int size = dtype == RDVB_F32 ? 4 : 2;
    auto widest = [&](int divides) {
        int w = 16 / size;
        while (w > 1 && divides % w) w /= 2;
        for (const void* q : ptrs)
            while (w > 1 && !aligned(q, static_cast<uintptr_t>(w) * size)) w /= 2;
        return w;
    };
    const int w = widest(c / groups);
    return w * size >= 4 ? Access{w, true} : Access{widest(c), false};
}

// f(element, vector width, one group an access, activation): silu has its own
// kernels where accesses are 16 bytes, the others take it at run time.
template <typename F>
void each_kind(int dtype, Access a, int act, F&& f) {
    using std::bool_constant;
    using std::integral_constant;
    auto with_act = [&](auto t, auto v, auto one) {
        if constexpr (decltype(v)::value * sizeof(t) == 16)
            if (act == kSilu) return f(t, v, one, integral_constant<int, kSilu>{});
        f(t, v, one, integral_constant<int, kRuntime>{});
    };
    auto with_one = [&](auto t, auto v) {
        if constexpr (decltype(v)::value * sizeof(t) >= 4)
            if (a.one) return with_act(t, v, bool_constant<true>{});
        with_act(t, v, bool_constant<false>{});
    };
    auto with_vec = [&](auto t) {
        if constexpr (sizeof(t) == 2)
            if (a.vec == 8) return with_one(t, integral_constant<int, 8>{});
        if (a.vec == 4) return with_one(t, integral_constant<int, 4>{});
        if (a.vec == 2) return with_one(t, integral_constant<int, 2>{});
        with_one(t, integral_constant<int, 1>{});
    };
    if (dtype == RDVB_F32) with_vec(float{});
    else if (dtype == RDVB_F16) with_vec(__half{});
    else with_vec(__nv_bfloat16{});
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

static int check_workspace(int64_t n, int64_t rows, int c, int groups, int backward, size_t have) {
    const int64_t need = rdvb_group_norm_workspace_bytes(n, rows, c, groups, backward);
    if (have < static_cast<size_t>(need))
        return fail(RDVB_ERR_INVALID_ARG, "workspace holds %zu bytes; %lld are needed", have, static_cast<long long>(need));
    return RDVB_OK;
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
    if (int rc = check_workspace(n, rows, c, groups, 0, workspace_bytes)) return rc;
    rdvb_host::Device dev;
    if (int rc = rdvb_host::device(&dev)) return rc;
    const Access w = access(dtype, c, groups, {x, y});
    const Plan a = plan(n, rows, c, groups, 0);
    Params p;
    fill(p, x, n, rows, c, groups, weight, bias, param_dtype, activation, eps, a, workspace);
    p.out = y;
    p.stats = stats;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // A block a sample in one launch: where the sample fits, in whole 16-byte pieces, and either the samples fill
    // the processors or they are so small that a second launch costs more than the idle ones.
    const int64_t sample = rows * c * static_cast<int64_t>(size);
    uint32_t* status = nullptr;
    if (w.one && c / w.vec <= kThreads && groups <= kThreads && sample <= kSmallBytes && sample % 16 == 0 &&
        aligned(x, 16) && (n >= dev.sm_count || sample <= kSmallBytes / 2))
        if (int rc = rdvb_host::status_word(&status)) return rc;
    const unsigned grid = static_cast<unsigned>(n * a.slabs);
    const size_t smem = static_cast<size_t>(groups) * 8;
    int rc = RDVB_OK;
    each_kind(dtype, w, activation, [&](auto t, auto v, auto one, auto act) {
        using T = decltype(t);
        constexpr int kVec = decltype(v)::value, kAct = decltype(act)::value;
        constexpr bool kOne = decltype(one)::value;
        if constexpr (kOne) {
            if (status) {
                auto kernel = small_kernel<T, kVec, kAct>;
                if ((rc = rdvb_host::allow_smem(reinterpret_cast<const void*>(kernel), kSmallBytes, dev.index))) return;
                kernel<<<static_cast<unsigned>(n), kThreads, static_cast<size_t>(sample), st>>>(p, status);
                rc = rdvb_host::launched("group_norm small_kernel");
                return;
            }
        }
        sums_kernel<T, kVec, kOne><<<grid, kThreads, groups * 12, st>>>(p);
        if ((rc = rdvb_host::launched("group_norm sums_kernel"))) return;
        apply_kernel<T, kVec, kOne, kAct><<<grid, kThreads, smem, st>>>(p);
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
    if (int rc = check_workspace(n, rows, c, groups, 1, workspace_bytes)) return rc;
    rdvb_host::Device dev;
    if (int rc = rdvb_host::device(&dev)) return rc;
    const Plan a = plan(n, rows, c, groups, 1);
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
    each_kind(dtype, access(dtype, c, groups, {x, dy, dx}), activation, [&](auto t, auto v, auto one, auto act) {
        using T = decltype(t);
        constexpr int kVec = decltype(v)::value, kAct = decltype(act)::value;
        constexpr bool kOne = decltype(one)::value;
        grad_sums_kernel<T, kVec, kOne, kAct><<<grid, kThreads, 0, st>>>(p);
        if ((rc = rdvb_host::launched("group_norm grad_sums_kernel"))) return;
        grad_apply_kernel<T, kVec, kOne, kAct><<<grid + more, kThreads, smem, st>>>(p);
        rc = rdvb_host::launched("group_norm grad_apply_kernel");
    });
    return rc;
}

}  // extern "C"
