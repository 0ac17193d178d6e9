// rdvb_dropout (include/rdvb.h).
#include <cmath>

#include "dropout.cuh"
#include "host.h"

using rdvb_host::aligned;
using rdvb_host::fail;

extern "C" int rdvb_dropout(const void* x, const void* residual, void* y, int dtype, int64_t n, double p,
                            uint64_t seed, uint64_t offset, void* stream) {
    using namespace rdvb::dropout;
    if (dtype != RDVB_F32 && dtype != RDVB_F16 && dtype != RDVB_BF16)
        return fail(RDVB_ERR_INVALID_ARG, "dtype %d is not RDVB_F32/F16/BF16", dtype);
    if (n < 0) return fail(RDVB_ERR_INVALID_ARG, "n must be >= 0");
    const double threshold = std::nearbyint(p * 4294967296.0);
    if (!(p >= 0.0) || !(threshold < 4294967296.0))
        return fail(RDVB_ERR_INVALID_ARG, "p must be in [0, 1 - 2^-32), got %g", p);
    if (n == 0) return RDVB_OK;
    if (!x || !y) return fail(RDVB_ERR_INVALID_ARG, "x and y must not be NULL");
    const uintptr_t size = dtype == RDVB_F32 ? 4 : 2;
    if (!aligned(x, size) || !aligned(y, size) || !aligned(residual, size))
        return fail(RDVB_ERR_INVALID_ARG, "x, residual and y must be aligned to their element size");
    rdvb_host::Device dev;
    if (int rc = rdvb_host::device(&dev)) return rc;
    Params a;
    a.x = x;
    a.residual = residual;
    a.y = y;
    a.n = n;
    a.offset = offset;
    a.key[0] = make_uint2(static_cast<uint32_t>(seed), static_cast<uint32_t>(seed >> 32));
    for (int r = 1; r < 10; ++r) a.key[r] = make_uint2(a.key[r - 1].x + 0x9E3779B9u, a.key[r - 1].y + 0xBB67AE85u);
    a.threshold = static_cast<uint32_t>(threshold);
    a.scale = static_cast<float>(1.0 / (1.0 - p));
    const bool wide = aligned(x, 16) && aligned(y, 16) && aligned(residual, 16);
    const int64_t per_block = kThreads * static_cast<int64_t>(16 / size);
    const int64_t blocks = (n + per_block - 1) / per_block;
    if (blocks > 0x7fffffffLL) return fail(RDVB_ERR_UNSUPPORTED, "n = %lld is too large", static_cast<long long>(n));
    const unsigned grid = static_cast<unsigned>(blocks);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto t) {
        using T = decltype(t);
        if (residual)
            wide ? dropout_kernel<T, true, true><<<grid, kThreads, 0, st>>>(a)
                 : dropout_kernel<T, false, true><<<grid, kThreads, 0, st>>>(a);
        else
            wide ? dropout_kernel<T, true, false><<<grid, kThreads, 0, st>>>(a)
                 : dropout_kernel<T, false, false><<<grid, kThreads, 0, st>>>(a);
    };
    if (dtype == RDVB_F32) go(float{});
    else if (dtype == RDVB_F16) go(__half{});
    else go(__nv_bfloat16{});
    return rdvb_host::launched("dropout_kernel");
}
