// rdvb_attention_* (include/rdvb.h).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "attention.cuh"
#include "host.h"

using rdvb_host::aligned;
using rdvb_host::fail;

namespace {
using namespace rdvb::attn;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round16(int64_t v) { return (v + 15) / 16 * 16; }

int check(const rdvb_attention* a) {
    if (!a) return fail(RDVB_ERR_INVALID_ARG, "the description must not be NULL");
    if (a->dtype != RDVB_F32 && a->dtype != RDVB_F16 && a->dtype != RDVB_BF16)
        return fail(RDVB_ERR_INVALID_ARG, "dtype %d is not RDVB_F32/F16/BF16", a->dtype);
    if (a->batch < 0 || a->q_len < 0 || a->kv_len < 0) return fail(RDVB_ERR_INVALID_ARG, "sizes must be >= 0");
    if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads)
        return fail(RDVB_ERR_INVALID_ARG, "kv_heads (%d) must divide heads (%d)", a->kv_heads, a->heads);
    if (a->dim < 1 || a->dim > 256)
        return fail(RDVB_ERR_UNSUPPORTED, "head dimension must be in [1, 256], got %d", a->dim);
    if (!std::isfinite(a->scale)) return fail(RDVB_ERR_INVALID_ARG, "scale must be finite");
    if (a->heads > 65535 || a->q_len > 0x7fffffffLL || a->kv_len > 0x7fffffffLL)
        return fail(RDVB_ERR_UNSUPPORTED, "heads, q_len or kv_len is too large");
    return RDVB_OK;
}

int check_pointers(const rdvb_attention* a) {
    const uintptr_t size = a->dtype == RDVB_F32 ? 4 : 2;
    if (!a->q || (a->kv_len > 0 && (!a->k || !a->v))) return fail(RDVB_ERR_INVALID_ARG, "q, k and v must not be NULL");
    if (!aligned(a->q, size) || !aligned(a->k, size) || !aligned(a->v, size) || !aligned(a->lengths, 4))
        return fail(RDVB_ERR_INVALID_ARG, "q, k, v and lengths must be aligned to their element size");
    return RDVB_OK;
}

int tile_of(int dim) { return dim > 128 ? 32 : 64; }

// Parts into which a launch of `tiles` blocks with `items` loop steps each is
// split: as many as fill the processors about twice, none of fewer than four
// steps, at most 32 (their join reads every part).
int splits_for(int64_t tiles, int64_t items) {
    const int64_t want = 2 * 148 / std::max<int64_t>(tiles, 1);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, items / 4, 32})));
}

struct Plan {
    int forward, dkv;  // splits
    int64_t forward_len, dkv_len;
    int64_t forward_bytes, backward_bytes;
    int64_t delta_bytes, dq_bytes;
};

Plan plan(const rdvb_attention* a) {
    Plan p;
    const int tile = tile_of(a->dim);
    const int64_t q_tiles = ceil_div(a->q_len, tile), k_tiles = ceil_div(a->kv_len, tile);
    const int64_t rows = static_cast<int64_t>(a->batch) * a->q_len * a->heads;
    const int64_t kv_rows = static_cast<int64_t>(a->batch) * a->kv_len * a->kv_heads;
    p.forward = splits_for(q_tiles * a->heads * a->batch, k_tiles);
    p.forward_len = ceil_div(k_tiles, p.forward) * tile;
    p.forward = static_cast<int>(std::max<int64_t>(1, ceil_div(a->kv_len, std::max<int64_t>(p.forward_len, 1))));
    const int64_t items = q_tiles * (a->heads / a->kv_heads);
    p.dkv = splits_for(k_tiles * a->kv_heads * a->batch, items);
    p.dkv_len = ceil_div(items, p.dkv);
    p.dkv = static_cast<int>(std::max<int64_t>(1, ceil_div(items, std::max<int64_t>(p.dkv_len, 1))));
    p.forward_bytes = p.forward > 1 ? round16(p.forward * rows * 8) + p.forward * rows * a->dim * 4 : 0;
    p.delta_bytes = round16(rows * 4);
    p.dq_bytes = p.forward > 1 ? p.forward * rows * a->dim * 4 : 0;
    const int64_t dkv_bytes = p.dkv > 1 ? 2 * p.dkv * kv_rows * a->dim * 4 : 0;
    p.backward_bytes = p.delta_bytes + std::max(p.dq_bytes, dkv_bytes);  // the two are joined in turn
    return p;
}

void fill(Params& p, const rdvb_attention* a) {
    memset(&p, 0, sizeof(p));
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.lengths = a->lengths;
    p.mask = a->mask;
    p.mask_stride = a->mask_stride;
    p.qs = {a->q_stride[0], a->q_stride[1], a->q_stride[2]};
    p.ks = {a->k_stride[0], a->k_stride[1], a->k_stride[2]};
    p.vs = {a->v_stride[0], a->v_stride[1], a->v_stride[2]};
    p.q_len = a->q_len;
    p.kv_len = a->kv_len;
    p.dtype = a->dtype;
    p.batch = a->batch;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.dim = a->dim;
    p.splits = 1;
    p.split_len = a->kv_len;
    p.scale = a->scale;
    const uintptr_t quad = a->dtype == RDVB_F32 ? 16 : 8;
    bool wide = aligned(a->q, quad) && aligned(a->k, quad) && aligned(a->v, quad) && a->dim % 4 == 0;
    for (int i = 0; i < 3; ++i) wide &= a->q_stride[i] % 4 == 0 && a->k_stride[i] % 4 == 0 && a->v_stride[i] % 4 == 0;
    p.wide = wide;
}

template <typename K>
int launch(K kernel, int64_t blocks, int smem, const Params& p, cudaStream_t st, const char* what) {
    if (blocks > 0x7fffffffLL) return fail(RDVB_ERR_UNSUPPORTED, "%s: too many blocks", what);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(RDVB_ERR_CUDA, "cudaFuncSetAttribute(%s): %s", what, cudaGetErrorString(e));
    kernel<<<static_cast<unsigned>(blocks), kThreads, smem, st>>>(p);
    return rdvb_host::launched(what);
}

#define RDVB_BY_DIM(kernel, bytes, ...)                                                                     \
    (a->dim <= 32    ? launch(kernel<32>, __VA_ARGS__ Shape<32>::bytes, p, st, #kernel)                     \
     : a->dim <= 64  ? launch(kernel<64>, __VA_ARGS__ Shape<64>::bytes, p, st, #kernel)                     \
     : a->dim <= 128 ? launch(kernel<128>, __VA_ARGS__ Shape<128>::bytes, p, st, #kernel)                   \
                     : launch(kernel<256>, __VA_ARGS__ Shape<256>::bytes, p, st, #kernel))

int simple_launch_check(int64_t blocks, const char* what) {
    return blocks > 0x7fffffffLL ? fail(RDVB_ERR_UNSUPPORTED, "%s: too many blocks", what) : RDVB_OK;
}

}  // namespace

extern "C" {

int64_t rdvb_attention_workspace_bytes(const rdvb_attention* a, int backward) {
    if (check(a)) return 0;
    const Plan l = plan(a);
    return backward ? l.backward_bytes : l.forward_bytes;
}

int rdvb_attention_forward(const rdvb_attention* a, void* out, float* lse, void* workspace, size_t workspace_bytes,
                           void* stream) {
    if (int rc = check(a)) return rc;
    if (a->batch == 0 || a->q_len == 0) return RDVB_OK;
    if (int rc = check_pointers(a)) return rc;
    const uintptr_t size = a->dtype == RDVB_F32 ? 4 : 2;
    if (!out || !aligned(out, size) || !aligned(lse, 4))
        return fail(RDVB_ERR_INVALID_ARG, "out must not be NULL, out and lse aligned to their elements");
    const Plan l = plan(a);
    if (l.forward_bytes > 0 && (!workspace || !aligned(workspace, 16) ||
                                workspace_bytes < static_cast<size_t>(l.forward_bytes)))
        return fail(RDVB_ERR_INVALID_ARG, "workspace must be a 16-byte aligned pointer to %lld bytes",
                    static_cast<long long>(l.forward_bytes));
    rdvb_host::Device dev;
    if (int rc = rdvb_host::device(&dev)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    Params p;
    fill(p, a);
    p.o = out;
    p.lse = lse;
    p.splits = l.forward;
    p.split_len = l.forward_len;
    const int64_t rows = static_cast<int64_t>(a->batch) * a->q_len * a->heads;
    p.part_stat = static_cast<float*>(workspace);
    p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + round16(p.splits * rows * 8));
    const int64_t blocks = ceil_div(a->q_len, tile_of(a->dim)) * a->heads * a->batch * p.splits;
    if (int rc = RDVB_BY_DIM(forward_kernel, kForwardBytes, blocks, )) return rc;
    if (p.splits > 1) {
        const int64_t join = ceil_div(rows, kThreads / 32);
        if (int rc = simple_launch_check(join, "join_forward_kernel")) return rc;
        join_forward_kernel<<<static_cast<unsigned>(join), kThreads, 0, st>>>(p);
        return rdvb_host::launched("join_forward_kernel");
    }
    return RDVB_OK;
}

int rdvb_attention_backward(const rdvb_attention* a, const void* dout, const void* out, const float* lse, void* dq,
                            void* dk, void* dv, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = check(a)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uintptr_t size = a->dtype == RDVB_F32 ? 4 : 2;
    const int64_t rows = static_cast<int64_t>(a->batch) * a->q_len * a->heads;
    const int64_t kv_rows = static_cast<int64_t>(a->batch) * a->kv_len * a->kv_heads;
    if ((rows > 0 && (!dq || !dout || !out || !lse)) || (kv_rows > 0 && (!dk || !dv)))
        return fail(RDVB_ERR_INVALID_ARG, "dout, out, lse, dq, dk and dv must not be NULL");
    if (!aligned(dout, size) || !aligned(out, size) || !aligned(dq, size) || !aligned(dk, size) ||
        !aligned(dv, size) || !aligned(lse, 4))
        return fail(RDVB_ERR_INVALID_ARG, "a pointer is not aligned to its element size");
    if (rows == 0 || kv_rows == 0) {  // no pair: zero gradients
        if (rows == 0 && kv_rows == 0) return RDVB_OK;
        rdvb_host::Device dev;
        if (int rc = rdvb_host::device(&dev)) return rc;
        const int64_t n = (rows + kv_rows) * a->dim * static_cast<int64_t>(size);
        for (void* g : {rows ? dq : dk, rows ? nullptr : dv}) {
            cudaError_t e = g ? cudaMemsetAsync(g, 0, static_cast<size_t>(n), st) : cudaSuccess;
            if (e != cudaSuccess) return fail(RDVB_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
        }
        return RDVB_OK;
    }
    if (int rc = check_pointers(a)) return rc;
    const Plan l = plan(a);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < static_cast<size_t>(l.backward_bytes))
        return fail(RDVB_ERR_INVALID_ARG, "workspace must be a 16-byte aligned pointer to %lld bytes",
                    static_cast<long long>(l.backward_bytes));
    rdvb_host::Device dev;
    if (int rc = rdvb_host::device(&dev)) return rc;
    Params p;
    fill(p, a);
    p.wide = p.wide && aligned(dout, 4 * size) && aligned(out, 4 * size);
    p.out = out;
    p.dout = dout;
    p.lse = const_cast<float*>(lse);
    p.delta = static_cast<float*>(workspace);
    p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.delta_bytes);
    p.dq = dq;
    p.dk = dk;
    p.dv = dv;
    const int64_t delta_blocks = ceil_div(rows, kThreads / 32);
    if (int rc = simple_launch_check(delta_blocks, "delta_kernel")) return rc;
    delta_kernel<<<static_cast<unsigned>(delta_blocks), kThreads, 0, st>>>(p);
    if (int rc = rdvb_host::launched("delta_kernel")) return rc;
    const int tile = tile_of(a->dim);
    auto join = [&](const float* part, int splits, int64_t pitch, int64_t n, void* to) -> int {
        const int64_t blocks = ceil_div(n, kThreads);
        if (int rc = simple_launch_check(blocks, "join_kernel")) return rc;
        join_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(part, splits, pitch, n, to, a->dtype);
        return rdvb_host::launched("join_kernel");
    };
    p.splits = l.forward;
    p.split_len = l.forward_len;
    int64_t blocks = ceil_div(a->q_len, tile) * a->heads * a->batch * p.splits;
    if (int rc = RDVB_BY_DIM(dq_kernel, kBackwardBytes, blocks, )) return rc;
    if (p.splits > 1)
        if (int rc = join(p.part, p.splits, rows * a->dim, rows * a->dim, dq)) return rc;
    p.splits = l.dkv;
    p.split_len = l.dkv_len;
    blocks = ceil_div(a->kv_len, tile) * a->kv_heads * a->batch * p.splits;
    if (int rc = RDVB_BY_DIM(dkv_kernel, kBackwardBytes, blocks, )) return rc;
    if (p.splits > 1) {
        const int64_t n = kv_rows * a->dim;
        if (int rc = join(p.part, p.splits, 2 * n, n, dk)) return rc;
        if (int rc = join(p.part + n, p.splits, 2 * n, n, dv)) return rc;
    }
    return RDVB_OK;
}

}  // extern "C"
