// rdvb_attention_* (include/rdvb.h).
#include <algorithm>
#include <cmath>
#include <cstring>

#define RDVB_STATUS_ELSEWHERE
#include "attention.cuh"
#include "attention_tc.cuh"
#include "attention_tc_grad.cuh"
#include "attention_few.cuh"
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

// Whether the tensor-core kernels take the call: 16-bit elements, a head
// dimension of whole 16-byte pieces up to 128, q, k and v as tensor maps take
// them (16-byte aligned, strides of whole 16-byte pieces; a sample or head
// stride of 0 is an axis of one) and a scale that keeps the scores' order.
bool tensor_core(const rdvb_attention* a) {
    if (a->dtype == RDVB_F32 || a->dim > 128 || a->dim % 8 || !(a->scale > 0.0f)) return false;
    if (a->kv_len == 0 || !aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16)) return false;
    auto fits = [](const int64_t* stride, int64_t batch, int64_t length, int64_t heads) {
        const int64_t extent[3] = {batch, length, heads};
        for (int i = 0; i < 3; ++i) {
            const int64_t s = stride[i];
            if (extent[i] > 1 && (s % 8 || s < 0 || s >= (1LL << 38) || (s == 0 && i == 1))) return false;
        }
        return true;
    };
    if (!fits(a->q_stride, a->batch, a->q_len, a->heads) || !fits(a->k_stride, a->batch, a->kv_len, a->kv_heads) ||
        !fits(a->v_stride, a->batch, a->kv_len, a->kv_heads))
        return false;
    return rdvb_host::tensor_map_encoder() != nullptr;
}

// Whether the few-row kernel takes the forward pass: at most eight rows a key
// head, rows of whole 16-byte pieces up to 128 dimensions, 16-byte aligned.
bool few_rows(const rdvb_attention* a) {
    const int vec = a->dtype == RDVB_F32 ? 4 : 8;
    if (a->q_len * (a->heads / a->kv_heads) > kFewRows || a->dim > 128 || a->dim % vec) return false;
    if (!aligned(a->q, 16) || !aligned(a->k, 16) || !aligned(a->v, 16)) return false;
    for (int i = 0; i < 3; ++i)
        if (a->q_stride[i] % vec || a->k_stride[i] % vec || a->v_stride[i] % vec) return false;
    return true;
}

// The map of [batch, length, heads, dim] that a tile of 128 positions of one
// head is loaded by, in atoms of 64 dimensions; past the ends it reads 0.
int encode(TcMap* out, const rdvb_attention* a, const void* base, const int64_t* stride, int64_t length, int heads) {
    out->head_step = heads > 1 && stride[2] != 0;
    out->batch_step = a->batch > 1 && stride[0] != 0;
    auto bytes = [](bool walked, int64_t s) -> cuuint64_t { return walked ? s * 2 : 16; };
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a->dim), static_cast<cuuint64_t>(out->head_step ? heads : 1),
                                static_cast<cuuint64_t>(length),
                                static_cast<cuuint64_t>(out->batch_step ? a->batch : 1)};
    const cuuint64_t strides[3] = {bytes(out->head_step, stride[2]), bytes(length > 1, stride[1]),
                                   bytes(out->batch_step, stride[0])};
    const cuuint32_t box[4] = {64, 1, kTcTile, 1}, one[4] = {1, 1, 1, 1};
    const CUresult rc = rdvb_host::tensor_map_encoder()(
        &out->map, a->dtype == RDVB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
        const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS)
        return fail(RDVB_ERR_CUDA, "cuTensorMapEncodeTiled returned %d", static_cast<int>(rc));
    return RDVB_OK;
}

int tile_of(const rdvb_attention* a, bool tc) { return tc ? kTcTile : a->dim > 128 ? 32 : 64; }

// Parts that the long axis is split into: those that make the launch
// shortest. `blocks` blocks of `steps` loop steps run `slots` at a time, a
// step takes step_us; parts are written and read once more by a join
// (part_bytes each, at 3 TB/s with their launches' ends, and 4 us of launch;
// the sum of dQ's row sums, 2.4 us, is not counted). At least two steps a part,
// at most 32 parts.
int splits_for(int64_t blocks, int64_t steps, int64_t slots, double step_us, double part_bytes) {
    int best = 1;
    double least = 0.0;
    for (int s = 1; s <= 32 && (s == 1 || 2 * s <= steps); ++s) {
        const double rounds = static_cast<double>(ceil_div(blocks * s, slots));
        const double us = rounds * static_cast<double>(ceil_div(steps, s)) * step_us +
                          (s > 1 ? 4.0 + 2.0 * s * part_bytes / 3e6 : 0.0);
        if (s == 1 || us < 0.97 * least) {
            best = s;
            least = us;
        }
    }
    return best;
}

struct Plan {
    bool tc, few;
    int forward, dq, dkv;  // splits
    int64_t forward_len, dq_len, dkv_len;
    int64_t forward_bytes, backward_bytes, delta_bytes, dq_bytes, q_pad;
};

Plan plan(const rdvb_attention* a) {
    Plan p;
    p.tc = tensor_core(a);
    const int tile = tile_of(a, p.tc), back = tile;
    const int64_t q_tiles = ceil_div(a->q_len, tile), k_tiles = ceil_div(a->kv_len, tile);
    const int64_t rows = static_cast<int64_t>(a->batch) * a->q_len * a->heads;
    const int64_t kv_rows = static_cast<int64_t>(a->batch) * a->kv_len * a->kv_heads;
    // The tensor-core kernels hold one block a processor (the forward one takes two query tiles). The CUDA-core ones
    // are counted as two; above 64 dimensions shared memory holds one (129 to 256 forward: two). Microseconds a step, measured: 128 keys against 256 queries, 128 x 128 for dQ and for dK and dV; 64 x 64.
    const int64_t slots = p.tc ? 148 : 296;
    const bool narrow = a->dim <= 64;
    const double row_bytes = static_cast<double>(a->dim) * 4;
    p.forward = splits_for((p.tc ? ceil_div(q_tiles, 2) : q_tiles) * a->heads * a->batch, k_tiles, slots,
                           p.tc ? (narrow ? 1.9 : 2.5) : 12.0, rows * row_bytes);
    p.forward_len = ceil_div(k_tiles, p.forward) * tile;
    p.few = few_rows(a);
    if (p.few) {
        // three blocks a processor stream the keys, 64 or more each (223 pairs of a sample and a key head, or more:
        // a block each)
        const int64_t heads = static_cast<int64_t>(a->batch) * a->kv_heads;
        const int64_t most = std::min<int64_t>(ceil_div(a->kv_len, 64), kMaxSplits);
        const int64_t want = std::max<int64_t>(1, std::min(most, 3 * 148 / std::max<int64_t>(heads, 1)));
        p.forward_len = ceil_div(ceil_div(a->kv_len, want), 64) * 64;
    }
    p.forward = static_cast<int>(std::max<int64_t>(1, ceil_div(a->kv_len, std::max<int64_t>(p.forward_len, 1))));
    p.forward_bytes = p.forward > 1 ? round16(p.forward * rows * 8) + p.forward * rows * a->dim * 4 : 0;
    // gradients
    const int64_t bq_tiles = ceil_div(a->q_len, back), bk_tiles = ceil_div(a->kv_len, back);
    p.dq = splits_for(bq_tiles * a->heads * a->batch, bk_tiles, slots,
                      p.tc ? (narrow ? 1.4 : 1.6) : 16.0, rows * row_bytes);
    p.dq_len = ceil_div(bk_tiles, p.dq) * back;
    p.dq = static_cast<int>(std::max<int64_t>(1, ceil_div(a->kv_len, std::max<int64_t>(p.dq_len, 1))));
    const int64_t items = bq_tiles * (a->heads / a->kv_heads);
    p.dkv = splits_for(bk_tiles * a->kv_heads * a->batch, items, slots,
                       p.tc ? (narrow ? 1.5 : 2.4) : 16.0, 2 * kv_rows * row_bytes);
    p.dkv_len = ceil_div(items, p.dkv);
    p.dkv = static_cast<int>(std::max<int64_t>(1, ceil_div(items, std::max<int64_t>(p.dkv_len, 1))));
    p.q_pad = bq_tiles * back;
    const int64_t stat_bytes = static_cast<int64_t>(a->batch) * a->heads * p.q_pad * 4;
    p.delta_bytes = p.tc ? (2 + (p.dq > 1 ? p.dq : 0)) * stat_bytes + kPrepBlocks * 8 : round16(rows * 4);
    const int64_t dq_bytes = p.dq > 1 ? p.dq * rows * a->dim * 4 : 0;
    const int64_t dkv_bytes = p.dkv > 1 ? 2 * p.dkv * kv_rows * a->dim * 4 : 0;
    p.dq_bytes = round16(dq_bytes);
    p.backward_bytes = p.delta_bytes + p.dq_bytes + dkv_bytes;
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
int launch(K kernel, int64_t blocks, int smem, const Params& p, int device, cudaStream_t st, const char* what) {
    if (blocks > 0x7fffffffLL) return fail(RDVB_ERR_UNSUPPORTED, "%s: too many blocks", what);
    if (int rc = rdvb_host::allow_smem(reinterpret_cast<const void*>(kernel), smem, device)) return rc;
    kernel<<<static_cast<unsigned>(blocks), kThreads, smem, st>>>(p);
    return rdvb_host::launched(what);
}

#define RDVB_BY_DIM(kernel, bytes, ...)                                                                     \
    (a->dim <= 32    ? launch(kernel<32>, __VA_ARGS__ Shape<32>::bytes, p, dev.index, st, #kernel)                     \
     : a->dim <= 64  ? launch(kernel<64>, __VA_ARGS__ Shape<64>::bytes, p, dev.index, st, #kernel)                     \
     : a->dim <= 128 ? launch(kernel<128>, __VA_ARGS__ Shape<128>::bytes, p, dev.index, st, #kernel)                   \
                     : launch(kernel<256>, __VA_ARGS__ Shape<256>::bytes, p, dev.index, st, #kernel))

int launch_tc_forward(const rdvb_attention* a, const Params& p, const rdvb_host::Device& dev, cudaStream_t st) {
    const int64_t items = ceil_div(a->q_len, 2 * kTcTile) * a->heads * a->batch * p.splits;
    if (items > 0x3fffffffLL) return fail(RDVB_ERR_UNSUPPORTED, "tc_forward_kernel: too many query tiles");
    TcParams t;
    t.a = p;
    if (int rc = rdvb_host::status_word(&t.status)) return rc;
    t.k_steps = static_cast<uint32_t>((a->dim + 15) / 16);
    t.n_pv = 16 * t.k_steps;
    t.guarded = a->lengths || a->mask;
    TcMap q, k, v;
    if (int rc = encode(&q, a, a->q, a->q_stride, a->q_len, a->heads)) return rc;
    if (int rc = encode(&k, a, a->k, a->k_stride, a->kv_len, a->kv_heads)) return rc;
    if (int rc = encode(&v, a, a->v, a->v_stride, a->kv_len, a->kv_heads)) return rc;
    auto go = [&](auto kernel, uint32_t smem) -> int {
        if (int rc = rdvb_host::allow_smem(reinterpret_cast<const void*>(kernel), static_cast<int>(smem), dev.index))
            return rc;
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(items, dev.sm_count));
        kernel<<<grid, kTcThreads, smem, st>>>(t, static_cast<uint32_t>(items), q, k, v);
        return rdvb_host::launched("tc_forward_kernel");
    };
    const bool bf16 = a->dtype == RDVB_BF16;
    if (a->dim <= 64)
        return bf16 ? go(tc_forward_kernel<64, true>, TcForward<64>::kBytes)
                    : go(tc_forward_kernel<64, false>, TcForward<64>::kBytes);
    return bf16 ? go(tc_forward_kernel<128, true>, TcForward<128>::kBytes)
                : go(tc_forward_kernel<128, false>, TcForward<128>::kBytes);
}

template <typename T>
int launch_few(const rdvb_attention* a, const Params& p, const rdvb_host::Device& dev, cudaStream_t st) {
    const int64_t blocks = static_cast<int64_t>(a->batch) * a->kv_heads * p.splits;
    if (blocks > 0x7fffffffLL) return fail(RDVB_ERR_UNSUPPORTED, "few_kernel: too many blocks");
    const int64_t rows = a->q_len * (a->heads / a->kv_heads), lanes = a->dim / static_cast<int>(16 / sizeof(T));
    auto run = [&](auto kernel, int smem) -> int {
        if (int rc = rdvb_host::allow_smem(reinterpret_cast<const void*>(kernel), smem, dev.index)) return rc;
        kernel<<<static_cast<unsigned>(blocks), kFewThreads, smem, st>>>(p);
        return rdvb_host::launched("few_kernel");
    };
    auto go = [&](auto n) -> int {
        constexpr int kLanes = decltype(n)::value;
        if (rows <= 1) return run(few_kernel<T, kLanes, 1>, Few<T, kLanes, 1>::kBytes);
        if (rows <= 2) return run(few_kernel<T, kLanes, 2>, Few<T, kLanes, 2>::kBytes);
        if (rows <= 4) return run(few_kernel<T, kLanes, 4>, Few<T, kLanes, 4>::kBytes);
        return run(few_kernel<T, kLanes, 8>, Few<T, kLanes, 8>::kBytes);
    };
    if (lanes <= 8) return go(std::integral_constant<int, 8>{});
    if constexpr (sizeof(T) == 4)
        if (lanes > 16) return go(std::integral_constant<int, 32>{});
    return go(std::integral_constant<int, 16>{});
}

int simple_launch_check(int64_t blocks, const char* what) {
    return blocks > 0x7fffffffLL ? fail(RDVB_ERR_UNSUPPORTED, "%s: too many blocks", what) : RDVB_OK;
}

// dQ, dK and dV, or their parts, of a call that tensor_core() takes.
int launch_tc_backward(const rdvb_attention* a, const Plan& l, Params p, void* workspace, const rdvb_host::Device& dev,
                       cudaStream_t st) {
    GradParams g;
    if (int rc = rdvb_host::status_word(&g.status)) return rc;
    const int64_t stats = static_cast<int64_t>(a->batch) * a->heads * l.q_pad;
    g.neg_lse = static_cast<float*>(workspace);
    g.neg_delta = g.neg_lse + stats;
    g.norms = reinterpret_cast<float2*>(g.neg_delta + stats);
    g.slips = reinterpret_cast<float*>(g.norms + kPrepBlocks);
    g.q_pad = l.q_pad;
    g.k_steps = static_cast<uint32_t>((a->dim + 15) / 16);
    g.n_pv = 16 * g.k_steps;
    g.guarded = a->lengths || a->mask;
    TcMap q, k, v, d;
    const int64_t dense[3] = {a->q_len * a->heads * a->dim, static_cast<int64_t>(a->heads) * a->dim, a->dim};
    if (int rc = encode(&q, a, a->q, a->q_stride, a->q_len, a->heads)) return rc;
    if (int rc = encode(&k, a, a->k, a->k_stride, a->kv_len, a->kv_heads)) return rc;
    if (int rc = encode(&v, a, a->v, a->v_stride, a->kv_len, a->kv_heads)) return rc;
    if (int rc = encode(&d, a, p.dout, dense, a->q_len, a->heads)) return rc;
    const bool bf16 = a->dtype == RDVB_BF16, narrow = a->dim <= 64;
    g.a = p;
    if (narrow)
        bf16 ? tc_prep_kernel<8, true><<<kPrepBlocks, kThreads, 0, st>>>(g)
             : tc_prep_kernel<8, false><<<kPrepBlocks, kThreads, 0, st>>>(g);
    else
        bf16 ? tc_prep_kernel<16, true><<<kPrepBlocks, kThreads, 0, st>>>(g)
             : tc_prep_kernel<16, false><<<kPrepBlocks, kThreads, 0, st>>>(g);
    if (int rc = rdvb_host::launched("tc_prep_kernel")) return rc;
    g.a.splits = l.dq;
    g.a.split_len = l.dq_len;
    const int64_t items = l.q_pad / kTcTile * a->heads * a->batch * l.dq;
    if (items > 0x3fffffffLL) return fail(RDVB_ERR_UNSUPPORTED, "tc_dq_kernel: too many query tiles");
    auto go_q = [&](auto kernel, uint32_t smem) -> int {
        if (int rc = rdvb_host::allow_smem(reinterpret_cast<const void*>(kernel), static_cast<int>(smem), dev.index))
            return rc;
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>(items, dev.sm_count));
        kernel<<<grid, kGradThreads, smem, st>>>(g, static_cast<uint32_t>(items), q, k, v, d);
        return rdvb_host::launched("tc_dq_kernel");
    };
    if (int rc = narrow ? (bf16 ? go_q(tc_dq_kernel<64, true>, TcDq<64>::kBytes)
                                : go_q(tc_dq_kernel<64, false>, TcDq<64>::kBytes))
                        : (bf16 ? go_q(tc_dq_kernel<128, true>, TcDq<128>::kBytes)
                                : go_q(tc_dq_kernel<128, false>, TcDq<128>::kBytes)))
        return rc;
    if (l.dq > 1) {
        const int64_t slip_blocks = ceil_div(stats, kThreads);
        if (int rc = simple_launch_check(slip_blocks, "tc_slips_kernel")) return rc;
        tc_slips_kernel<<<static_cast<unsigned>(slip_blocks), kThreads, 0, st>>>(g);
        if (int rc = rdvb_host::launched("tc_slips_kernel")) return rc;
    }
    g.a.splits = l.dkv;
    g.a.split_len = l.dkv_len;
    const int64_t blocks = ceil_div(a->kv_len, kTcTile) * a->kv_heads * a->batch * l.dkv;
    if (blocks > 0x7fffffffLL) return fail(RDVB_ERR_UNSUPPORTED, "tc_dkv_kernel: too many blocks");
    auto go = [&](auto kernel, uint32_t smem) -> int {
        if (int rc = rdvb_host::allow_smem(reinterpret_cast<const void*>(kernel), static_cast<int>(smem), dev.index))
            return rc;
        kernel<<<static_cast<unsigned>(blocks), kGradThreads, smem, st>>>(g, q, k, v, d);
        return rdvb_host::launched("tc_dkv_kernel");
    };
    return narrow ? (bf16 ? go(tc_dkv_kernel<64, true>, TcDkv<64>::kBytes) : go(tc_dkv_kernel<64, false>, TcDkv<64>::kBytes))
                  : (bf16 ? go(tc_dkv_kernel<128, true>, TcDkv<128>::kBytes)
                          : go(tc_dkv_kernel<128, false>, TcDkv<128>::kBytes));
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
    if (!out || !aligned(out, 16) || !aligned(lse, 4))
        return fail(RDVB_ERR_INVALID_ARG, "out must be a 16-byte aligned pointer, lse 4-byte aligned");
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
    const int64_t blocks = ceil_div(a->q_len, tile_of(a, l.tc)) * a->heads * a->batch * p.splits;
    if (l.few) {
        const int rc = a->dtype == RDVB_F32   ? launch_few<float>(a, p, dev, st)
                       : a->dtype == RDVB_F16 ? launch_few<__half>(a, p, dev, st)
                                              : launch_few<__nv_bfloat16>(a, p, dev, st);
        if (rc) return rc;
    } else if (l.tc) {
        if (int rc = launch_tc_forward(a, p, dev, st)) return rc;
    } else if (int rc = RDVB_BY_DIM(forward_kernel, kForwardBytes, blocks, )) {
        return rc;
    }
    if (p.splits > 1) {
        const int64_t join = ceil_div(rows * ceil_div(a->dim, 32), kThreads / 32);
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
    if (!aligned(dout, 16) || !aligned(out, 16) || !aligned(dq, 16) || !aligned(dk, 16) || !aligned(dv, 16) ||
        !aligned(lse, 4))
        return fail(RDVB_ERR_INVALID_ARG, "dout, out, dq, dk and dv must be 16-byte aligned, lse 4-byte aligned");
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
    p.out = out;
    p.dout = dout;
    p.lse = const_cast<float*>(lse);
    p.delta = static_cast<float*>(workspace);
    p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.delta_bytes);
    p.dq = dq;
    p.dk = dk;
    p.dv = dv;
    p.part_kv = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.delta_bytes + l.dq_bytes);
    if (l.tc) {
        if (int rc = launch_tc_backward(a, l, p, workspace, dev, st)) return rc;
    } else {
        const int64_t delta_blocks = ceil_div(rows, kThreads / 32);
        if (int rc = simple_launch_check(delta_blocks, "delta_kernel")) return rc;
        delta_kernel<<<static_cast<unsigned>(delta_blocks), kThreads, 0, st>>>(p);
        if (int rc = rdvb_host::launched("delta_kernel")) return rc;
        const int tile = tile_of(a, false);
        p.splits = l.dq;
        p.split_len = l.dq_len;
        int64_t blocks = ceil_div(a->q_len, tile) * a->heads * a->batch * p.splits;
        if (int rc = RDVB_BY_DIM(dq_kernel, kBackwardBytes, blocks, )) return rc;
        p.splits = l.dkv;
        p.split_len = l.dkv_len;
        blocks = ceil_div(a->kv_len, tile) * a->kv_heads * a->batch * p.splits;
        if (int rc = RDVB_BY_DIM(dkv_kernel, kBackwardBytes, blocks, )) return rc;
    }
    if (l.dq == 1 && l.dkv == 1) return RDVB_OK;
    const int64_t nq = rows * a->dim, nk = kv_rows * a->dim;
    Joins j;
    j.g[0] = {p.part, dq, nq, nq, l.dq > 1 ? l.dq : 0};
    j.g[1] = {p.part_kv, dk, nk, 2 * nk, l.dkv > 1 ? l.dkv : 0};
    j.g[2] = {p.part_kv + nk, dv, nk, 2 * nk, l.dkv > 1 ? l.dkv : 0};
    j.dtype = a->dtype;
    j.wide = nq % 4 == 0 && nk % 4 == 0;
    const int64_t most = std::max(l.dq > 1 ? nq : 0, l.dkv > 1 ? nk : 0);
    const int64_t blocks = ceil_div(most, 4 * (j.wide ? 4 * kThreads : kThreads));
    if (int rc = simple_launch_check(blocks, "join_kernel")) return rc;
    join_kernel<<<dim3(static_cast<unsigned>(blocks), 3), kThreads, 0, st>>>(j);
    return rdvb_host::launched("join_kernel");
}

}  // extern "C"
