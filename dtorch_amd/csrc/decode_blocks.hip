// Single-token decode over listed blocks of tokens (semantics: dtattn.h, "attention over selected key blocks"): the arithmetic of
// SdpaOp::Compute (dtorch/core/operators/standard/scaled_dot_product_attention_op.cc:107-109) at Lq = 1 over the tokens of the blocks that
// select_blocks_kernel, or a caller, lists for each kv head.  The reference has no KV cache.
//
// Bound by HBM: the listed rows are read once.  Each (sequence, kv head) has the same number of units, so that shares need no
// prefix sum; a sequence inside one share is written directly, the others' records are merged by a second launch.
#include <algorithm>

#include "decode_parts.hpp"

namespace dtattn {

template <typename T, int D, bool TWO>
__global__ void __launch_bounds__(64 * kPartWaves, 2) decode_blocks_kernel(const PartsParams p) {
    __shared__ __attribute__((aligned(16))) float red_o[kPartWaves][16][D + 4];
    __shared__ float red_m[kPartWaves][16], red_l[kPartWaves][16];
    const int U = p.B * part_places(p.list_units);
    const PartShares sh(U * p.Hkv * p.nsub[1], p.shares);
    if ((int)blockIdx.x < sh.n) decode_part<T, D, kListPart, TWO>(p, PartLengths{}, PartScan{}, U, sh, blockIdx.x, red_o, red_m, red_l);
}

namespace {

struct BlocksPlan {
    int32_t kernel_d, nsub, units, shares;
    size_t rec_o, rec_ml;
};

BlocksPlan plan_blocks(const dtattn_decode_blocks_args* a, int cus) {
    BlocksPlan r;
    r.kernel_d = a->D <= 64 ? 64 : 128;
    r.nsub = (int32_t)((a->Hq / a->Hkv + 15) / 16);
    r.units = (int32_t)((a->n_blocks * a->block + kPartUnit - 1) / kPartUnit);
    const int64_t places = a->B * a->Hkv * r.nsub * (int64_t)(r.units + kPartExtra);
    r.shares = (int32_t)std::max<int64_t>(1, std::min<int64_t>((int64_t)2 * cus, places / kPartLeast));
    const size_t records = (size_t)2 * r.shares * 16;
    r.rec_o = part_up(records * r.kernel_d * sizeof(float));
    r.rec_ml = part_up(records * sizeof(float2));
    return r;
}

template <typename T, int D>
int launch_blocks(const PartsParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)p.shares), block(64 * kPartWaves);
    if (p.block_shift < 5) hipLaunchKernelGGL((decode_blocks_kernel<T, D, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((decode_blocks_kernel<T, D, false>), grid, block, 0, stream, p);
    const int st = check_launch("decode_blocks_kernel");
    if (st != DTATTN_OK) return st;
    const int64_t pairs = (int64_t)p.B * p.Hq;
    if (pairs <= 256) hipLaunchKernelGGL((decode_parts_merge_kernel<T, D, 4, false>), dim3((unsigned)pairs), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((decode_parts_merge_kernel<T, D, 1, false>), dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, stream, p);
    return check_launch("decode_parts_merge_kernel");
}

}  // namespace

}  // namespace dtattn

using namespace dtattn;

extern "C" size_t dtattn_decode_blocks_workspace_size(const dtattn_decode_blocks_args* a, void* stream) {
    if (a == nullptr || a->B <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->D <= 0 || a->n_blocks <= 0 || a->block <= 0) return 0;
    const int cus = stream_cus(reinterpret_cast<hipStream_t>(stream));
    const BlocksPlan plan = plan_blocks(a, cus > 0 ? cus : 256);
    return plan.rec_o + plan.rec_ml;
}

extern "C" int dtattn_decode_blocks(const dtattn_decode_blocks_args* a, void* stream_) {
    const char* who = "decode_blocks";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (a->B < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->D <= 0 || a->B > (1 << 24) || a->Hq > (1 << 20) || a->n_blocks <= 0 || a->n_blocks > (1 << 25))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
    if (a->Hq % a->Hkv != 0) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: Hq is not a multiple of Hkv", who);
    if (a->block < 16 || a->block > 256 || (a->block & (a->block - 1)) != 0)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: block %d must be a power of two from 16 to 256", who, a->block);
    // a unit's place in the list is a 32-bit number of tokens
    if (a->n_blocks * a->block > (1 << 30)) return fail(DTATTN_ERR_UNSUPPORTED, "%s: %lld listed tokens (up to 2^30)", who, (long long)(a->n_blocks * a->block));
    const bool paged = a->block_table != nullptr;
    if (paged) {
        if (a->page_size < 16 || (a->page_size & (a->page_size - 1)) != 0 || a->page_size > (1 << 20))
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: page_size %lld must be a power of two >= 16", who, (long long)a->page_size);
        if (a->page_size < a->block)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: a page of %lld tokens does not hold a block of %d", who, (long long)a->page_size, a->block);
        if (a->num_pages <= 0 || a->max_pages <= 0 || a->num_pages > 0x7fffffff || a->max_pages > (1 << 29) / a->page_size)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad page counts", who);
    } else if (a->S_max <= 0 || a->S_max > (1 << 29)) {
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad capacity", who);
    }
    const int64_t strides[10] = {a->q_stride[0], a->q_stride[1], a->o_stride[0], a->o_stride[1], a->k_stride[0],
                                 a->k_stride[1], a->k_stride[2], a->v_stride[0], a->v_stride[1], a->v_stride[2]};
    const int64_t rows[2] = {a->k_stride[2], a->v_stride[2]};
    int st = part_tensor_checks(a->D, a->dtype, strides, 10, rows, 2,
                                reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->o) | reinterpret_cast<uintptr_t>(a->k_cache) |
                                    reinterpret_cast<uintptr_t>(a->v_cache), who);
    if (st != DTATTN_OK) return st;
    ScalePlan sp;
    st = plan_scale(a->scale, a->D, a->dtype == DTATTN_FP32 ? kSign32 : kSign16, &sp);
    if (st != DTATTN_OK || a->B == 0) return st;
    if (a->q == nullptr || a->o == nullptr || a->k_cache == nullptr || a->v_cache == nullptr || a->lengths == nullptr || a->blocks == nullptr)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    const int cus = stream_cus(stream);
    if (cus <= 0) return fail(DTATTN_ERR_DEVICE, "%s: cannot tell the stream's device", who);
    const BlocksPlan plan = plan_blocks(a, cus);
    if (a->B * a->Hkv * plan.nsub * (int64_t)(plan.units + kPartExtra) >= ((int64_t)1 << 31) || a->B * a->Hq > 0x7fffffff)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: too many blocks", who);
    const size_t need = plan.rec_o + plan.rec_ml;
    if (a->workspace == nullptr || a->workspace_bytes < need)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, need, a->workspace_bytes);
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);

    PartsParams p = {};
    const int64_t esz = a->dtype == DTATTN_FP32 ? 4 : 2;
    p.q = reinterpret_cast<const char*>(a->q), p.o = reinterpret_cast<char*>(a->o), p.lse = a->lse;
    p.k[1] = reinterpret_cast<const char*>(a->k_cache), p.v[1] = reinterpret_cast<const char*>(a->v_cache);
    p.k_b[1] = a->k_stride[0] * esz, p.k_h[1] = a->k_stride[1] * esz, p.k_s[1] = a->k_stride[2] * esz;
    p.v_b[1] = a->v_stride[0] * esz, p.v_h[1] = a->v_stride[1] * esz, p.v_s[1] = a->v_stride[2] * esz;
    if (paged) {
        p.table = a->block_table, p.bt_s = a->block_table_stride;
        p.page_shift = __builtin_ctzll((unsigned long long)a->page_size), p.num_pages = (int32_t)a->num_pages;
    }
    p.capacity[1] = (int32_t)(paged ? a->max_pages * a->page_size : a->S_max);
    p.lengths = a->lengths, p.list = a->blocks;
    p.list_b = a->blocks_stride[0], p.list_h = a->blocks_stride[1];
    p.n_list = (int32_t)a->n_blocks, p.list_units = plan.units, p.block_shift = __builtin_ctz((unsigned)a->block);
    p.nsub[1] = plan.nsub, p.shares = plan.shares, p.columns[1] = 16;
    p.rec_o[1] = reinterpret_cast<float*>(a->workspace);
    p.rec_ml[1] = reinterpret_cast<float2*>(reinterpret_cast<char*>(a->workspace) + plan.rec_o);
    p.q_b = a->q_stride[0], p.q_h = a->q_stride[1], p.o_b = a->o_stride[0], p.o_h = a->o_stride[1];
    p.lse_b = a->lse != nullptr ? a->lse_stride[0] : 0;
    p.B = (int32_t)a->B, p.Hq = (int32_t)a->Hq, p.Hkv = (int32_t)a->Hkv, p.group = (int32_t)(a->Hq / a->Hkv);
    p.groups = p.B, p.per = 1;
    p.d = (int32_t)a->D;
    p.c = sp.scale * kLog2e;
    p.q_and = sp.q_and, p.q_xor = sp.q_xor;
    const bool wide = plan.kernel_d == 128;
    switch (a->dtype) {
        case DTATTN_BF16: return wide ? launch_blocks<bf16_t, 128>(p, stream) : launch_blocks<bf16_t, 64>(p, stream);
        case DTATTN_FP16: return wide ? launch_blocks<f16_t, 128>(p, stream) : launch_blocks<f16_t, 64>(p, stream);
        default: return wide ? launch_blocks<float, 128>(p, stream) : launch_blocks<float, 64>(p, stream);
    }
}
