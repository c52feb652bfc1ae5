// Single-token decode of sequences that share a prefix (semantics: dtattn.h, "attention over a shared prefix"): the arithmetic of
// SdpaOp::Compute (dtorch/core/operators/standard/scaled_dot_product_attention_op.cc:107-109) at Lq = 1.  The reference has no KV cache.
//
// The prefix's keys meet the query heads of all sequences of a group as one matrix product, so they are
// read once per so many query rows instead of once per sequence; a long prefix of many sequences is bound by the matrix cores and the
// instructions around them, the sequences' own tokens by HBM.  Both write records (a base, a row sum
// and an undivided sum of P V each), which one more launch merges.
// 64 sequences of 32 heads and 8 kv heads, 16 to 1500 own tokens each behind 8192 shared ones, bf16, head dim 128 (233 MB of keys and
// values): 60 us, 3.9 TB/s.  4 samples of one prompt of 2000 tokens: 16 us, of which 11 are the first launch and 8000 cycles of those the
// lengths, the shares and the first loads.
#include <algorithm>

#include "decode_parts.hpp"

namespace dtattn {

namespace {

// Workgroups of the prefix, in eighths of all: as its units' cost is to that of all, with one of either kind at least where there is
// any work for it.  Rounded up, for a short part on too few workgroups is what all wait for: 96 sequences of up to 560 tokens of 20 heads
// behind 7 to 30 shared ones take 43 us, and 69 rounded to nearest; 64 behind 8192 60 and 62.
__device__ __forceinline__ int prefix_shares(float cost0, float cost1, int most) {
    const int eighth = most / 8;
    if (cost0 == 0.f) return 0;
    if (cost1 == 0.f) return most;
    return 8 * min(max((int)(cost0 / (cost0 + cost1) * (float)eighth) + 1, 1), eighth - 1);
}

}  // namespace

// One launch for both parts.  Workgroups go to the XCDs in turn; of those on an XCD the first ones take the prefix, so that a CU has some
// of both, and consecutive shares, whose column sets read the same keys, lie on one XCD and its L2.
// NC: the prefix by rows (16-bit types), 16 NC of them a wave; 0: by keys.
template <typename T, int D, int NC, bool TWO>
__global__ void __launch_bounds__(64 * kPartWaves, 2) decode_shared_kernel(const PartsParams p) {
    constexpr size_t kMeet = sizeof(float) * kPartWaves * 16 * (D + 4), kRing = NC > 0 ? sizeof(T) * 2 * 2 * kStageTokens * D : 0;
    __shared__ __attribute__((aligned(1024))) char lds[kMeet > kRing ? kMeet : kRing];
    float (*const red_o)[16][D + 4] = reinterpret_cast<float (*)[16][D + 4]>(lds);
    __shared__ float red_m[kPartWaves][16], red_l[kPartWaves][16];
    __shared__ int least[kPartGroups], lead[kPartGroups], said[kPartGroups];
    const PartLengths lens = part_lengths(p, least, lead, said);
    const bool tells = blockIdx.x == 0 && threadIdx.x < 64;
    PartScan scan[2];
    const int U0 = part_total<kPrefixPart>(p, lens, tells, scan[0]), U1 = part_total<kOwnPart>(p, lens, tells, scan[1]);
    const int V0 = U0 * p.Hkv * p.nsub[0], V1 = U1 * p.Hkv * p.nsub[1];
    const int most0 = prefix_shares((float)V0 * (float)p.weight[0], (float)V1 * (float)p.weight[1], p.shares), most1 = p.shares - most0;
    if (tells && threadIdx.x == 0) {
        const PartShares s0(V0, most0), s1(V1, most1);
        p.meta[0][0] = U0, p.meta[0][1] = s0.n, p.meta[0][2] = s0.q, p.meta[0][3] = s0.rem;
        p.meta[1][0] = U1, p.meta[1][1] = s1.n, p.meta[1][2] = s1.q, p.meta[1][3] = s1.rem;
    }
    const int x = blockIdx.x & 7, y = blockIdx.x >> 3;
    const bool first = y < most0 / 8;
    const PartShares sh(first ? V0 : V1, first ? most0 : most1);
    const int per = (sh.n + 7) / 8, at = first ? y : y - most0 / 8;  // shares of an XCD
    const int r = first && p.nsub[0] > 1 ? x * per + at : at * 8 + x;
    if ((first ? V0 : V1) == 0 || at >= per || r >= sh.n) return;
    if (first) {
        if constexpr (NC > 0) decode_part_rows<T, D, NC>(p, lens, scan[0], U0, sh, r, reinterpret_cast<T (*)[2][kStageTokens * D]>(lds));
        else decode_part<T, D, kPrefixPart, TWO>(p, lens, scan[0], U0, sh, r, red_o, red_m, red_l);
        return;
    }
    decode_part<T, D, kOwnPart, TWO>(p, lens, scan[1], U1, sh, r, red_o, red_m, red_l);
}

namespace {

struct SharedPlan {
    int32_t kernel_d, nc, nsub[2], shares, columns[2], weight[2];
    size_t meta[2], rec_o[2], rec_ml[2], whole_o, whole_ml, bytes;
};

// Places of a segment of so many tokens.
int64_t places_in(int64_t tokens) { return (tokens + kPartUnit - 1) / kPartUnit + kPartExtra; }

SharedPlan plan_shared(const dtattn_decode_shared_args* a, int cus) {
    SharedPlan r = {};
    const int64_t group = a->Hq / a->Hkv, rows = a->B / a->groups * group;
    r.kernel_d = a->D <= 64 ? 64 : 128;
    const bool f32 = a->dtype == DTATTN_FP32;
    // Many rows share a stage of keys in LDS, few divide the keys among the waves.  us with a prefix of 8192 tokens, by keys and by rows: 32
    // rows 23.6 and 25.6, 64 28.2 and 27.8, 256 57.9 and 42.0.  16 rows a wave up to 128, which leave the waves more to hide behind, 32 beyond,
    // where the stages count: 128 rows 29.1 and 34.0, 256 65.9 and 63.5 (with up to 1500 own tokens), 512 74.7 and 70.7 (500).
    r.nc = f32 || rows <= 32 ? 0 : rows <= 128 ? 1 : 2;
    r.columns[0] = r.nc > 0 ? 16 * r.nc * kPartWaves : 16, r.columns[1] = 16;
    // What a unit of the prefix costs, and one of the own tokens, of which the workgroups' division follows.  us at these weights and at others:
    // by keys 33.2 and (1:1) 36.1 (32 rows, 1000 to 4000 own tokens), 16 rows a wave 29.3 and (3:2) 33.1 (64 rows, up to 1500), 32 rows a wave
    // 70.7 and (1:1) 78.7 (512 rows, up to 500).
    r.weight[0] = r.nc == 0 ? 2 : r.nc == 1 ? 1 : 3, r.weight[1] = r.nc == 0 ? 3 : r.nc == 1 ? 1 : 2;
    r.shares = std::max(2 * cus / 8 * 8, 16);
    const int64_t cols[2] = {rows, group}, sets[2] = {a->groups, a->B};
    for (int s = 0; s < 2; ++s) {
        r.nsub[s] = (int32_t)((cols[s] + r.columns[s] - 1) / r.columns[s]);
        const size_t records = (size_t)2 * r.shares * r.columns[s];
        r.meta[s] = part_up((4 + 2 * (size_t)sets[s]) * sizeof(int32_t));
        r.rec_o[s] = part_up(records * r.kernel_d * sizeof(float));
        r.rec_ml[s] = part_up(records * sizeof(float2));
    }
    r.whole_o = part_up((size_t)a->B * a->Hq * r.kernel_d * sizeof(float));
    r.whole_ml = part_up((size_t)a->B * a->Hq * sizeof(float2));
    r.bytes = 2 * (r.whole_o + r.whole_ml);
    for (int s = 0; s < 2; ++s) r.bytes += r.meta[s] + r.rec_o[s] + r.rec_ml[s];
    return r;
}

template <typename T, int D, int NC>
void launch_parts(const PartsParams& p, hipStream_t stream) {
    const dim3 grid((unsigned)p.shares), block(64 * kPartWaves);
    if (p.table != nullptr && p.page_shift < 5) hipLaunchKernelGGL((decode_shared_kernel<T, D, NC, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((decode_shared_kernel<T, D, NC, false>), grid, block, 0, stream, p);
}

template <typename T, int D>
int launch_shared(const PartsParams& p, int nc, hipStream_t stream) {
    if constexpr (sizeof(T) == 2) {
        if (nc == 0) launch_parts<T, D, 0>(p, stream);
        else if (nc == 1) launch_parts<T, D, 1>(p, stream);
        else launch_parts<T, D, 2>(p, stream);
    } else {
        launch_parts<T, D, 0>(p, stream);
    }
    const int st = check_launch("decode_shared_kernel");
    if (st != DTATTN_OK) return st;
    const int64_t pairs = (int64_t)p.B * p.Hq;
    // Few pairs are cut into many records each: four waves to a pair.  Up to `most` records of the prefix; us of a call with four waves and
    // with one: 256 pairs 26.2 and 29.4, 512 29.4 and 31.9, 1024 40.9 and 40.6, 2048 67.2 and 62.1.
    const int64_t most = p.shares / ((int64_t)p.Hkv * p.nsub[0] * p.groups);
    if (pairs <= 256 || (pairs <= 1024 && most > 8)) hipLaunchKernelGGL((decode_parts_merge_kernel<T, D, 4, true>), dim3((unsigned)pairs), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((decode_parts_merge_kernel<T, D, 1, true>), dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, stream, p);
    return check_launch("decode_parts_merge_kernel");
}

}  // namespace

}  // namespace dtattn

using namespace dtattn;

extern "C" size_t dtattn_decode_shared_workspace_size(const dtattn_decode_shared_args* a, void* stream) {
    if (a == nullptr || a->B <= 0 || a->groups <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->D <= 0 || a->Hq < a->Hkv || a->B < a->groups) return 0;
    const int cus = stream_cus(reinterpret_cast<hipStream_t>(stream));
    return plan_shared(a, cus > 0 ? cus : 256).bytes;
}

extern "C" int dtattn_decode_shared(const dtattn_decode_shared_args* a, void* stream_) {
    const char* who = "decode_shared";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (a->B < 0 || a->groups <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->D <= 0 || a->B > (1 << 24) || a->Hq > (1 << 20))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
    if (a->Hq % a->Hkv != 0) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: Hq is not a multiple of Hkv", who);
    if (a->B % a->groups != 0) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: %lld sequences are not %lld equal groups", who, (long long)a->B, (long long)a->groups);
    if (a->groups > kPartGroups) return fail(DTATTN_ERR_UNSUPPORTED, "%s: %lld groups (up to %d)", who, (long long)a->groups, kPartGroups);
    const bool paged = a->block_table != nullptr;
    if (paged) {
        if (a->page_size < 16 || (a->page_size & (a->page_size - 1)) != 0 || a->page_size > (1 << 20))
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: page_size %lld must be a power of two >= 16", who, (long long)a->page_size);
        if (a->num_pages <= 0 || a->max_pages <= 0 || a->num_pages > 0x7fffffff || a->max_pages > (1 << 29) / a->page_size)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad page counts", who);
    } else if (a->S_prefix <= 0 || a->S_max <= 0 || a->S_prefix > (1 << 29) || a->S_max > (1 << 29)) {
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad capacities", who);
    }
    const int64_t strides[16] = {a->q_stride[0], a->q_stride[1], a->o_stride[0], a->o_stride[1], a->k_stride[0], a->k_stride[1], a->k_stride[2],
                                 a->v_stride[0], a->v_stride[1], a->v_stride[2], a->k_prefix_stride[0], a->k_prefix_stride[1], a->k_prefix_stride[2],
                                 a->v_prefix_stride[0], a->v_prefix_stride[1], a->v_prefix_stride[2]};
    const int64_t rows[4] = {a->k_stride[2], a->v_stride[2], a->k_prefix_stride[2], a->v_prefix_stride[2]};
    uintptr_t bits = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->o) | reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache);
    if (!paged) bits |= reinterpret_cast<uintptr_t>(a->k_prefix) | reinterpret_cast<uintptr_t>(a->v_prefix);
    int st = part_tensor_checks(a->D, a->dtype, strides, paged ? 10 : 16, rows, paged ? 2 : 4, bits, who);
    if (st != DTATTN_OK) return st;
    ScalePlan sp;
    st = plan_scale(a->scale, a->D, a->dtype == DTATTN_FP32 ? kSign32 : kSign16, &sp);
    if (st != DTATTN_OK || a->B == 0) return st;
    if (a->q == nullptr || a->o == nullptr || a->k_cache == nullptr || a->v_cache == nullptr || a->lengths == nullptr || a->prefix_lengths == nullptr ||
        (!paged && (a->k_prefix == nullptr || a->v_prefix == nullptr)))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    const int cus = stream_cus(stream);
    if (cus <= 0) return fail(DTATTN_ERR_DEVICE, "%s: cannot tell the stream's device", who);
    const SharedPlan plan = plan_shared(a, cus);
    const int64_t capacity = paged ? a->max_pages * a->page_size : a->S_max, most_prefix = paged ? capacity : a->S_prefix;
    if (a->groups * a->Hkv * plan.nsub[0] * places_in(most_prefix) >= ((int64_t)1 << 31) ||
        a->B * a->Hkv * plan.nsub[1] * places_in(capacity) >= ((int64_t)1 << 31) || a->B * a->Hq > 0x7fffffff)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: cache too large", who);
    if (a->workspace == nullptr || a->workspace_bytes < plan.bytes)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, plan.bytes, a->workspace_bytes);
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);

    PartsParams p = {};
    const int64_t esz = a->dtype == DTATTN_FP32 ? 4 : 2;
    p.q = reinterpret_cast<const char*>(a->q), p.o = reinterpret_cast<char*>(a->o), p.lse = a->lse;
    p.k[1] = reinterpret_cast<const char*>(a->k_cache), p.v[1] = reinterpret_cast<const char*>(a->v_cache);
    p.k_b[1] = a->k_stride[0] * esz, p.k_h[1] = a->k_stride[1] * esz, p.k_s[1] = a->k_stride[2] * esz;
    p.v_b[1] = a->v_stride[0] * esz, p.v_h[1] = a->v_stride[1] * esz, p.v_s[1] = a->v_stride[2] * esz;
    if (paged) {
        p.k[0] = p.k[1], p.k_b[0] = p.k_b[1], p.k_h[0] = p.k_h[1], p.k_s[0] = p.k_s[1];
        p.v[0] = p.v[1], p.v_b[0] = p.v_b[1], p.v_h[0] = p.v_h[1], p.v_s[0] = p.v_s[1];
        p.table = a->block_table, p.bt_s = a->block_table_stride;
        p.page_shift = __builtin_ctzll((unsigned long long)a->page_size), p.num_pages = (int32_t)a->num_pages;
    } else {
        p.k[0] = reinterpret_cast<const char*>(a->k_prefix), p.v[0] = reinterpret_cast<const char*>(a->v_prefix);
        p.k_b[0] = a->k_prefix_stride[0] * esz, p.k_h[0] = a->k_prefix_stride[1] * esz, p.k_s[0] = a->k_prefix_stride[2] * esz;
        p.v_b[0] = a->v_prefix_stride[0] * esz, p.v_h[0] = a->v_prefix_stride[1] * esz, p.v_s[0] = a->v_prefix_stride[2] * esz;
    }
    p.capacity[0] = (int32_t)most_prefix, p.capacity[1] = (int32_t)capacity;
    p.lengths = a->lengths, p.prefix = a->prefix_lengths;
    char* ws = reinterpret_cast<char*>(a->workspace);
    auto take = [&](size_t bytes) {
        char* at = ws;
        ws += bytes;
        return at;
    };
    for (int s = 0; s < 2; ++s) {
        p.nsub[s] = plan.nsub[s], p.columns[s] = plan.columns[s], p.weight[s] = plan.weight[s];
        p.meta[s] = reinterpret_cast<int32_t*>(take(plan.meta[s]));
        p.rec_o[s] = reinterpret_cast<float*>(take(plan.rec_o[s]));
        p.rec_ml[s] = reinterpret_cast<float2*>(take(plan.rec_ml[s]));
        p.whole_o[s] = reinterpret_cast<float*>(take(plan.whole_o));
        p.whole_ml[s] = reinterpret_cast<float2*>(take(plan.whole_ml));
    }
    p.shares = plan.shares;
    p.q_b = a->q_stride[0], p.q_h = a->q_stride[1], p.o_b = a->o_stride[0], p.o_h = a->o_stride[1];
    p.lse_b = a->lse != nullptr ? a->lse_stride[0] : 0;
    p.B = (int32_t)a->B, p.Hq = (int32_t)a->Hq, p.Hkv = (int32_t)a->Hkv, p.group = (int32_t)(a->Hq / a->Hkv);
    p.groups = (int32_t)a->groups, p.per = (int32_t)(a->B / a->groups);
    p.per_inv = 1.f / (float)p.per;
    p.d = (int32_t)a->D;
    p.c = sp.scale * kLog2e;
    p.q_and = sp.q_and, p.q_xor = sp.q_xor;
    const bool wide = plan.kernel_d == 128;
    switch (a->dtype) {
        case DTATTN_BF16: return wide ? launch_shared<bf16_t, 128>(p, plan.nc, stream) : launch_shared<bf16_t, 64>(p, plan.nc, stream);
        case DTATTN_FP16: return wide ? launch_shared<f16_t, 128>(p, plan.nc, stream) : launch_shared<f16_t, 64>(p, plan.nc, stream);
        default: return wide ? launch_shared<float, 128>(p, plan.nc, stream) : launch_shared<float, 64>(p, plan.nc, stream);
    }
}
