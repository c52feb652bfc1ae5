// Eviction from a KV cache by accumulated attention weight (the rule and its ties: dtattn_kv_evict in dtattn.h).
//
// No counterpart in the reference, which keeps no KV cache (python/dtorch/test/modules/llama.py:126-156).
//
// kv_evict_select_kernel: one workgroup per (sequence, kv head) finds the weight of the last block that stays by a radix
// select over the blocks' weights (as unsigned numbers in their order, 8 bits a round), takes of the blocks at that
// weight the first ones, and writes the list of blocks that stay, in order.
// kv_evict_move_kernel: one workgroup per (sequence, kv head, K / V / weights and scales) moves rows to the front in
// place.  Row i of the result comes from a row at or past i, so a tile of rows may be written as soon as the tile itself
// has been read: what a write covers belongs to rows already read.
#include <algorithm>

#include "dtattn_common.hpp"

namespace dtattn {

struct EvictParams {
    char* kv[2];
    float* scale[2];  // NULL: none
    float* w;
    int32_t* lengths;
    int32_t* kept;
    uint32_t* order;  // [B, Hkv, S_max / block]: candidates' weights in unsigned order
    int64_t kv_b[2], kv_h[2], kv_s[2];  // bytes
    int64_t s_b[2], s_h[2], w_b, w_h;
    int32_t B, Hkv, S_max, keep, recent;  // keep and recent in blocks
    int32_t block_shift, scale_shift;     // tokens per block; scale blocks per block
    int32_t chunks;                       // 16-byte chunks per row
    int32_t blocks_max;                   // ceil(S_max / block)
};

namespace {

constexpr int kSelect = 1024;

// Floats as unsigned numbers of the same order; NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) x = kNegInf;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the workgroup (kSelect threads), and the total.
__device__ __forceinline__ int scan_all(int v, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d, 64);
        if (lane >= d) s += o;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kSelect / 64; ++i) {
        const int t = lds[i];
        before += i < wave ? t : 0;
        total += t;
    }
    return before + s - v;
}

// Every wave's loads have returned (a barrier alone orders what they see, not when they are done).
__device__ __forceinline__ void read_all() {
    wait_vmem();
    __syncthreads();
}

__device__ __forceinline__ int tokens_of(const EvictParams& p, int64_t b) { return min(max(p.lengths[b], 0), p.S_max); }

}  // namespace

__global__ void __launch_bounds__(kSelect) kv_evict_select_kernel(const EvictParams p) {
    __shared__ int hist[256];
    __shared__ int waves[kSelect / 64];
    __shared__ int found[2];
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x, b = bh / p.Hkv;
    const int h = (int)(bh % p.Hkv);
    const int n = tokens_of(p, b);
    const int blocks = (n + (1 << p.block_shift) - 1) >> p.block_shift;
    int32_t* kept = p.kept + bh * p.keep;
    if (blocks <= p.keep) {
        for (int i = tid; i < p.keep; i += kSelect) kept[i] = i < blocks ? i : -1;
        return;
    }
    const int cand = blocks - p.recent;  // candidates: 0 .. cand - 1, all of them whole blocks
    int need = p.keep - p.recent;        // of which so many stay; fewer than cand
    uint32_t* order = p.order + bh * p.blocks_max;
    const float* w = p.w + b * p.w_b + h * p.w_h;
    for (int i = tid; i < cand; i += kSelect) {
        float m;
        if (p.block_shift == 0) {
            m = w[i];
        } else {
            double s = 0.;
            const float* x = w + ((int64_t)i << p.block_shift);
            for (int j = 0; j < (1 << p.block_shift); ++j) s += (double)x[j];
            m = (float)s;
        }
        order[i] = ordered(m);
    }
    __syncthreads();
    // The need-th largest, 8 bits a round: `prefix` holds the bits found so far, and `need` how many stay of those that share them
    uint32_t prefix = 0, mask = 0;
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < cand; i += kSelect) {
                const uint32_t u = order[i];
                if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & 255u], 1);
            }
            __syncthreads();
            const int mine = tid < 256 ? hist[255 - tid] : 0;  // from the largest down
            int total;
            const int before = scan_all(mine, waves, total);
            if (tid < 256 && before < need && before + mine >= need) {
                found[0] = 255 - tid;
                found[1] = need - before;
            }
            __syncthreads();
            prefix |= (uint32_t)found[0] << shift;
            mask |= 255u << shift;
            need = found[1];
            __syncthreads();
        }
    } else {
        prefix = 0xffffffffu;  // above every weight
    }
    // those above stay, and the first `need` of those at it; a thread takes a run of candidates
    const int run = (cand + kSelect - 1) / kSelect;
    const int i0 = min(tid * run, cand), i1 = min(i0 + run, cand);
    int above = 0, at = 0;
    for (int i = i0; i < i1; ++i) {
        above += order[i] > prefix;
        at += order[i] == prefix;
    }
    int total;
    const int at0 = scan_all(at, waves, total);
    const int mine = above + min(max(need - at0, 0), at);
    int out = scan_all(mine, waves, total);
    int left = need - at0;
    for (int i = i0; i < i1; ++i) {
        const uint32_t u = order[i];
        const bool stays = u > prefix || (u == prefix && left-- > 0);
        if (stays) kept[out++] = i;
    }
    for (int i = tid; i < p.recent; i += kSelect) kept[p.keep - p.recent + i] = cand + i;
}

__global__ void __launch_bounds__(1024) kv_evict_move_kernel(const EvictParams p) {
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x, b = bh / p.Hkv;
    const int h = (int)(bh % p.Hkv), what = blockIdx.y;
    const int n = tokens_of(p, b);
    const int blocks = (n + (1 << p.block_shift) - 1) >> p.block_shift;
    if (blocks <= p.keep) return;
    const int32_t* kept = p.kept + bh * p.keep;
    const int left = ((p.keep - 1) << p.block_shift) + n - ((blocks - 1) << p.block_shift);  // tokens that stay
    const int inner = (1 << p.block_shift) - 1;
    auto source = [&](int row) { return (kept[row >> p.block_shift] << p.block_shift) + (row & inner); };
    if (what < 2) {
        constexpr int PER = 4;  // chunks per thread and tile
        char* base = p.kv[what] + b * p.kv_b[what] + h * p.kv_h[what];
        const int64_t pitch = p.kv_s[what];
        const int64_t cells = (int64_t)left * p.chunks;
        for (int64_t c0 = 0; c0 < cells; c0 += 1024 * PER) {
            u32x4 v[PER];
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int64_t c = c0 + k * 1024 + tid;
                if (c < cells) v[k] = ld16(base + source((int)(c / p.chunks)) * pitch + (c % p.chunks) * 16);
            }
            read_all();
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int64_t c = c0 + k * 1024 + tid;
                if (c < cells) st16(base + (c / p.chunks) * pitch + (c % p.chunks) * 16, v[k]);
            }
        }
        return;
    }
    float* w = p.w + b * p.w_b + h * p.w_h;
    for (int r0 = 0; r0 < left; r0 += 1024) {
        const int r = r0 + tid;
        const float v = r < left ? w[source(r)] : 0.f;
        read_all();
        if (r < left) w[r] = v;
    }
    __syncthreads();
    for (int r = left + tid; r < n; r += 1024) w[r] = 0.f;
    if (p.scale[0] != nullptr) {
        // scale blocks move as tokens do: all of a block's, of the last one those it has
        const int sub = (1 << p.scale_shift) - 1;
        const int per_block = p.block_shift - p.scale_shift;  // log2 tokens per scale
        const int have = (left + (1 << per_block) - 1) >> per_block;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            float* s = p.scale[kv] + b * p.s_b[kv] + h * p.s_h[kv];
            for (int r0 = 0; r0 < have; r0 += 1024) {
                const int r = r0 + tid;
                const float v = r < have ? s[(kept[r >> p.scale_shift] << p.scale_shift) + (r & sub)] : 0.f;
                read_all();
                if (r < have) s[r] = v;
            }
        }
    }
}

__global__ void __launch_bounds__(256) kv_evict_lengths_kernel(const EvictParams p) {
    const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (b >= p.B) return;
    const int n = tokens_of(p, b);
    const int blocks = (n + (1 << p.block_shift) - 1) >> p.block_shift;
    if (blocks > p.keep) p.lengths[b] = ((p.keep - 1) << p.block_shift) + n - ((blocks - 1) << p.block_shift);
}

static size_t evict_workspace(const dtattn_kv_evict_args* a) {
    const int64_t blocks = (a->S_max + a->block - 1) / a->block;
    return ((size_t)a->B * a->Hkv * blocks * sizeof(uint32_t) + 255) & ~(size_t)255;
}

}  // namespace dtattn

using namespace dtattn;

extern "C" size_t dtattn_kv_evict_workspace_size(const dtattn_kv_evict_args* a) {
    if (a == nullptr || a->B <= 0 || a->Hkv <= 0 || a->S_max <= 0 || a->block <= 0) return 0;
    return evict_workspace(a);
}

extern "C" int dtattn_kv_evict(const dtattn_kv_evict_args* a, void* stream_) {
    const char* who = "kv_evict";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    if (a->B < 0 || a->Hkv <= 0 || a->S_max <= 0 || a->S_max > (1 << 29) || a->row_bytes <= 0)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
    if (a->block < 1 || a->block > 256 || (a->block & (a->block - 1)) != 0)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: block %lld must be a power of two up to 256", who, (long long)a->block);
    if (a->recent < a->block || a->keep < a->recent || a->keep % a->block != 0 || a->recent % a->block != 0 || a->keep > (1 << 29))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: keep %lld and recent %lld must be multiples of the block of %lld tokens with block <= recent <= keep",
                    who, (long long)a->keep, (long long)a->recent, (long long)a->block);
    if (a->row_bytes % 16 != 0 || a->row_bytes > (1 << 20))
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: a row of %lld bytes is not a multiple of 16", who, (long long)a->row_bytes);
    const bool scales = a->k_scale != nullptr || a->v_scale != nullptr;
    if (scales && (a->k_scale == nullptr || a->v_scale == nullptr))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: K and V both have scales or neither has", who);
    if (scales && (a->scale_block < 1 || (a->scale_block & (a->scale_block - 1)) != 0 || a->block % a->scale_block != 0 || a->S_max % a->scale_block != 0))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: the block of %lld tokens must be a multiple of the %lld tokens of a scale", who,
                    (long long)a->block, (long long)a->scale_block);
    for (int i = 0; i < 3; ++i)
        if (a->k_stride[i] % 16 != 0 || a->v_stride[i] % 16 != 0)
            return fail(DTATTN_ERR_UNSUPPORTED, "%s: cache strides must be multiples of 16 bytes", who);
    if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15u)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: caches must be 16-byte aligned", who);
    if (a->B == 0) return DTATTN_OK;
    if (a->k_cache == nullptr || a->v_cache == nullptr || a->weights == nullptr || a->lengths == nullptr || a->kept == nullptr)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    if (a->B * a->Hkv > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
    const size_t need = evict_workspace(a);
    if (a->workspace == nullptr || a->workspace_bytes < need)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, need, a->workspace_bytes);
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return fail(DTATTN_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
    EvictParams p = {};
    p.kv[0] = reinterpret_cast<char*>(a->k_cache), p.kv[1] = reinterpret_cast<char*>(a->v_cache);
    p.scale[0] = a->k_scale, p.scale[1] = a->v_scale;
    p.w = a->weights, p.lengths = a->lengths, p.kept = a->kept;
    p.order = reinterpret_cast<uint32_t*>(a->workspace);
    p.kv_b[0] = a->k_stride[0], p.kv_h[0] = a->k_stride[1], p.kv_s[0] = a->k_stride[2];
    p.kv_b[1] = a->v_stride[0], p.kv_h[1] = a->v_stride[1], p.kv_s[1] = a->v_stride[2];
    p.s_b[0] = a->k_scale_stride[0], p.s_h[0] = a->k_scale_stride[1];
    p.s_b[1] = a->v_scale_stride[0], p.s_h[1] = a->v_scale_stride[1];
    p.w_b = a->w_stride[0], p.w_h = a->w_stride[1];
    p.B = (int32_t)a->B, p.Hkv = (int32_t)a->Hkv, p.S_max = (int32_t)a->S_max;
    p.keep = (int32_t)(a->keep / a->block), p.recent = (int32_t)(a->recent / a->block);
    p.block_shift = __builtin_ctzll((unsigned long long)a->block);
    p.scale_shift = scales ? p.block_shift - __builtin_ctzll((unsigned long long)a->scale_block) : 0;
    p.chunks = (int32_t)(a->row_bytes / 16);
    p.blocks_max = (int32_t)((a->S_max + a->block - 1) / a->block);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const unsigned heads = (unsigned)(a->B * a->Hkv);
    hipLaunchKernelGGL(kv_evict_select_kernel, dim3(heads), dim3(kSelect), 0, stream, p);
    int st = check_launch("kv_evict_select_kernel");
    if (st != DTATTN_OK) return st;
    hipLaunchKernelGGL(kv_evict_move_kernel, dim3(heads, 3), dim3(1024), 0, stream, p);
    st = check_launch("kv_evict_move_kernel");
    if (st != DTATTN_OK) return st;
    hipLaunchKernelGGL(kv_evict_lengths_kernel, dim3((unsigned)((a->B + 255) / 256)), dim3(256), 0, stream, p);
    return check_launch("kv_evict_lengths_kernel");
}
