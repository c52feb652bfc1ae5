// Eviction from a KV cache by accumulated attention weight (the rule and its ties: dtattn_kv_evict in dtattn.h).
//
// No counterpart in the reference, which keeps no KV cache (python/dtorch/test/modules/llama.py:126-156).
//
// kv_evict_select_kernel: one workgroup per (sequence, kv head) finds the weight of the last block that stays by a radix
// select over the blocks' weights (as unsigned numbers in their order; 11, 11 and 10 bits a round), takes of the blocks at that
// weight the first ones, and writes the list of blocks that stay, in order.  Up to 16384 candidates are held in registers.
// kv_evict_move_kernel: moves rows to the front in place.  Row i of the result comes from a row at or past i, so a tile
// of rows may be written as soon as the tile itself has been read: what a write covers belongs to rows already read.  A workgroup
// has the next tile's loads in flight while it writes one, and that tile's list entries before them.  Few heads share a row's chunks
// among several workgroups, all on one XCD, whose L2 puts the lines together again.  Bound by HBM.
#include <algorithm>

#include "decode_params.hpp"
#include "fp8_cache.hpp"

namespace dtattn {

struct EvictParams {
    char* kv[2];
    float* scale[2];  // NULL: none
    float* w;
    int32_t* lengths;
    int32_t* kept;
    uint32_t* order;  // [B, Hkv, S_max / block]: candidates' weights in unsigned order (where registers do not hold them)
    int2* plan;       // [B, Hkv]: tokens before, and after (equal: nothing moves)
    int64_t kv_b[2], kv_h[2], kv_s[2];  // bytes
    int64_t s_b[2], s_h[2], w_b, w_h;
    int32_t B, Hkv, S_max, keep, recent;  // keep and recent in blocks
    int32_t block_shift, scale_shift;     // tokens per block; scale blocks per block
    int32_t chunks, width, groups;        // 16-byte chunks per row, of which a workgroup moves `width`, `groups` of them a row
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

// Exclusive prefix sum over the workgroup (kSelect threads), and the total.  `lds` is not in use before the call or, until every
// thread is past a barrier, after it.
__device__ __forceinline__ int scan_all(int v, int* lds, int& total) {
    const int wave = threadIdx.x >> 6;
    const int s = scan64(v);
    if ((threadIdx.x & 63) == 63) lds[wave] = s;
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

// The candidates' weights: PER per thread in registers (candidate PER * tid + k), or PER = 0 in memory.
template <int PER>
__global__ void __launch_bounds__(kSelect) kv_evict_select_kernel(const EvictParams p) {
    constexpr int BINS = 2048;
    __shared__ int hist[3][BINS];  // one a round: nothing is cleared between them
    __shared__ int waves[4][kSelect / 64];
    __shared__ int found[3][2];
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x, b = bh / p.Hkv;
    const int h = (int)(bh % p.Hkv);
    const int n = tokens_of(p, b);
    const int blocks = (n + (1 << p.block_shift) - 1) >> p.block_shift;
    int32_t* kept = p.kept + bh * p.keep;
    const int left = blocks <= p.keep ? n : ((p.keep - 1) << p.block_shift) + n - ((blocks - 1) << p.block_shift);
    if (tid == 0) p.plan[bh] = make_int2(n, left);
    if (blocks <= p.keep) {
        for (int i = tid; i < p.keep; i += kSelect) kept[i] = i < blocks ? i : -1;
        return;
    }
    const int cand = blocks - p.recent;  // candidates: 0 .. cand - 1, all of them whole blocks
    int need = p.keep - p.recent;        // of which so many stay; fewer than cand
    uint32_t* order = p.order + bh * p.blocks_max;
    const float* w = p.w + b * p.w_b + h * p.w_h;
    auto weight = [&](int i) {
        if (p.block_shift == 0) return ordered(w[i]);
        double s = 0.;
        const float* x = w + ((int64_t)i << p.block_shift);
#pragma unroll 16
        for (int j = 0; j < (1 << p.block_shift); ++j) s += (double)x[j];
        return ordered((float)s);
    };
    uint32_t mine[PER > 0 ? PER : 1];
    if constexpr (PER > 0) {
#pragma unroll
        for (int k = 0; k < PER; ++k) mine[k] = PER * tid + k < cand ? weight(PER * tid + k) : 0u;
    } else {
        for (int i = tid; i < cand; i += kSelect) order[i] = weight(i);
    }
    for (int i = tid; i < 3 * BINS; i += kSelect) (&hist[0][0])[i] = 0;
    __syncthreads();
    // The need-th largest, some bits a round: `prefix` holds the bits found so far, and `need` how many stay of those that share them
    uint32_t prefix = 0, mask = 0;
    if (need > 0) {
#pragma unroll
        for (int round = 0; round < 3; ++round) {
            const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bins = round < 2 ? 2048 : 1024;
            auto count = [&](uint32_t u) {
                if ((u & mask) == prefix) atomicAdd(&hist[round][(u >> shift) & (bins - 1)], 1);
            };
            if constexpr (PER > 0) {
#pragma unroll
                for (int k = 0; k < PER; ++k)
                    if (PER * tid + k < cand) count(mine[k]);
            } else {
                for (int i = tid; i < cand; i += kSelect) count(order[i]);
            }
            __syncthreads();
            // two bins a thread, from the largest down
            const int hi = hist[round][BINS - 1 - 2 * tid], lo = hist[round][BINS - 2 - 2 * tid];
            int total;
            const int before = scan_all(hi + lo, waves[round], total);
            if (before < need && before + hi + lo >= need) {
                const bool upper = before + hi >= need;
                found[round][0] = BINS - 1 - 2 * tid - (upper ? 0 : 1);
                found[round][1] = need - before - (upper ? 0 : hi);
            }
            __syncthreads();
            prefix |= (uint32_t)found[round][0] << shift;
            mask |= (uint32_t)(bins - 1) << shift;
            need = found[round][1];
        }
    } else {
        prefix = 0xffffffffu;  // above every weight
    }
    // those above stay, and the first `need` of those at it
    if constexpr (PER > 0) {
        int counts = 0;  // above << 16, and at it: up to 16384 of both
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (PER * tid + k < cand) counts += mine[k] > prefix ? 1 << 16 : mine[k] == prefix ? 1 : 0;
        int total;
        const int before = scan_all(counts, waves[3], total);
        int above = before >> 16, at = before & 0xffff;
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (PER * tid + k < cand) {
                const bool over = mine[k] > prefix, same = mine[k] == prefix;
                if (over || (same && at < need)) kept[above + min(at, need)] = PER * tid + k;
                above += over, at += same;
            }
    } else {
        int above = 0, at = 0;  // of the candidates before: one row of kSelect after another
        for (int i0 = 0; i0 < cand; i0 += kSelect) {
            const uint32_t u = i0 + tid < cand ? order[i0 + tid] : 0u;
            const bool over = i0 + tid < cand && u > prefix, same = i0 + tid < cand && u == prefix;
            int total;
            const int before = scan_all(((int)over << 16) + (int)same, waves[3], total);
            const int mine_at = at + (before & 0xffff);
            if (over || (same && mine_at < need)) kept[above + (before >> 16) + min(mine_at, need)] = i0 + tid;
            above += total >> 16, at += total & 0xffff;
            __syncthreads();
        }
    }
    for (int i = tid; i < p.recent; i += kSelect) kept[p.keep - p.recent + i] = cand + i;
}

// A workgroup per (sequence, kv head, K or V, group of chunks), eight of them in a row on different XCDs; blockIdx.y = 1: the
// weights and scales of a (sequence, kv head).
__global__ void __launch_bounds__(1024) kv_evict_move_kernel(const EvictParams p) {
    const int tid = threadIdx.x;
    const int64_t heads = (int64_t)p.B * p.Hkv;
    int64_t item = blockIdx.x;
    int group = 0;
    if (blockIdx.y == 0) {
        const int64_t lot = item / (8 * p.groups);  // eight items' groups
        group = (int)(item / 8 % p.groups);
        item = lot * 8 + item % 8;
        if (item >= 2 * heads) return;
    } else if (item >= heads) {
        return;
    }
    const int what = blockIdx.y == 0 ? (int)(item & 1) : 2;
    const int64_t bh = blockIdx.y == 0 ? item >> 1 : item, b = bh / p.Hkv;
    const int h = (int)(bh % p.Hkv);
    const int2 plan = p.plan[bh];
    const int n = plan.x, left = plan.y;
    if (what == 2 && h == 0 && tid == 0 && left < n) p.lengths[b] = left;
    if (left == n) return;
    const int32_t* kept = p.kept + bh * p.keep;
    const int inner = (1 << p.block_shift) - 1;
    auto source = [&](int row) { return (kept[row >> p.block_shift] << p.block_shift) + (row & inner); };
    if (what < 2) {
        constexpr int PER = 4;  // rows per thread and tile
        const int64_t pitch = p.kv_s[what];
        const int c = tid % p.width, step = 1024 / p.width;  // this thread's chunk, and rows that the threads cover at once
        const int chunk = group * p.width + c;
        const bool works = tid < step * p.width && chunk < p.chunks;
        char* base = p.kv[what] + b * p.kv_b[what] + h * p.kv_h[what] + chunk * 16;
        const int first = works ? tid / p.width : left;  // row of the first pass
        const int tile = PER * step;
        u32x4 v[2][PER];
        int src[PER];
        auto look = [&](int r0) {  // where the rows of the tile at r0 come from
#pragma unroll
            for (int k = 0; k < PER; ++k) src[k] = source(min(first + r0 + k * step, left - 1));
        };
        auto load = [&](u32x4* x) {
#pragma unroll
            for (int k = 0; k < PER; ++k)
                if (works) x[k] = ld16_nt(base + src[k] * pitch);
        };
        auto store = [&](u32x4* x, int r0) {
#pragma unroll
            for (int k = 0; k < PER; ++k) asm volatile("" : "+v"(x[k]));  // the tile has been read
            lds_barrier();                                              // by every wave
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const int r = first + r0 + k * step;
                if (r < left) st16(base + r * pitch, x[k]);
            }
        };
        look(0);
        load(v[0]);
        look(tile);
        for (int r0 = 0; r0 < left; r0 += 2 * tile) {
            if (r0 + tile < left) load(v[1]);
            look(r0 + 2 * tile);
            store(v[0], r0);
            if (r0 + tile >= left) break;
            if (r0 + 2 * tile < left) load(v[0]);
            look(r0 + 3 * tile);
            store(v[1], r0 + tile);
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

struct EvictSpace {
    size_t plan, order;  // bytes
};

constexpr int kHeldRows = 16;  // candidates a thread holds

static EvictSpace evict_workspace(const dtattn_kv_evict_args* a) {
    const int64_t blocks = (a->S_max + a->block - 1) / a->block;
    const size_t heads = (size_t)a->B * a->Hkv;
    EvictSpace r;
    r.plan = (heads * sizeof(int2) + 255) & ~(size_t)255;
    r.order = blocks > kHeldRows * kSelect ? ((heads * blocks * sizeof(uint32_t) + 255) & ~(size_t)255) : 0;
    return r;
}

}  // namespace dtattn

using namespace dtattn;

extern "C" size_t dtattn_kv_evict_workspace_size(const dtattn_kv_evict_args* a) {
    if (a == nullptr || a->B <= 0 || a->Hkv <= 0 || a->S_max <= 0 || a->block <= 0) return 0;
    const EvictSpace r = evict_workspace(a);
    return r.plan + r.order;
}

extern "C" int dtattn_kv_evict(const dtattn_kv_evict_args* a, void* stream_) {
    const char* who = "kv_evict";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    if (a->B < 0 || a->Hkv <= 0 || a->B > 0x7fffffff || a->Hkv > 0x7fffffff || a->S_max <= 0 || a->S_max > (1 << 29) || a->row_bytes <= 0)
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
    if (a->k_cache == a->v_cache || (scales && a->k_scale == a->v_scale))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: keys and values are both moved in place and cannot share memory", who);
    if (a->B * a->Hkv > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
    const EvictSpace space = evict_workspace(a);
    const size_t need = space.plan + space.order;
    if (a->workspace == nullptr || a->workspace_bytes < need)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, need, a->workspace_bytes);
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return fail(DTATTN_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
    EvictParams p = {};
    p.kv[0] = reinterpret_cast<char*>(a->k_cache), p.kv[1] = reinterpret_cast<char*>(a->v_cache);
    p.scale[0] = a->k_scale, p.scale[1] = a->v_scale;
    p.w = a->weights, p.lengths = a->lengths, p.kept = a->kept;
    p.plan = reinterpret_cast<int2*>(a->workspace);
    p.order = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(a->workspace) + space.plan);
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
    // Candidates in registers, as few a thread as hold them, or in memory.  us of the launch: 64 heads of 4096 tokens, four a thread
    // 7.3, sixteen 11.6, in memory 10.8; 16 of 10319, sixteen 13.5, in memory 21.1; 8 of 16384 17.7, 28.2; 128 of 256 blocks of 32,
    // one 5.8, four 16.8, in memory 6.8.
    if (p.blocks_max <= kSelect) hipLaunchKernelGGL(kv_evict_select_kernel<1>, dim3(heads), dim3(kSelect), 0, stream, p);
    else if (p.blocks_max <= 4 * kSelect) hipLaunchKernelGGL(kv_evict_select_kernel<4>, dim3(heads), dim3(kSelect), 0, stream, p);
    else if (p.blocks_max <= kHeldRows * kSelect) hipLaunchKernelGGL(kv_evict_select_kernel<kHeldRows>, dim3(heads), dim3(kSelect), 0, stream, p);
    else hipLaunchKernelGGL(kv_evict_select_kernel<0>, dim3(heads), dim3(kSelect), 0, stream, p);
    int st = check_launch("kv_evict_select_kernel");
    if (st != DTATTN_OK) return st;
    // A row's chunks are halved among workgroups until three CUs in four have one, or each chunk has one.  us where that bound is no CU /
    // half of them / three in four / all / all twice, heads of 128 bf16, 8192 -> 4096 tokens: 1 sequence of 8 heads 45 / 29 / 33 / 33 / 34,
    // 3 61 / 44 / 44 / 49 / 62, 6 68 / 52 / 52 / 69 / 80, 8 72 / 72 / 64 / 63 / 81, 12 81 / 81 / 81 / 83 / 109.  Workgroups double, so one
    // sequence goes from 128 of them, which half of the CUs would take, to 256 of single chunks: 33 us, and not the 29 of two.
    const int wanted = std::max(stream_cus(stream) * 3 / 4, 1);
    p.width = p.chunks;
    while (p.width > 1 && 2 * (int64_t)heads * ((p.chunks + p.width - 1) / p.width) < wanted) p.width = (p.width + 1) / 2;
    p.width = std::min(p.width, 1024);
    p.groups = (p.chunks + p.width - 1) / p.width;
    const int64_t lots = (2 * (int64_t)heads + 7) / 8;
    const int64_t grid = std::max<int64_t>(lots * 8 * p.groups, heads);
    if (grid > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
    hipLaunchKernelGGL(kv_evict_move_kernel, dim3((unsigned)grid, 2), dim3(1024), 0, stream, p);
    return check_launch("kv_evict_move_kernel");
}
