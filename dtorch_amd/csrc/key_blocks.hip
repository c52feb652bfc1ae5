// Key bounds of a cache's blocks, and the selection of blocks by them (formulas: dtattn.h, "attention over selected key blocks").
//
// No counterpart in the reference, which keeps no KV cache (python/dtorch/test/modules/llama.py:126-156).
//
// The bound: a token's key lies between k_min and k_max in every dimension, so q . k <= sum_d q_d x_d with x_d = k_max_d where
// q_d > 0 and k_min_d elsewhere.  Reading 2 D values per block instead of D per token, it says which blocks can hold large scores.
//
// key_bounds_kernel: a wave or a workgroup per (block, sequence and kv head); every 16-byte chunk of a row belongs to one column of
// threads, which meet by lane exchanges and, of several waves, in LDS.  Bound by HBM: the rows are read once (4 x 4000 tokens of 8 heads of 128 dims, 34 MB, 8.0
// us, 4.1 TB/s; the last block of 64 sequences' steps 5.0, a launch).
// score_blocks_kernel: eight lanes to a block, with the query's heads in LDS as 64-bit numbers.  Sums are taken in 64 bits, so that scores next to
// one another are told apart: exact, and alike in any order, where the products of a 16-bit type lie within 2^24 (fp16, 22 bits each) or 2^30
// (bf16, 16 bits) of the largest one, and off by at most D 2^-53 sum |q x| elsewhere.  The vector units' 64-bit rate is that of 32 bits.
// select_blocks_kernel: one workgroup per (sequence, kv head) takes the largest scores by a radix select.
#include <algorithm>

#include "decode_params.hpp"
#include "radix_select.hpp"

namespace dtattn {

struct BlockCache {  // where blocks lie
    const int32_t* table;  // NULL: padded
    const int32_t* lengths;
    int64_t bt_s;
    int32_t capacity, page_shift, num_pages, block_shift;
};

struct BoundsParams {
    BlockCache c;
    const char* k;
    char* lo;
    char* hi;
    int64_t k_b, k_h, k_s, lo_b, lo_h, lo_s, hi_b, hi_h, hi_s;  // bytes
    int32_t Hkv, n_new, chunks;
    int32_t first;  // of the blocks that the new tokens touch, this launch's
};

struct SelectParams {
    BlockCache c;
    const char* q;
    const char* lo;
    const char* hi;
    uint32_t* order;  // [B, Hkv, blocks_max]: scores in unsigned order
    int32_t* kept;
    int64_t q_b, q_h;  // elements
    int64_t lo_b, lo_h, lo_s, hi_b, hi_h, hi_s;  // bytes
    int32_t Hkv, group, d, keep, recent, blocks_max;
    uint32_t q_and, q_xor;
};

namespace {

__device__ __forceinline__ int tokens_in(const BlockCache& c, int64_t b) { return min(max(c.lengths[b], 0), c.capacity); }

}  // namespace

// W: chunks of a row's columns of threads, a power of two.  WAVES: of a block; with one, a workgroup has four blocks.
template <typename T, int W, int WAVES>
__global__ void __launch_bounds__(256) key_bounds_kernel(const BoundsParams p) {
    constexpr int E = 16 / (int)sizeof(T), ROWS = 64 * WAVES / W;
    __shared__ float red[4][2][W * E];
    const int tid = threadIdx.x % (64 * WAVES), col = tid % W, row = tid / W;
    const int64_t bh = blockIdx.x, b = bh / p.Hkv;
    const int h = (int)(bh % p.Hkv);
    const int n = tokens_in(p.c, b);
    const int block = 1 << p.c.block_shift;
    const int64_t j = (max(n - p.n_new, 0) >> p.c.block_shift) + p.first + (int64_t)blockIdx.y * (4 / WAVES) + threadIdx.x / (64 * WAVES);
    const int64_t t0 = j << p.c.block_shift;
    if (t0 >= n) return;
    const int rows = (int)min((int64_t)block, n - t0);
    int64_t slot = b, r0 = t0;
    if (p.c.table != nullptr) {
        slot = p.c.table[b * p.c.bt_s + (t0 >> p.c.page_shift)];
        r0 = t0 & ((1 << p.c.page_shift) - 1);
        if (slot < 0 || slot >= p.c.num_pages) return;
    }
    const char* k = p.k + slot * p.k_b + h * p.k_h + r0 * p.k_s + col * 16;
    float lo[E], hi[E];
#pragma unroll
    for (int e = 0; e < E; ++e) lo[e] = __builtin_inff(), hi[e] = kNegInf;
    if (col < p.chunks) {
        constexpr int PER = 4;  // rows in flight
        for (int r = row; r < rows; r += ROWS * PER) {
            u32x4 w[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) w[i] = ld16(k + min(r + ROWS * i, rows - 1) * p.k_s);  // a row twice changes nothing
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                float x[E];
                if constexpr (sizeof(T) == 4) {
                    const f32x4 f = __builtin_bit_cast(f32x4, w[i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = f[e];
                } else {
                    unpack8<T>(w[i], x);
                }
#pragma unroll
                for (int e = 0; e < E; ++e) lo[e] = fminf(lo[e], x[e]), hi[e] = fmaxf(hi[e], x[e]);  // NaN is passed over
            }
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (W == 8) lo[e] = fminf(lo[e], dpp_f<0x128>(lo[e])), hi[e] = fmaxf(hi[e], dpp_f<0x128>(hi[e]));  // lane ^ 8
        if (W <= 16) lo[e] = -max_xor16(-lo[e]), hi[e] = max_xor16(hi[e]);
        lo[e] = -max_xor32(-lo[e]), hi[e] = max_xor32(hi[e]);
    }
    const int64_t jb = r0 >> p.c.block_shift;
    T* out_lo = reinterpret_cast<T*>(p.lo + slot * p.lo_b + h * p.lo_h + jb * p.lo_s);
    T* out_hi = reinterpret_cast<T*>(p.hi + slot * p.hi_b + h * p.hi_h + jb * p.hi_s);
    if constexpr (WAVES == 1) {
        if (tid < p.chunks) {
            __attribute__((aligned(16))) T x[2][E];
#pragma unroll
            for (int e = 0; e < E; ++e) x[0][e] = Elem<T>::from_f32(lo[e]), x[1][e] = Elem<T>::from_f32(hi[e]);
            *reinterpret_cast<u32x4*>(out_lo + col * E) = *reinterpret_cast<const u32x4*>(x[0]);
            *reinterpret_cast<u32x4*>(out_hi + col * E) = *reinterpret_cast<const u32x4*>(x[1]);
        }
        return;
    }
    if ((tid & 63) < W) {
#pragma unroll
        for (int e = 0; e < E; ++e) red[tid >> 6][0][col * E + e] = lo[e], red[tid >> 6][1][col * E + e] = hi[e];
    }
    __syncthreads();
    for (int i = tid; i < p.chunks * E; i += 256) {
        out_lo[i] = Elem<T>::from_f32(fminf(fminf(red[0][0][i], red[1][0][i]), fminf(red[2][0][i], red[3][0][i])));
        out_hi[i] = Elem<T>::from_f32(fmaxf(fmaxf(red[0][1][i], red[1][1][i]), fmaxf(red[2][1][i], red[3][1][i])));
    }
}

// A workgroup scores kScoreBlocks blocks of one (sequence, kv head) at a time, kScoreLanes lanes to a block; HB: heads at a time.
// For every head a value is chosen by a mask (for 16-bit types two values at once), converted and multiplied with a query value from
// LDS; which of these it waits for has not been told apart.  The 64-bit matrix cores, at the vector units' rate with 16 columns for a
// group's 4 heads, take 29 us where this takes 17
// (32 sequences of 3000 to 32000 tokens in blocks of 64).  us with 4, 8 and 16 lanes (selection and attention included): one sequence
// of 30000 22.2, 20.9 and 20.6, eight 34.1, 33.0 and 36.0; two blocks to four lanes, which read the query from LDS half as often, 108.4 instead
// of 107.3 for those 32, and 40.4 instead of 32.0 for 64 sequences of 32 heads of up to 104 tokens.
constexpr int kScoreHeads = 16;
constexpr int kScoreLanes = 8, kScoreBlocks = 256 / kScoreLanes;

template <typename T, int D, int HB>
__global__ void __launch_bounds__(256) score_blocks_kernel(const SelectParams p) {
    constexpr int E = 16 / (int)sizeof(T), NI = D / E / kScoreLanes;  // chunks of a row per lane
    __shared__ __attribute__((aligned(16))) double qd[kScoreHeads][D];
    __shared__ __attribute__((aligned(16))) uint32_t qm[kScoreHeads][D * sizeof(T) / 4];  // all ones where q > 0
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x, b = bh / p.Hkv;
    const int h = (int)(bh % p.Hkv);
    const int n = tokens_in(p.c, b);
    const int blocks = (n + (1 << p.c.block_shift) - 1) >> p.c.block_shift;
    const int cand = blocks - p.recent, first = blockIdx.y * kScoreBlocks;
    if (blocks <= p.keep || first >= cand) return;
    uint32_t* order = p.order + bh * p.blocks_max;
    const int mine = tid / kScoreLanes, l = tid % kScoreLanes;
    const int in_page = p.c.page_shift - p.c.block_shift;  // log2 of a page's blocks
    u32x4 wl[NI], wh[NI];
    auto load = [&](int j0) {
        const int j = min(j0 + mine, cand - 1);
        int64_t slot = b, jb = j;
        if (p.c.table != nullptr) {
            slot = min(max(p.c.table[b * p.c.bt_s + (j >> in_page)], 0), p.c.num_pages - 1);
            jb = j & ((1 << in_page) - 1);
        }
        const char* lo = p.lo + slot * p.lo_b + h * p.lo_h + jb * p.lo_s;
        const char* hi = p.hi + slot * p.hi_b + h * p.hi_h + jb * p.hi_s;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = l + kScoreLanes * i;
            const bool there = E * c < p.d;
            wl[i] = ld16_nt(lo + (there ? 16 * c : 0));
            wh[i] = ld16_nt(hi + (there ? 16 * c : 0));
            if (!there) wl[i] = wh[i] = u32x4{0u, 0u, 0u, 0u};
        }
    };
    load(first);  // on their way while the query is laid out
    for (int g0 = 0; g0 < p.group; g0 += kScoreHeads) {
        const int heads = min(p.group - g0, kScoreHeads);
        if (g0 > 0) __syncthreads();  // the last heads have been used
        for (int i = tid; i < (heads + HB - 1) / HB * HB * D / E; i += 256) {
            const int g = i / (D / E), dim = i % (D / E) * E;
            u32x4 w = {0u, 0u, 0u, 0u}, mask;
            if (g < heads && dim < p.d)
                w = q_bits(ld16(reinterpret_cast<const T*>(p.q) + b * p.q_b + (h * p.group + g0 + g) * p.q_h + dim), p.q_and, p.q_xor);
            if constexpr (sizeof(T) == 4) {
                const f32x4 x = __builtin_bit_cast(f32x4, w);
#pragma unroll
                for (int e = 0; e < 4; ++e) qd[g][dim + e] = x[e], mask[e] = x[e] > 0.f ? 0xffffffffu : 0u;
            } else {
                float x[E];
                unpack8<T>(w, x);
#pragma unroll
                for (int e = 0; e < E; ++e) qd[g][dim + e] = x[e];
#pragma unroll
                for (int e = 0; e < 4; ++e) mask[e] = (x[2 * e] > 0.f ? 0xffffu : 0u) | (x[2 * e + 1] > 0.f ? 0xffff0000u : 0u);
            }
            *reinterpret_cast<u32x4*>(&qm[g][dim * (int)sizeof(T) / 4]) = mask;
        }
        __syncthreads();
        for (int j0 = first; j0 < cand; j0 += gridDim.y * kScoreBlocks) {
            if (g0 > 0 || j0 > first) load(j0);
            float best = kNegInf;
            for (int hb = 0; hb < heads; hb += HB) {
                double s[HB];
#pragma unroll
                for (int g = 0; g < HB; ++g) s[g] = 0.;
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int dim = (l + kScoreLanes * i) * E;
#pragma unroll
                    for (int g = 0; g < HB; ++g) {
                        const u32x4 mask = *reinterpret_cast<const u32x4*>(&qm[hb + g][dim * (int)sizeof(T) / 4]);
                        const u32x4 x = (wh[i] & mask) | (wl[i] & ~mask);
                        float f[E];
                        if constexpr (sizeof(T) == 4) {
                            const f32x4 v = __builtin_bit_cast(f32x4, x);
#pragma unroll
                            for (int e = 0; e < 4; ++e) f[e] = v[e];
                        } else {
                            unpack8<T>(x, f);
                        }
#pragma unroll
                        for (int e = 0; e < E; ++e) s[g] = __builtin_fma(qd[hb + g][dim + e], (double)f[e], s[g]);
                    }
                }
#pragma unroll
                for (int g = 0; g < HB; ++g) {
#pragma unroll
                    for (int x = 1; x < kScoreLanes; x *= 2) s[g] += __shfl_xor(s[g], x, 64);
                    if (hb + g < heads) best = fmaxf(best, (float)s[g]);  // NaN is passed over
                }
            }
            const int j = j0 + mine;
            if (l == 0 && j < cand) {
                const uint32_t u = ordered(best);
                order[j] = g0 == 0 ? u : max(order[j], u);
            }
        }
    }
}

// The scores: PER per thread in registers, or PER = 0 in memory.
template <int PER>
__global__ void __launch_bounds__(kSelect) select_blocks_kernel(const SelectParams p) {
    const int64_t bh = blockIdx.x, b = bh / p.Hkv;
    const int n = tokens_in(p.c, b);
    const int blocks = (n + (1 << p.c.block_shift) - 1) >> p.c.block_shift;
    int32_t* kept = p.kept + bh * p.keep;
    if (blocks <= p.keep) {
        for (int i = threadIdx.x; i < p.keep; i += kSelect) kept[i] = i < blocks ? i : -1;
        return;
    }
    uint32_t* order = p.order + bh * p.blocks_max;
    select_largest<PER>(blocks - p.recent, p.keep - p.recent, p.recent, order, kept, [&](int i) { return order[i]; });
}

namespace {

struct BlockSizes {
    int64_t S_max, num_pages, page_size, max_pages, block_table_stride;
    const int32_t* table;
    const int32_t* lengths;
    int32_t block;
};

int block_checks(const BlockSizes& a, const char* who, BlockCache* out) {
    if (a.block < 16 || a.block > 256 || (a.block & (a.block - 1)) != 0)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: block %d must be a power of two from 16 to 256", who, a.block);
    out->table = a.table;
    out->lengths = a.lengths;
    out->bt_s = a.block_table_stride;
    out->block_shift = __builtin_ctz((unsigned)a.block);
    out->page_shift = 0, out->num_pages = 0;
    if (a.table != nullptr) {
        if (a.page_size < 16 || (a.page_size & (a.page_size - 1)) != 0 || a.page_size > (1 << 20))
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: page_size %lld must be a power of two >= 16", who, (long long)a.page_size);
        if (a.page_size < a.block)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: a page of %lld tokens does not hold a block of %d", who, (long long)a.page_size, a.block);
        if (a.num_pages <= 0 || a.max_pages <= 0 || a.num_pages > 0x7fffffff || a.max_pages > (1 << 29) / a.page_size)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad page counts", who);
        out->capacity = (int32_t)(a.max_pages * a.page_size);
        out->page_shift = __builtin_ctzll((unsigned long long)a.page_size);
        out->num_pages = (int32_t)a.num_pages;
    } else {
        if (a.S_max <= 0 || a.S_max > (1 << 29) || a.S_max % a.block != 0)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: S_max=%lld must be a positive multiple of the block of %d tokens", who, (long long)a.S_max, a.block);
        out->capacity = (int32_t)a.S_max;
    }
    return DTATTN_OK;
}

// Rows of 16-byte chunks at 16-byte strides, D up to 128.
int row_checks(int64_t D, int32_t dtype, const int64_t* strides, int n, uintptr_t bits, const char* who) {
    if (dtype != DTATTN_BF16 && dtype != DTATTN_FP16 && dtype != DTATTN_FP32)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: dtype %d not supported (bf16, fp16, fp32)", who, dtype);
    const int64_t esz = dtype == DTATTN_FP32 ? 4 : 2;
    if (D <= 0 || D > 128 || (D * esz) % 16 != 0)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: head dim %lld not supported (up to 128, a multiple of 16 bytes)", who, (long long)D);
    for (int i = 0; i < n; ++i)
        if (strides[i] < 0 || (strides[i] * esz) % 16 != 0)
            return fail(DTATTN_ERR_UNSUPPORTED, "%s: strides must be multiples of 16 bytes", who);
    if (bits & 15) return fail(DTATTN_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned", who);
    return DTATTN_OK;
}

template <typename T, int WAVES>
void launch_bounds_waves(const BoundsParams& p, unsigned heads, unsigned groups, hipStream_t stream) {
    const dim3 grid(heads, groups);
    if (p.chunks <= 8) hipLaunchKernelGGL((key_bounds_kernel<T, 8, WAVES>), grid, dim3(256), 0, stream, p);
    else if (p.chunks <= 16) hipLaunchKernelGGL((key_bounds_kernel<T, 16, WAVES>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((key_bounds_kernel<T, 32, WAVES>), grid, dim3(256), 0, stream, p);
}
template <typename T>
void launch_bounds_of(BoundsParams p, unsigned heads, int64_t blocks, hipStream_t stream) {
    // A wave to a block of up to 64 tokens, whose waves would have a load each before they meet.  us with one wave and with four, 4 x 4000
    // tokens: blocks of 16 8.9 and 21.2, of 32 8.3 and 12.1, of 64 8.0 and 8.6, of 256 10.7 and 8.1.
    const bool one = p.c.block_shift <= 6;
    const int64_t each = one ? 4 : 1, most = 65535 * each;  // blocks of a workgroup, and of a launch
    for (int64_t b0 = 0; b0 < blocks; b0 += most) {
        p.first = (int32_t)b0;
        const unsigned groups = (unsigned)((std::min(most, blocks - b0) + each - 1) / each);
        if (one) launch_bounds_waves<T, 1>(p, heads, groups, stream);
        else launch_bounds_waves<T, 4>(p, heads, groups, stream);
    }
}

template <typename T, int D, int HB>
void launch_score(const SelectParams& p, unsigned heads, int64_t cus, hipStream_t stream) {
    // As many workgroups as have blocks, up to 16 to a CU.  us of those 32 sequences with 8, 16 and 64: 109.2, 107.7 and 107.6
    const int64_t most = std::max<int64_t>((16 * cus + heads - 1) / heads, 1), parts = (p.blocks_max + kScoreBlocks - 1) / kScoreBlocks;
    hipLaunchKernelGGL((score_blocks_kernel<T, D, HB>), dim3(heads, (unsigned)std::min(parts, most)), dim3(256), 0, stream, p);
}
template <typename T>
void score(const SelectParams& p, unsigned heads, int64_t cus, hipStream_t stream) {
    if (p.d <= 64) p.group == 1 ? launch_score<T, 64, 1>(p, heads, cus, stream) : launch_score<T, 64, 4>(p, heads, cus, stream);
    else p.group == 1 ? launch_score<T, 128, 1>(p, heads, cus, stream) : launch_score<T, 128, 4>(p, heads, cus, stream);
}

template <typename Args>
BlockSizes sizes_of(const Args* a) {
    return {a->S_max, a->num_pages, a->page_size, a->max_pages, a->block_table_stride, a->block_table, a->lengths, a->block};
}

int64_t blocks_max_of(const dtattn_select_blocks_args* a) {
    const int64_t capacity = a->block_table != nullptr ? a->max_pages * a->page_size : a->S_max;
    return (capacity + a->block - 1) / a->block;
}

}  // namespace

}  // namespace dtattn

using namespace dtattn;

extern "C" int dtattn_key_bounds(const dtattn_key_bounds_args* a, void* stream_) {
    const char* who = "key_bounds";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    if (a->B < 0 || a->Hkv <= 0 || a->B > (1 << 24) || a->Hkv > (1 << 20) || a->n_new < 0) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
    BoundsParams p = {};
    int st = block_checks(sizes_of(a), who, &p.c);
    if (st != DTATTN_OK) return st;
    const int64_t strides[9] = {a->k_stride[0], a->k_stride[1], a->k_stride[2], a->min_stride[0], a->min_stride[1], a->min_stride[2],
                                a->max_stride[0], a->max_stride[1], a->max_stride[2]};
    st = row_checks(a->D, a->dtype, strides, 9,
                    reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->k_min) | reinterpret_cast<uintptr_t>(a->k_max), who);
    if (st != DTATTN_OK || a->B == 0 || a->n_new == 0) return st;
    if (a->k_cache == nullptr || a->k_min == nullptr || a->k_max == nullptr || a->lengths == nullptr)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    if (a->k_min == a->k_max || a->k_min == a->k_cache || a->k_max == a->k_cache)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: keys and bounds cannot share memory", who);
    const int64_t esz = a->dtype == DTATTN_FP32 ? 4 : 2;
    p.k = reinterpret_cast<const char*>(a->k_cache);
    p.lo = reinterpret_cast<char*>(a->k_min), p.hi = reinterpret_cast<char*>(a->k_max);
    p.k_b = a->k_stride[0] * esz, p.k_h = a->k_stride[1] * esz, p.k_s = a->k_stride[2] * esz;
    p.lo_b = a->min_stride[0] * esz, p.lo_h = a->min_stride[1] * esz, p.lo_s = a->min_stride[2] * esz;
    p.hi_b = a->max_stride[0] * esz, p.hi_h = a->max_stride[1] * esz, p.hi_s = a->max_stride[2] * esz;
    p.Hkv = (int32_t)a->Hkv, p.chunks = (int32_t)(a->D * esz / 16);
    const int64_t n = std::min<int64_t>(a->n_new, p.c.capacity);
    p.n_new = (int32_t)n;
    const int64_t blocks = (n + a->block - 2) / a->block + 1, heads = a->B * a->Hkv;  // that n tokens touch, at most
    if (heads > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    switch (a->dtype) {
        case DTATTN_BF16: launch_bounds_of<bf16_t>(p, (unsigned)heads, blocks, stream); break;
        case DTATTN_FP16: launch_bounds_of<f16_t>(p, (unsigned)heads, blocks, stream); break;
        default: launch_bounds_of<float>(p, (unsigned)heads, blocks, stream);
    }
    return check_launch("key_bounds_kernel");
}

extern "C" size_t dtattn_select_key_blocks_workspace_size(const dtattn_select_blocks_args* a) {
    if (a == nullptr || a->B <= 0 || a->Hkv <= 0 || a->block <= 0) return 0;
    return ((size_t)a->B * a->Hkv * blocks_max_of(a) * sizeof(uint32_t) + 255) & ~(size_t)255;
}

extern "C" int dtattn_select_key_blocks(const dtattn_select_blocks_args* a, void* stream_) {
    const char* who = "select_key_blocks";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    if (a->B < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->B > (1 << 24) || a->Hq > (1 << 20)) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
    if (a->Hq % a->Hkv != 0) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: Hq is not a multiple of Hkv", who);
    SelectParams p = {};
    int st = block_checks(sizes_of(a), who, &p.c);
    if (st != DTATTN_OK) return st;
    if (a->recent < a->block || a->keep < a->recent || a->keep % a->block != 0 || a->recent % a->block != 0 || a->keep > (1 << 29))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: keep %lld and recent %lld must be multiples of the block of %d tokens with block <= recent <= keep",
                    who, (long long)a->keep, (long long)a->recent, a->block);
    const int64_t strides[8] = {a->q_stride[0], a->q_stride[1], a->min_stride[0], a->min_stride[1], a->min_stride[2],
                                a->max_stride[0], a->max_stride[1], a->max_stride[2]};
    st = row_checks(a->D, a->dtype, strides, 8,
                    reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k_min) | reinterpret_cast<uintptr_t>(a->k_max), who);
    if (st != DTATTN_OK) return st;
    ScalePlan sp;
    st = plan_scale(a->scale, a->D, a->dtype == DTATTN_FP32 ? kSign32 : kSign16, &sp);
    if (st != DTATTN_OK || a->B == 0) return st;
    if (a->q == nullptr || a->k_min == nullptr || a->k_max == nullptr || a->lengths == nullptr || a->blocks == nullptr)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    if (a->B * a->Hkv > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
    const size_t need = dtattn_select_key_blocks_workspace_size(a);
    if (a->workspace == nullptr || a->workspace_bytes < need)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, need, a->workspace_bytes);
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return fail(DTATTN_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
    const int64_t esz = a->dtype == DTATTN_FP32 ? 4 : 2;
    p.q = reinterpret_cast<const char*>(a->q);
    p.lo = reinterpret_cast<const char*>(a->k_min), p.hi = reinterpret_cast<const char*>(a->k_max);
    p.order = reinterpret_cast<uint32_t*>(a->workspace);
    p.kept = a->blocks;
    p.q_b = a->q_stride[0], p.q_h = a->q_stride[1];
    p.lo_b = a->min_stride[0] * esz, p.lo_h = a->min_stride[1] * esz, p.lo_s = a->min_stride[2] * esz;
    p.hi_b = a->max_stride[0] * esz, p.hi_h = a->max_stride[1] * esz, p.hi_s = a->max_stride[2] * esz;
    p.Hkv = (int32_t)a->Hkv, p.group = (int32_t)(a->Hq / a->Hkv), p.d = (int32_t)a->D;
    p.keep = (int32_t)(a->keep / a->block), p.recent = (int32_t)(a->recent / a->block);
    p.blocks_max = (int32_t)blocks_max_of(a);
    p.q_and = sp.q_and, p.q_xor = sp.q_xor;
    const unsigned heads = (unsigned)(a->B * a->Hkv);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const int64_t cus = std::max(stream_cus(stream), 1);
    switch (a->dtype) {
        case DTATTN_BF16: score<bf16_t>(p, heads, cus, stream); break;
        case DTATTN_FP16: score<f16_t>(p, heads, cus, stream); break;
        default: score<float>(p, heads, cus, stream);
    }
    st = check_launch("score_blocks_kernel");
    if (st != DTATTN_OK) return st;
    // as few a thread as hold them
    if (p.blocks_max <= kSelect) hipLaunchKernelGGL(select_blocks_kernel<1>, dim3(heads), dim3(kSelect), 0, stream, p);
    else if (p.blocks_max <= 4 * kSelect) hipLaunchKernelGGL(select_blocks_kernel<4>, dim3(heads), dim3(kSelect), 0, stream, p);
    else if (p.blocks_max <= 16 * kSelect) hipLaunchKernelGGL(select_blocks_kernel<16>, dim3(heads), dim3(kSelect), 0, stream, p);
    else hipLaunchKernelGGL(select_blocks_kernel<0>, dim3(heads), dim3(kSelect), 0, stream, p);
    return check_launch("select_blocks_kernel");
}
