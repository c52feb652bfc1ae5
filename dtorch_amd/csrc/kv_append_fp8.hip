// Quantised KV-cache append: new keys and values as e4m3fn codes with one power-of-two scale per block of tokens.
//
// No counterpart in the reference, which keeps no KV cache (python/dtorch/test/modules/llama.py:126-156).  With
// amax = max |x| over the finite new values of a block, the block needs s = 2^k, the smallest power of two with
// amax <= 448 s; code = e4m3_rne(x / s).  A floating code loses nothing by a power of two (its relative precision does not
// depend on the scale, only the range below the block's maximum does, and that is 2^-9 at the least), and a block that
// grows over several appends then re-encodes its older rows by an exact shift instead of rounding them again each time.
//
// HBM-bound: an item per (sequence, kv head, K or V, touched block), whose threads hold its new rows in four chunks of 8
// elements each, so that they are read once: a wave for up to 16 rows of 128, a workgroup of 2 to 16 waves for more.  A
// thread runs the code once, so short code matters: 16 chunks per lane, one wave to a block of 64, took 20 us where this takes
// 12 (4 x 2000 tokens of 8 heads of 128, bf16).  Few items per sequence (a decode step) run as one workgroup per
// sequence, which also advances the length; with more a second launch on the same stream does.
#include <algorithm>

#include "fp8_cache.hpp"

namespace dtattn {

struct Append8Params {
    const char* src[2];  // new K, new V
    char* dst[2];        // codes: cache base, or page pool base
    float* scale[2];
    const int32_t* block_table;  // paged only
    int32_t* lengths;
    int64_t n_b[2], n_h[2], n_s[2];  // byte strides of the new tokens
    int64_t d_b[2], d_h[2], d_s[2];  // byte strides of the codes: (batch | page), head, row
    int64_t s_b[2], s_h[2];          // element strides of the scales
    int64_t bt_s, items;
    int32_t Hkv, n_new, cpr;  // cpr: chunks of 8 elements per token row
    int32_t nblk;             // most blocks that a sequence's new tokens touch
    int32_t capacity, page_shift, num_pages, block_shift;
};

namespace {

constexpr int kHeld = 4;  // chunks of 8 elements that a lane holds: a wave holds 16 rows of 128

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < __builtin_inff(); }

// The smallest power of two s >= 2^-126 with m <= 448 s.  m = f 2^e with 1 <= f < 2: 448 = 1.75 * 2^8.  For m = 0 that is 2^-126, which
// no other value's scale is below: tokens without a finite value other than 0 leave the scale to those before and behind them.
__device__ __forceinline__ float scale_for(float m) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, m);
    const int k = (int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);  // biased by 127
    return __builtin_bit_cast(float, (uint32_t)max(k, 1) << 23);
}

__device__ __forceinline__ uint32_t codes4(const float* x) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
}

// 8 values times `inv` as codes, NaN for values that are not finite (their product with inv may be).
__device__ __forceinline__ u32x2 encode8(const float* x, float inv) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = finite(x[e]) ? x[e] * inv : __builtin_nanf("");
    return u32x2{codes4(y), codes4(y + 4)};
}

// Largest magnitude as bits: those of elements without their sign, which order as the values do, infinities and NaN on top.
// Two 16-bit elements go at a time.
template <typename T>
__device__ __forceinline__ uint32_t max_bits(uint32_t m, const Chunk<T>& c) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(c.v) / sizeof(c.v[0])); ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) m = max(m, c.v[i][j] & 0x7fffffffu);
            else m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m), __builtin_bit_cast(u16x2, c.v[i][j] & 0x7fff7fffu)));
        }
    return m;
}
// The value of max_bits over a wave's lanes.
template <typename T>
__device__ __forceinline__ float wave_max_bits(uint32_t m) {
    if constexpr (sizeof(T) == 2) m = max(m & 0xffffu, m >> 16);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d, 64));
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, m);
    else return Elem<T>::to_f32(__builtin_bit_cast(T, (uint16_t)m));
}

// 8 values of 16 bits, all finite, over a power of two s that holds them: one conversion per pair, which divides and rounds
// once (the same codes as encode8's, checked over every value of both types).
template <typename T>
__device__ __forceinline__ u32x2 encode8_pow2(const Chunk<T>& c, float s) {
    typedef T pair __attribute__((ext_vector_type(2)));
    typedef short s16x2 __attribute__((ext_vector_type(2)));
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = c.v[0][i];
        const pair x = __builtin_bit_cast(pair, w);
        s16x2 r = {};
        if constexpr (__is_same(T, f16_t)) r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(r, x, s, false);
        else r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, x, s, false);
        o[i] = __builtin_bit_cast(uint32_t, r);
    }
    return u32x2{pack_lo_hi(o[0], o[1], 0), pack_lo_hi(o[2], o[3], 0)};
}

// 4 codes times `f`, rounded to codes again.
__device__ __forceinline__ uint32_t recode4(uint32_t w, float f) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    const float y[4] = {a[0] * f, a[1] * f, b[0] * f, b[1] * f};
    return codes4(y);
}

// An item: block i of those that the new tokens of (b, h) touch, of K (kv = 0) or V.  WAVES: one wave's, or a workgroup's.
template <typename T, bool PAGED, bool WAVES>
__device__ __forceinline__ void append8_item(const Append8Params& p, int64_t b, int h, int kv, int i, int length) {
    const int t = WAVES ? threadIdx.x & 63 : threadIdx.x, threads = WAVES ? 64 : blockDim.x;
    const int start = max(length, 0);
    if (start >= p.capacity) return;
    const int t0 = ((start >> p.block_shift) + i) << p.block_shift;
    const int first = max(start, t0);
    const int stop = min((int)min((int64_t)start + p.n_new, (int64_t)p.capacity), t0 + (1 << p.block_shift));
    if (first >= stop) return;
    int64_t slot = b;
    int row0 = t0;
    if constexpr (PAGED) {
        const int page = p.block_table[b * p.bt_s + (t0 >> p.page_shift)];
        if (page < 0 || page >= p.num_pages) return;  // not a page of the pool: the tokens are dropped
        slot = page;
        row0 = t0 & ((1 << p.page_shift) - 1);
    }
    char* dst = p.dst[kv] + slot * p.d_b[kv] + h * p.d_h[kv] + row0 * p.d_s[kv];  // the block's first row
    float* sp = p.scale[kv] + slot * p.s_b[kv] + h * p.s_h[kv] + (row0 >> p.block_shift);
    const char* src = p.src[kv] + b * p.n_b[kv] + h * p.n_h[kv] + (int64_t)(first - start) * p.n_s[kv];
    const float old = first > t0 ? *sp : 0.f;
    // a thread's chunks: number c of rows r, r + step, ...; the launch has no more than kHeld * step rows in a block
    const int step = threads / p.cpr, r = t / p.cpr, c = t - r * p.cpr;
    const int rows = r < step ? stop - first : 0;  // threads past the last whole row idle
    Chunk<T> raw[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        raw[k] = Chunk<T>{};
        if (r + k * step < rows) raw[k] = load_chunk<T, false>(reinterpret_cast<const T*>(src + (r + k * step) * p.n_s[kv]) + c * 8);
    }
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) top = max_bits<T>(top, raw[k]);
    __shared__ float red[2][16];
    auto largest = [&](float m, int which) {
        if constexpr (!WAVES) {
            if ((t & 63) == 0) red[which][t >> 6] = m;
            __syncthreads();
            for (int w = 0; w < threads >> 6; ++w) {  // NaN bits count as the largest here
                const float x = red[which][w];
                m = x != x || x > m ? x : m;
            }
        }
        return m;
    };
    float m = largest(wave_max_bits<T>(top), 0);
    const bool clean = finite(m);
    if (!clean) {  // of the others, then
        m = 0.f;
#pragma unroll
        for (int k = 0; k < kHeld; ++k) {
            float x[8];
            unpack_chunk<T>(raw[k], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, finite(x[e]) ? fabsf(x[e]) : 0.f);
        }
        m = largest(wave_max(m), 1);
    }
    float s = scale_for(m);
    if (first > t0) {
        s = fmaxf(old, s);
        if (s != old) {  // the block's older rows at its new scale
            const float f = old / s;
            for (int i = r; i < (r < step ? first - t0 : 0); i += step) {
                u32x2* at = reinterpret_cast<u32x2*>(dst + i * p.d_s[kv] + c * 8);
                const u32x2 w = *at;
                *at = u32x2{recode4(w.x, f), recode4(w.y, f)};
            }
        }
    }
    if (t == 0) *sp = s;
    const float inv = 1.f / s;
    char* to = dst + (first - t0) * p.d_s[kv] + c * 8;
    auto put = [&](auto encode) {
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (r + k * step < rows) *reinterpret_cast<u32x2*>(to + (r + k * step) * p.d_s[kv]) = encode(raw[k]);
    };
    if constexpr (sizeof(T) == 2) {
        // an older scale of the caller's own need not be a power of two
        if (clean && (__builtin_bit_cast(uint32_t, s) & 0x7fffffu) == 0) {
            put([&](const Chunk<T>& w) { return encode8_pow2<T>(w, s); });
            return;
        }
    }
    put([&](const Chunk<T>& w) {
        float x[8];
        unpack_chunk<T>(w, x);
        return encode8(x, inv);
    });
}

}  // namespace

template <typename T, bool PAGED, bool WAVES>
__global__ void __launch_bounds__(WAVES ? 256 : 1024) kv_append_fp8_kernel(const Append8Params p) {
    const int64_t item = WAVES ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
    if (item >= p.items) return;
    const int64_t bh = item / (2 * p.nblk), b = bh / p.Hkv;
    const int r = (int)(item % (2 * p.nblk));
    append8_item<T, PAGED, WAVES>(p, b, (int)(bh % p.Hkv), r & 1, r >> 1, p.lengths[b]);
}

// One sequence per workgroup, and its length.
template <typename T, bool PAGED>
__global__ void __launch_bounds__(1024) kv_append_fp8_step_kernel(const Append8Params p) {
    const int64_t b = blockIdx.x;
    const int length = p.lengths[b];
    const int per = 2 * p.nblk, items = p.Hkv * per;
    for (int it = threadIdx.x >> 6; it < items; it += blockDim.x >> 6)
        append8_item<T, PAGED, true>(p, b, it / per, (it % per) & 1, (it % per) >> 1, length);
    __syncthreads();  // every thread has read the length
    if (threadIdx.x == 0) p.lengths[b] = (int)min((int64_t)max(length, 0) + p.n_new, (int64_t)p.capacity);
}

__global__ void __launch_bounds__(256) kv_lengths_fp8_kernel(int32_t* lengths, int64_t B, int32_t n_new, int32_t capacity) {
    const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (b < B) lengths[b] = (int)min((int64_t)max(lengths[b], 0) + n_new, (int64_t)capacity);
}

template <typename T, bool PAGED>
static int launch_append8(const Append8Params& p, int64_t B, hipStream_t stream) {
    const int64_t per_seq = p.items / B;
    // One launch for few items of few rows (a wave holds 16 rows of 128): us with 16 / 32 / 64 / 128 items a sequence against two
    // launches 6.0 and 8.8 / 7.8 and 9.1 / 11.5 and 9.0 / 19.3 and 9.5 (1 token, 64 to 16 sequences of 8 to 64 heads).
    const int held = kHeld * (64 / p.cpr);
    if (p.n_new > 0 && per_seq <= 32 && p.n_new <= held && B <= 0x7fffffff) {
        const unsigned waves = (unsigned)(per_seq < 16 ? per_seq : 16);
        hipLaunchKernelGGL((kv_append_fp8_step_kernel<T, PAGED>), dim3((unsigned)B), dim3(64 * waves), 0, stream, p);
        return check_launch("kv_append_fp8_step_kernel");
    }
    if (p.n_new > 0) {
        // a wave for a block that it holds, or else as many as hold it; 256 rows of 128 are 16 waves' (kHeld * (threads / cpr) rows)
        const int rows = std::min(1 << p.block_shift, p.n_new);
        unsigned waves = 1;
        while (kHeld * (64 * (int)waves / p.cpr) < rows) ++waves;
        const int64_t blocks = waves == 1 ? (p.items + 3) / 4 : p.items;
        if (blocks > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "kv_append_fp8: grid too large");
        if (waves == 1) hipLaunchKernelGGL((kv_append_fp8_kernel<T, PAGED, true>), dim3((unsigned)blocks), dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((kv_append_fp8_kernel<T, PAGED, false>), dim3((unsigned)blocks), dim3(64 * waves), 0, stream, p);
        const int st = check_launch("kv_append_fp8_kernel");
        if (st != DTATTN_OK) return st;
    }
    hipLaunchKernelGGL(kv_lengths_fp8_kernel, dim3((unsigned)((B + 255) / 256)), dim3(256), 0, stream, p.lengths, B, p.n_new, p.capacity);
    return check_launch("kv_lengths_fp8_kernel");
}

}  // namespace dtattn

using namespace dtattn;

extern "C" int dtattn_kv_append_fp8(const dtattn_kv_append_fp8_args* a, void* stream_) {
    const char* who = "kv_append_fp8";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    if (a->B < 0 || a->Hkv <= 0 || a->n_new < 0 || a->D <= 0 || a->Hkv > (1 << 20) || a->B > (1 << 24))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
    Append8Params p = {};
    Fp8Cache c;
    int st = fp8_cache_checks(a, a->block_table != nullptr, who, &c);
    if (st != DTATTN_OK) return st;
    if (a->dtype != DTATTN_BF16 && a->dtype != DTATTN_FP16 && a->dtype != DTATTN_FP32)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: dtype %d not supported (bf16, fp16, fp32)", who, a->dtype);
    if (a->n_new > 0x3fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: too many new tokens", who);
    if (a->B == 0) return DTATTN_OK;
    if (a->lengths == nullptr || (a->n_new > 0 && (a->k_new == nullptr || a->v_new == nullptr)))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    if (a->k_cache == a->v_cache || a->k_scale == a->v_scale)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: keys and values are both written and cannot share memory", who);
    const int64_t esz = a->dtype == DTATTN_FP32 ? 4 : 2;
    for (int i = 0; i < 3; ++i)
        if ((a->k_new_stride[i] * esz) % 16 != 0 || (a->v_new_stride[i] * esz) % 16 != 0)
            return fail(DTATTN_ERR_UNSUPPORTED, "%s: strides of the new tokens must be multiples of 16 bytes", who);
    if ((reinterpret_cast<uintptr_t>(a->k_new) | reinterpret_cast<uintptr_t>(a->v_new)) & 15u)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: new tokens must be 16-byte aligned", who);
    const void* src[2] = {a->k_new, a->v_new};
    void* dst[2] = {a->k_cache, a->v_cache};
    float* scale[2] = {a->k_scale, a->v_scale};
    const int64_t* ns[2] = {a->k_new_stride, a->v_new_stride};
    const int64_t* ds[2] = {a->k_stride, a->v_stride};
    const int64_t* ss[2] = {a->k_scale_stride, a->v_scale_stride};
    for (int i = 0; i < 2; ++i) {
        p.src[i] = reinterpret_cast<const char*>(src[i]);
        p.dst[i] = reinterpret_cast<char*>(dst[i]);
        p.scale[i] = scale[i];
        p.n_b[i] = ns[i][0] * esz, p.n_h[i] = ns[i][1] * esz, p.n_s[i] = ns[i][2] * esz;
        p.d_b[i] = ds[i][0], p.d_h[i] = ds[i][1], p.d_s[i] = ds[i][2];
        p.s_b[i] = ss[i][0], p.s_h[i] = ss[i][1];
    }
    p.block_table = a->block_table;
    p.bt_s = a->block_table_stride;
    p.lengths = a->lengths;
    p.Hkv = (int32_t)a->Hkv;
    p.n_new = (int32_t)a->n_new;
    p.cpr = (int32_t)(a->D / 8);
    p.capacity = c.capacity;
    p.page_shift = c.page_shift;
    p.num_pages = c.num_pages;
    p.block_shift = c.block_shift;
    // the first new token may be the last row of its block
    p.nblk = a->n_new == 0 ? 0 : (int32_t)((a->block - 1 + a->n_new - 1) / a->block + 1);
    if (a->B * a->Hkv > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
    p.items = a->B * a->Hkv * 2 * p.nblk;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    const bool paged = a->block_table != nullptr;
    switch (a->dtype) {
        case DTATTN_BF16: return paged ? launch_append8<bf16_t, true>(p, a->B, stream) : launch_append8<bf16_t, false>(p, a->B, stream);
        case DTATTN_FP16: return paged ? launch_append8<f16_t, true>(p, a->B, stream) : launch_append8<f16_t, false>(p, a->B, stream);
        default: return paged ? launch_append8<float, true>(p, a->B, stream) : launch_append8<float, false>(p, a->B, stream);
    }
}
