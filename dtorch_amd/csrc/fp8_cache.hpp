// What the entry points over an 8-bit KV cache check alike, and the small device helpers that they share.
#pragma once
#include "dtattn_common.hpp"

namespace dtattn {

struct Fp8Cache {
    int32_t capacity, page_shift, num_pages, block_shift;
};

// Sizes, strides and alignment of the code and scale arrays of dtattn_kv_append_fp8_args / dtattn_decode_fp8_args.
template <typename Args>
static int fp8_cache_checks(const Args* a, bool paged, const char* who, Fp8Cache* out) {
    if (a->D % 16 != 0 || a->D > 128)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: head dim %lld not supported (a multiple of 16 up to 128)", who, (long long)a->D);
    if (a->block < 16 || a->block > 256 || (a->block & (a->block - 1)) != 0)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: block %d must be a power of two from 16 to 256", who, a->block);
    out->block_shift = __builtin_ctz((unsigned)a->block);
    out->page_shift = 0;
    out->num_pages = 0;
    if (paged) {
        if (a->page_size < 16 || (a->page_size & (a->page_size - 1)) != 0 || a->page_size > (1 << 20))
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: page_size %lld must be a power of two >= 16", who, (long long)a->page_size);
        if (a->page_size < a->block)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: a page of %lld tokens does not hold a block of %d", who, (long long)a->page_size, a->block);
        if (a->num_pages <= 0 || a->max_pages <= 0 || a->num_pages > 0x7fffffff || a->max_pages > (1 << 29) / a->page_size)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad page counts", who);
        out->capacity = (int32_t)(a->max_pages * a->page_size);
        out->page_shift = __builtin_ctzll((unsigned long long)a->page_size);
        out->num_pages = (int32_t)a->num_pages;
    } else {
        if (a->S_max <= 0 || a->S_max > (1 << 29) || a->S_max % a->block != 0)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: S_max=%lld must be a positive multiple of the block of %d tokens", who,
                        (long long)a->S_max, a->block);
        out->capacity = (int32_t)a->S_max;
    }
    if (a->B == 0) return DTATTN_OK;
    if (a->k_cache == nullptr || a->v_cache == nullptr || a->k_scale == nullptr || a->v_scale == nullptr)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null cache pointer", who);
    if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15u)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: caches must be 16-byte aligned", who);
    for (int i = 0; i < 3; ++i)
        if (a->k_stride[i] % 16 != 0 || a->v_stride[i] % 16 != 0)
            return fail(DTATTN_ERR_UNSUPPORTED, "%s: cache strides must be multiples of 16 bytes", who);
    // the 32 rows of a decode unit are addressed with 32-bit offsets below 2^30, and what must not be read with offsets from 3 * 2^30 on
    if (a->k_stride[2] < a->D || a->v_stride[2] < a->D || a->k_stride[2] > (1 << 24) || a->v_stride[2] > (1 << 24))
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: the row stride of a cache must be from D to 2^24 bytes", who);
    return DTATTN_OK;
}

// Two codes of a word (its low or high half) as two 16-bit floats: exact.
template <typename T, bool HIGH>
__device__ __forceinline__ uint32_t codes_to_pair(uint32_t w) {
    if constexpr (__is_same(T, f16_t)) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
}
// Eight codes as a matrix operand.
template <typename T>
__device__ __forceinline__ typename Elem<T>::vec8 codes_to_vec8(uint32_t lo, uint32_t hi) {
    return __builtin_bit_cast(typename Elem<T>::vec8, u32x4{codes_to_pair<T, false>(lo), codes_to_pair<T, true>(lo), codes_to_pair<T, false>(hi), codes_to_pair<T, true>(hi)});
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Inclusive prefix sum over the wave's lanes, by DPP: within rows of 16, then the last lanes of rows to those behind.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int scan64(int v) {
    v = dpp_add<0x111, 0xf>(v);  // row_shr:1
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    return dpp_add<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
}

// The three bf16 parts of an fp32 value, each the rest rounded to nearest: 24 bits of mantissa as 8 + 8 + 8, so that their sum is the
// value (parts below the smallest bf16 normal apart), with the second at most 2^-8 and the third 2^-16 of it.  A value that is
// not finite is its first part; of one that would round to infinity that is cut off instead.
__device__ __forceinline__ void split3(float x, bf16_t out[3]) {
    const float mag = fabsf(x);
    const bool finite = mag < __builtin_inff();
    const bool cut = finite && mag > 0x1.fep127f;
    out[0] = static_cast<bf16_t>(cut ? __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xffff0000u) : x);
    float r = finite ? x - static_cast<float>(out[0]) : 0.f;
    out[1] = static_cast<bf16_t>(r);
    r -= static_cast<float>(out[1]);
    out[2] = static_cast<bf16_t>(r);
}

}  // namespace dtattn
