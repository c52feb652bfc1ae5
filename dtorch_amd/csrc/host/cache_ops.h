// Host operators over the 8-bit KV cache and the bounded one (dtattn.h, "KV cache in 8 bits" and "a bounded KV cache").
//
// New operators without a reference counterpart: the reference keeps no KV cache
// (python/dtorch/test/modules/llama.py:126-156).  They follow the operator contract of sdpa_op.h.
#pragma once

#include "sdpa_op.h"

namespace dtorch_amd {
namespace core {

struct KvCacheAppendFp8Param : KvCacheAppendParam {};
struct KvCacheAppendFp8PagedParam : KvCacheAppendParam {};

// SdpaDecodeFp8 / SdpaDecodeFp8Paged: softmax scale (none: 1/sqrt(D)).
struct SdpaDecodeFp8Param {
    std::optional<double> scale = std::nullopt;

    SdpaDecodeFp8Param() = default;
    explicit SdpaDecodeFp8Param(std::optional<double> scale_) : scale(scale_) {}

    template <class Archive>
    void serialize(Archive& ar, const unsigned int /*version*/) {
        ar & scale;
    }
};
struct SdpaDecodeFp8PagedParam : SdpaDecodeFp8Param {
    using SdpaDecodeFp8Param::SdpaDecodeFp8Param;
    SdpaDecodeFp8PagedParam() = default;
};

// AttentionWeights: softmax scale, causal rule and the position of the first query.
struct AttentionWeightsParam {
    std::optional<double> scale = std::nullopt;
    bool isCausal = false;
    int64_t qOffset = 0;

    AttentionWeightsParam() = default;
    AttentionWeightsParam(std::optional<double> scale_, bool isCausal_, int64_t qOffset_)
        : scale(scale_), isCausal(isCausal_), qOffset(qOffset_) {}

    template <class Archive>
    void serialize(Archive& ar, const unsigned int /*version*/) {
        ar & scale;
        ar & isCausal;
        ar & qOffset;
    }
};

// KvCacheEvict: tokens that stay, how many of them are the last ones, and the tokens of a block (0: those of a scale, or 1).
struct KvCacheEvictParam {
    int64_t keep = 1;
    int64_t recent = 1;
    int64_t block = 0;

    KvCacheEvictParam() = default;
    KvCacheEvictParam(int64_t keep_, int64_t recent_, int64_t block_) : keep(keep_), recent(recent_), block(block_) {}

    template <class Archive>
    void serialize(Archive& ar, const unsigned int /*version*/) {
        ar & keep;
        ar & recent;
        ar & block;
    }
};

// {k_cache, v_cache, k_scale, v_scale, lengths, k_new, v_new} -> {k_cache, v_cache, k_scale, v_scale, lengths}, updated in
// place: codes float8_e4m3fn [B, Hkv, S_max, D], scales fp32 [B, Hkv, S_max / block].
class KvCacheAppendFp8Op {
public:
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;
};

// {k_pages, v_pages, k_scale, v_scale, block_table, lengths, k_new, v_new} -> the first four and lengths: pools
// [num_pages, Hkv, page, D], scales [num_pages, Hkv, page / block].
class KvCacheAppendFp8PagedOp {
public:
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;
};

// {q[B,Hq,1,D], k_cache, v_cache, k_scale, v_scale, lengths[B] int32} -> {O[B,Hq,1,D], LSE[B,Hq]}
class SdpaDecodeFp8Op {
public:
    explicit SdpaDecodeFp8Op(SdpaDecodeFp8Param param) : mParam(std::move(param)) {}
    const SdpaDecodeFp8Param& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    SdpaDecodeFp8Param mParam;
};

// {q, k_pages, v_pages, k_scale, v_scale, block_table[B,max_pages] int32, lengths} -> {O, LSE}
class SdpaDecodeFp8PagedOp {
public:
    explicit SdpaDecodeFp8PagedOp(SdpaDecodeFp8PagedParam param) : mParam(std::move(param)) {}
    const SdpaDecodeFp8PagedParam& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    SdpaDecodeFp8PagedParam mParam;
};

// {weights[B,Hkv,S] fp32, q[B,Hq,L,D], k[B,Hkv,S,D], lse[B,Hq,L] or [B,Hq], lengths?, k_scale?} -> {weights}, in place.
class AttentionWeightsOp {
public:
    explicit AttentionWeightsOp(AttentionWeightsParam param) : mParam(std::move(param)) {}
    const AttentionWeightsParam& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    AttentionWeightsParam mParam;
};

// {k_cache, v_cache, lengths, weights, k_scale?, v_scale?} -> {kept[B,Hkv,keep/block] int32}; the inputs are updated in place.
class KvCacheEvictOp {
public:
    explicit KvCacheEvictOp(KvCacheEvictParam param) : mParam(std::move(param)) {}
    const KvCacheEvictParam& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    KvCacheEvictParam mParam;
};

}  // namespace core
}  // namespace dtorch_amd
