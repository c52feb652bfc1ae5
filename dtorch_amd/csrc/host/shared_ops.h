// Host operators over a KV cache whose pages are shared and which is read in part (dtattn.h, "pages that sequences share",
// "attention over a shared prefix" and "attention over selected key blocks").
//
// New operators without a reference counterpart: the reference keeps no KV cache
// (python/dtorch/test/modules/llama.py:126-156).  They follow the operator contract of sdpa_op.h.
#pragma once

#include "cache_ops.h"

namespace dtorch_amd {
namespace core {

struct KvPagesForkParam : KvCacheAppendParam {};
struct KvPagesCompactParam : KvCacheAppendParam {};

// KvPagesReserve and KeyBounds: how many tokens.
struct TokenCountParam {
    int64_t tokens = 1;

    TokenCountParam() = default;
    explicit TokenCountParam(int64_t tokens_) : tokens(tokens_) {}

    template <class Archive>
    void serialize(Archive& ar, const unsigned int /*version*/) {
        ar & tokens;
    }
};

// SdpaDecodeShared / SdpaDecodeSharedPaged: softmax scale (none: 1/sqrt(D)).
struct SdpaDecodeSharedParam : SdpaDecodeFp8Param {
    using SdpaDecodeFp8Param::SdpaDecodeFp8Param;
    SdpaDecodeSharedParam() = default;
};

// SelectKeyBlocks: tokens of the selected blocks, how many of them are the last ones, tokens of a block, and the softmax scale.
struct SelectKeyBlocksParam {
    int64_t keep = 16;
    int64_t recent = 16;
    int64_t block = 16;
    std::optional<double> scale = std::nullopt;

    SelectKeyBlocksParam() = default;
    SelectKeyBlocksParam(int64_t keep_, int64_t recent_, int64_t block_, std::optional<double> scale_)
        : keep(keep_), recent(recent_), block(block_), scale(scale_) {}

    template <class Archive>
    void serialize(Archive& ar, const unsigned int /*version*/) {
        ar & keep;
        ar & recent;
        ar & block;
        ar & scale;
    }
};

// SdpaDecodeBlocks: tokens of a block and the softmax scale.
struct SdpaDecodeBlocksParam {
    int64_t block = 16;
    std::optional<double> scale = std::nullopt;

    SdpaDecodeBlocksParam() = default;
    SdpaDecodeBlocksParam(int64_t block_, std::optional<double> scale_) : block(block_), scale(scale_) {}

    template <class Archive>
    void serialize(Archive& ar, const unsigned int /*version*/) {
        ar & block;
        ar & scale;
    }
};

// {block_table[B,max_pages], lengths[B], page_refs[num_pages], parents[B]}, all int32 -> {block_table, lengths, page_refs}, in place.
class KvPagesForkOp {
public:
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;
};

// {block_table, lengths, page_refs, pool...} -> {short[1] int32}; the first pool is [num_pages, Hkv, page_size, D], the others hold rows
// per token or per block of tokens.  The table, the counts and the pools are updated in place.
class KvPagesReserveOp {
public:
    explicit KvPagesReserveOp(TokenCountParam param) : mParam(std::move(param)) {}
    const TokenCountParam& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    TokenCountParam mParam;
};

// {block_table, page_refs, pool...} -> {used[1] int32}, the inputs in place.
class KvPagesCompactOp {
public:
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;
};

// {q[B,Hq,1,D], k_prefix[G,Hkv,S,D], v_prefix, prefix_lengths[G], k_cache[B,Hkv,S_max,D], v_cache, lengths[B]} -> {O, LSE[B,Hq]}
class SdpaDecodeSharedOp {
public:
    explicit SdpaDecodeSharedOp(SdpaDecodeSharedParam param) : mParam(std::move(param)) {}
    const SdpaDecodeSharedParam& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    SdpaDecodeSharedParam mParam;
};

// {q, k_pages, v_pages, block_table[B,max_pages], lengths[B], prefix_lengths[G]} -> {O, LSE}
class SdpaDecodeSharedPagedOp {
public:
    explicit SdpaDecodeSharedPagedOp(SdpaDecodeSharedParam param) : mParam(std::move(param)) {}
    const SdpaDecodeSharedParam& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    SdpaDecodeSharedParam mParam;
};

// {k_cache or k_pages, k_min, k_max, lengths, block_table?} -> {k_min, k_max}, in place.
class KeyBoundsOp {
public:
    explicit KeyBoundsOp(TokenCountParam param) : mParam(std::move(param)) {}
    const TokenCountParam& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    TokenCountParam mParam;
};

// {q, k_min, k_max, lengths, block_table?} -> {blocks[B,Hkv,keep/block] int32}
class SelectKeyBlocksOp {
public:
    explicit SelectKeyBlocksOp(SelectKeyBlocksParam param) : mParam(std::move(param)) {}
    const SelectKeyBlocksParam& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    SelectKeyBlocksParam mParam;
};

// {q, k_cache or k_pages, v_cache or v_pages, lengths, blocks[B,Hkv,n] int32, block_table?} -> {O, LSE}
class SdpaDecodeBlocksOp {
public:
    explicit SdpaDecodeBlocksOp(SdpaDecodeBlocksParam param) : mParam(std::move(param)) {}
    const SdpaDecodeBlocksParam& Param() const { return mParam; }
    void Compute(const TorchTensorOptArray& inputs, TorchTensorArray& outputs) const;

private:
    SdpaDecodeBlocksParam mParam;
};

}  // namespace core
}  // namespace dtorch_amd
