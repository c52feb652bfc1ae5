// Host operators over the 8-bit KV cache and the bounded one (see cache_ops.h): validation, outputs and workspaces from the
// c10 caching allocator, and launches on the thread's current stream, as in sdpa_op.cc.
#include "cache_ops.h"

#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <cmath>
#include <cstring>

#include "op_common.h"

namespace dtorch_amd {
namespace core {

namespace {

float ScaleOf(const std::optional<double>& scale) {
    if (scale.has_value() && !std::isfinite(scale.value())) Throw("scale must be finite");
    return scale.has_value() ? (float)scale.value() : std::nanf("");  // NaN: 1/sqrt(D)
}

// A tensor written in place holds each element once.
void CheckNotExpanded(const at::Tensor& t, const char* name) {
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) == 0) Throw(std::string(name) + " is updated in place and must not be expanded");
}

// Codes and scales: [slots, Hkv, rows, D] and [slots, Hkv, rows / block]; the block comes from the two row counts.
int32_t CheckFp8Cache(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs) {
    CheckCacheLayout(kc, "the key codes");
    CheckCacheLayout(vc, "the value codes");
    if (kc.sizes() != vc.sizes()) Throw("key and value code shapes differ");
    if (kc.scalar_type() != at::kFloat8_e4m3fn || vc.scalar_type() != at::kFloat8_e4m3fn)
        Throw("the codes of an 8-bit cache are float8_e4m3fn");
    if (ks.dim() != 3 || ks.sizes() != vs.sizes() || ks.scalar_type() != at::kFloat || vs.scalar_type() != at::kFloat)
        Throw("k_scale and v_scale must be fp32 tensors of the same shape [batch or pages, Hkv, blocks]");
    if (ks.size(0) != kc.size(0) || ks.size(1) != kc.size(1)) Throw("code and scale shapes do not match");
    if (ks.size(2) <= 0 || kc.size(2) % ks.size(2) != 0) Throw("the rows of a cache must be a whole number of blocks, one scale each");
    for (const at::Tensor* t : {&ks, &vs})
        if (t->size(2) > 1 && t->stride(2) != 1) Throw("scales need a unit stride between blocks");
    return (int32_t)std::min<int64_t>(kc.size(2) / ks.size(2), 1 << 30);
}

// The fields that dtattn_kv_append_fp8_args and dtattn_decode_fp8_args share.
template <typename Args>
void FillCache(Args& a, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs, const at::Tensor* table) {
    a.k_cache = kc.data_ptr(), a.v_cache = vc.data_ptr();
    a.k_scale = ks.data_ptr<float>(), a.v_scale = vs.data_ptr<float>();
    a.Hkv = kc.size(1), a.D = kc.size(3);
    for (int i = 0; i < 3; ++i) a.k_stride[i] = kc.stride(i), a.v_stride[i] = vc.stride(i);
    for (int i = 0; i < 2; ++i) a.k_scale_stride[i] = ks.stride(i), a.v_scale_stride[i] = vs.stride(i);
    if (table != nullptr) {
        a.block_table = table->data_ptr<int32_t>();
        a.block_table_stride = table->stride(0);
        a.num_pages = kc.size(0), a.page_size = kc.size(2), a.max_pages = table->size(1);
    } else {
        a.S_max = kc.size(2);
    }
}

at::Tensor CheckTable(const at::Tensor& bt, int64_t B) {
    if (bt.scalar_type() != at::kInt || bt.dim() != 2 || bt.size(0) != B) Throw("block_table must be an int32 tensor of shape [B, max_pages]");
    if (bt.size(1) == 0) Throw("block_table has no pages");
    return bt.stride(1) == 1 ? bt : bt.contiguous();
}

void AppendFp8(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs, const at::Tensor* bt,
               const at::Tensor& len, const at::Tensor& kn, const at::Tensor& vn, TorchTensorArray& outputs) {
    c10::DeviceGuard guard(kc.device());
    const int32_t block = CheckFp8Cache(kc, vc, ks, vs);
    for (const at::Tensor* t : {&kc, &vc, &ks, &vs}) CheckNotExpanded(*t, "an 8-bit cache");
    const int64_t B = len.dim() == 1 ? len.size(0) : -1;
    CheckLengths(len, B);
    if (bt == nullptr && kc.size(0) != B) Throw("lengths must have one entry per sequence of the cache");
    if (kn.dim() != 4 || vn.dim() != 4 || kn.sizes() != vn.sizes())
        Throw("k_new and v_new must be 4-D tensors of the same shape [B, Hkv, n_new, D]");
    if (kn.size(0) != B || kn.size(1) != kc.size(1) || kn.size(3) != kc.size(3)) Throw("k_new must be [B, Hkv, n_new, D] matching the cache");
    const c10::ScalarType st = kn.scalar_type();
    if (vn.scalar_type() != st || (st != at::kBFloat16 && st != at::kHalf && st != at::kFloat))
        Throw("new tokens must both be bf16, fp16 or fp32");
    const at::Tensor table = bt != nullptr ? CheckTable(*bt, B) : at::Tensor();
    View4 k = MakeView4(kn, "k_new"), v = MakeView4(vn, "v_new");
    dtattn_kv_append_fp8_args a;
    std::memset(&a, 0, sizeof(a));
    FillCache(a, kc, vc, ks, vs, bt != nullptr ? &table : nullptr);
    a.k_new = k.t.data_ptr(), a.v_new = v.t.data_ptr();
    a.k_new_stride[0] = k.sb, a.k_new_stride[1] = k.sh, a.k_new_stride[2] = k.ss;
    a.v_new_stride[0] = v.sb, a.v_new_stride[1] = v.sh, a.v_new_stride[2] = v.ss;
    a.lengths = len.data_ptr<int32_t>();
    a.B = B, a.n_new = kn.size(2);
    a.block = block;
    a.dtype = DtypeCode(st);
    Check(dtattn_kv_append_fp8(&a, CurrentStream(kc)), "dtattn_kv_append_fp8");
    for (const at::Tensor* t : {&kc, &vc, &ks, &vs, &len}) outputs.push_back(*t);
}

void DecodeFp8(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
               const at::Tensor* bt, const at::Tensor& len, const std::optional<double>& scale, TorchTensorArray& outputs) {
    c10::DeviceGuard guard(q.device());
    const int32_t block = CheckFp8Cache(kc, vc, ks, vs);
    if (q.dim() != 4 || q.size(2) != 1) Throw("decode query must have one token per sequence ([B, Hq, 1, D])");
    const int64_t B = q.size(0);
    if (bt == nullptr && kc.size(0) != B) Throw("query and cache batch sizes differ");
    if (q.size(3) != kc.size(3)) Throw("query and cache head dims differ");
    if (kc.size(1) <= 0 || q.size(1) % kc.size(1) != 0) Throw("number of query heads must be a multiple of kv heads");
    if (len.scalar_type() != at::kInt || len.dim() != 1 || len.size(0) != B) Throw("lengths must be an int32 tensor of shape [B]");
    const c10::ScalarType st = q.scalar_type();
    if (st != at::kBFloat16 && st != at::kHalf && st != at::kFloat) Throw("decode supports bf16, fp16 and fp32 queries");
    const float s = ScaleOf(scale);
    const at::Tensor table = bt != nullptr ? CheckTable(*bt, B) : at::Tensor();
    at::Tensor o = at::empty(q.sizes(), q.options());
    at::Tensor lse = at::empty({B, q.size(1)}, q.options().dtype(at::kFloat));
    if (o.numel() > 0) {
        View4 qv = MakeView4(q, "query");
        at::Tensor lc = len.contiguous();
        dtattn_decode_fp8_args a;
        std::memset(&a, 0, sizeof(a));
        FillCache(a, kc, vc, ks, vs, bt != nullptr ? &table : nullptr);
        a.q = qv.t.data_ptr(), a.o = o.data_ptr(), a.lse = lse.data_ptr<float>();
        a.lengths = lc.data_ptr<int32_t>();
        a.B = B, a.Hq = q.size(1);
        a.q_stride[0] = qv.sb, a.q_stride[1] = qv.sh;
        a.o_stride[0] = q.size(1) * q.size(3), a.o_stride[1] = q.size(3);
        a.lse_stride[0] = q.size(1);
        a.block = block;
        a.dtype = DtypeCode(st);
        a.scale = s;
        void* stream = CurrentStream(q);
        const size_t ws = dtattn_decode_fp8_workspace_size(&a, stream);
        at::Tensor wst = at::empty({(int64_t)std::max<size_t>(ws, 1)}, q.options().dtype(at::kByte));
        a.workspace = wst.data_ptr();
        a.workspace_bytes = ws;
        Check(dtattn_decode_fp8(&a, stream), "dtattn_decode_fp8");
    }
    outputs.push_back(o);
    outputs.push_back(lse);
}

const at::Tensor* Optional(const TorchTensorOptArray& inputs, size_t i) {
    return inputs[i].has_value() && inputs[i]->defined() ? &*inputs[i] : nullptr;
}

void CheckAll(const TorchTensorOptArray& inputs, size_t required, size_t total, const char* what) {
    if (inputs.size() != total) Throw(what);
    std::vector<const at::Tensor*> ts;
    for (size_t i = 0; i < total; ++i) {
        const at::Tensor* t = Optional(inputs, i);
        if (t == nullptr && i < required) Throw(what);
        if (t != nullptr) ts.push_back(t);
    }
    CheckDevice(ts);
}

}  // namespace

void KvCacheAppendFp8Op::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    CheckAll(in, 7, 7, "KvCacheAppendFp8Op expects 7 inputs {k_cache, v_cache, k_scale, v_scale, lengths, k_new, v_new}");
    AppendFp8(*in[0], *in[1], *in[2], *in[3], nullptr, *in[4], *in[5], *in[6], outputs);
}

void KvCacheAppendFp8PagedOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    CheckAll(in, 8, 8, "KvCacheAppendFp8PagedOp expects 8 inputs {k_pages, v_pages, k_scale, v_scale, block_table, lengths, k_new, v_new}");
    AppendFp8(*in[0], *in[1], *in[2], *in[3], &*in[4], *in[5], *in[6], *in[7], outputs);
}

void SdpaDecodeFp8Op::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    CheckAll(in, 6, 6, "SdpaDecodeFp8Op expects 6 inputs {query, k_cache, v_cache, k_scale, v_scale, lengths}");
    DecodeFp8(*in[0], *in[1], *in[2], *in[3], *in[4], nullptr, *in[5], mParam.scale, outputs);
}

void SdpaDecodeFp8PagedOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    CheckAll(in, 7, 7, "SdpaDecodeFp8PagedOp expects 7 inputs {query, k_pages, v_pages, k_scale, v_scale, block_table, lengths}");
    DecodeFp8(*in[0], *in[1], *in[2], *in[3], *in[4], &*in[5], *in[6], mParam.scale, outputs);
}

void AttentionWeightsOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    CheckAll(in, 4, 6, "AttentionWeightsOp expects {weights, query, key, lse, lengths or none, key_scale or none}");
    const at::Tensor &w = *in[0], &q = *in[1], &k = *in[2], &lse_ = *in[3];
    const at::Tensor *len = Optional(in, 4), *ks = Optional(in, 5);
    c10::DeviceGuard guard(w.device());
    if (q.dim() != 4 || k.dim() != 4) Throw("query and key must be 4-D [B, H, tokens, D]");
    const int64_t B = q.size(0), Hq = q.size(1), L = q.size(2), Hkv = k.size(1), S = k.size(2);
    if (k.size(0) != B || k.size(3) != q.size(3)) Throw("query and key shapes do not match");
    if (Hkv <= 0 || Hq % Hkv != 0) Throw("number of query heads must be a multiple of key heads");
    if (w.scalar_type() != at::kFloat || w.dim() != 3 || w.size(0) != B || w.size(1) != Hkv || w.size(2) != S)
        Throw("weights must be an fp32 tensor of shape [B, Hkv, S]");
    if (w.size(2) > 1 && w.stride(2) != 1) Throw("weights need a unit stride along the keys (they are updated in place)");
    CheckNotExpanded(w, "weights");
    const bool flat = lse_.dim() == 2 && L == 1;
    if (lse_.scalar_type() != at::kFloat || !(flat || lse_.dim() == 3) || lse_.size(0) != B || lse_.size(1) != Hq || (!flat && lse_.size(2) != L))
        Throw("lse must be an fp32 tensor of shape [B, Hq, L], or [B, Hq] for one query");
    at::Tensor lse = flat ? lse_.unsqueeze(2) : lse_;
    if (L > 1 && lse.stride(2) != 1) lse = lse.contiguous();
    if (len != nullptr && (len->scalar_type() != at::kInt || len->dim() != 1 || len->size(0) != B))
        Throw("lengths must be an int32 tensor of shape [B]");
    const c10::ScalarType st = q.scalar_type();
    if (st != at::kBFloat16 && st != at::kHalf && st != at::kFloat) Throw("queries must be bf16, fp16 or fp32");
    const bool codes = k.scalar_type() == at::kFloat8_e4m3fn;
    if (!codes && k.scalar_type() != st) Throw("keys must have the query's dtype, or be float8_e4m3fn codes");
    if (codes != (ks != nullptr)) Throw("float8_e4m3fn keys, and only they, take key_scale");
    const float s = ScaleOf(mParam.scale);
    dtattn_weights_args a;
    std::memset(&a, 0, sizeof(a));
    if (codes) {
        if (ks->scalar_type() != at::kFloat || ks->dim() != 3 || ks->size(0) != B || ks->size(1) != Hkv || ks->size(2) <= 0 || S % ks->size(2) != 0)
            Throw("key_scale must be an fp32 tensor of shape [B, Hkv, S / block]");
        if (ks->size(2) > 1 && ks->stride(2) != 1) Throw("key_scale needs a unit stride between blocks");
        a.k_scale = ks->data_ptr<float>();
        a.k_scale_stride[0] = ks->stride(0), a.k_scale_stride[1] = ks->stride(1);
        a.block = (int32_t)std::min<int64_t>(S / ks->size(2), 1 << 30);
    }
    View4 qv = MakeView4(q, "query"), kv = MakeView4(k, "key");
    at::Tensor lc = len != nullptr ? len->contiguous() : at::Tensor();
    a.weights = w.data_ptr<float>();
    a.q = qv.t.data_ptr(), a.k = kv.t.data_ptr();
    a.lse = lse.data_ptr<float>();
    a.lengths = len != nullptr ? lc.data_ptr<int32_t>() : nullptr;
    a.B = B, a.Hq = Hq, a.Hkv = Hkv, a.L = L, a.S = S, a.D = q.size(3);
    a.w_stride[0] = w.stride(0), a.w_stride[1] = w.stride(1);
    a.q_stride[0] = qv.sb, a.q_stride[1] = qv.sh, a.q_stride[2] = qv.ss;
    a.k_stride[0] = kv.sb, a.k_stride[1] = kv.sh, a.k_stride[2] = kv.ss;
    a.lse_stride[0] = lse.stride(0), a.lse_stride[1] = lse.stride(1);
    a.q_offset = mParam.qOffset;
    a.causal = mParam.isCausal ? 1 : 0;
    a.q_dtype = DtypeCode(st);
    a.k_dtype = DtypeCode(k.scalar_type());
    a.scale = s;
    void* stream = CurrentStream(w);
    const size_t ws = dtattn_attention_weights_workspace_size(&a, stream);
    at::Tensor wst;
    if (ws > 0) {
        wst = at::empty({(int64_t)ws}, w.options().dtype(at::kByte));
        a.workspace = wst.data_ptr();
        a.workspace_bytes = ws;
    }
    Check(dtattn_attention_weights(&a, stream), "dtattn_attention_weights");
    outputs.push_back(w);
}

void KvCacheEvictOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    CheckAll(in, 4, 6, "KvCacheEvictOp expects {k_cache, v_cache, lengths, weights, k_scale or none, v_scale or none}");
    const at::Tensor &kc = *in[0], &vc = *in[1], &len = *in[2], &w = *in[3];
    const at::Tensor *ks = Optional(in, 4), *vs = Optional(in, 5);
    c10::DeviceGuard guard(kc.device());
    if ((ks != nullptr) != (vs != nullptr)) Throw("k_scale and v_scale go together");
    const bool codes = ks != nullptr;
    int64_t scaleBlock = 1;
    if (codes) {
        scaleBlock = CheckFp8Cache(kc, vc, *ks, *vs);
        CheckNotExpanded(*ks, "k_scale");
        CheckNotExpanded(*vs, "v_scale");
    } else {
        CheckCacheLayout(kc, "k_cache");
        CheckCacheLayout(vc, "v_cache");
        if (kc.sizes() != vc.sizes() || kc.scalar_type() != vc.scalar_type()) Throw("k_cache and v_cache differ in shape or dtype");
        const c10::ScalarType st = kc.scalar_type();
        if (st != at::kBFloat16 && st != at::kHalf && st != at::kFloat)
            Throw("the KV cache must be bf16, fp16 or fp32, or float8_e4m3fn with k_scale and v_scale");
    }
    CheckNotExpanded(kc, "k_cache");
    CheckNotExpanded(vc, "v_cache");
    const int64_t B = kc.size(0), Hkv = kc.size(1), S = kc.size(2);
    CheckLengths(len, B);
    if (w.scalar_type() != at::kFloat || w.dim() != 3 || w.size(0) != B || w.size(1) != Hkv || w.size(2) != S)
        Throw("weights must be an fp32 tensor of shape [B, Hkv, S_max]");
    if (w.size(2) > 1 && w.stride(2) != 1) Throw("weights need a unit stride along the tokens (they are updated in place)");
    CheckNotExpanded(w, "weights");
    if (mParam.block < 0) Throw("block must not be negative");
    const int64_t block = mParam.block > 0 ? mParam.block : scaleBlock;
    dtattn_kv_evict_args a;
    std::memset(&a, 0, sizeof(a));
    a.B = B, a.Hkv = Hkv, a.S_max = S;
    a.keep = mParam.keep, a.recent = mParam.recent, a.block = block, a.scale_block = scaleBlock;
    a.row_bytes = kc.size(3) * kc.element_size();
    a.k_cache = kc.data_ptr(), a.v_cache = vc.data_ptr();
    for (int i = 0; i < 3; ++i) a.k_stride[i] = kc.stride(i) * kc.element_size(), a.v_stride[i] = vc.stride(i) * vc.element_size();
    if (codes) {
        a.k_scale = ks->data_ptr<float>(), a.v_scale = vs->data_ptr<float>();
        for (int i = 0; i < 2; ++i) a.k_scale_stride[i] = ks->stride(i), a.v_scale_stride[i] = vs->stride(i);
    }
    a.weights = w.data_ptr<float>();
    a.w_stride[0] = w.stride(0), a.w_stride[1] = w.stride(1);
    a.lengths = len.data_ptr<int32_t>();
    if (block < 1 || mParam.keep < 1 || mParam.keep % block != 0 || mParam.keep > (int64_t)1 << 29)
        Throw("keep must be a positive multiple of the block of " + std::to_string(block) + " tokens");
    at::Tensor kept = at::empty({B, Hkv, mParam.keep / block}, len.options());
    const size_t ws = dtattn_kv_evict_workspace_size(&a);
    at::Tensor wst = at::empty({(int64_t)std::max<size_t>(ws, 1)}, len.options().dtype(at::kByte));
    a.workspace = wst.data_ptr();
    a.workspace_bytes = ws;
    a.kept = kept.data_ptr<int32_t>();
    Check(dtattn_kv_evict(&a, CurrentStream(kc)), "dtattn_kv_evict");
    outputs.push_back(kept);
}

}  // namespace core
}  // namespace dtorch_amd
