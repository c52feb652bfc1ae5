// Host operators over shared pages, a shared prefix and selected key blocks (see shared_ops.h): validation, outputs and workspaces from
// the c10 caching allocator, and launches on the thread's current stream, as in sdpa_op.cc.
#include "shared_ops.h"

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

// All inputs on one device; those from `required` on may be missing.
std::vector<const at::Tensor*> Inputs(const TorchTensorOptArray& inputs, size_t required, size_t total, const char* what) {
    if (inputs.size() < required || inputs.size() > total) Throw(what);
    std::vector<const at::Tensor*> all, there;
    for (size_t i = 0; i < inputs.size(); ++i) {
        const at::Tensor* t = inputs[i].has_value() && inputs[i]->defined() ? &*inputs[i] : nullptr;
        if (t == nullptr && i < required) Throw(what);
        if (t != nullptr) there.push_back(t);
        all.push_back(t);
    }
    all.resize(total, nullptr);
    CheckDevice(there);
    return all;
}

// A tensor written in place holds each element once.
void CheckOnce(const at::Tensor& t, const char* name) {
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) == 0) Throw(std::string(name) + " is updated in place and must not be expanded");
}

// A table that is updated where it lies.
void CheckTableInPlace(const at::Tensor& bt) {
    if (bt.scalar_type() != at::kInt || bt.dim() != 2) Throw("block_table must be an int32 tensor of shape [B, max_pages]");
    if (bt.size(1) == 0) Throw("block_table has no pages");
    if (bt.size(1) > 1 && bt.stride(1) != 1) Throw("block_table needs a unit stride along the pages (it is updated in place)");
    CheckOnce(bt, "block_table");
}

int64_t TableStride(const at::Tensor& bt) { return bt.size(0) > 1 ? bt.stride(0) : bt.size(1); }

// A table that is read.
at::Tensor ReadTable(const at::Tensor& bt, int64_t B) {
    if (bt.scalar_type() != at::kInt || bt.dim() != 2 || bt.size(0) != B) Throw("block_table must be an int32 tensor of shape [B, max_pages]");
    if (bt.size(1) == 0) Throw("block_table has no pages");
    return bt.size(1) == 1 || bt.stride(1) == 1 ? bt : bt.contiguous();
}

int64_t CheckRefs(const at::Tensor& refs) {
    if (refs.scalar_type() != at::kInt || refs.dim() != 1 || refs.size(0) == 0 || !refs.is_contiguous())
        Throw("page_refs must be a contiguous int32 tensor of shape [num_pages] (it is updated in place)");
    return refs.size(0);
}

at::Tensor Whole(const at::Tensor& t, int64_t n, const char* name) {
    if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n)
        Throw(std::string(name) + " must be an int32 tensor of shape [" + std::to_string(n) + "]");
    return t.contiguous();
}

bool FloatType(c10::ScalarType st) { return st == at::kBFloat16 || st == at::kHalf || st == at::kFloat; }

// Pools of pages: the first one [num_pages, heads, page_size, D]; the others [num_pages, heads, rows] or [num_pages, heads, rows, D].
int64_t FillPools(dtattn_page_pool* pools, int32_t& n, const std::vector<const at::Tensor*>& ts, size_t first, int64_t numPages) {
    n = 0;
    int64_t pageSize = 0;
    for (size_t i = first; i < ts.size(); ++i) {
        if (ts[i] == nullptr) continue;
        const at::Tensor& t = *ts[i];
        if (n >= DTATTN_MAX_PAGE_POOLS) Throw("too many pools of pages");
        if (n == 0 && t.dim() != 4) Throw("the first pool must be [num_pages, Hkv, page_size, D]");
        if ((t.dim() != 3 && t.dim() != 4) || t.size(0) != numPages || t.numel() == 0)
            Throw("pools must be [num_pages, Hkv, rows, D] or [num_pages, Hkv, rows], with as many pages as page_refs");
        if (n == 0) pageSize = t.size(2);
        if (pageSize % t.size(2) != 0) Throw("the rows of a pool must divide the tokens of a page");
        if (t.dim() == 4 && t.size(3) > 1 && t.stride(3) != 1) Throw("pools need a unit stride along D");
        CheckOnce(t, "a pool of pages");
        const int64_t esz = t.element_size();
        dtattn_page_pool& p = pools[n++];
        p.data = t.data_ptr();
        p.heads = t.size(1);
        p.row_bytes = (t.dim() == 4 ? t.size(3) : 1) * esz;
        p.row_tokens = pageSize / t.size(2);
        p.row_stride = t.size(2) > 1 ? t.stride(2) * esz : p.row_bytes;
        p.head_stride = t.size(1) > 1 ? t.stride(1) * esz : p.row_stride * t.size(2);
        p.page_stride = t.size(0) > 1 ? t.stride(0) * esz : p.head_stride * t.size(1);
    }
    if (n == 0) Throw("no pool of pages");
    return pageSize;
}

// The caches, or pools of pages, of a decode: k and v alike.
void CheckCaches(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const char* what) {
    CheckCacheLayout(k, (std::string("k_") + what).c_str());
    CheckCacheLayout(v, (std::string("v_") + what).c_str());
    if (k.sizes() != v.sizes()) Throw(std::string("k_") + what + " and v_" + what + " differ in shape");
    if (!FloatType(q.scalar_type()) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
        Throw("query and caches must be of one dtype: bf16, fp16 or fp32");
    if (q.size(3) != k.size(3)) Throw("query and cache head dims differ");
    if (k.size(1) <= 0 || q.size(1) % k.size(1) != 0) Throw("number of query heads must be a multiple of kv heads");
}

void CheckQuery(const at::Tensor& q) {
    if (q.dim() != 4 || q.size(2) != 1) Throw("decode query must have one token per sequence ([B, Hq, 1, D])");
}

// Strides of an axis of one element are free: the natural ones keep them multiples of 16 bytes.
void Strides(const at::Tensor& t, int64_t out[3]) {
    out[2] = t.size(2) > 1 ? t.stride(2) : t.size(3);
    out[1] = t.size(1) > 1 ? t.stride(1) : out[2] * t.size(2);
    out[0] = t.size(0) > 1 ? t.stride(0) : out[1] * t.size(1);
}

template <typename Args>
void FillQuery(Args& a, const View4& qv, at::Tensor& o, at::Tensor& lse, c10::ScalarType st, float scale) {
    a.q = qv.t.data_ptr(), a.o = o.data_ptr(), a.lse = lse.data_ptr<float>();
    a.q_stride[0] = qv.sb, a.q_stride[1] = qv.sh;
    a.o_stride[0] = o.size(1) * o.size(3), a.o_stride[1] = o.size(3);
    a.lse_stride[0] = o.size(1);
    a.dtype = DtypeCode(st);
    a.scale = scale;
}

template <typename Args>
void FillCaches(Args& a, const at::Tensor& k, const at::Tensor& v, const at::Tensor* table) {
    a.k_cache = k.data_ptr(), a.v_cache = v.data_ptr();
    a.Hkv = k.size(1), a.D = k.size(3);
    Strides(k, a.k_stride);
    Strides(v, a.v_stride);
    if (table != nullptr) {
        a.block_table = table->data_ptr<int32_t>();
        a.block_table_stride = TableStride(*table);
        a.num_pages = k.size(0), a.page_size = k.size(2), a.max_pages = table->size(1);
    } else {
        a.S_max = k.size(2);
    }
}

at::Tensor Bytes(size_t n, const at::Tensor& like) { return at::empty({(int64_t)std::max<size_t>(n, 1)}, like.options().dtype(at::kByte)); }

// Bounds [slots, Hkv, blocks, D] that go with keys or queries of dtype `st`.
void CheckBounds(const at::Tensor& lo, const at::Tensor& hi, c10::ScalarType st) {
    CheckCacheLayout(lo, "k_min");
    CheckCacheLayout(hi, "k_max");
    if (lo.sizes() != hi.sizes()) Throw("k_min and k_max differ in shape");
    if (!FloatType(st) || lo.scalar_type() != st || hi.scalar_type() != st) Throw("keys, queries and bounds must be of one dtype: bf16, fp16 or fp32");
    if (lo.size(2) <= 0) Throw("the bounds have no blocks");
}

}  // namespace

void KvPagesForkOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    const auto t = Inputs(in, 4, 4, "KvPagesForkOp expects 4 inputs {block_table, lengths, page_refs, parents}");
    const at::Tensor &bt = *t[0], &len = *t[1], &refs = *t[2];
    c10::DeviceGuard guard(bt.device());
    CheckTableInPlace(bt);
    const int64_t B = bt.size(0);
    CheckLengths(len, B);
    const at::Tensor parents = Whole(*t[3], B, "parents");
    dtattn_kv_fork_args a;
    std::memset(&a, 0, sizeof(a));
    a.num_pages = CheckRefs(refs);
    a.block_table = bt.data_ptr<int32_t>(), a.lengths = len.data_ptr<int32_t>(), a.page_refs = refs.data_ptr<int32_t>();
    a.parents = parents.data_ptr<int32_t>();
    a.B = B, a.max_pages = bt.size(1), a.block_table_stride = TableStride(bt);
    Check(dtattn_kv_pages_fork(&a, CurrentStream(bt)), "dtattn_kv_pages_fork");
    for (const at::Tensor* x : {&bt, &len, &refs}) outputs.push_back(*x);
}

void KvPagesReserveOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    const auto t = Inputs(in, 4, 3 + DTATTN_MAX_PAGE_POOLS, "KvPagesReserveOp expects {block_table, lengths, page_refs, pools of pages}");
    const at::Tensor &bt = *t[0], &len = *t[1], &refs = *t[2];
    c10::DeviceGuard guard(bt.device());
    CheckTableInPlace(bt);
    const int64_t B = bt.size(0);
    const at::Tensor lengths = Whole(len, B, "lengths");
    if (mParam.tokens < 0) Throw("the number of new tokens must not be negative");
    dtattn_kv_reserve_args a;
    std::memset(&a, 0, sizeof(a));
    a.num_pages = CheckRefs(refs);
    a.page_size = FillPools(a.pools, a.n_pools, t, 3, a.num_pages);
    a.block_table = bt.data_ptr<int32_t>(), a.lengths = lengths.data_ptr<int32_t>(), a.page_refs = refs.data_ptr<int32_t>();
    a.B = B, a.max_pages = bt.size(1), a.block_table_stride = TableStride(bt);
    a.n_new = mParam.tokens;
    at::Tensor shortBy = at::empty({1}, len.options());
    a.short_by = shortBy.data_ptr<int32_t>();
    const size_t ws = dtattn_kv_pages_reserve_workspace_size(&a);
    at::Tensor wst = Bytes(ws, bt);
    a.workspace = wst.data_ptr();
    a.workspace_bytes = ws;
    Check(dtattn_kv_pages_reserve(&a, CurrentStream(bt)), "dtattn_kv_pages_reserve");
    outputs.push_back(shortBy);
}

void KvPagesCompactOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    const auto t = Inputs(in, 3, 2 + DTATTN_MAX_PAGE_POOLS, "KvPagesCompactOp expects {block_table, page_refs, pools of pages}");
    const at::Tensor &bt = *t[0], &refs = *t[1];
    c10::DeviceGuard guard(bt.device());
    CheckTableInPlace(bt);
    dtattn_kv_compact_args a;
    std::memset(&a, 0, sizeof(a));
    a.num_pages = CheckRefs(refs);
    a.page_size = FillPools(a.pools, a.n_pools, t, 2, a.num_pages);
    a.block_table = bt.data_ptr<int32_t>(), a.page_refs = refs.data_ptr<int32_t>();
    a.B = bt.size(0), a.max_pages = bt.size(1), a.block_table_stride = TableStride(bt);
    at::Tensor used = at::empty({1}, refs.options());
    a.used = used.data_ptr<int32_t>();
    const size_t ws = dtattn_kv_pages_compact_workspace_size(&a);
    at::Tensor wst = Bytes(ws, bt);
    a.workspace = wst.data_ptr();
    a.workspace_bytes = ws;
    Check(dtattn_kv_pages_compact(&a, CurrentStream(bt)), "dtattn_kv_pages_compact");
    outputs.push_back(used);
}

namespace {

// prefix caches: NULL for a paged cache
void DecodeShared(const at::Tensor& q, const at::Tensor* kp, const at::Tensor* vp, const at::Tensor& prefix, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor* bt, const at::Tensor& len, const std::optional<double>& scale, TorchTensorArray& outputs) {
    c10::DeviceGuard guard(q.device());
    CheckQuery(q);
    CheckCaches(q, k, v, bt != nullptr ? "pages" : "cache");
    const int64_t B = q.size(0);
    if (prefix.dim() != 1 || prefix.size(0) <= 0 || B % prefix.size(0) != 0) Throw("prefix_lengths must be [groups], and the sequences as many in each group");
    const int64_t G = prefix.size(0);
    if (bt == nullptr) {
        CheckCaches(q, *kp, *vp, "prefix");
        if (kp->size(0) != G || kp->size(1) != k.size(1)) Throw("k_prefix must be [groups, Hkv, S, D] matching prefix_lengths and the cache");
        if (k.size(0) != B) Throw("query and cache batch sizes differ");
    }
    const at::Tensor pl = Whole(prefix, G, "prefix_lengths"), lc = Whole(len, B, "lengths");
    const at::Tensor table = bt != nullptr ? ReadTable(*bt, B) : at::Tensor();
    const float s = ScaleOf(scale);
    at::Tensor o = at::empty(q.sizes(), q.options());
    at::Tensor lse = at::empty({B, q.size(1)}, q.options().dtype(at::kFloat));
    if (o.numel() > 0) {
        View4 qv = MakeView4(q, "query");
        dtattn_decode_shared_args a;
        std::memset(&a, 0, sizeof(a));
        FillQuery(a, qv, o, lse, q.scalar_type(), s);
        FillCaches(a, k, v, bt != nullptr ? &table : nullptr);
        a.B = B, a.groups = G, a.Hq = q.size(1);
        if (bt == nullptr) {
            a.k_prefix = kp->data_ptr(), a.v_prefix = vp->data_ptr();
            a.S_prefix = kp->size(2);
            Strides(*kp, a.k_prefix_stride);
            Strides(*vp, a.v_prefix_stride);
        }
        a.prefix_lengths = pl.data_ptr<int32_t>(), a.lengths = lc.data_ptr<int32_t>();
        void* stream = CurrentStream(q);
        const size_t ws = dtattn_decode_shared_workspace_size(&a, stream);
        at::Tensor wst = Bytes(ws, q);
        a.workspace = wst.data_ptr();
        a.workspace_bytes = ws;
        Check(dtattn_decode_shared(&a, stream), "dtattn_decode_shared");
    }
    outputs.push_back(o);
    outputs.push_back(lse);
}

}  // namespace

void SdpaDecodeSharedOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    const auto t = Inputs(in, 7, 7, "SdpaDecodeSharedOp expects 7 inputs {query, k_prefix, v_prefix, prefix_lengths, k_cache, v_cache, lengths}");
    DecodeShared(*t[0], t[1], t[2], *t[3], *t[4], *t[5], nullptr, *t[6], mParam.scale, outputs);
}

void SdpaDecodeSharedPagedOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    const auto t = Inputs(in, 6, 6, "SdpaDecodeSharedPagedOp expects 6 inputs {query, k_pages, v_pages, block_table, lengths, prefix_lengths}");
    DecodeShared(*t[0], nullptr, nullptr, *t[5], *t[1], *t[2], t[3], *t[4], mParam.scale, outputs);
}

void KeyBoundsOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    const auto t = Inputs(in, 4, 5, "KeyBoundsOp expects {keys, k_min, k_max, lengths, block_table or none}");
    const at::Tensor &k = *t[0], &lo = *t[1], &hi = *t[2], &len = *t[3];
    const at::Tensor* bt = t[4];
    c10::DeviceGuard guard(k.device());
    CheckCacheLayout(k, "the keys");
    CheckBounds(lo, hi, k.scalar_type());
    CheckOnce(lo, "k_min");
    CheckOnce(hi, "k_max");
    if (lo.size(0) != k.size(0) || lo.size(1) != k.size(1) || lo.size(3) != k.size(3) || k.size(2) % lo.size(2) != 0)
        Throw("bounds must be [batch or pages, Hkv, rows / block, D] of the keys");
    if (mParam.tokens < 0) Throw("the number of new tokens must not be negative");
    const int64_t B = len.dim() == 1 ? len.size(0) : -1;
    const at::Tensor lc = Whole(len, B, "lengths");
    if (bt == nullptr && k.size(0) != B) Throw("lengths must have one entry per sequence of the cache");
    const at::Tensor table = bt != nullptr ? ReadTable(*bt, B) : at::Tensor();
    dtattn_key_bounds_args a;
    std::memset(&a, 0, sizeof(a));
    a.k_cache = k.data_ptr(), a.k_min = lo.data_ptr(), a.k_max = hi.data_ptr();
    a.lengths = lc.data_ptr<int32_t>();
    a.B = B, a.Hkv = k.size(1), a.D = k.size(3), a.n_new = mParam.tokens;
    Strides(k, a.k_stride);
    Strides(lo, a.min_stride);
    Strides(hi, a.max_stride);
    if (bt != nullptr) {
        a.block_table = table.data_ptr<int32_t>(), a.block_table_stride = TableStride(table);
        a.num_pages = k.size(0), a.page_size = k.size(2), a.max_pages = table.size(1);
    } else {
        a.S_max = k.size(2);
    }
    a.block = (int32_t)std::min<int64_t>(k.size(2) / lo.size(2), 1 << 30);
    a.dtype = DtypeCode(k.scalar_type());
    Check(dtattn_key_bounds(&a, CurrentStream(k)), "dtattn_key_bounds");
    outputs.push_back(lo);
    outputs.push_back(hi);
}

void SelectKeyBlocksOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    const auto t = Inputs(in, 4, 5, "SelectKeyBlocksOp expects {query, k_min, k_max, lengths, block_table or none}");
    const at::Tensor &q = *t[0], &lo = *t[1], &hi = *t[2], &len = *t[3];
    const at::Tensor* bt = t[4];
    c10::DeviceGuard guard(q.device());
    CheckQuery(q);
    CheckBounds(lo, hi, q.scalar_type());
    const int64_t B = q.size(0), Hkv = lo.size(1);
    if (q.size(3) != lo.size(3)) Throw("query and bounds head dims differ");
    if (Hkv <= 0 || q.size(1) % Hkv != 0) Throw("number of query heads must be a multiple of kv heads");
    if (bt == nullptr && lo.size(0) != B) Throw("query and bounds batch sizes differ");
    const at::Tensor lc = Whole(len, B, "lengths");
    const at::Tensor table = bt != nullptr ? ReadTable(*bt, B) : at::Tensor();
    const int64_t block = mParam.block;
    if (block < 1 || block > 256 || mParam.keep < 1 || mParam.keep % block != 0 || mParam.keep > (int64_t)1 << 29)
        Throw("keep must be a positive multiple of the block of " + std::to_string(block) + " tokens (at most 256)");
    const float s = ScaleOf(mParam.scale);
    at::Tensor blocks = at::empty({B, Hkv, mParam.keep / block}, len.options());
    if (B > 0) {
        View4 qv = MakeView4(q, "query");
        dtattn_select_blocks_args a;
        std::memset(&a, 0, sizeof(a));
        a.q = qv.t.data_ptr(), a.k_min = lo.data_ptr(), a.k_max = hi.data_ptr();
        a.lengths = lc.data_ptr<int32_t>(), a.blocks = blocks.data_ptr<int32_t>();
        a.B = B, a.Hq = q.size(1), a.Hkv = Hkv, a.D = q.size(3), a.keep = mParam.keep, a.recent = mParam.recent;
        a.q_stride[0] = qv.sb, a.q_stride[1] = qv.sh;
        Strides(lo, a.min_stride);
        Strides(hi, a.max_stride);
        if (bt != nullptr) {
            a.block_table = table.data_ptr<int32_t>(), a.block_table_stride = TableStride(table);
            a.num_pages = lo.size(0), a.page_size = lo.size(2) * block, a.max_pages = table.size(1);
        } else {
            a.S_max = lo.size(2) * block;
        }
        a.block = (int32_t)block;
        a.dtype = DtypeCode(q.scalar_type());
        a.scale = s;
        const size_t ws = dtattn_select_key_blocks_workspace_size(&a);
        at::Tensor wst = Bytes(ws, q);
        a.workspace = wst.data_ptr();
        a.workspace_bytes = ws;
        Check(dtattn_select_key_blocks(&a, CurrentStream(q)), "dtattn_select_key_blocks");
    }
    outputs.push_back(blocks);
}

void SdpaDecodeBlocksOp::Compute(const TorchTensorOptArray& in, TorchTensorArray& outputs) const {
    const auto t = Inputs(in, 5, 6, "SdpaDecodeBlocksOp expects {query, keys, values, lengths, blocks, block_table or none}");
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &len = *t[3], &list = *t[4];
    const at::Tensor* bt = t[5];
    c10::DeviceGuard guard(q.device());
    CheckQuery(q);
    CheckCaches(q, k, v, bt != nullptr ? "pages" : "cache");
    const int64_t B = q.size(0), Hkv = k.size(1);
    if (bt == nullptr && k.size(0) != B) Throw("query and cache batch sizes differ");
    const at::Tensor lc = Whole(len, B, "lengths");
    if (list.scalar_type() != at::kInt || list.dim() != 3 || list.size(0) != B || list.size(1) != Hkv || list.size(2) == 0)
        Throw("blocks must be an int32 tensor of shape [B, Hkv, n]");
    const at::Tensor blocks = list.size(2) == 1 || list.stride(2) == 1 ? list : list.contiguous();
    const at::Tensor table = bt != nullptr ? ReadTable(*bt, B) : at::Tensor();
    const float s = ScaleOf(mParam.scale);
    if (mParam.block < 1 || mParam.block > 256) Throw("the tokens of a block must be a power of two from 16 to 256");
    at::Tensor o = at::empty(q.sizes(), q.options());
    at::Tensor lse = at::empty({B, q.size(1)}, q.options().dtype(at::kFloat));
    if (o.numel() > 0) {
        View4 qv = MakeView4(q, "query");
        dtattn_decode_blocks_args a;
        std::memset(&a, 0, sizeof(a));
        FillQuery(a, qv, o, lse, q.scalar_type(), s);
        FillCaches(a, k, v, bt != nullptr ? &table : nullptr);
        a.B = B, a.Hq = q.size(1);
        a.lengths = lc.data_ptr<int32_t>(), a.blocks = blocks.data_ptr<int32_t>();
        a.n_blocks = blocks.size(2);
        a.blocks_stride[0] = blocks.stride(0), a.blocks_stride[1] = blocks.stride(1);
        a.block = (int32_t)mParam.block;
        void* stream = CurrentStream(q);
        const size_t ws = dtattn_decode_blocks_workspace_size(&a, stream);
        at::Tensor wst = Bytes(ws, q);
        a.workspace = wst.data_ptr();
        a.workspace_bytes = ws;
        Check(dtattn_decode_blocks(&a, stream), "dtattn_decode_blocks");
    }
    outputs.push_back(o);
    outputs.push_back(lse);
}

}  // namespace core
}  // namespace dtorch_amd
