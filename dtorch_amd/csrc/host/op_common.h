// Argument checks and tensor views shared by the host operators.
#pragma once

#include <c10/hip/HIPStream.h>
#include <torch/torch.h>

#include <sstream>
#include <stdexcept>
#include <string>
#include <vector>

#include "dtattn.h"

namespace dtorch_amd {
namespace core {

[[noreturn]] inline void Throw(const std::string& msg) { throw std::invalid_argument("dtorch_amd: " + msg); }

inline void Check(int status, const char* what) {
    if (status == DTATTN_OK) return;
    std::ostringstream os;
    os << what << " failed (status " << status << "): " << dtattn_last_error();
    if (status == DTATTN_ERR_LAUNCH || status == DTATTN_ERR_DEVICE) throw std::runtime_error("dtorch_amd: " + os.str());
    Throw(os.str());
}

inline void* CurrentStream(const at::Tensor& t) {
    return reinterpret_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

inline int32_t DtypeCode(c10::ScalarType st) {
    switch (st) {
        case c10::ScalarType::BFloat16: return DTATTN_BF16;
        case c10::ScalarType::Half: return DTATTN_FP16;
        case c10::ScalarType::Float8_e4m3fn: return DTATTN_FP8_E4M3FN;
        case c10::ScalarType::Float: return DTATTN_FP32;
        default: return -1;
    }
}

// A tensor viewed as [B, H, S, D] (leading axes folded into B), last-axis stride 1, 16-byte aligned
// strides and base pointer.  Anything else is made contiguous first (a layout copy, not compute).
struct View4 {
    at::Tensor t;
    int64_t B, H, S, D;
    int64_t sb, sh, ss;
};

// The leading (batch) axes 0 .. nd-4 fold into one axis of stride `sb` iff the axes of size > 1 form
// one arithmetic progression: for consecutive such axes i < j, stride(i) == stride(j) * size(j).
// Size-1 axes carry no stride information and are skipped; `sb` is then the stride of the innermost
// batch axis of size > 1 (any value works when the folded batch is 1, since it is never multiplied
// by a non-zero index).
inline bool FoldBatch(const at::Tensor& t, int64_t& sb) {
    const int64_t nd = t.dim();
    int64_t prev = -1;
    sb = 0;
    for (int64_t i = 0; i < nd - 3; ++i) {
        if (t.size(i) == 1) continue;
        if (prev >= 0 && t.stride(prev) != t.stride(i) * t.size(i)) return false;
        prev = i;
        sb = t.stride(i);
    }
    return true;
}

inline View4 MakeView4(const at::Tensor& in, const char* name) {
    if (in.dim() < 4) Throw(std::string(name) + " must have at least 4 dimensions [..., H, S, D]");
    at::Tensor t = in;
    const int64_t esz = t.element_size();
    int64_t sb = 0;
    auto ok = [&](const at::Tensor& x) {
        if (x.stride(-1) != 1 || !FoldBatch(x, sb)) return false;
        if ((reinterpret_cast<uintptr_t>(x.data_ptr()) & 15u) != 0) return false;
        for (int64_t i = 0; i < x.dim() - 1; ++i)
            if (x.size(i) > 1 && (x.stride(i) * esz) % 16 != 0) return false;
        return true;
    };
    if (!ok(t)) {
        t = t.contiguous();
        FoldBatch(t, sb);  // always foldable once contiguous
    }
    View4 v;
    v.t = t;
    const int64_t nd = t.dim();
    v.B = 1;
    for (int64_t i = 0; i < nd - 3; ++i) v.B *= t.size(i);
    v.H = t.size(nd - 3);
    v.S = t.size(nd - 2);
    v.D = t.size(nd - 1);
    // Size-1 axes are never indexed past 0, so their strides are free: give them the contiguous
    // values, which keeps every stride the kernels see a multiple of 16 bytes.
    v.ss = v.S > 1 ? t.stride(nd - 2) : v.D;
    v.sh = v.H > 1 ? t.stride(nd - 3) : v.S * v.ss;
    // A folded batch of 1 is never indexed past 0: give it the extent of one (H, S, D) slab.
    v.sb = v.B > 1 ? sb : v.H * v.sh;
    return v;
}

inline void CheckDevice(const std::vector<const at::Tensor*>& ts) {
    const at::Device dev = ts[0]->device();
    if (!dev.is_cuda())
        Throw("the MI355X attention kernels take device tensors; CPU meshes keep DTorch's libtorch path");
    for (const at::Tensor* t : ts)
        if (t->device() != dev) Throw("all tensors must be on the same device");
}

// A cache written in place: it cannot be copied to fix its layout, so the layout is checked instead.
inline void CheckCacheLayout(const at::Tensor& c, const char* name) {
    if (c.dim() != 4) Throw(std::string(name) + " must be 4-D");
    if (c.stride(3) != 1) Throw(std::string(name) + " needs a unit stride along D");
    for (int i = 0; i < 3; ++i)
        if ((c.stride(i) * c.element_size()) % 16 != 0)
            Throw(std::string(name) + " strides must be multiples of 16 bytes (it is updated in place)");
    if ((reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) != 0) Throw(std::string(name) + " must be 16-byte aligned");
}

inline void CheckLengths(const at::Tensor& len, int64_t B) {
    if (len.scalar_type() != at::kInt || len.dim() != 1 || len.size(0) != B || !len.is_contiguous())
        Throw("lengths must be a contiguous int32 tensor of shape [B] (it is updated in place)");
}

}  // namespace core
}  // namespace dtorch_amd
