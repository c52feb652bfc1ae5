// Single-token decode over an 8-bit KV cache (e4m3fn codes, one fp32 scale per block of tokens and kv head).
//
// O_b = softmax(scale * q_b K_b^T) V_b over the first lengths[b] tokens with GQA, K = code * k_scale, V = code * v_scale:
// the arithmetic of SdpaOp::Compute (dtorch/core/operators/standard/scaled_dot_product_attention_op.cc:107-109) at
// Lq = 1.  The reference has no KV cache.
//
// Bound by HBM: 2 D bytes per token and kv head, read once.  The cache goes from memory to registers to matrix
// operands, without LDS: a lane loads 16 bytes of one token's keys, which are two operands of the 16x16x32 MFMA (the
// order of the head dims inside a product is free, so long as the query's is the same), and for the values 8 (D = 128)
// or 4 bytes of each of 8 tokens, whose bytes pair up by token with one v_perm for four of them.  Codes become
// 16-bit floats exactly (e4m3 has 4 significant bits); scales are applied to scores, and to P through its exponent, in
// fp32, so any positive scale does.  Per 32 tokens: 80 conversions and permutes, 16 MFMAs and about 150 other
// instructions for 8 KB.
//
// fp32 queries: q and P are each the sum of three bf16 numbers (8 mantissa bits apiece, exact), and codes are exact in
// bf16, so three MFMAs give the fp32 product.
//
// All (kv head, sequence, 32-token unit) triples are laid end to end by a prefix sum of the lengths and cut in equal
// shares, one per wave.  What a share cuts (its first and its last sequence) goes to a record per head, which
// decode_fp8_merge_kernel merges by LSE; sequences inside one share are written directly.
#include <algorithm>
#include <cmath>

#include "decode_params.hpp"
#include "fp8_cache.hpp"

namespace dtattn {

struct Decode8Params {
    const char* q;
    const uint8_t* k;
    const uint8_t* v;
    const float* ks;
    const float* vs;
    const int32_t* block_table;  // NULL: padded cache
    const int32_t* lengths;
    char* o;
    float* lse;
    float* part_o;    // [2 * shares, 16, kernel D]
    float* part_lse;  // [2 * shares, 16]
    int64_t q_b, q_h;            // elements
    int64_t k_b, k_h, k_s;       // bytes: (batch | page), head, row
    int64_t v_b, v_h, v_s;
    int64_t ks_b, ks_h, vs_b, vs_h;
    int64_t o_b, o_h, lse_b, bt_s;
    int32_t B, Hq, Hkv, group, nsub;  // nsub: 16-head column sets of a kv head's query heads
    int32_t capacity, page_shift, num_pages, block_shift;
    int32_t d, shares;
    float c;  // scale * log2(e)
    uint32_t q_and, q_xor;
};

namespace {

constexpr int kUnit8 = 32;  // tokens per step: two tiles of 16

__device__ __forceinline__ int units8(const Decode8Params& p, int64_t b) {
    return (min(max(p.lengths[b], 0), p.capacity) + kUnit8 - 1) / kUnit8;
}

// Inclusive prefix sum over the wave's lanes.
__device__ __forceinline__ int scan64(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    return v;
}

// V units in `n` shares of V / n or one more (all the longer ones first); the host keeps V below 2^31.
struct Shares8 {
    int n, q, rem;
    __device__ __forceinline__ Shares8(int V, int most) {
        n = min(most, max(1, V));
        q = V / n;
        rem = V - q * n;
    }
    __device__ __forceinline__ int start(int r) const { return r * q + min(r, rem); }
    __device__ __forceinline__ int of(int x) const {  // the share of unit x
        const int big = rem * (q + 1);
        return x < big ? x / (q + 1) : rem + (x - big) / q;
    }
};

// Operand types by query type: bf16 products for bf16 and (in three parts) fp32 queries, fp16 ones for fp16.
template <typename T>
struct Q8 {
    typedef T E;
    static constexpr int parts = 1;
};
template <>
struct Q8<float> {
    typedef bf16_t E;
    static constexpr int parts = 3;
};

// x[0..7] as `parts` operands whose sum they are.
template <typename T>
__device__ __forceinline__ void operands(const float* x, typename Elem<typename Q8<T>::E>::vec8* out) {
    typedef typename Q8<T>::E E;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (Q8<T>::parts == 1) {
            out[0][e] = Elem<E>::from_f32(x[e]);
        } else {
            bf16_t t[3];
            split3(x[e], t);
#pragma unroll
            for (int i = 0; i < 3; ++i) out[i][e] = t[i];
        }
    }
}

// Largest and sum over the four lane groups that hold a column.
__device__ __forceinline__ float colmax(float x) { return max_across_groups<16>(x); }
__device__ __forceinline__ float colsum(float x) { return sum_across_groups<16>(x); }

template <int D>
struct Stage8 {
    u32x4 k[2][D / 64];
    uint32_t v[8][D / 64];
    float ks[2], vs[2];
};

}  // namespace

template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(64, 2) decode_fp8_kernel(const Decode8Params p) {
    typedef typename Q8<T>::E E;
    typedef typename Elem<E>::vec8 V8;
    constexpr int NP = Q8<T>::parts, DH = D / 64, DPL = D / 16;  // DPL: V bytes (dims) per lane and token
    const int lane = threadIdx.x;
    const int col = lane & 15, g4 = lane >> 4;

    const int own0 = lane < p.B ? units8(p, lane) : 0;
    const int pre0 = scan64(own0);
    int U = __shfl(pre0, 63, 64);
    for (int j0 = 64; j0 < p.B; j0 += 64) U += __shfl(scan64(j0 + lane < p.B ? units8(p, j0 + lane) : 0), 63, 64);
    U = __builtin_amdgcn_readfirstlane(U);
    if (U == 0) return;
    const Shares8 sh(U * p.Hkv * p.nsub, p.shares);
    const int r = blockIdx.x;
    if (r >= sh.n) return;
    const int u0 = sh.start(r), n = sh.start(r + 1) - u0;  // first unit and units of this wave

    struct At {
        int slot, b, tok, L;  // slot: kv head * nsub + column set
        bool first;           // the unit starts a segment
        int page[2];          // PAGED: of its two tiles
    };
    typedef const __attribute__((address_space(4))) int32_t cint32;
    typedef const __attribute__((address_space(4))) float cfloat;
    cint32* const lengths = (cint32*)p.lengths;
    cint32* const table = (cint32*)p.block_table;
    cfloat* const kscale = (cfloat*)p.ks;
    cfloat* const vscale = (cfloat*)p.vs;
    auto length = [&](int b) { return min(max(lengths[b], 0), p.capacity); };
    // a tile past the sequence's end stands for its last token: no row of it is read
    auto tile_token = [&](const At& a, int tt) { return min(a.tok + 16 * tt, a.L - 1); };
    auto pages = [&](At& a) {
        if constexpr (PAGED) {
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) a.page[tt] = table[a.b * p.bt_s + (tile_token(a, tt) >> p.page_shift)];
        }
    };
    At at;
    at.slot = u0 / U;
    int x = u0 - at.slot * U;
    at.b = 0;
    for (int j0 = 0;; j0 += 64) {
        const int own = j0 == 0 ? own0 : j0 + lane < p.B ? units8(p, j0 + lane) : 0;
        const int s = j0 == 0 ? pre0 : scan64(own);
        const uint64_t hit = __ballot(s > x);  // sequences ending past x
        if (hit != 0) {
            const int l = __builtin_ctzll(hit);
            at.b = __builtin_amdgcn_readfirstlane(j0 + l);
            x -= __builtin_amdgcn_readfirstlane(__shfl(s - own, l, 64));
            break;
        }
        x -= __builtin_amdgcn_readfirstlane(__shfl(s, 63, 64));
    }
    at.tok = x * kUnit8;
    at.L = length(at.b);
    at.first = true;
    pages(at);
    auto next = [&](At a) {
        a.tok += kUnit8;
        a.first = false;
        if (a.tok >= a.L) {
            a.tok = 0;
            a.first = true;
            do {  // a unit follows, so a sequence with tokens does
                if (++a.b == p.B) a.b = 0, ++a.slot;
                a.L = length(a.b);
            } while (a.L == 0);
        }
        pages(a);
        return a;
    };

    // byte offsets of this lane's loads in a tile of 16 rows; chunks past the real head dim lie past any tile
    const uint32_t kp = (uint32_t)p.k_s, vp = (uint32_t)p.v_s;
    uint32_t koff[DH];
#pragma unroll
    for (int h = 0; h < DH; ++h) koff[h] = 64 * h + 16 * g4 < p.d ? (uint32_t)col * kp + (uint32_t)(64 * h + 16 * g4) : 0xfffffff0u;
    uint32_t voff[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) voff[e] = DPL * col < p.d ? (uint32_t)(4 * g4 + e) * vp + (uint32_t)(DPL * col) : 0xfffffff0u;

    auto load = [&](Stage8<D>& st, const At& a) {
        const int hk = a.slot / p.nsub;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const int tok = tile_token(a, tt), rows = min(max(a.L - a.tok - 16 * tt, 0), 16);
            int64_t slot = a.b;
            int row = tok;
            if constexpr (PAGED) {
                slot = min(max(a.page[tt], 0), p.num_pages - 1);
                row = tok & ((1 << p.page_shift) - 1);
            }
            const int blk = row >> p.block_shift;
            row &= ~15;  // the tile's first row (tiles past the end read nothing)
            const auto krs = make_rsrc(p.k + slot * p.k_b + hk * p.k_h + row * p.k_s, rows > 0 ? (uint32_t)(rows - 1) * kp + (uint32_t)p.d : 0u);
            const auto vrs = make_rsrc(p.v + slot * p.v_b + hk * p.v_h + row * p.v_s, rows > 0 ? (uint32_t)(rows - 1) * vp + (uint32_t)p.d : 0u);
#pragma unroll
            for (int h = 0; h < DH; ++h) st.k[tt][h] = buf_ld16_nt(krs, koff[h]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (D == 128) {
                    const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(vrs, voff[e], 0, 2));
                    st.v[4 * tt + e][0] = w.x, st.v[4 * tt + e][DH - 1] = w.y;
                } else {
                    st.v[4 * tt + e][0] = __builtin_amdgcn_raw_buffer_load_b32(vrs, voff[e], 0, 2);
                }
            }
            st.ks[tt] = kscale[slot * p.ks_b + hk * p.ks_h + blk];
            st.vs[tt] = vscale[slot * p.vs_b + hk * p.vs_h + blk];
        }
    };

    float ML = kNegInf, l = 0.f;            // running max of the scores, and the row sum on that base
    float ER = kNegInf, eb = kNegInf;       // running max of score + log2(v scale), and the accumulators' base
    f32x4 acc[DPL];
    V8 qf[NP][2 * DH];
    int start = 0;          // the segment's first token
    bool cut_first = true;  // the segment is the share's first

    auto compute = [&](const Stage8<D>& st, const At& cur, int s) {
        const int hk = cur.slot / p.nsub, sub = cur.slot - hk * p.nsub;
        const int heads = min(p.group - 16 * sub, 16);
        const int hq = hk * p.group + 16 * sub + col;  // this lane's query head, where col < heads
        if (cur.first || s == 0) {
            const T* qp = reinterpret_cast<const T*>(p.q) + cur.b * p.q_b + (hk * p.group + 16 * sub + min(col, heads - 1)) * p.q_h;
#pragma unroll
            for (int k = 0; k < 2 * DH; ++k) {
                const int dim = 64 * (k >> 1) + 16 * g4 + 8 * (k & 1);
                Chunk<T> w = load_chunk<T, false>(qp + (dim < p.d ? dim : 0));
                float f[8];
#pragma unroll
                for (int i = 0; i < (int)(sizeof(w.v) / sizeof(w.v[0])); ++i) w.v[i] = dim < p.d ? q_bits(w.v[i], p.q_and, p.q_xor) : u32x4{0u, 0u, 0u, 0u};
                if constexpr (NP == 1) {
                    qf[0][k] = __builtin_bit_cast(V8, w.v[0]);
                } else {
                    unpack_chunk<T>(w, f);
                    V8 t[NP];
                    operands<T>(f, t);
#pragma unroll
                    for (int i = 0; i < NP; ++i) qf[i][k] = t[i];
                }
            }
            ML = ER = eb = kNegInf;
            l = 0.f;
#pragma unroll
            for (int j = 0; j < DPL; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            start = cur.tok;
            cut_first = s == 0;
        }
        const int left = cur.L - cur.tok;
        f32x4 sc[2];
        float lv[2], tm[2];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 2 * DH; ++k) {
                const u32x4 w = st.k[tt][k >> 1];
                const V8 kf = k & 1 ? codes_to_vec8<E>(w.z, w.w) : codes_to_vec8<E>(w.x, w.y);
#pragma unroll
                for (int i = 0; i < NP; ++i) a = mfma16(kf, qf[i][k], a);
            }
            const float c = p.c * st.ks[tt];
            lv[tt] = __log2f(st.vs[tt]);
            tm[tt] = kNegInf;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[tt][i] = 16 * tt + 4 * g4 + i < left ? a[i] * c : kNegInf;
                tm[tt] = fmaxf(tm[tt], sc[tt][i]);
            }
            tm[tt] = colmax(tm[tt]);
        }
        // The row sum is on the running max of the scores.  P is on a base of its own, E, where the exponents of a tile's
        // scores and of its V scale add up, so the product of P and codes needs no scaling.  E is the unit's own largest
        // value, so that the largest P is a power of two and rounds exactly, but at most 2^24 below the running one, which
        // keeps alpha and the accumulators finite.  That power is 1, and in fp16 2^15: its subnormals then begin 2^-29
        // below the largest P and not 2^-14, and a small P next to it keeps its precision.
        const float Mn = fmaxf(ML, fmaxf(tm[0], tm[1]));
        const float Mb = Mn == kNegInf ? 0.f : Mn;
        const float e0 = fmaxf(tm[0] + lv[0], tm[1] + lv[1]);
        ER = fmaxf(ER, e0);
        const float en = fmaxf(e0, ER - 24.f) - (__is_same(E, f16_t) ? 15.f : 0.f);
        const float base = en == kNegInf ? 0.f : en;
        const float alpha = fast_exp2(eb - base);
        eb = en;
        float us = 0.f;
        float pf[8];
#pragma unroll
        for (int tt = 0; tt < 2; ++tt) {
            const float pb = base - lv[tt];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                us += fast_exp2(sc[tt][i] - Mb);
                pf[4 * tt + i] = fast_exp2(sc[tt][i] - pb);
            }
        }
        l = __builtin_fmaf(l, fast_exp2(ML - Mb), us);
        ML = Mn;
        V8 pk[NP];
        operands<T>(pf, pk);
#pragma unroll
        for (int h = 0; h < DH; ++h) {
            // four dims of eight tokens: bytes paired by token, then two dims of one pair per conversion
            uint32_t w[4][4];  // [dim][token pair]
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t lo = __builtin_amdgcn_perm(st.v[2 * t + 1][h], st.v[2 * t][h], 0x05010400u);
                const uint32_t hi = __builtin_amdgcn_perm(st.v[2 * t + 1][h], st.v[2 * t][h], 0x07030602u);
                w[0][t] = codes_to_pair<E, false>(lo), w[1][t] = codes_to_pair<E, true>(lo);
                w[2][t] = codes_to_pair<E, false>(hi), w[3][t] = codes_to_pair<E, true>(hi);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const V8 vf = __builtin_bit_cast(V8, u32x4{w[j][0], w[j][1], w[j][2], w[j][3]});
                f32x4 a = acc[4 * h + j] * alpha;
#pragma unroll
                for (int i = 0; i < NP; ++i) a = mfma16(vf, pk[i], a);
                acc[4 * h + j] = a;
            }
        }
        const bool ends = left <= kUnit8;  // the sequence's last unit
        if (ends || s + 1 == n) {
            const float lt = colsum(l);
            if (col < heads) {
                const float lse = __builtin_fmaf(ML, kLn2, __log2f(lt) * kLn2);
                const bool whole = ends && start == 0;
                // every score -inf: a record of O = 0 at the LSE of -inf, which drops it in the merge; the output itself is 0 / 0
                const float f = lt == 0.f && !whole ? 0.f : fast_exp2(eb - ML) / lt;
                const int rec = 2 * r + (cut_first ? 0 : 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int dim = DPL * (4 * g4 + i);
                    float o[DPL];
#pragma unroll
                    for (int j = 0; j < DPL; ++j) o[j] = acc[j][i] * f;
                    if (whole) {
                        T* op = reinterpret_cast<T*>(p.o) + cur.b * p.o_b + hq * p.o_h + dim;
                        if (dim < p.d) {
#pragma unroll
                            for (int j = 0; j < DPL; j += 4) {
                                if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(op + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
                                else *reinterpret_cast<u32x2*>(op + j) = u32x2{pack2<T>(o[j], o[j + 1]), pack2<T>(o[j + 2], o[j + 3])};
                            }
                        }
                    } else {
                        float* op = p.part_o + ((int64_t)rec * 16 + col) * D + dim;
#pragma unroll
                        for (int j = 0; j < DPL; j += 4) *reinterpret_cast<f32x4*>(op + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
                    }
                }
                if (g4 == 0) {
                    if (!whole) p.part_lse[rec * 16 + col] = lse;
                    else if (p.lse != nullptr) p.lse[cur.b * p.lse_b + hq] = lse;
                }
            }
        }
    };

    // two stages in registers: while one is computed the other is in flight
    Stage8<D> s0, s1;
    At a0 = at, a1 = at;
    load(s0, a0);
    for (int s = 0; s < n; s += 2) {
        if (s + 1 < n) {
            a1 = next(a0);
            load(s1, a1);
        }
        compute(s0, a0, s);
        if (s + 1 >= n) break;
        if (s + 2 < n) {
            a0 = next(a1);
            load(s0, a0);
        }
        compute(s1, a1, s + 1);
    }
}

// Merges the records of the shares that cut a sequence, one (b, query head) per wave.
template <typename T, int D>
__global__ void __launch_bounds__(256) decode_fp8_merge_kernel(const Decode8Params p) {
    constexpr int DL = D / 64;  // dims per lane
    const int lane = threadIdx.x & 63;
    const int64_t pair = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (pair >= (int64_t)p.B * p.Hq) return;
    const int b = (int)(pair / p.Hq), hq = (int)(pair % p.Hq), hk = hq / p.group, g = hq - hk * p.group;
    int U = 0, before = 0, own = 0;
    for (int j0 = 0; j0 < p.B; j0 += 64) {
        const int u = j0 + lane < p.B ? units8(p, j0 + lane) : 0;
        const int s = scan64(u);
        if (b >= j0 && b < j0 + 64) {
            own = __shfl(u, b - j0, 64);
            before = U + __shfl(s, b - j0, 64) - own;
        }
        U += __shfl(s, 63, 64);
    }
    T* op = reinterpret_cast<T*>(p.o) + b * p.o_b + hq * p.o_h;
    if (own == 0) {  // empty sequence: O = 0, LSE = -inf
#pragma unroll
        for (int e = 0; e < DL; ++e)
            if (DL * lane + e < p.d) op[DL * lane + e] = Elem<T>::from_f32(0.f);
        if (p.lse != nullptr && lane == 0) p.lse[b * p.lse_b + hq] = kNegInf;
        return;
    }
    const Shares8 sh(U * p.Hkv * p.nsub, p.shares);
    const int x0 = (hk * p.nsub + g / 16) * U + before, r0 = sh.of(x0), r1 = sh.of(x0 + own - 1);
    if (r0 == r1) return;
    const int ns = r1 - r0 + 1;
    // share r0 holds this sequence in its first segment only if it begins with it
    const int slot0 = sh.start(r0) < x0 ? 1 : 0;
    auto rec = [&](int j) { return (int64_t)(2 * (r0 + j) + (j == 0 ? slot0 : 0)) * 16 + g % 16; };
    float mx = kNegInf;
    for (int j = lane; j < ns; j += 64) mx = fmaxf(mx, p.part_lse[rec(j)]);
    mx = wave_max(mx);
    float sum = 0.f;
    for (int j = lane; j < ns; j += 64) sum += __expf(p.part_lse[rec(j)] - mx);
    sum = wave_sum(sum);
    const float inv = 1.f / sum;
    float acc[DL] = {};
    constexpr int MB = 8;  // records in flight
    for (int j0 = 0; j0 < ns; j0 += MB) {
        float lw[MB], v[MB][DL];
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const int64_t q = rec(min(j0 + j, ns - 1));
            lw[j] = p.part_lse[q];
#pragma unroll
            for (int e = 0; e < DL; ++e) v[j][e] = p.part_o[q * D + DL * lane + e];
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const float w = j0 + j < ns ? __expf(lw[j] - mx) * inv : 0.f;
#pragma unroll
            for (int e = 0; e < DL; ++e) acc[e] = __builtin_fmaf(w, v[j][e], acc[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < DL; ++e)
        if (DL * lane + e < p.d) op[DL * lane + e] = Elem<T>::from_f32(acc[e]);
    if (p.lse != nullptr && lane == 0) p.lse[b * p.lse_b + hq] = mx + __logf(sum);
}

namespace {

struct Plan8 {
    int32_t nsub, shares, kernel_d;
    size_t bytes;
};

// Shares: eight waves per CU, and no more than there can be units.
Plan8 plan8(const dtattn_decode_fp8_args* a, int64_t capacity, int cus) {
    Plan8 r;
    r.kernel_d = a->D <= 64 ? 64 : 128;
    r.nsub = (int32_t)((a->Hq / a->Hkv + 15) / 16);
    const int64_t units = a->B * a->Hkv * r.nsub * ((capacity + kUnit8 - 1) / kUnit8);
    r.shares = (int32_t)std::max<int64_t>(1, std::min<int64_t>(8 * (int64_t)cus, units));
    const size_t records = (size_t)2 * r.shares * 16;
    r.bytes = (records * (r.kernel_d + 1) * sizeof(float) + 255) & ~(size_t)255;
    return r;
}

int64_t capacity_of(const dtattn_decode_fp8_args* a) { return a->block_table != nullptr ? a->max_pages * a->page_size : a->S_max; }

template <typename T, int D>
int launch8(const Decode8Params& p, hipStream_t stream) {
    if (p.block_table != nullptr)
        hipLaunchKernelGGL((decode_fp8_kernel<T, D, true>), dim3((unsigned)p.shares), dim3(64), 0, stream, p);
    else
        hipLaunchKernelGGL((decode_fp8_kernel<T, D, false>), dim3((unsigned)p.shares), dim3(64), 0, stream, p);
    const int st = check_launch("decode_fp8_kernel");
    if (st != DTATTN_OK) return st;
    const int64_t pairs = (int64_t)p.B * p.Hq;
    hipLaunchKernelGGL((decode_fp8_merge_kernel<T, D>), dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, stream, p);
    return check_launch("decode_fp8_merge_kernel");
}

}  // namespace

}  // namespace dtattn

using namespace dtattn;

extern "C" size_t dtattn_decode_fp8_workspace_size(const dtattn_decode_fp8_args* a, void* stream) {
    if (a == nullptr || a->B <= 0 || a->Hq <= 0 || a->Hkv <= 0 || a->D <= 0) return 0;
    const int cus = stream_cus(reinterpret_cast<hipStream_t>(stream));
    return plan8(a, std::max<int64_t>(capacity_of(a), 1), cus > 0 ? cus : 256).bytes;
}

extern "C" int dtattn_decode_fp8(const dtattn_decode_fp8_args* a, void* stream_) {
    const char* who = "decode_fp8";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    if (a->B < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->D <= 0 || a->B > (1 << 24) || a->Hq > (1 << 20))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
    if (a->Hq % a->Hkv != 0) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: Hq is not a multiple of Hkv", who);
    if (a->dtype != DTATTN_BF16 && a->dtype != DTATTN_FP16 && a->dtype != DTATTN_FP32)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: dtype %d not supported (bf16, fp16, fp32)", who, a->dtype);
    Fp8Cache c;
    int st = fp8_cache_checks(a, a->block_table != nullptr, who, &c);
    if (st != DTATTN_OK) return st;
    ScalePlan sp;
    st = plan_scale(a->scale, a->D, a->dtype == DTATTN_FP32 ? kSign32 : kSign16, &sp);
    if (st != DTATTN_OK) return st;
    if (a->B == 0) return DTATTN_OK;
    if (a->q == nullptr || a->lengths == nullptr || a->o == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    const int64_t esz = a->dtype == DTATTN_FP32 ? 4 : 2;
    for (int i = 0; i < 2; ++i)
        if ((a->q_stride[i] * esz) % 16 != 0 || (a->o_stride[i] * esz) % 16 != 0)
            return fail(DTATTN_ERR_UNSUPPORTED, "%s: query and output strides must be multiples of 16 bytes", who);
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->o)) & 15u)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: query and output must be 16-byte aligned", who);
    const int cus = stream_cus(stream);
    if (cus <= 0) return fail(DTATTN_ERR_DEVICE, "%s: cannot tell the stream's device", who);
    const Plan8 plan = plan8(a, c.capacity, cus);
    if (a->B * a->Hkv * plan.nsub * (((int64_t)c.capacity + kUnit8 - 1) / kUnit8) >= ((int64_t)1 << 31))
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: cache too large", who);
    if (a->workspace == nullptr || a->workspace_bytes < plan.bytes)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, plan.bytes, a->workspace_bytes);
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);

    Decode8Params p = {};
    p.q = reinterpret_cast<const char*>(a->q);
    p.k = reinterpret_cast<const uint8_t*>(a->k_cache), p.v = reinterpret_cast<const uint8_t*>(a->v_cache);
    p.ks = a->k_scale, p.vs = a->v_scale;
    p.block_table = a->block_table;
    p.lengths = a->lengths;
    p.o = reinterpret_cast<char*>(a->o), p.lse = a->lse;
    p.part_o = reinterpret_cast<float*>(a->workspace);
    p.part_lse = p.part_o + (int64_t)2 * plan.shares * 16 * plan.kernel_d;
    p.q_b = a->q_stride[0], p.q_h = a->q_stride[1];
    p.k_b = a->k_stride[0], p.k_h = a->k_stride[1], p.k_s = a->k_stride[2];
    p.v_b = a->v_stride[0], p.v_h = a->v_stride[1], p.v_s = a->v_stride[2];
    p.ks_b = a->k_scale_stride[0], p.ks_h = a->k_scale_stride[1];
    p.vs_b = a->v_scale_stride[0], p.vs_h = a->v_scale_stride[1];
    p.o_b = a->o_stride[0], p.o_h = a->o_stride[1];
    p.lse_b = a->lse ? a->lse_stride[0] : 0;
    p.bt_s = a->block_table_stride;
    p.B = (int32_t)a->B, p.Hq = (int32_t)a->Hq, p.Hkv = (int32_t)a->Hkv, p.group = (int32_t)(a->Hq / a->Hkv);
    p.nsub = plan.nsub, p.shares = plan.shares;
    p.capacity = c.capacity, p.page_shift = c.page_shift, p.num_pages = c.num_pages, p.block_shift = c.block_shift;
    p.d = (int32_t)a->D;
    p.c = sp.scale * kLog2e;
    p.q_and = sp.q_and, p.q_xor = sp.q_xor;
    const bool wide = plan.kernel_d == 128;
    switch (a->dtype) {
        case DTATTN_BF16: return wide ? launch8<bf16_t, 128>(p, stream) : launch8<bf16_t, 64>(p, stream);
        case DTATTN_FP16: return wide ? launch8<f16_t, 128>(p, stream) : launch8<f16_t, 64>(p, stream);
        default: return wide ? launch8<float, 128>(p, stream) : launch8<float, 64>(p, stream);
    }
}
