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
// fp32, so any positive scale does.
//
// fp32 queries: q and P are each the sum of three bf16 numbers (8 mantissa bits apiece, exact), and codes are exact in
// bf16, so three MFMAs give the fp32 product.  16-bit queries: P is two numbers of their type, which leaves 2^-16 (bf16) or 2^-22
// (fp16) of it, far below the one rounding of the output; P rounded to 16 bits would add half a step of the type.  The second
// part costs 1% (us without it and with: 64 sequences of 512 to 8192 in pages 103.0 and 103.4, 16 of 20000 to 32768 136.2 and 137.8,
// one of 4000 12.0 and 12.2).
//
// All (kv head, sequence, 32-token unit) triples are laid end to end by a prefix sum of the lengths and cut in equal
// shares, one per workgroup, whose four waves take its units in turn and meet in LDS where a sequence ends.  What a share cuts (its
// first and its last sequence) goes to a record per head, which decode_fp8_merge_kernel merges by LSE; sequences inside
// one share are written directly.  The keys of the next unit are loaded when this one's scores are done, its values when P V
// is.  Waves that stream shares of their own (four times the streams and records) take 14.3 us where this takes 12.8 (1x4000),
// and 106 where this takes 104 (64 of 512 to 8192); more waves per CU only slow the memory down (16: 234 instead of 150 us for
// 16 of 20000 to 32768).
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
    int32_t d, shares;  // shares: at most so many
    float c;  // scale * log2(e)
    uint32_t q_and, q_xor;
};

namespace {

constexpr int kTiles8 = 2;             // tiles of 16 tokens per step of a wave
constexpr int kUnit8 = 16 * kTiles8;
constexpr int kWaves8 = 4;             // waves of a workgroup, which take the units of its share in turn
// Shares per CU, and units that a share has at least.  us, 1x4000 / 64 sequences of 512 to 8192 in 16-token pages / 16 of
// 20000 to 32768 (8 kv heads of 128): one share per CU 14.4 / 128 / 165, two 12.8 / 104 / 144, three 14.6 / 103 / 147; two units
// at least 15.6 / 104 / 144, eight 15.8 / 105 / 144.
constexpr int kSharesPerCu = 2;
constexpr int kShareLeast = kWaves8;

__device__ __forceinline__ int tokens8(const Decode8Params& p, int64_t b) { return min(max(p.lengths[b], 0), p.capacity); }
__device__ __forceinline__ int units8(const Decode8Params& p, int64_t b) { return (tokens8(p, b) + kUnit8 - 1) / kUnit8; }

// V units in `n` shares of V / n or one more (all the longer ones first); the host keeps V below 2^31.
struct Shares8 {
    int n, q, rem;
    __device__ __forceinline__ Shares8(int V, int most) {
        n = min(most, max(1, V / kShareLeast));
        q = V / n;
        rem = V - q * n;
    }
    __device__ __forceinline__ int start(int r) const { return r * q + min(r, rem); }
    __device__ __forceinline__ int of(int x) const {  // the share of unit x
        const int big = rem * (q + 1);
        return x < big ? x / (q + 1) : rem + (x - big) / q;
    }
};

// Operand types by query type: bf16 products for bf16 and fp32 queries, fp16 ones for fp16; parts of a query and of P.
template <typename T>
struct Q8 {
    typedef T E;
    static constexpr int parts = 1, pparts = 2;
};
template <>
struct Q8<float> {
    typedef bf16_t E;
    static constexpr int parts = 3, pparts = 3;
};

// x[0..7] as the two or three operands whose sum they are.
template <typename T>
__device__ __forceinline__ void operands(const float* x, typename Elem<typename Q8<T>::E>::vec8* out) {
    typedef typename Q8<T>::E E;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (Q8<T>::pparts == 2) {
            out[0][e] = Elem<E>::from_f32(x[e]);
            out[1][e] = Elem<E>::from_f32(x[e] - Elem<E>::to_f32(out[0][e]));
        } else {
            bf16_t t[3];
            split3(x[e], t);
#pragma unroll
            for (int i = 0; i < 3; ++i) out[i][e] = t[i];
        }
    }
}

// log2 of any float >= 0: the instruction takes a subnormal for 0.
__device__ __forceinline__ float log2_any(float x) {
    const bool small = __builtin_bit_cast(uint32_t, x) < 0x00800000u;
    return __log2f(small ? x * 0x1p24f : x) - (small ? 24.f : 0.f);
}

// Largest and sum over the four lane groups that hold a column.
__device__ __forceinline__ float colmax(float x) { return max_across_groups<16>(x); }
__device__ __forceinline__ float colsum(float x) { return sum_across_groups<16>(x); }

// Bits of 4 bytes of 8 tokens (two tiles' rows 4 g4 .. 4 g4 + 3) as operands of 4 dims: bytes paired by token, then two dims of
// one pair per conversion.
template <typename E>
__device__ __forceinline__ void transpose4x8(const uint32_t (&v)[8], typename Elem<E>::vec8 (&out)[4]) {
    uint32_t w[4][4];  // [dim][token pair]
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const uint32_t lo = __builtin_amdgcn_perm(v[2 * t + 1], v[2 * t], 0x05010400u);
        const uint32_t hi = __builtin_amdgcn_perm(v[2 * t + 1], v[2 * t], 0x07030602u);
        w[0][t] = codes_to_pair<E, false>(lo), w[1][t] = codes_to_pair<E, true>(lo);
        w[2][t] = codes_to_pair<E, false>(hi), w[3][t] = codes_to_pair<E, true>(hi);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = __builtin_bit_cast(typename Elem<E>::vec8, u32x4{w[j][0], w[j][1], w[j][2], w[j][3]});
}

}  // namespace

// PAGES: 0, a padded cache; 1, pages of a whole unit or more; 2, smaller pages.
template <typename T, int D, int PAGES>
__global__ void __launch_bounds__(64 * kWaves8, kSharesPerCu) decode_fp8_kernel(const Decode8Params p) {
    typedef typename Q8<T>::E E;
    typedef typename Elem<E>::vec8 V8;
    constexpr int NT = kTiles8;
    constexpr int NP = Q8<T>::parts, PP = Q8<T>::pparts, DH = D / 64, DPL = D / 16;  // DPL: V bytes (dims) per lane and token
    constexpr int NR = PAGES == 2 ? NT : 1;  // buffer resources of a unit
    constexpr int RP = D + 4;  // floats per row of red_o: rows 16 bytes apart in the banks
    __shared__ __attribute__((aligned(16))) float red_o[kWaves8][16][RP];
    __shared__ float red_m[kWaves8][16], red_l[kWaves8][16], red_e[kWaves8][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g4 = lane >> 4;

    // units of all sequences (the first 64 are kept: their prefix finds the share's start)
    const int len0 = lane < p.B ? tokens8(p, lane) : 0;
    const int own0 = (len0 + kUnit8 - 1) / kUnit8;
    const int pre0 = scan64(own0);
    int U = __builtin_amdgcn_readlane(pre0, 63);
    for (int j0 = 64; j0 < p.B; j0 += 64) U += __builtin_amdgcn_readlane(scan64(j0 + lane < p.B ? units8(p, j0 + lane) : 0), 63);
    if (U == 0) return;
    const Shares8 sh(U * p.Hkv * p.nsub, p.shares);
    const int r = blockIdx.x;
    if (r >= sh.n) return;
    const int u0 = sh.start(r), n = sh.start(r + 1) - u0;  // first unit and units of this workgroup

    typedef const __attribute__((address_space(4))) int32_t cint32;
    typedef const __attribute__((address_space(4))) float cfloat;
    cint32* const lengths = (cint32*)p.lengths;
    cint32* const table = (cint32*)p.block_table;
    auto length = [&](int b) { return min(max(lengths[b], 0), p.capacity); };
    // Where a unit lies (cur: of the workgroup's segment; nx: the next that this wave loads).  Lengths, page ids and scales are scalar loads, which leave the vector loads in flight alone.
    struct At {
        int slot, hk, b, tok, L;  // slot: kv head * nsub + column set
        const uint8_t* k;         // PAGES 0: first rows
        const uint8_t* v;
        cfloat* ks;               // PAGES 0: scales of the head
        cfloat* vs;
        int page[NR];             // PAGES 1, 2
    };
    // a tile past the sequence's end stands for its last token: no row of it is read
    auto tile_token = [&](const At& a, int tt) { return min(a.tok + 16 * tt, a.L - 1); };
    auto enter = [&](At& a) {  // a segment
        a.hk = p.nsub == 1 ? a.slot : a.slot / p.nsub;
        if constexpr (PAGES == 0) {
            a.k = p.k + a.b * p.k_b + a.hk * p.k_h + a.tok * p.k_s;
            a.v = p.v + a.b * p.v_b + a.hk * p.v_h + a.tok * p.v_s;
            a.ks = (cfloat*)p.ks + a.b * p.ks_b + a.hk * p.ks_h;
            a.vs = (cfloat*)p.vs + a.b * p.vs_b + a.hk * p.vs_h;
        }
    };
    auto pages = [&](At& a) {
        if constexpr (PAGES != 0) {
#pragma unroll
            for (int i = 0; i < NR; ++i) a.page[i] = table[a.b * p.bt_s + (tile_token(a, i) >> p.page_shift)];
        }
    };
    At at;
    at.slot = u0 / U;
    int x = u0 - at.slot * U;
    at.b = 0;
    for (int j0 = 0;; j0 += 64) {
        const int len = j0 == 0 ? len0 : j0 + lane < p.B ? tokens8(p, j0 + lane) : 0;
        const int own = (len + kUnit8 - 1) / kUnit8;
        const int s = j0 == 0 ? pre0 : scan64(own);
        const uint64_t hit = __ballot(s > x);  // sequences ending past x
        if (hit != 0) {
            const int l = __builtin_ctzll(hit);
            at.b = j0 + l;
            at.L = __builtin_amdgcn_readlane(len, l);
            x -= __builtin_amdgcn_readlane(s - own, l);
            break;
        }
        x -= __builtin_amdgcn_readlane(s, 63);
    }
    at.tok = x * kUnit8;
    auto advance = [&](At& a, int units) {
        a.tok += units * kUnit8;
        if (a.tok < a.L) {
            if constexpr (PAGES == 0) {
                a.k += units * kUnit8 * p.k_s;
                a.v += units * kUnit8 * p.v_s;
            }
            return;
        }
        do {  // a unit follows, so a sequence with tokens does
            a.tok -= (a.L + kUnit8 - 1) & -kUnit8;
            if (++a.b == p.B) a.b = 0, ++a.slot;
            a.L = length(a.b);
        } while (a.tok >= a.L);
        enter(a);
    };

    // byte offsets of this lane's loads from a unit's (PAGES 2: a tile's) first row; chunks past the real head dim lie past any
    const uint32_t kp = (uint32_t)p.k_s, vp = (uint32_t)p.v_s;
    uint32_t koff[DH], voff[4];
#pragma unroll
    for (int h = 0; h < DH; ++h) koff[h] = 64 * h + 16 * g4 < p.d ? (uint32_t)col * kp + (uint32_t)(64 * h + 16 * g4) : 0xc0000000u;
#pragma unroll
    for (int e = 0; e < 4; ++e) voff[e] = DPL * col < p.d ? (uint32_t)(4 * g4 + e) * vp + (uint32_t)(DPL * col) : 0xc0000000u;

    u32x4 kr[NT][DH];
    uint32_t vr[NT / 2][DH][8];  // by pairs of tiles
    float ks[NT], vs[NT];
    // rows of a resource that hold tokens: of the unit, or of tile i
    auto rows_of = [&](const At& a, int i) { return min(max(a.L - a.tok - (NR > 1 ? 16 * i : 0), 0), NR > 1 ? 16 : kUnit8); };
    auto slot_of = [&](const At& a, int i) { return (int64_t)min(max(a.page[i], 0), p.num_pages - 1); };
    auto row_of = [&](const At& a, int i) { return (tile_token(a, i) & ((1 << p.page_shift) - 1)) & ~15; };
    auto load_k = [&](const At& a) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int rows = rows_of(a, i);
            const uint8_t* base;
            if constexpr (PAGES == 0) base = a.k;
            else base = p.k + slot_of(a, i) * p.k_b + a.hk * p.k_h + row_of(a, i) * p.k_s;
            const auto rs = make_rsrc(base, rows > 0 ? (uint32_t)(rows - 1) * kp + (uint32_t)p.d : 0u);
#pragma unroll
            for (int tt = NR > 1 ? i : 0; tt < (NR > 1 ? i + 1 : NT); ++tt)
#pragma unroll
                for (int h = 0; h < DH; ++h) kr[tt][h] = buf_ld16_nt(rs, koff[h] + (NR > 1 ? 0u : 16u * tt * kp));
        }
    };
    auto load_v = [&](const At& a) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int rows = rows_of(a, i);
            const uint8_t* base;
            if constexpr (PAGES == 0) base = a.v;
            else base = p.v + slot_of(a, i) * p.v_b + a.hk * p.v_h + row_of(a, i) * p.v_s;
            const auto rs = make_rsrc(base, rows > 0 ? (uint32_t)(rows - 1) * vp + (uint32_t)p.d : 0u);
#pragma unroll
            for (int tt = NR > 1 ? i : 0; tt < (NR > 1 ? i + 1 : NT); ++tt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t off = voff[e] + (NR > 1 ? 0u : 16u * tt * vp);
                    if constexpr (D == 128) {
                        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, 2));
                        vr[tt / 2][0][4 * (tt & 1) + e] = w.x, vr[tt / 2][DH - 1][4 * (tt & 1) + e] = w.y;
                    } else {
                        vr[tt / 2][0][4 * (tt & 1) + e] = __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 2);
                    }
                }
        }
    };
    auto load_scales = [&](const At& a) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            if constexpr (PAGES == 0) {
                const int blk = tile_token(a, tt) >> p.block_shift;
                ks[tt] = a.ks[blk];
                vs[tt] = a.vs[blk];
            } else {
                const int64_t slot = slot_of(a, NR > 1 ? tt : 0);
                const int blk = (tile_token(a, tt) & ((1 << p.page_shift) - 1)) >> p.block_shift;
                ks[tt] = ((cfloat*)p.ks)[slot * p.ks_b + a.hk * p.ks_h + blk];
                vs[tt] = ((cfloat*)p.vs)[slot * p.vs_b + a.hk * p.vs_h + blk];
            }
        }
    };

    float ML = kNegInf, l = 0.f;       // running max of the scores, and the row sum on that base
    float ER = kNegInf, eb = kNegInf;  // running max of score + log2(v scale), and the accumulators' base
    f32x4 acc[DPL];
    V8 qf[NP][2 * DH];
    At cur = at, nx = at;
    cur.hk = p.nsub == 1 ? cur.slot : cur.slot / p.nsub;
    if (wave < n) {
        enter(nx);
        if (wave > 0) advance(nx, wave);
        pages(nx);
        load_k(nx);
        load_v(nx);
        load_scales(nx);
    }
    int s = wave;  // this wave's next unit of the share
    for (int u = 0; u < n;) {
      const int m = min((cur.L - cur.tok + kUnit8 - 1) / kUnit8, n - u);  // units of the segment
      const int hk = cur.hk, b = cur.b, sub = cur.slot - hk * p.nsub;
      const int heads = min(p.group - 16 * sub, 16);
      ML = ER = eb = kNegInf;
      l = 0.f;
#pragma unroll
      for (int j = 0; j < DPL; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (s < u + m) {
        const T* qp = reinterpret_cast<const T*>(p.q) + b * p.q_b + (hk * p.group + 16 * sub + min(col, heads - 1)) * p.q_h;
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
      }
      for (; s < u + m; s += kWaves8) {
        const int left = cur.L - cur.tok - (s - u) * kUnit8;
        const bool more = s + kWaves8 < n;
        if (more) {
            advance(nx, kWaves8);
            pages(nx);
        }
        f32x4 sc[NT];
        float tm[NT], lv[NT];
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 2 * DH; ++k) {
                const u32x4 w = kr[tt][k >> 1];
                const V8 kf = k & 1 ? codes_to_vec8<E>(w.z, w.w) : codes_to_vec8<E>(w.x, w.y);
#pragma unroll
                for (int i = 0; i < NP; ++i) a = mfma16(kf, qf[i][k], a);
            }
            sc[tt] = a * (p.c * ks[tt]);
            lv[tt] = log2_any(vs[tt]);
        }
        if (more) load_k(nx);  // the keys are used up
        if (left < kUnit8) {
#pragma unroll
            for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (16 * tt + 4 * g4 + i >= left) sc[tt][i] = kNegInf;
        }
        if (more) load_scales(nx);
        // The row sum is on the running max of the scores.  P is on a base of its own, E, where the exponents of a tile's
        // scores and of its V scale add up, so the product of P and codes needs no scaling.  E is the unit's own largest
        // value, so that the largest P is a power of two, but at most 2^24 below the running one, which
        // keeps alpha and the accumulators finite.  That power is 1, and in fp16 2^15: its subnormals then begin 2^-29
        // below the largest P and not 2^-14, and a small P and its second part keep their precision.
        float Mn = ML, e0 = kNegInf;
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            tm[tt] = fmaxf(fmaxf(sc[tt][0], sc[tt][1]), fmaxf(sc[tt][2], sc[tt][3]));
            Mn = fmaxf(Mn, tm[tt]);
            e0 = fmaxf(e0, tm[tt] + lv[tt]);
        }
        Mn = colmax(Mn);
        e0 = colmax(e0);
        const float Mb = Mn == kNegInf ? 0.f : Mn;
        ER = fmaxf(ER, e0);
        const float en = fmaxf(e0, ER - 24.f) - (__is_same(E, f16_t) ? 15.f : 0.f);
        const float base = en == kNegInf ? 0.f : en;
        const float alpha = fast_exp2(eb - base);
        eb = en;
        float us = 0.f;
        V8 pk[NT / 2][PP];
#pragma unroll
        for (int tp = 0; tp < NT / 2; ++tp) {
            float pf[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int tt = 2 * tp + (i >> 2);
                us += fast_exp2(sc[tt][i & 3] - Mb);
                pf[i] = fast_exp2(sc[tt][i & 3] - (base - lv[tt]));
            }
            operands<T>(pf, pk[tp]);
        }
        l = __builtin_fmaf(l, fast_exp2(ML - Mb), us);
        ML = Mn;
#pragma unroll
        for (int j = 0; j < DPL; ++j) acc[j] *= alpha;
#pragma unroll
        for (int tp = 0; tp < NT / 2; ++tp)
#pragma unroll
            for (int h = 0; h < DH; ++h) {
                V8 vf[4];
                transpose4x8<E>(vr[tp][h], vf);
#pragma unroll
                for (int i = 0; i < PP; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[4 * h + j] = mfma16(vf[j], pk[tp][i], acc[4 * h + j]);
            }
        if (more) load_v(nx);
      }
      // the waves meet: each leaves its accumulators and their bases
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < DPL; j += 4)
            *reinterpret_cast<f32x4*>(&red_o[wave][col][DPL * (4 * g4 + i) + j]) = f32x4{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
      const float lw = colsum(l);
      if (g4 == 0) red_m[wave][col] = ML, red_l[wave][col] = lw, red_e[wave][col] = eb;
      lds_barrier();
      const int g = tid >> 4;  // a head, and DPL of its dims
      if (g < heads) {
        float M = kNegInf, X = kNegInf;
#pragma unroll
        for (int w = 0; w < kWaves8; ++w) M = fmaxf(M, red_m[w][g]), X = fmaxf(X, red_e[w][g]);
        float lt = 0.f, o[DPL] = {};
#pragma unroll
        for (int w = 0; w < kWaves8; ++w) {
            const float mw = red_m[w][g], ew = red_e[w][g];
            lt += (mw == kNegInf ? 0.f : fast_exp2(mw - M)) * red_l[w][g];
            const float f = ew == kNegInf ? 0.f : fast_exp2(ew - X);
#pragma unroll
            for (int j = 0; j < DPL; j += 4) {
                const f32x4 a = *reinterpret_cast<const f32x4*>(&red_o[w][g][DPL * (tid & 15) + j]);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[j + i] = __builtin_fmaf(a[i], f, o[j + i]);
            }
        }
        const int hq = hk * p.group + 16 * sub + g, dim = DPL * (tid & 15);
        const float lse = __builtin_fmaf(M, kLn2, __log2f(lt) * kLn2);
        const bool whole = cur.tok == 0 && u + m <= n && m * kUnit8 >= cur.L;
        // every score -inf: a record of O = 0 at the LSE of -inf, which drops it in the merge; the output itself is 0 / 0
        // (2^(X - M), which the smallest scales of V take below what the instruction gives, is the product of two powers)
        const float f = lt == 0.f && !whole ? 0.f : fast_exp2(fmaxf(X - M, -100.f)) / lt, small = fast_exp2(fminf(X - M + 100.f, 0.f));
#pragma unroll
        for (int j = 0; j < DPL; ++j) o[j] = o[j] * f * small;
        if (whole) {
            T* op = reinterpret_cast<T*>(p.o) + b * p.o_b + hq * p.o_h + dim;
            if (dim < p.d) {
#pragma unroll
                for (int j = 0; j < DPL; j += 4) {
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<f32x4*>(op + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
                    else *reinterpret_cast<u32x2*>(op + j) = u32x2{pack2<T>(o[j], o[j + 1]), pack2<T>(o[j + 2], o[j + 3])};
                }
            }
            if (p.lse != nullptr && (tid & 15) == 0) p.lse[b * p.lse_b + hq] = lse;
        } else {
            const int rec = 2 * r + (u == 0 ? 0 : 1);
            float* op = p.part_o + ((int64_t)rec * 16 + g) * D + dim;
#pragma unroll
            for (int j = 0; j < DPL; j += 4) *reinterpret_cast<f32x4*>(op + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
            if ((tid & 15) == 0) p.part_lse[rec * 16 + g] = lse;
        }
      }
      u += m;
      if (u < n) {
        lds_barrier();  // every wave has read the others' before they write again
        cur.tok = 0;
        do {  // a unit follows, so a sequence with tokens does
            if (++cur.b == p.B) cur.b = 0, ++cur.slot;
            cur.L = length(cur.b);
        } while (cur.L == 0);
        cur.hk = p.nsub == 1 ? cur.slot : cur.slot / p.nsub;
      }
    }
}

// Merges the records of the shares that cut a sequence: one (b, query head) per W waves.
template <typename T, int D, int W>
__global__ void __launch_bounds__(256) decode_fp8_merge_kernel(const Decode8Params p) {
    constexpr int DL = D / 64;  // dims per lane
    __shared__ float red[W > 1 ? W : 1][D];
    const int lane = threadIdx.x & 63, wave = W > 1 ? threadIdx.x >> 6 : 0;
    const int64_t pair = W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
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
        U += __builtin_amdgcn_readlane(s, 63);
    }
    T* op = reinterpret_cast<T*>(p.o) + b * p.o_b + hq * p.o_h;
    if (own == 0) {  // empty sequence: O = 0, LSE = -inf
        if (wave > 0) return;
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
    for (int j0 = wave; j0 < ns; j0 += W * MB) {
        float lw[MB], v[MB][DL];
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const int64_t q = rec(min(j0 + W * j, ns - 1));
            lw[j] = p.part_lse[q];
#pragma unroll
            for (int e = 0; e < DL; ++e) v[j][e] = p.part_o[q * D + DL * lane + e];
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const float w = j0 + W * j < ns ? __expf(lw[j] - mx) * inv : 0.f;
#pragma unroll
            for (int e = 0; e < DL; ++e) acc[e] = __builtin_fmaf(w, v[j][e], acc[e]);
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int e = 0; e < DL; ++e) red[wave][DL * lane + e] = acc[e];
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int w = 1; w < W; ++w)
#pragma unroll
            for (int e = 0; e < DL; ++e) acc[e] += red[w][DL * lane + e];
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

// Shares: no more than there can be units for.
Plan8 plan8(const dtattn_decode_fp8_args* a, int64_t capacity, int cus) {
    Plan8 r;
    r.kernel_d = a->D <= 64 ? 64 : 128;
    r.nsub = (int32_t)((a->Hq / a->Hkv + 15) / 16);
    const int64_t units = a->B * a->Hkv * r.nsub * ((capacity + kUnit8 - 1) / kUnit8);
    r.shares = (int32_t)std::max<int64_t>(1, std::min<int64_t>(kSharesPerCu * (int64_t)cus, units / kShareLeast));
    const size_t records = (size_t)2 * r.shares * 16;
    r.bytes = (records * (r.kernel_d + 1) * sizeof(float) + 255) & ~(size_t)255;
    return r;
}

int64_t capacity_of(const dtattn_decode_fp8_args* a) { return a->block_table != nullptr ? a->max_pages * a->page_size : a->S_max; }

template <typename T, int D>
int launch8(const Decode8Params& p, hipStream_t stream) {
    const dim3 grid((unsigned)p.shares);
    if (p.block_table == nullptr) hipLaunchKernelGGL((decode_fp8_kernel<T, D, 0>), grid, dim3(64 * kWaves8), 0, stream, p);
    else if ((1 << p.page_shift) >= kUnit8) hipLaunchKernelGGL((decode_fp8_kernel<T, D, 1>), grid, dim3(64 * kWaves8), 0, stream, p);
    else hipLaunchKernelGGL((decode_fp8_kernel<T, D, 2>), grid, dim3(64 * kWaves8), 0, stream, p);
    const int st = check_launch("decode_fp8_kernel");
    if (st != DTATTN_OK) return st;
    const int64_t pairs = (int64_t)p.B * p.Hq;
    // Few pairs are cut into many records each: four waves to a pair.  us with four and with one at 32 pairs 12.8 and 14.4, 256 21.3
    // and 21.9, 512 30.6 and 30.1, 1024 50.0 and 48.6.
    if (pairs <= 256) hipLaunchKernelGGL((decode_fp8_merge_kernel<T, D, 4>), dim3((unsigned)pairs), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((decode_fp8_merge_kernel<T, D, 1>), dim3((unsigned)((pairs + 3) / 4)), dim3(256), 0, stream, p);
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
    if (a->B * a->Hq > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
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
