// Decode attention by parts: the kernel that decode_shared.hip and decode_blocks.hip instantiate for a prefix that sequences share, for
// their own tokens behind it, and for listed blocks of tokens; and the kernel that merges what its shares leave.
//
// A part is a set of segments, (column set, sequence or group) pairs with a number of 32-token units each.  All units are laid end to
// end, each segment's behind places that stand for its own cost, and cut in equal shares, one per workgroup, whose four waves take its
// units in turn and meet in LDS where a segment ends.
// A segment's columns are query rows that read the same keys: the query heads of a kv head (a sequence's own tokens and listed blocks), or
// those of all sequences of a group (the prefix), 16 of them a set, or 64 and 128 where the prefix is read by rows.
//
// K and V go from memory to registers to matrix operands, without LDS.  Keys are the matrix rows: a lane loads 16-byte pieces of one
// key, in an order of the head dims that the query shares.  Scores come out with a lane's four keys of a tile in registers, which is
// where the second product wants P, and a lane's values of eight (16-bit) or four (fp32) tokens are its other operand: for 16 bits
// pairs of tokens are put side by side by v_perm, 4 D / 128 of them per token and lane.
//
// P in 16-bit types is two numbers, its rounding and the remainder's, so that the output is rounded once: P rounded to bf16 would add
// as much again (error of O against 64 bits 1.7e-3 of its size with the remainder, which is that of the output's rounding, and
// 2.4e-3 without).  For fp16 P is 2^15 times larger, whose subnormals begin at 2^-29 of the largest P.
#pragma once
#include "decode_params.hpp"
#include "fp8_cache.hpp"

namespace dtattn {

enum PartKind { kPrefixPart = 0, kOwnPart = 1, kListPart = 2 };

struct PartsParams {
    const char* q;
    char* o;
    float* lse;
    // [0]: a padded cache's prefix; [1]: the cache (or pool of pages)
    const char* k[2];
    const char* v[2];
    int64_t k_b[2], k_h[2], k_s[2], v_b[2], v_h[2], v_s[2];  // bytes: (sequence, group | page), head, row
    const int32_t* table;  // NULL: padded
    const int32_t* lengths;
    const int32_t* prefix;
    const int32_t* list;
    // [0]: prefix, [1]: own tokens or listed blocks
    float* rec_o[2];    // [2 * shares, columns, kernel D]: segments that a share cuts (its first and its last)
    float2* rec_ml[2];
    float* whole_o[2];  // [B, Hq, kernel D]: segments inside one share
    float2* whole_ml[2];
    int32_t* meta[2];   // places of a column set, and the shares; then of each group or sequence: places before it, and its units
    int32_t nsub[2], columns[2];  // column sets of a kv head; columns of a set
    int32_t shares;     // of both parts, or of the listed blocks, at most
    int32_t weight[2];  // what a unit of each part costs
    int32_t capacity[2];
    int64_t q_b, q_h, o_b, o_h, lse_b, bt_s, list_b, list_h;  // elements
    int32_t B, Hq, Hkv, group, groups, per;  // per: sequences of a group
    int32_t page_shift, num_pages;
    int32_t n_list, list_units, block_shift;
    int32_t d;
    float c;  // scale * log2(e)
    float per_inv;
    uint32_t q_and, q_xor;
};

namespace {

constexpr int kPartUnit = 32;  // tokens
constexpr int kPartWaves = 4;
// Places of a share, at least: a unit for each wave.  us with 4, with 5 (a second turn for one wave) and with 2: 4 samples of one prompt 16.1,
// 16.7 and 17.9, 2048 listed tokens of one sequence (scores and choice included) 21.6, 22.9 and 22.0.
constexpr int kPartLeast = kPartWaves;
constexpr int kPartGroups = 1024;
// What a segment costs besides its units, in units: its waves meet, and the last of them take turns that others have no unit for.  64
// sequences of one or two tokens behind 8192 take 62.5 us with 0 and 48.7 with 4.
constexpr int kPartExtra = 4;

// V places in `n` shares of V / n or one more (all the longer ones first); the host keeps V below 2^31.
struct PartShares {
    int n, q, rem;
    __device__ __forceinline__ PartShares(int n_, int q_, int rem_) : n(n_), q(q_), rem(rem_) {}
    __device__ __forceinline__ PartShares(int V, int most) {
        n = max(1, min(most, V / kPartLeast));
        q = V / n;
        rem = V - q * n;
    }
    __device__ __forceinline__ int start(int r) const { return r * q + min(r, rem); }
    __device__ __forceinline__ int of(int x) const {  // the share of place x
        const int big = rem * (q + 1);
        const bool longer = x < big;
        return (longer ? 0 : rem) + (longer ? x : x - big) / (longer ? q + 1 : q);
    }
};

template <typename T>
struct PartType {  // 16 bits
    typedef typename Elem<T>::vec8 vec8;
    static constexpr int parts = 2;
    static constexpr float offset = __is_same(T, f16_t) ? 15.f : 0.f;  // log2 of what P is multiplied by
};
template <>
struct PartType<float> {
    typedef u32x4 vec8;  // not used
    static constexpr int parts = 1;
    static constexpr float offset = 0.f;
};

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

}  // namespace

__device__ __forceinline__ int part_clamp(int n, int most) { return min(max(n, 0), most); }

// The group of sequence z.  Below 2^20 the float quotient is off by less than its distance of 0.5 / per from a whole number.
__device__ __forceinline__ int part_group(const PartsParams& p, int z) {
    if (p.groups == 1) return 0;
    return z < (1 << 20) ? (int)(((float)z + 0.5f) * p.per_inv) : z / p.per;
}

// What both parts of a shared call need to know of the lengths.
struct PartLengths {
    // LDS, paged: of each group the least tokens of its sequences with tokens, the first of those, and what it is said to share
    int* least;
    int* lead;
    int* said;
    int own0, pre0;  // this lane's of the first 64 lengths and prefixes

    // Tokens that a group of a paged cache shares: whole pages that each of its sequences with tokens has.
    __device__ __forceinline__ int shared(const PartsParams& p, int g) const {
        const int n = least[g] == 0x7fffffff ? 0 : min(least[g], said[g]);
        return n >> p.page_shift << p.page_shift;
    }
};

__device__ __forceinline__ PartLengths part_lengths(const PartsParams& p, int* least, int* lead, int* said) {
    const int tid = threadIdx.x, lane = tid & 63;
    PartLengths r = {least, lead, said, 0, 0};
    r.own0 = lane < p.B ? p.lengths[lane] : 0;
    r.pre0 = lane < p.groups ? p.prefix[lane] : 0;
    if (p.table != nullptr) {
        for (int g = tid; g < p.groups; g += 256) least[g] = lead[g] = 0x7fffffff;
        for (int g = tid; g < p.groups; g += 256) said[g] = max(g < 64 ? r.pre0 : p.prefix[g], 0);
        __syncthreads();
        for (int b = tid; b < p.B; b += 256) {
            const int n = part_clamp(b < 64 ? r.own0 : p.lengths[b], p.capacity[1]);
            if (n > 0) {
                const int g = part_group(p, b);
                atomicMin(&least[g], n);
                atomicMin(&lead[g], b);
            }
        }
        __syncthreads();
    }
    r.own0 = part_clamp(r.own0, p.capacity[1]);
    r.pre0 = part_clamp(r.pre0, p.capacity[0]);
    return r;
}

// Units of group or sequence z, per lane (z = lane or beyond the first 64).
template <int KIND>
__device__ __forceinline__ int part_units(const PartsParams& p, const PartLengths& at, int z) {
    const bool paged = p.table != nullptr;
    int n;
    if constexpr (KIND == kPrefixPart) n = paged ? at.shared(p, z) : z < 64 ? at.pre0 : part_clamp(p.prefix[z], p.capacity[0]);
    else n = (z < 64 ? at.own0 : part_clamp(p.lengths[z], p.capacity[1])) - (paged ? at.shared(p, part_group(p, z)) : 0);
    return (max(n, 0) + kPartUnit - 1) / kPartUnit;
}

// Places of units and of what segments cost besides.
__device__ __forceinline__ int part_places(int units) { return units > 0 ? units + kPartExtra : 0; }

// The first 64 groups or sequences, one a lane: units, and sums of places and of units up to them.
struct PartScan {
    int units, places, sum;
};
template <int KIND>
__device__ __forceinline__ PartScan part_scan(const PartsParams& p, const PartLengths& at, int j0) {
    const int lane = threadIdx.x & 63;
    PartScan r;
    r.units = j0 + lane < (KIND == kPrefixPart ? p.groups : p.B) ? part_units<KIND>(p, at, j0 + lane) : 0;
    r.places = scan64(part_places(r.units));
    r.sum = scan64(r.units);
    return r;
}

// Places of all groups or sequences; the wave that `tells` leaves them for the merge.
template <int KIND>
__device__ __forceinline__ int part_total(const PartsParams& p, const PartLengths& at, bool tells, PartScan& first) {
    const int Z = KIND == kPrefixPart ? p.groups : p.B, lane = threadIdx.x & 63;
    int32_t* meta = p.meta[KIND == kPrefixPart ? 0 : 1];
    int U = 0;
    for (int j0 = 0; j0 < Z; j0 += 64) {
        const PartScan s = part_scan<KIND>(p, at, j0);
        if (j0 == 0) first = s;
        if (tells && j0 + lane < Z) {
            meta[4 + 2 * (j0 + lane)] = U + s.places - part_places(s.units);
            meta[5 + 2 * (j0 + lane)] = s.units;
        }
        U += __builtin_amdgcn_readlane(s.places, 63);
    }
    return U;
}

// Walks the units of one part.  Lengths, page ids and lists are scalar loads, which leave the vector loads in flight alone.
// NR: tiles of a unit that are found apart.
template <int KIND, int NR>
struct PartWalk {
    static constexpr int S = KIND == kPrefixPart ? 0 : 1;
    typedef const __attribute__((address_space(4))) int32_t cint32;
    struct At {              // a unit
        int slot, hk, z;     // slot: kv head * nsub + column set
        int u, units;        // of the segment
        int start, end, row; // the segment's tokens; its row of the table
        int t[NR], rows[NR], page[NR];
    };
    const PartsParams& p;
    const PartLengths& lens;
    const PartScan& scan0;
    const int U, Z;
    const bool paged;

    __device__ __forceinline__ PartWalk(const PartsParams& p_, const PartLengths& lens_, const PartScan& scan0_, int U_)
        : p(p_), lens(lens_), scan0(scan0_), U(U_), Z(KIND == kPrefixPart ? p_.groups : p_.B), paged(p_.table != nullptr) {}

    // a segment's tokens: from `start` to before `end`
    __device__ __forceinline__ int start_of(int z) const {
        return KIND == kOwnPart && paged ? __builtin_amdgcn_readfirstlane(lens.shared(p, part_group(p, z))) : 0;
    }
    __device__ __forceinline__ int end_of(int z) const {
        if constexpr (KIND == kPrefixPart) {
            if (paged) return __builtin_amdgcn_readfirstlane(lens.shared(p, z));
            return z < 64 ? __builtin_amdgcn_readlane(lens.pre0, z) : part_clamp(((cint32*)p.prefix)[z], p.capacity[0]);
        } else {
            return KIND == kOwnPart && z < 64 ? __builtin_amdgcn_readlane(lens.own0, z) : part_clamp(((cint32*)p.lengths)[z], p.capacity[1]);
        }
    }
    __device__ __forceinline__ void enter(At& a) const {
        a.hk = p.nsub[S] == 1 ? a.slot : a.slot / p.nsub[S];
        a.start = start_of(a.z);
        a.end = end_of(a.z);
        a.units = KIND == kListPart ? p.list_units : (max(a.end - a.start, 0) + kPartUnit - 1) / kPartUnit;
        a.row = KIND == kPrefixPart && paged && a.units > 0 ? __builtin_amdgcn_readfirstlane(lens.lead[a.z]) : a.z;
    }
    // The next segment with units.  There is one, unless somebody changes the lengths meanwhile, which must cost no more than the results:
    // behind the last segment lie units without tokens.
    __device__ __forceinline__ void next(At& a) const {
        do {
            if (++a.z == Z) {
                a.z = 0;
                if (++a.slot == p.Hkv * p.nsub[S]) {
                    --a.slot;
                    a.start = a.end = 0, a.units = 1 << 30;
                    return;
                }
            }
            enter(a);
        } while (a.units == 0);
    }
    __device__ __forceinline__ void advance(At& a, int k) const {
        a.u += k;
        while (a.u >= a.units) {
            a.u -= a.units;
            next(a);
        }
    }
    // The tokens of a unit's tile i, from `skip` on, of up to `most`; and the page that holds them.
    __device__ __forceinline__ void find_tile(At& a, int i, int skip, int most) const {
        cint32* const list = (cint32*)p.list;
        const int x = a.u * kPartUnit + skip;
        if constexpr (KIND == kListPart) {
            const int e = x >> p.block_shift;
            const int j = e < p.n_list ? list[a.z * p.list_b + a.hk * p.list_h + e] : -1;
            const bool there = (uint32_t)j < (uint32_t)((a.end + (1 << p.block_shift) - 1) >> p.block_shift);
            a.t[i] = there ? (j << p.block_shift) + (x & ((1 << p.block_shift) - 1)) : 0;
            a.rows[i] = there ? part_clamp(a.end - a.t[i], most) : 0;
        } else {
            a.t[i] = a.start + x;
            a.rows[i] = part_clamp(a.end - a.t[i], most);
            if (a.rows[i] == 0) a.t[i] = 0;
        }
        a.page[i] = paged ? ((cint32*)p.table)[a.row * p.bt_s + (a.t[i] >> p.page_shift)] : a.z;
    }
    __device__ __forceinline__ void find(At& a) const {
#pragma unroll
        for (int i = 0; i < NR; ++i) find_tile(a, i, 16 * i, kPartUnit / NR);
    }
    // The first row of a tile.
    __device__ __forceinline__ const char* base(const At& a, int i, const char* x, int64_t sb, int64_t s_h, int64_t ss) const {
        const int64_t where = paged ? part_clamp(a.page[i], p.num_pages - 1) : a.page[i];
        const int row = paged ? a.t[i] & ((1 << p.page_shift) - 1) : a.t[i];
        return x + where * sb + a.hk * s_h + row * ss;
    }
    // The first unit at or behind a place, and its index among all.
    __device__ __forceinline__ int locate(int place, At& a) const {
        a.slot = place / U;
        int x = place - a.slot * U, before;
        if constexpr (KIND == kListPart) {
            const int each = part_places(p.list_units);
            a.z = x / each;
            x -= a.z * each;
            before = (a.slot * p.B + a.z) * p.list_units;
        } else {
            int total = 0, left = 0;  // units of all groups or sequences, and of those before z
            bool found = false;
            a.z = Z - 1;
            for (int j0 = 0; j0 < Z; j0 += 64) {
                const PartScan s = j0 == 0 ? scan0 : part_scan<KIND>(p, lens, j0);
                const uint64_t hit = __ballot(s.places > x);  // segments ending past x
                if (!found && hit != 0) {
                    const int l = __builtin_ctzll(hit);
                    found = true;
                    a.z = j0 + l;
                    left = total + __builtin_amdgcn_readlane(s.sum - s.units, l);
                    x -= __builtin_amdgcn_readlane(s.places - part_places(s.units), l);
                } else if (!found) {
                    x -= __builtin_amdgcn_readlane(s.places, 63);
                }
                total += __builtin_amdgcn_readlane(s.sum, 63);
            }
            before = a.slot * total + left;
        }
        a.u = max(x - kPartExtra, 0);
        return before + a.u;
    }
    // A share's first unit, and how many it has.
    __device__ __forceinline__ int units(const PartShares& sh, int r, At& a) const {
        const int all = U * p.Hkv * p.nsub[S], end = sh.start(r + 1);
        At behind;
        const int u0 = locate(sh.start(r), a);
        const int n = (end < all ? locate(end, behind) : locate(all - 1, behind) + 1) - u0;
        // said to be the same in every lane, so that what follows from them stays in scalar registers
        a.slot = __builtin_amdgcn_readfirstlane(a.slot), a.z = __builtin_amdgcn_readfirstlane(a.z), a.u = __builtin_amdgcn_readfirstlane(a.u);
        return __builtin_amdgcn_readfirstlane(n);
    }
    __device__ __forceinline__ int rows_of_head() const { return KIND == kPrefixPart ? p.per * p.group : p.group; }
    // The sequence and head of a segment's row.
    __device__ __forceinline__ void where(int z, int hk, int row, int& b, int& hq) const {
        const int i = KIND == kPrefixPart ? row / p.group : 0;
        b = KIND == kPrefixPart ? z * p.per + i : z;
        hq = hk * p.group + row - i * p.group;
    }
};

// A row of the query, in pieces of 16 bytes whose order the keys share: piece 4 k + lane / 16 in w[k].
template <typename T, int NK>
__device__ __forceinline__ void part_query(const PartsParams& p, int b, int hq, u32x4 (&w)[NK]) {
    const int g4 = (threadIdx.x & 63) >> 4, row_bytes = p.d * (int)sizeof(T);
    const char* qp = p.q + (b * p.q_b + hq * p.q_h) * (int64_t)sizeof(T);
#pragma unroll
    for (int k = 0; k < NK; ++k) {
        const int at16 = 16 * (4 * k + g4);
        w[k] = ld16(qp + (at16 < row_bytes ? at16 : 0));
    }
}
// The same once it has arrived: signed, and zeros past the head dim.
template <typename T, int NK>
__device__ __forceinline__ void part_query_bits(const PartsParams& p, u32x4 (&w)[NK]) {
    const int g4 = (threadIdx.x & 63) >> 4, row_bytes = p.d * (int)sizeof(T);
#pragma unroll
    for (int k = 0; k < NK; ++k) w[k] = 16 * (4 * k + g4) < row_bytes ? q_bits(w[k], p.q_and, p.q_xor) : u32x4{0u, 0u, 0u, 0u};
}

// The running maxima of NC sets of columns rise to those of NT tiles' scores; what was summed on the old base is scaled to the new one.
template <int NC, int NT, int DPL>
__device__ __forceinline__ void part_rise(const f32x4 (&sc)[NC][NT], float scale, float (&M)[NC], float (&l)[NC], f32x4 (&acc)[NC][DPL]) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float mx = kNegInf;
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) mx = fmaxf(mx, fmaxf(fmaxf(sc[c][tt][0], sc[c][tt][1]), fmaxf(sc[c][tt][2], sc[c][tt][3])));
        const float Mn = fmaxf(M[c], max_across_groups<16>(mx) * scale);
        const float alpha = fast_exp2(M[c] - (Mn == kNegInf ? 0.f : Mn));
        M[c] = Mn;
        l[c] *= alpha;
#pragma unroll
        for (int j = 0; j < DPL; ++j) acc[c][j] *= alpha;
    }
}

// P of a unit's scores in one set of columns, as numbers and (16 bits) as two matrix operands, and its part of the row sum.
template <typename T>
__device__ __forceinline__ void part_weights(const f32x4* sc, float scale, float M, float& l, float (&pf)[8],
                                             typename PartType<T>::vec8 (&pk)[PartType<T>::parts]) {
    const float base = (M == kNegInf ? 0.f : M) - PartType<T>::offset;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        pf[i] = fast_exp2(__builtin_fmaf(sc[i >> 2][i & 3], scale, -base));
        l += pf[i];
    }
    if constexpr (sizeof(T) == 2) {
        // two at a time: one conversion rounds a pair
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            hi[i] = pack2<T>(pf[2 * i], pf[2 * i + 1]);
            float a, b;
            if constexpr (__is_same(T, bf16_t)) {
                a = __builtin_bit_cast(float, hi[i] << 16), b = __builtin_bit_cast(float, hi[i] & 0xffff0000u);
            } else {
                const f16x2 h = __builtin_bit_cast(f16x2, hi[i]);
                a = (float)h[0], b = (float)h[1];
            }
            lo[i] = pack2<T>(pf[2 * i] - a, pf[2 * i + 1] - b);
        }
        pk[0] = __builtin_bit_cast(typename PartType<T>::vec8, u32x4{hi[0], hi[1], hi[2], hi[3]});
        pk[1] = __builtin_bit_cast(typename PartType<T>::vec8, u32x4{lo[0], lo[1], lo[2], lo[3]});
    }
}

// Share r of the segments of one part, U places in each of Hkv * nsub column sets.
// TWO: a unit's two tiles of 16 tokens may lie apart (pages or blocks of 16 tokens).
template <typename T, int D, int KIND, bool TWO>
__device__ void decode_part(const PartsParams& p, const PartLengths& lens, const PartScan& scan0, int U, const PartShares& sh, int r, float (*red_o)[16][D + 4],
                            float (*red_m)[16], float (*red_l)[16]) {
    typedef typename PartType<T>::vec8 V8;
    constexpr bool kF32 = sizeof(T) == 4;
    constexpr int S = KIND == kPrefixPart ? 0 : 1;
    constexpr int NK = D * (int)sizeof(T) / 64;  // 16-byte loads of a key per lane
    constexpr int DPL = D / 16;                  // dims of a token's values per lane
    constexpr int VW = DPL * (int)sizeof(T) / 4; // words of them
    constexpr int NR = TWO ? 2 : 1;              // buffer resources of a unit
    constexpr int PP = PartType<T>::parts;
    // Sums of an fp32 score, as many as there are registers for: one chain of D products is off by more (O against 64 bits 5.4e-7 of its size
    // with one sum, 2.8e-7 with four, D = 64).
    constexpr int SUMS = D == 64 ? 4 : 2;
    constexpr float kOff = PartType<T>::offset;
    typedef PartWalk<KIND, NR> Walk;
    typedef typename Walk::At At;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g4 = lane >> 4;
    const Walk walk(p, lens, scan0, U);
    At at;
    const int n = walk.units(sh, r, at);  // units of this workgroup
    if (n == 0) return;
    walk.enter(at);

    // byte offsets of this lane's loads from a tile's first row; pieces past the real head dim lie past any resource
    const int row_bytes = p.d * (int)sizeof(T);
    const uint32_t kp = (uint32_t)p.k_s[S], vp = (uint32_t)p.v_s[S];
    uint32_t koff[NK], voff[4];
#pragma unroll
    for (int k = 0; k < NK; ++k) koff[k] = 16 * (4 * k + g4) < row_bytes ? (uint32_t)col * kp + (uint32_t)(16 * (4 * k + g4)) : 0xc0000000u;
#pragma unroll
    for (int e = 0; e < 4; ++e) voff[e] = 4 * VW * col < row_bytes ? (uint32_t)(4 * g4 + e) * vp + (uint32_t)(4 * VW * col) : 0xc0000000u;
    const uint32_t vsecond = 4 * VW * col + 16 < row_bytes ? 16u : 0xc0000000u;  // fp32, D = 128: the lane's second piece

    u32x4 kr[2][NK];
    uint32_t vr[8][VW];
    auto ld16b = [&](__amdgpu_buffer_rsrc_t rs, uint32_t off) { return KIND == kPrefixPart ? buf_ld16(rs, off) : buf_ld16_nt(rs, off); };
    auto load_k = [&](const At& a) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const auto rs = make_rsrc(walk.base(a, i, p.k[S], p.k_b[S], p.k_h[S], p.k_s[S]), a.rows[i] > 0 ? (uint32_t)(a.rows[i] - 1) * kp + (uint32_t)row_bytes : 0u);
#pragma unroll
            for (int tt = TWO ? i : 0; tt < (TWO ? i + 1 : 2); ++tt)
#pragma unroll
                for (int k = 0; k < NK; ++k) kr[tt][k] = ld16b(rs, koff[k] + (TWO ? 0u : 16u * tt * kp));
        }
    };
    auto load_v = [&](const At& a) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const auto rs = make_rsrc(walk.base(a, i, p.v[S], p.v_b[S], p.v_h[S], p.v_s[S]), a.rows[i] > 0 ? (uint32_t)(a.rows[i] - 1) * vp + (uint32_t)row_bytes : 0u);
#pragma unroll
            for (int tt = TWO ? i : 0; tt < (TWO ? i + 1 : 2); ++tt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t off = voff[e] + (TWO ? 0u : 16u * tt * vp);
                    uint32_t* w = vr[4 * tt + e];
                    if constexpr (VW == 2) {
                        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, off, 0, KIND == kPrefixPart ? 0 : 2));
                        w[0] = v.x, w[1] = v.y;
                    } else {
#pragma unroll
                        for (int h = 0; h < VW / 4; ++h) {
                            const u32x4 v = ld16b(rs, h == 0 ? off : off + vsecond);
                            w[4 * h] = v.x, w[4 * h + 1] = v.y, w[4 * h + 2] = v.z, w[4 * h + 3] = v.w;
                        }
                    }
                }
        }
    };

    f32x4 acc[1][DPL];
    float M[1], l[1];  // running max, and this lane's part of the row sum on that base
    u32x4 qf[NK];
    At cur = at, nx = at;
    if (wave < n) {
        if (wave > 0) walk.advance(nx, wave);
        walk.find(nx);
        load_k(nx);
        load_v(nx);
    }
    const int R = walk.rows_of_head();
    auto load_q = [&](const At& a) {
        int b, hq;
        walk.where(a.z, a.hk, min(16 * (a.slot - a.hk * p.nsub[S]) + col, R - 1), b, hq);
        part_query<T, NK>(p, b, hq, qf);
    };
    load_q(cur);
    int s = wave;  // this wave's next unit of the share
    for (int u = 0; u < n;) {
        const int m = max(min(cur.units - cur.u, n - u), 1);  // units of the segment
        const int hk = cur.hk, z = cur.z, R0 = 16 * (cur.slot - hk * p.nsub[S]);
        const bool whole = cur.u == 0 && m == cur.units;
        bool seen = false;
        M[0] = kNegInf, l[0] = 0.f;
#pragma unroll
        for (int j = 0; j < DPL; ++j) acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        part_query_bits<T, NK>(p, qf);
        for (; s < u + m; s += kPartWaves) {
            int rows[NR];
#pragma unroll
            for (int i = 0; i < NR; ++i) rows[i] = nx.rows[i], seen |= rows[i] > 0;
            const bool more = s + kPartWaves < n;
            if (more) {
                walk.advance(nx, kPartWaves);
                walk.find(nx);
            }
            f32x4 sc[1][2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                sc[0][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
                f32x4 part[SUMS] = {};
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    if constexpr (kF32) {
                        const f32x4 kf = __builtin_bit_cast(f32x4, kr[tt][k]), q = __builtin_bit_cast(f32x4, qf[k]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) part[e % SUMS] = mfma_f32(kf[e], q[e], part[e % SUMS]);
                    } else {
                        sc[0][tt] = mfma16(__builtin_bit_cast(V8, kr[tt][k]), __builtin_bit_cast(V8, qf[k]), sc[0][tt]);
                    }
                }
                if constexpr (kF32) {
#pragma unroll
                    for (int e = 0; e < SUMS; ++e) sc[0][tt] += part[e];
                }
            }
            if (more) load_k(nx);  // the keys are used up
            if (rows[0] < kPartUnit / NR || (TWO && rows[NR - 1] < 16)) {
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if ((TWO ? 0 : 16 * tt) + 4 * g4 + i >= rows[TWO ? tt : 0]) sc[0][tt][i] = kNegInf;
            }
            part_rise(sc, p.c, M, l, acc);
            V8 pk[PP];
            float pf[8];
            if constexpr (kF32) {
                part_weights<T>(sc[0], p.c, M[0], l[0], pf, pk);
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int j = 0; j < DPL; ++j) acc[0][j] = mfma_f32(__builtin_bit_cast(float, vr[i][j]), pf[i], acc[0][j]);
                if (more) load_v(nx);
            } else {
                // two tokens' values of one dim side by side, all of them, so that the values' registers take the next unit's at once
                V8 vf[DPL];
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    uint32_t a[4], b[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        a[t] = __builtin_amdgcn_perm(vr[2 * t + 1][w], vr[2 * t][w], 0x05040100u);
                        b[t] = __builtin_amdgcn_perm(vr[2 * t + 1][w], vr[2 * t][w], 0x07060302u);
                    }
                    vf[2 * w] = __builtin_bit_cast(V8, u32x4{a[0], a[1], a[2], a[3]});
                    vf[2 * w + 1] = __builtin_bit_cast(V8, u32x4{b[0], b[1], b[2], b[3]});
                }
                if (more) load_v(nx);
                part_weights<T>(sc[0], p.c, M[0], l[0], pf, pk);
#pragma unroll
                for (int h = 0; h < PP; ++h)
#pragma unroll
                    for (int j = 0; j < DPL; ++j) acc[0][j] = mfma16(vf[j], pk[h], acc[0][j]);
            }
        }
        // the next segment's query is on its way while this one's waves meet
        const bool cut_first = u == 0;
        u += m;
        if (u < n) {
            cur.u = 0;
            walk.next(cur);
            load_q(cur);
        }
        // the waves meet
        const bool any = KIND != kListPart || __syncthreads_or(seen);
        const int heads = min(R - R0, 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float* at_o = &red_o[wave][col][DPL * (4 * g4 + i)];
#pragma unroll
            for (int j = 0; j < DPL; j += 4) *reinterpret_cast<f32x4*>(at_o + j) = f32x4{acc[0][j][i], acc[0][j + 1][i], acc[0][j + 2][i], acc[0][j + 3][i]};
        }
        const float lw = sum_across_groups<16>(l[0]);
        if (g4 == 0) red_m[wave][col] = M[0], red_l[wave][col] = lw;
        lds_barrier();
        const int g = tid >> 4;  // a column, and DPL of its dims
        if (g < heads) {
            float X = kNegInf, lt = 0.f, o[DPL] = {};
#pragma unroll
            for (int w = 0; w < kPartWaves; ++w) X = fmaxf(X, red_m[w][g]);
#pragma unroll
            for (int w = 0; w < kPartWaves; ++w) {
                const float mw = red_m[w][g];
                const float f = mw == kNegInf ? 0.f : fast_exp2(mw - X);
                lt = __builtin_fmaf(red_l[w][g], f, lt);
#pragma unroll
                for (int j = 0; j < DPL; j += 4) {
                    const f32x4 a = *reinterpret_cast<const f32x4*>(&red_o[w][g][DPL * (tid & 15) + j]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[j + i] = __builtin_fmaf(a[i], f, o[j + i]);
                }
            }
            int b, hq;
            walk.where(z, hk, R0 + g, b, hq);
            const int dim = DPL * (tid & 15);
            if (KIND == kListPart && whole) {
                const float inv = any ? 1.f / lt : 0.f;
#pragma unroll
                for (int j = 0; j < DPL; ++j) o[j] *= inv;
                T* op = reinterpret_cast<T*>(p.o) + b * p.o_b + hq * p.o_h + dim;
#pragma unroll
                for (int j = 0; j < DPL; j += 4)
                    if (dim + j < p.d) {
                        if constexpr (kF32) *reinterpret_cast<f32x4*>(op + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
                        else *reinterpret_cast<u32x2*>(op + j) = u32x2{pack2<T>(o[j], o[j + 1]), pack2<T>(o[j + 2], o[j + 3])};
                    }
                if (p.lse != nullptr && (tid & 15) == 0) p.lse[b * p.lse_b + hq] = __builtin_fmaf(X - kOff, kLn2, __log2f(lt) * kLn2);
            } else {
                const int64_t rec = whole ? (int64_t)b * p.Hq + hq : (int64_t)(2 * r + (cut_first ? 0 : 1)) * 16 + g;
                float* op = (whole ? p.whole_o[S] : p.rec_o[S]) + rec * D + dim;
#pragma unroll
                for (int j = 0; j < DPL; j += 4) *reinterpret_cast<f32x4*>(op + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
                if ((tid & 15) == 0) (whole ? p.whole_ml[S] : p.rec_ml[S])[rec] = make_float2(X - kOff, lt);
            }
        }
        if (u < n) lds_barrier();  // every wave has read the others' before they write again
    }
}

// 16-byte chunk c of row r of a tile in LDS lies at c ^ part_swizzle(r): without bank conflicts for the 16-byte reads of keys (16 rows, one
// chunk) and the 8-byte transposed ones of values (rows 16 apart alike).
template <int D>
__device__ __forceinline__ int part_swizzle(int r) { return D == 128 ? 2 * (r & 7) + ((r >> 3) & 1) : (r >> 1) & 7; }

// Share r of the prefix for many rows (16-bit types): the four waves hold 16 NC rows each, and keys and values go through LDS once for all
// of them, two units a stage, by direct loads into one of two buffers while the other is worked on.  A unit then costs a wave a third of
// the instructions of the form above: no addresses of its own, no pairing of values, which a transposed read replaces, and one
// rescaling for two units.
constexpr int kStageTokens = 2 * kPartUnit;

template <typename T, int D, int NC>
__device__ void decode_part_rows(const PartsParams& p, const PartLengths& lens, const PartScan& scan0, int U, const PartShares& sh, int r,
                                 T (*kv)[2][kStageTokens * D]) {
    typedef typename Elem<T>::vec8 V8;
    typedef typename Elem<T>::vec4 V4;
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    typedef PartWalk<kPrefixPart, 1> Walk;
    typedef typename Walk::At At;
    constexpr int NK = D / 32, NV = D / 16, CH = D / 8, RPL = 64 / CH, NL = 16 / RPL;  // CH: chunks of a row; a wave's 16 rows: NL loads of RPL
    constexpr int NT = kStageTokens / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g4 = lane >> 4;
    const Walk walk(p, lens, scan0, U);
    At cur;
    const int n = walk.units(sh, r, cur);
    if (n == 0) return;
    walk.enter(cur);

    // each wave loads a tile of a stage
    const uint32_t kp = (uint32_t)p.k_s[0], vp = (uint32_t)p.v_s[0];
    uint32_t koff[NL], voff[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int row = RPL * i + lane / CH, c = (lane % CH) ^ part_swizzle<D>(row);
        const bool there = 8 * c < p.d;  // chunks past the real head dim come as zeros
        koff[i] = there ? (uint32_t)row * kp + (uint32_t)(16 * c) : 0xc0000000u;
        voff[i] = there ? (uint32_t)row * vp + (uint32_t)(16 * c) : 0xc0000000u;
    }
    // the stage to be loaded next: its units lie in one segment
    At nx = cur;
    int nx_left = n;                                   // units of the share from it on
    int nx_here = max(min(cur.units - cur.u, nx_left), 1);  // of its segment
    // 64 page ids from page `ids_from` of row `ids_row` on, one a lane: a scalar load a stage would be waited for before its first key
    int ids = 0, ids_from = 0, ids_row = -1;
    auto issue = [&](int buf) {
        // a second unit that is not there is loaded as no rows
        const int t = nx.u * kPartUnit + 16 * wave;
        nx.rows[0] = wave < 2 || nx_here > 1 ? part_clamp(nx.end - t, 16) : 0;
        nx.t[0] = nx.rows[0] > 0 ? t : 0;
        nx.page[0] = nx.z;
        if (walk.paged) {
            const int page = nx.t[0] >> p.page_shift, first = (nx.u * kPartUnit) >> p.page_shift;  // of this wave's tile, and of the unit
            if (nx.row != ids_row || first < ids_from || first + 4 > ids_from + 64) {
                ids_row = nx.row, ids_from = first;
                const int64_t at = (int64_t)(p.capacity[0] >> p.page_shift) - 1;
                ids = p.table[nx.row * p.bt_s + min((int64_t)first + lane, at)];
            }
            if (nx.rows[0] > 0) nx.page[0] = __builtin_amdgcn_readlane(ids, page - ids_from);
        }
        const uint32_t row_bytes = (uint32_t)(p.d * (int)sizeof(T));
        const auto krs = make_rsrc(walk.base(nx, 0, p.k[0], p.k_b[0], p.k_h[0], p.k_s[0]), nx.rows[0] > 0 ? (uint32_t)(nx.rows[0] - 1) * kp + row_bytes : 0u);
        const auto vrs = make_rsrc(walk.base(nx, 0, p.v[0], p.v_b[0], p.v_h[0], p.v_s[0]), nx.rows[0] > 0 ? (uint32_t)(nx.rows[0] - 1) * vp + row_bytes : 0u);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            buf_ld16_lds_async(krs, &kv[buf][0][(16 * wave + RPL * i) * D], koff[i]);
            buf_ld16_lds_async(vrs, &kv[buf][1][(16 * wave + RPL * i) * D], voff[i]);
        }
        const int took = min(nx_here, 2);
        nx_left -= took, nx_here -= took, nx.u += took;
        if (nx_here == 0 && nx_left > 0) {
            walk.next(nx);
            nx.u = 0;
            nx_here = min(nx.units, nx_left);
        }
    };
    const int R = walk.rows_of_head();
    u32x4 qf[NC][NK];
    auto row_of = [&](const At& a, int c) { return 16 * NC * (kPartWaves * (a.slot - a.hk * p.nsub[0]) + wave) + 16 * c + col; };
    auto load_q = [&](const At& a) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            int b, hq;
            walk.where(a.z, a.hk, min(row_of(a, c), R - 1), b, hq);
            part_query<T, NK>(p, b, hq, qf[c]);
        }
    };
    load_q(cur);
    issue(0);
    f32x4 acc[NC][NV];
    float M[NC], l[NC];
    int buf = 0;
    for (int u = 0; u < n;) {
        const int m = max(min(cur.units - cur.u, n - u), 1);
        const bool whole = cur.u == 0 && m == cur.units, cut_first = u == 0;
        const At seg = cur;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            M[c] = kNegInf, l[c] = 0.f;
#pragma unroll
            for (int j = 0; j < NV; ++j) acc[c][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            part_query_bits<T, NK>(p, qf[c]);
        }
        for (int i = 0; i < m; i += 2) {
            wait_vmem();    // this wave's loads of the stage have landed
            lds_barrier();  // everybody's have, and the other buffer has been read
            if (nx_left > 0) issue(buf ^ 1);
            const T* K = kv[buf][0];
            const T* V = kv[buf][1];
            f32x4 sc[NC][NT];
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) {
                V8 kf[NK];
#pragma unroll
                for (int k = 0; k < NK; ++k) kf[k] = __builtin_bit_cast(V8, ld16(K + (16 * tt + col) * D + 8 * ((4 * k + g4) ^ part_swizzle<D>(col))));
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    sc[c][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < NK; ++k) sc[c][tt] = mfma16(kf[k], __builtin_bit_cast(V8, qf[c][k]), sc[c][tt]);
                }
            }
            const int left = __builtin_amdgcn_readfirstlane(min(seg.end - seg.start - (seg.u + i) * kPartUnit, (m - i) * kPartUnit));
            if (left < kStageTokens) {
#pragma unroll
                for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (16 * tt + 4 * g4 + e >= left) {
#pragma unroll
                            for (int c = 0; c < NC; ++c) sc[c][tt][e] = kNegInf;
                        }
            }
            part_rise(sc, p.c, M, l, acc);
#pragma unroll
            for (int t2 = 0; t2 < NT / 2; ++t2) {
                V8 pk[NC][2];
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    float pf[8];
                    part_weights<T>(&sc[c][2 * t2], p.c, M[c], l[c], pf, pk[c]);
                }
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int row = 4 * g4 + (col >> 2), ch = (2 * j + ((col & 3) >> 1)) ^ part_swizzle<D>(row);
                    const int off = (32 * t2 + row) * D + 8 * ch + 4 * (col & 1);
                    const V4 lo = __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(V + off)));
                    const V4 hi = __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(V + off + 16 * D)));
                    const V8 vf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int c = 0; c < NC; ++c) acc[c][j] = mfma16(vf, pk[c][h], acc[c][j]);
                }
            }
            buf ^= 1;
        }
        u += m;
        if (u < n) {
            walk.next(cur);
            cur.u = 0;
            load_q(cur);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float lt = sum_across_groups<16>(l[c]);
            const int row = row_of(seg, c);
            if (row < R) {
                int b, hq;
                walk.where(seg.z, seg.hk, row, b, hq);
                const int in_set = 16 * NC * wave + 16 * c + col;
                const int64_t rec = whole ? (int64_t)b * p.Hq + hq : (int64_t)(2 * r + (cut_first ? 0 : 1)) * (16 * NC * kPartWaves) + in_set;
                float* op = (whole ? p.whole_o[0] : p.rec_o[0]) + rec * D + 4 * g4;
#pragma unroll
                for (int j = 0; j < NV; ++j) *reinterpret_cast<f32x4*>(op + 16 * j) = acc[c][j];
                if (g4 == 0) (whole ? p.whole_ml[0] : p.rec_ml[0])[rec] = make_float2(M[c] - PartType<T>::offset, lt);
            }
        }
    }
}

// Merges a query head's records: of the prefix and of its own tokens (SHARED), or of listed blocks that several shares hold.  W waves
// to a (sequence, query head).  A record holds the sum of P V, the maximum that P is based on (times log2 e) and the row sum: an LSE in fp32
// would be off by half a step of its own value, 5e-7 of a weight between 8 and 16.
template <typename T, int D, int W, bool SHARED>
__global__ void __launch_bounds__(256) decode_parts_merge_kernel(const PartsParams p) {
    constexpr int DL = D / 64;  // dims per lane
    __shared__ float red[W > 1 ? W : 1][D + 2];
    const int lane = threadIdx.x & 63, wave = W > 1 ? threadIdx.x >> 6 : 0;
    const int pair = __builtin_amdgcn_readfirstlane(W > 1 ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 6));
    if (pair >= p.B * p.Hq) return;
    const int b = pair / p.Hq, hq = pair - b * p.Hq, hk = hq / p.group, g = hq - hk * p.group;
    struct Part {
        int n;                // records
        int64_t first, later; // that of the part's first share, and of the one behind it
        const float* o;
        const float2* ml;
    };
    auto part = [&](int S, int z, int row) {
        Part r = {0, 0, 0, nullptr, nullptr};
        const int* meta = p.meta[S];
        const int U = SHARED ? meta[0] : p.B * part_places(p.list_units);
        const int before = SHARED ? meta[4 + 2 * z] : b * part_places(p.list_units), own = SHARED ? meta[5 + 2 * z] : p.list_units;
        if (own == 0) return r;
        const int cols = p.columns[S], sub = row / cols;
        const PartShares sh = SHARED ? PartShares(meta[1], meta[2], meta[3]) : PartShares(U * p.Hkv * p.nsub[S], p.shares);
        const int x0 = (hk * p.nsub[S] + sub) * U + before + kPartExtra, r0 = sh.of(x0), r1 = sh.of(x0 + own - 1);
        const bool whole = r0 == r1;
        r.n = r1 - r0 + 1;
        // the segment is share r0's first, unless units of another lie before it there
        r.first = whole ? pair : (int64_t)(2 * r0 + (sh.start(r0) < x0 - kPartExtra ? 1 : 0)) * cols + row - sub * cols;
        r.later = (int64_t)2 * (r0 + 1) * cols + row - sub * cols;
        r.o = whole ? p.whole_o[S] : p.rec_o[S];
        r.ml = whole ? p.whole_ml[S] : p.rec_ml[S];
        return r;
    };
    Part pre = {0, 0, 0, nullptr, nullptr}, own = part(1, b, g);
    if (!SHARED && own.n == 1) return;  // written directly
    if constexpr (SHARED) {
        const int z = b / p.per;
        pre = part(0, z, (b - z * p.per) * p.group + g);
        // a padded prefix is read for every sequence; a paged one holds the first of a sequence's tokens, if it has any
        if (p.table != nullptr && p.lengths[b] <= 0) pre.n = own.n = 0;
    }
    const int n = pre.n + own.n;
    T* op = reinterpret_cast<T*>(p.o) + b * p.o_b + hq * p.o_h;
    float M = kNegInf, sum = 0.f, acc[DL] = {};
    constexpr int MB = 8;  // records in flight
    for (int j0 = wave; j0 < n; j0 += W * MB) {
        float2 ml[MB];
        float v[MB][DL], top = M;
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const int i = min(j0 + W * j, n - 1);
            const bool is_own = !SHARED || i >= pre.n;
            const int k = i - (SHARED && is_own ? pre.n : 0);
            const int64_t q = k == 0 ? (is_own ? own.first : pre.first) : (is_own ? own.later : pre.later) + (int64_t)(k - 1) * 2 * p.columns[is_own ? 1 : 0];
            ml[j] = (is_own ? own.ml : pre.ml)[q];
            const float* o = (is_own ? own.o : pre.o) + q * D + DL * lane;
#pragma unroll
            for (int e = 0; e < DL; ++e) v[j][e] = o[e];
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            if (j0 + W * j >= n) ml[j].x = kNegInf;
            top = fmaxf(top, ml[j].x);
        }
        const float base = top == kNegInf ? 0.f : top, alpha = fast_exp2(M - base);
        M = top;
        sum *= alpha;
#pragma unroll
        for (int e = 0; e < DL; ++e) acc[e] *= alpha;
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const float w = fast_exp2(ml[j].x - base);
            sum = __builtin_fmaf(w, ml[j].y, sum);
#pragma unroll
            for (int e = 0; e < DL; ++e) acc[e] = __builtin_fmaf(w, v[j][e], acc[e]);
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int e = 0; e < DL; ++e) red[wave][DL * lane + e] = acc[e];
        if (lane == 0) red[wave][D] = M, red[wave][D + 1] = sum;
        __syncthreads();
        if (wave > 0) return;
        float top = kNegInf;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, red[w][D]);
        const float base = top == kNegInf ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int e = 0; e < DL; ++e) acc[e] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = fast_exp2(red[w][D] - base);
            sum = __builtin_fmaf(red[w][D + 1], f, sum);
#pragma unroll
            for (int e = 0; e < DL; ++e) acc[e] = __builtin_fmaf(red[w][DL * lane + e], f, acc[e]);
        }
        M = top;
    }
    bool nothing = n == 0;  // no token: O = 0, LSE = -inf
    if (!SHARED && M == kNegInf) {  // no listed block with a token, or scores of -inf
        const int tokens = part_clamp(p.lengths[b], p.capacity[1]), blocks = (tokens + (1 << p.block_shift) - 1) >> p.block_shift;
        bool there = false;
        for (int j = lane; j < p.n_list; j += 64) there |= (uint32_t)p.list[b * p.list_b + hk * p.list_h + j] < (uint32_t)blocks;
        nothing = __ballot(there) == 0;
    }
    const float inv = nothing ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < DL; ++e)
        if (DL * lane + e < p.d) op[DL * lane + e] = Elem<T>::from_f32(nothing ? 0.f : acc[e] * inv);
    if (p.lse != nullptr && lane == 0) p.lse[b * p.lse_b + hq] = __builtin_fmaf(M, kLn2, __log2f(sum) * kLn2);
}

namespace {

// Types, head dims, strides and alignment of the tensors of both entry points.
int part_tensor_checks(int64_t D, int32_t dtype, const int64_t* strides, int n, const int64_t* rows, int n_rows, uintptr_t bits, const char* who) {
    if (dtype != DTATTN_BF16 && dtype != DTATTN_FP16 && dtype != DTATTN_FP32)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: dtype %d not supported (bf16, fp16, fp32)", who, dtype);
    const int64_t esz = dtype == DTATTN_FP32 ? 4 : 2;
    if (D <= 0 || D > 128 || (D * esz) % 16 != 0)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: head dim %lld not supported (up to 128, a multiple of 16 bytes)", who, (long long)D);
    for (int i = 0; i < n; ++i)
        if ((strides[i] * esz) % 16 != 0) return fail(DTATTN_ERR_UNSUPPORTED, "%s: strides must be multiples of 16 bytes", who);
    // the 32 rows of a unit are addressed with 32-bit offsets below 2^30, and what must not be read with offsets from 3 * 2^30 on
    for (int i = 0; i < n_rows; ++i)
        if (rows[i] < D || rows[i] * esz > (1 << 24)) return fail(DTATTN_ERR_UNSUPPORTED, "%s: the row stride of a cache must be from D elements to 2^24 bytes", who);
    if (bits & 15) return fail(DTATTN_ERR_UNSUPPORTED, "%s: tensors must be 16-byte aligned", who);
    return DTATTN_OK;
}

size_t part_up(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

}  // namespace dtattn
