// Decode attention by parts: the kernel that decode_shared.hip and decode_blocks.hip instantiate for a prefix that sequences share, for
// their own tokens behind it, and for listed blocks of tokens; and the kernel that merges what its shares leave.
//
// A part is a set of segments, (column set, sequence or group) pairs with a number of 32-token units each.  All units are laid end to
// end and cut in equal shares, one per workgroup, whose four waves take its units in turn and meet in LDS where a segment ends.
// A segment's columns are query rows that read the same keys: the query heads of a kv head (a sequence's own tokens and listed blocks), or
// those of all sequences of a group (the prefix), 16 NC of them.
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
    float* rec_lse[2];
    float* whole_o[2];  // [B, Hq, kernel D]: segments inside one share
    float* whole_lse[2];
    int32_t* meta[2];   // units of all; then of each group or sequence: units before it, and its own
    int32_t nsub[2], shares[2], columns[2];  // column sets of a kv head; shares at most; columns of a set
    int32_t capacity[2];
    int64_t q_b, q_h, o_b, o_h, lse_b, bt_s, list_b, list_h;  // elements
    int32_t B, Hq, Hkv, group, groups, per;  // per: sequences of a group
    int32_t page_shift, num_pages;
    int32_t n_list, list_units, block_shift;
    int32_t d;
    float c;  // scale * log2(e)
    uint32_t q_and, q_xor;
};

namespace {

constexpr int kPartUnit = 32;  // tokens
constexpr int kPartWaves = 4;
constexpr int kPartLeast = kPartWaves;  // units of a share, at least
constexpr int kPartGroups = 2048;

// V units in `n` shares of V / n or one more (all the longer ones first); the host keeps V below 2^31.
struct PartShares {
    int n, q, rem;
    __device__ __forceinline__ PartShares(int V, int most) {
        n = min(most, max(1, V / kPartLeast));
        q = V / n;
        rem = V - q * n;
    }
    __device__ __forceinline__ int start(int r) const { return r * q + min(r, rem); }
    __device__ __forceinline__ int of(int x) const {  // the share of unit x
        const int big = rem * (q + 1);
        return x < big ? x / (q + 1) : rem + (x - big) / q;
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

// NC: sets of 16 columns.  TWO: a unit's two tiles of 16 tokens may lie apart (pages or blocks of 16 tokens).
template <typename T, int D, int NC, int KIND, bool TWO>
__device__ void decode_part(const PartsParams& p, int share, float (*red_o)[16][D + 4], float (*red_m)[16], float (*red_l)[16], int* eff, int* lead) {
    typedef typename PartType<T>::vec8 V8;
    constexpr bool kF32 = sizeof(T) == 4;
    constexpr int S = KIND == kPrefixPart ? 0 : 1;
    constexpr int NK = D * (int)sizeof(T) / 64;  // 16-byte loads of a key per lane
    constexpr int DPL = D / 16;                  // dims of a token's values per lane
    constexpr int VW = DPL * (int)sizeof(T) / 4; // words of them
    constexpr int NR = TWO ? 2 : 1;              // buffer resources of a unit
    constexpr int PP = PartType<T>::parts;
    constexpr float kOff = PartType<T>::offset;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g4 = lane >> 4;
    typedef const __attribute__((address_space(4))) int32_t cint32;
    cint32* const lengths = (cint32*)p.lengths;
    cint32* const prefix = (cint32*)p.prefix;
    cint32* const table = (cint32*)p.table;
    cint32* const list = (cint32*)p.list;
    const bool paged = p.table != nullptr;
    const int Z = KIND == kPrefixPart ? p.groups : p.B;
    auto clamped = [](int n, int most) { return min(max(n, 0), most); };

    // Tokens that a group shares: whole pages that each of its sequences with tokens has, and the first of those sequences
    if constexpr (KIND != kListPart) {
        if (paged) {
            for (int g = tid; g < p.groups; g += 256) eff[g] = lead[g] = 0x7fffffff;
            __syncthreads();
            for (int b = tid; b < p.B; b += 256) {
                const int n = clamped(p.lengths[b], p.capacity[1]);
                if (n > 0) {
                    atomicMin(&eff[b / p.per], n);
                    atomicMin(&lead[b / p.per], b);
                }
            }
            __syncthreads();
            for (int g = tid; g < p.groups; g += 256) {
                const int n = eff[g] == 0x7fffffff ? 0 : min(eff[g], max(p.prefix[g], 0));
                eff[g] = n >> p.page_shift << p.page_shift;
            }
            __syncthreads();
        }
    }
    // a segment's tokens: from `start` to before `end`
    auto start_of = [&](int z) { return KIND == kOwnPart && paged ? __builtin_amdgcn_readfirstlane(eff[z / p.per]) : 0; };
    auto end_of = [&](int z) {
        if constexpr (KIND == kPrefixPart) return paged ? __builtin_amdgcn_readfirstlane(eff[z]) : clamped(prefix[z], p.capacity[0]);
        else return clamped(lengths[z], p.capacity[1]);
    };
    auto units_of = [&](int z) {  // per lane
        int n;
        if constexpr (KIND == kPrefixPart) n = paged ? eff[z] : clamped(p.prefix[z], p.capacity[0]);
        else n = clamped(p.lengths[z], p.capacity[1]) - (paged ? eff[z / p.per] : 0);
        return (max(n, 0) + kPartUnit - 1) / kPartUnit;
    };
    int U = 0, own0 = 0, pre0 = 0;
    if constexpr (KIND == kListPart) {
        U = p.B * p.list_units;
    } else {
        const bool tells = share == 0 && wave == 0;
        for (int j0 = 0; j0 < Z; j0 += 64) {
            const int own = j0 + lane < Z ? units_of(j0 + lane) : 0;
            const int s = scan64(own);
            if (j0 == 0) own0 = own, pre0 = s;
            if (tells && j0 + lane < Z) {
                p.meta[S][1 + 2 * (j0 + lane)] = U + s - own;
                p.meta[S][2 + 2 * (j0 + lane)] = own;
            }
            U += __builtin_amdgcn_readlane(s, 63);
        }
        if (tells && lane == 0) p.meta[S][0] = U;
    }
    if (U == 0) return;
    const PartShares sh(U * p.Hkv * p.nsub[S], p.shares[S]);
    const int r = share;
    if (r >= sh.n) return;
    const int u0 = sh.start(r), n = sh.start(r + 1) - u0;  // first unit and units of this workgroup

    struct At {  // a unit
        int slot, hk, z;     // slot: kv head * nsub + column set
        int u, units;        // of the segment
        int start, end, row; // row: of the table
        int t[NR], rows[NR], page[NR];
    };
    auto enter = [&](At& a) {
        a.hk = p.nsub[S] == 1 ? a.slot : a.slot / p.nsub[S];
        a.start = start_of(a.z);
        a.end = end_of(a.z);
        a.units = KIND == kListPart ? p.list_units : (max(a.end - a.start, 0) + kPartUnit - 1) / kPartUnit;
        a.row = KIND == kPrefixPart && paged && a.units > 0 ? __builtin_amdgcn_readfirstlane(lead[a.z]) : a.z;
    };
    auto next = [&](At& a) {  // the next segment with units; there is one
        do {
            if (++a.z == Z) a.z = 0, ++a.slot;
            enter(a);
        } while (a.units == 0);
    };
    auto advance = [&](At& a, int k) {
        a.u += k;
        while (a.u >= a.units) {
            a.u -= a.units;
            next(a);
        }
    };
    auto find = [&](At& a) {  // the tokens of a unit, and the pages that hold them
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int x = a.u * kPartUnit + 16 * i;
            if constexpr (KIND == kListPart) {
                const int e = x >> p.block_shift;
                const int j = e < p.n_list ? list[a.z * p.list_b + a.hk * p.list_h + e] : -1;
                const bool there = (uint32_t)j < (uint32_t)((a.end + (1 << p.block_shift) - 1) >> p.block_shift);
                a.t[i] = there ? (j << p.block_shift) + (x & ((1 << p.block_shift) - 1)) : 0;
                a.rows[i] = there ? clamped(a.end - a.t[i], kPartUnit / NR) : 0;
            } else {
                a.t[i] = a.start + x;
                a.rows[i] = clamped(a.end - a.t[i], kPartUnit / NR);
                if (a.rows[i] == 0) a.t[i] = 0;
            }
            a.page[i] = paged ? table[a.row * p.bt_s + (a.t[i] >> p.page_shift)] : a.z;
        }
    };
    At at;
    at.slot = u0 / U;
    int x = u0 - at.slot * U;
    if constexpr (KIND == kListPart) {
        at.z = x / p.list_units;
        x -= at.z * p.list_units;
    } else {
        for (int j0 = 0;; j0 += 64) {
            const int own = j0 == 0 ? own0 : j0 + lane < Z ? units_of(j0 + lane) : 0;
            const int s = j0 == 0 ? pre0 : scan64(own);
            const uint64_t hit = __ballot(s > x);  // segments ending past x
            if (hit != 0) {
                const int l = __builtin_ctzll(hit);
                at.z = j0 + l;
                x -= __builtin_amdgcn_readlane(s - own, l);
                break;
            }
            x -= __builtin_amdgcn_readlane(s, 63);
        }
    }
    at.u = x;
    enter(at);

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
    auto base_of = [&](const At& a, int i, const char* x, int64_t sb, int64_t s_h, int64_t ss) {
        const int64_t where = paged ? clamped(a.page[i], p.num_pages - 1) : a.page[i];
        const int row = paged ? a.t[i] & ((1 << p.page_shift) - 1) : a.t[i];
        return x + where * sb + a.hk * s_h + row * ss;
    };
    auto ld16b = [&](__amdgpu_buffer_rsrc_t rs, uint32_t off) { return KIND == kPrefixPart ? buf_ld16(rs, off) : buf_ld16_nt(rs, off); };
    auto load_k = [&](const At& a) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const auto rs = make_rsrc(base_of(a, i, p.k[S], p.k_b[S], p.k_h[S], p.k_s[S]), a.rows[i] > 0 ? (uint32_t)(a.rows[i] - 1) * kp + (uint32_t)row_bytes : 0u);
#pragma unroll
            for (int tt = TWO ? i : 0; tt < (TWO ? i + 1 : 2); ++tt)
#pragma unroll
                for (int k = 0; k < NK; ++k) kr[tt][k] = ld16b(rs, koff[k] + (TWO ? 0u : 16u * tt * kp));
        }
    };
    auto load_v = [&](const At& a) {
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const auto rs = make_rsrc(base_of(a, i, p.v[S], p.v_b[S], p.v_h[S], p.v_s[S]), a.rows[i] > 0 ? (uint32_t)(a.rows[i] - 1) * vp + (uint32_t)row_bytes : 0u);
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

    f32x4 acc[NC][DPL];
    float M[NC], l[NC];  // running max, and this lane's part of the row sum on that base
    u32x4 qf[NC][NK];
    At cur = at, nx = at;
    if (wave < n) {
        if (wave > 0) advance(nx, wave);
        find(nx);
        load_k(nx);
        load_v(nx);
    }
    int s = wave;  // this wave's next unit of the share
    for (int u = 0; u < n;) {
        const int m = min(cur.units - cur.u, n - u);  // units of the segment
        const int hk = cur.hk, z = cur.z, sub = cur.slot - hk * p.nsub[S];
        const int R = KIND == kPrefixPart ? p.per * p.group : p.group;
        const int R0 = 16 * NC * sub;
        bool seen = false;
        auto where = [&](int row, int& b, int& hq) {  // the sequence and head of a row
            const int i = KIND == kPrefixPart ? row / p.group : 0;
            b = KIND == kPrefixPart ? z * p.per + i : z;
            hq = hk * p.group + row - i * p.group;
        };
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            M[c] = kNegInf, l[c] = 0.f;
#pragma unroll
            for (int j = 0; j < DPL; ++j) acc[c][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (s < u + m) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                int b, hq;
                where(min(R0 + 16 * c + col, R - 1), b, hq);
                const char* qp = p.q + (b * p.q_b + hq * p.q_h) * (int64_t)sizeof(T);
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    const int at16 = 16 * (4 * k + g4);
                    const u32x4 w = ld16(qp + (at16 < row_bytes ? at16 : 0));
                    qf[c][k] = at16 < row_bytes ? q_bits(w, p.q_and, p.q_xor) : u32x4{0u, 0u, 0u, 0u};
                }
            }
        }
        for (; s < u + m; s += kPartWaves) {
            int rows[NR];
#pragma unroll
            for (int i = 0; i < NR; ++i) rows[i] = nx.rows[i], seen |= rows[i] > 0;
            const bool more = s + kPartWaves < n;
            if (more) {
                advance(nx, kPartWaves);
                find(nx);
            }
            f32x4 sc[NC][2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
                for (int c = 0; c < NC; ++c) sc[c][tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    if constexpr (kF32) {
                        const f32x4 kf = __builtin_bit_cast(f32x4, kr[tt][k]);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int c = 0; c < NC; ++c) sc[c][tt] = mfma_f32(kf[e], __builtin_bit_cast(f32x4, qf[c][k])[e], sc[c][tt]);
                    } else {
#pragma unroll
                        for (int c = 0; c < NC; ++c)
                            sc[c][tt] = mfma16(__builtin_bit_cast(V8, kr[tt][k]), __builtin_bit_cast(V8, qf[c][k]), sc[c][tt]);
                    }
                }
            }
            if (more) load_k(nx);  // the keys are used up
            if (rows[0] < kPartUnit / NR || (TWO && rows[NR - 1] < 16)) {
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if ((TWO ? 0 : 16 * tt) + 4 * g4 + i >= rows[TWO ? tt : 0]) {
#pragma unroll
                            for (int c = 0; c < NC; ++c) sc[c][tt][i] = kNegInf;
                        }
            }
            float Mn[NC];
            bool grows = false;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                float mx = kNegInf;
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) mx = fmaxf(mx, fmaxf(fmaxf(sc[c][tt][0], sc[c][tt][1]), fmaxf(sc[c][tt][2], sc[c][tt][3])));
                Mn[c] = fmaxf(M[c], max_across_groups<16>(mx) * p.c);
                grows |= Mn[c] > M[c];
            }
            if (__ballot(grows) != 0) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const float alpha = fast_exp2(M[c] - (Mn[c] == kNegInf ? 0.f : Mn[c]));
                    M[c] = Mn[c];
                    l[c] *= alpha;
#pragma unroll
                    for (int j = 0; j < DPL; ++j) acc[c][j] *= alpha;
                }
            }
            V8 vf[kF32 ? 1 : DPL];
            if constexpr (!kF32) {
                // two tokens' values of one dim side by side
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
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const float base = (M[c] == kNegInf ? 0.f : M[c]) - kOff;
                float pf[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    pf[i] = fast_exp2(__builtin_fmaf(sc[c][i >> 2][i & 3], p.c, -base));
                    l[c] += pf[i];
                }
                if constexpr (kF32) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int j = 0; j < DPL; ++j) acc[c][j] = mfma_f32(__builtin_bit_cast(float, vr[i][j]), pf[i], acc[c][j]);
                } else {
                    V8 pk[PP];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        pk[0][i] = Elem<T>::from_f32(pf[i]);
                        pk[PP - 1][i] = Elem<T>::from_f32(pf[i] - Elem<T>::to_f32(pk[0][i]));
                    }
#pragma unroll
                    for (int h = 0; h < PP; ++h)
#pragma unroll
                        for (int j = 0; j < DPL; ++j) acc[c][j] = mfma16(vf[j], pk[h], acc[c][j]);
                }
            }
            if (kF32 && more) load_v(nx);
        }
        // the waves meet, 16 columns at a time
        const bool whole = cur.u == 0 && m == cur.units;
        const bool any = KIND != kListPart || __syncthreads_or(seen);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int heads = min(R - R0 - 16 * c, 16);
            if (heads <= 0) break;
            if (c > 0) lds_barrier();  // the last columns have been read
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float* at_o = &red_o[wave][col][DPL * (4 * g4 + i)];
#pragma unroll
                for (int j = 0; j < DPL; j += 4) *reinterpret_cast<f32x4*>(at_o + j) = f32x4{acc[c][j][i], acc[c][j + 1][i], acc[c][j + 2][i], acc[c][j + 3][i]};
            }
            const float lw = sum_across_groups<16>(l[c]);
            if (g4 == 0) red_m[wave][col] = M[c], red_l[wave][col] = lw;
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
                where(R0 + 16 * c + g, b, hq);
                const int dim = DPL * (tid & 15);
                const bool direct = KIND == kListPart && whole;
                const float lse = __builtin_fmaf(X - kOff, kLn2, __log2f(lt) * kLn2);
                // every score -inf: a record of O = 0 at the LSE of -inf, which drops it in the merge; the output itself is 0 / 0
                const float inv = (lt == 0.f && !direct) || !any ? 0.f : 1.f / lt;
#pragma unroll
                for (int j = 0; j < DPL; ++j) o[j] *= inv;
                if (direct) {
                    T* op = reinterpret_cast<T*>(p.o) + b * p.o_b + hq * p.o_h + dim;
#pragma unroll
                    for (int j = 0; j < DPL; j += 4)
                        if (dim + j < p.d) {
                            if constexpr (kF32) *reinterpret_cast<f32x4*>(op + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
                            else *reinterpret_cast<u32x2*>(op + j) = u32x2{pack2<T>(o[j], o[j + 1]), pack2<T>(o[j + 2], o[j + 3])};
                        }
                    if (p.lse != nullptr && (tid & 15) == 0) p.lse[b * p.lse_b + hq] = lse;
                } else {
                    const int64_t rec = whole ? (int64_t)b * p.Hq + hq : (int64_t)(2 * r + (u == 0 ? 0 : 1)) * (16 * NC) + 16 * c + g;
                    float* op = (whole ? p.whole_o[S] : p.rec_o[S]) + rec * D + dim;
#pragma unroll
                    for (int j = 0; j < DPL; j += 4) *reinterpret_cast<f32x4*>(op + j) = f32x4{o[j], o[j + 1], o[j + 2], o[j + 3]};
                    if ((tid & 15) == 0) (whole ? p.whole_lse[S] : p.rec_lse[S])[rec] = lse;
                }
            }
        }
        u += m;
        if (u < n) {
            lds_barrier();  // every wave has read the others' before they write again
            cur.u = 0;
            next(cur);
        }
    }
}

// Merges a query head's records: of the prefix and of its own tokens (SHARED), or of listed blocks that several shares hold.  W waves
// to a (sequence, query head).
template <typename T, int D, int W, bool SHARED>
__global__ void __launch_bounds__(256) decode_parts_merge_kernel(const PartsParams p) {
    constexpr int DL = D / 64;  // dims per lane
    __shared__ float red[W > 1 ? W : 1][D];
    const int lane = threadIdx.x & 63, wave = W > 1 ? threadIdx.x >> 6 : 0;
    const int64_t pair = W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (pair >= (int64_t)p.B * p.Hq) return;
    const int b = (int)(pair / p.Hq), hq = (int)(pair % p.Hq), hk = hq / p.group, g = hq - hk * p.group;
    int64_t first[2] = {0, 0}, later[2] = {0, 0};  // the record of a part's first share, and of the one behind it
    int ns[2] = {0, 0};
    bool whole[2] = {false, false};
#pragma unroll
    for (int S = SHARED ? 0 : 1; S < 2; ++S) {
        const int z = S == 0 ? b / p.per : b;
        const int row = S == 0 ? (b - z * p.per) * p.group + g : g;
        const int U = SHARED ? p.meta[S][0] : p.B * p.list_units;
        const int before = SHARED ? p.meta[S][1 + 2 * z] : b * p.list_units, own = SHARED ? p.meta[S][2 + 2 * z] : p.list_units;
        if (own == 0) continue;
        const int cols = p.columns[S], sub = row / cols;
        const PartShares sh(U * p.Hkv * p.nsub[S], p.shares[S]);
        const int x0 = (hk * p.nsub[S] + sub) * U + before, r0 = sh.of(x0), r1 = sh.of(x0 + own - 1);
        ns[S] = r1 - r0 + 1;
        whole[S] = r0 == r1;
        // share r0 holds the segment first only if it begins with it
        first[S] = whole[S] ? pair : (int64_t)(2 * r0 + (sh.start(r0) < x0 ? 1 : 0)) * cols + row - sub * cols;
        later[S] = (int64_t)2 * (r0 + 1) * cols + row - sub * cols;
    }
    if (!SHARED && ns[1] == 1) return;  // written directly
    // a padded prefix is read for every sequence; a paged one holds the first of a sequence's tokens, if it has any
    if (SHARED && p.table != nullptr && p.lengths[b] <= 0) ns[0] = ns[1] = 0;
    const int n = ns[0] + ns[1];
    T* op = reinterpret_cast<T*>(p.o) + b * p.o_b + hq * p.o_h;
    auto nothing = [&]() {  // no token: O = 0, LSE = -inf
        if (wave > 0) return;
#pragma unroll
        for (int e = 0; e < DL; ++e)
            if (DL * lane + e < p.d) op[DL * lane + e] = Elem<T>::from_f32(0.f);
        if (p.lse != nullptr && lane == 0) p.lse[b * p.lse_b + hq] = kNegInf;
    };
    if (n == 0) return nothing();
    struct Rec {
        const float* o;
        const float* lse;
    };
    auto rec = [&](int j) {
        const int S = SHARED && j < ns[0] ? 0 : 1, i = S == 1 ? j - ns[0] : j;
        const int64_t q = i == 0 ? first[S] : later[S] + (int64_t)(i - 1) * 2 * p.columns[S];
        return Rec{(whole[S] ? p.whole_o[S] : p.rec_o[S]) + q * D, (whole[S] ? p.whole_lse[S] : p.rec_lse[S]) + q};
    };
    float mx = kNegInf;
    for (int j = lane; j < n; j += 64) mx = fmaxf(mx, *rec(j).lse);
    mx = wave_max(mx);
    if (!SHARED && mx == kNegInf) {  // no listed block with a token, or scores of -inf
        const int tokens = min(max(p.lengths[b], 0), p.capacity[1]), blocks = (tokens + (1 << p.block_shift) - 1) >> p.block_shift;
        bool there = false;
        for (int j = lane; j < p.n_list; j += 64) there |= (uint32_t)p.list[b * p.list_b + hk * p.list_h + j] < (uint32_t)blocks;
        if (__ballot(there) == 0) return nothing();
    }
    float sum = 0.f;
    for (int j = lane; j < n; j += 64) sum += __expf(*rec(j).lse - mx);
    sum = wave_sum(sum);
    const float inv = 1.f / sum;
    float acc[DL] = {};
    constexpr int MB = 8;  // records in flight
    for (int j0 = wave; j0 < n; j0 += W * MB) {
        float lw[MB], v[MB][DL];
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const Rec q = rec(min(j0 + W * j, n - 1));
            lw[j] = *q.lse;
#pragma unroll
            for (int e = 0; e < DL; ++e) v[j][e] = q.o[DL * lane + e];
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            const float w = j0 + W * j < n ? __expf(lw[j] - mx) * inv : 0.f;
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
