// Accumulated attention weights: weights[b, hk, j] += sum over the query heads h of hk and the queries i that see key j
// of exp(scale * q[b, h, i] . k[b, hk, j] - lse[b, h, i]), lse being what the attention returned.
//
// No counterpart in the reference, which keeps no KV cache (python/dtorch/test/modules/llama.py:126-156); the weights are
// what dtattn_kv_evict chooses by.
//
// One query per sequence (decode) is bound by HBM: the keys are read once.  A prompt is bound by its products and
// exponentials.  Both keep a wave's keys in registers as MFMA operands (64 keys: four tiles of 16) and pass the queries
// by in sets of 16 (query, head) columns, so that the sum over queries stays in registers too and no two waves add
// to one weight: the result does not depend on timing.
#include <algorithm>
#include <type_traits>

#include "decode_params.hpp"
#include "fp8_cache.hpp"

namespace dtattn {

struct WeightParams {
    float* w;
    const char* q;
    const char* k;
    const float* ks;
    const float* lse;
    const int32_t* lengths;  // may be NULL
    int64_t w_b, w_h;
    int64_t q_b, q_h, q_s;  // elements
    int64_t k_b, k_h, k_s;
    int64_t ks_b, ks_h, lse_b, lse_h;
    int64_t q_offset;
    int32_t B, Hkv, group, L, S, d, block_shift;
    float c;  // scale * log2(e)
    uint32_t q_and, q_xor;
    float* part;               // prompts whose columns several workgroups share: [parts, B * Hkv, S]
    int32_t parts, part_tiles; // and the column tiles of each
    int32_t key_blocks;
};

namespace {

constexpr int kFewColumns = 64;

// How a wave holds one tile's 16 keys (B operand: lane & 15 is the key) and one set's 16 queries (A operand), and their product: a
// lane has queries 4 (lane / 16) .. + 3 of key lane & 15, so a sum over queries is three adds and two exchanges.
// 16-bit and 8-bit keys: 16x16x32 MFMAs on 16-bit operands; codes are exact there, and fp32 queries over codes are
// three bf16 parts.  Keys are loaded as they are, from rows and chunks that exist (what stands for a head dim past the last
// meets a zero of the query), so that nothing stands between their loads and the next ones.
template <typename TQ, typename TK, int D>
struct Operands {
    typedef typename std::conditional<std::is_same<TQ, f16_t>::value, f16_t, bf16_t>::type E;
    typedef typename Elem<E>::vec8 V8;
    static constexpr bool codes = sizeof(TK) == 1;
    static constexpr int parts = std::is_same<TQ, float>::value ? 3 : 1;
    static constexpr int steps = D / 32, loads = codes ? D / 64 : D / 32;
    struct Keys { u32x4 v[loads]; };
    struct Queries { V8 v[parts][steps]; };
    // first head dim of the 8 of step s: chunks of 16 bytes of keys
    static __device__ __forceinline__ int dim(int g4, int s) { return codes ? 64 * (s >> 1) + 16 * g4 + 8 * (s & 1) : 32 * s + 8 * g4; }
    static __device__ __forceinline__ void keys(Keys& f, const TK* row, int g4, int d) {
#pragma unroll
        for (int i = 0; i < loads; ++i) {
            const int x = dim(g4, codes ? 2 * i : i);
            f.v[i] = ld16_nt(row + (x < d ? x : 0));
        }
    }
    // none: a query of zeros
    static __device__ __forceinline__ void queries(Queries& f, const TQ* row, int g4, int d, bool none, uint32_t q_and, uint32_t q_xor) {
        Chunk<TQ> w[steps];
#pragma unroll
        for (int s = 0; s < steps; ++s) w[s] = load_chunk<TQ, false>(row + (dim(g4, s) < d ? dim(g4, s) : 0));
#pragma unroll
        for (int s = 0; s < steps; ++s) {
#pragma unroll
            for (int i = 0; i < (int)(sizeof(w[s].v) / sizeof(w[s].v[0])); ++i)
                w[s].v[i] = dim(g4, s) < d && !none ? q_bits(w[s].v[i], q_and, q_xor) : u32x4{0u, 0u, 0u, 0u};
            if constexpr (parts == 1) {
                f.v[0][s] = __builtin_bit_cast(V8, w[s].v[0]);
            } else {
                float y[8];
                unpack_chunk<TQ>(w[s], y);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    bf16_t t[3];
                    split3(y[e], t);
#pragma unroll
                    for (int i = 0; i < 3; ++i) f.v[i][s][e] = t[i];
                }
            }
        }
    }
    static __device__ __forceinline__ f32x4 product(const Keys& k, const Queries& q) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < steps; ++s) {
            V8 kf;
            if constexpr (codes) kf = s & 1 ? codes_to_vec8<E>(k.v[s >> 1].z, k.v[s >> 1].w) : codes_to_vec8<E>(k.v[s >> 1].x, k.v[s >> 1].y);
            else kf = __builtin_bit_cast(V8, k.v[s]);
#pragma unroll
            for (int i = 0; i < parts; ++i) a = mfma16(q.v[i][s], kf, a);
        }
        return a;
    }
};
// fp32 keys: the fp32 matrix cores
template <int D>
struct Operands<float, float, D> {
    static constexpr int steps = D / 16;
    struct Keys { f32x4 v[steps]; };
    struct Queries { f32x4 v[steps]; };
    static __device__ __forceinline__ void keys(Keys& f, const float* row, int g4, int d) {
#pragma unroll
        for (int s = 0; s < steps; ++s) f.v[s] = __builtin_bit_cast(f32x4, ld16_nt(row + (16 * s + 4 * g4 < d ? 16 * s + 4 * g4 : 0)));
    }
    static __device__ __forceinline__ void queries(Queries& f, const float* row, int g4, int d, bool none, uint32_t q_and, uint32_t q_xor) {
        u32x4 w[steps];
#pragma unroll
        for (int s = 0; s < steps; ++s) w[s] = ld16(row + (16 * s + 4 * g4 < d ? 16 * s + 4 * g4 : 0));
#pragma unroll
        for (int s = 0; s < steps; ++s)
            f.v[s] = 16 * s + 4 * g4 < d && !none ? __builtin_bit_cast(f32x4, q_bits(w[s], q_and, q_xor)) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    static __device__ __forceinline__ f32x4 product(const Keys& k, const Queries& q) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < steps; ++s)
#pragma unroll
            for (int e = 0; e < 4; ++e) a = __builtin_amdgcn_mfma_f32_16x16x4f32(q.v[s][e], k.v[s][e], a, 0, 0, 0);
        return a;
    }
};

}  // namespace

// Few queries (up to kFewColumns of a kv head).  Grid: (workgroups of a (sequence, kv head), kv heads, sequences); the waves of those
// workgroups take the chunks of TILES tiles in turn, whatever the sequence's length.  Column c of a set is (query, head) number
// 16 * set + c, query-major: query c / group, head c % group.  A wave loads the next chunk's keys and weights when it
// has this one's scores.
template <typename TQ, typename TK, int D, bool CAUSAL, int TILES>
__global__ void __launch_bounds__(256) attn_weights_kernel(const WeightParams p) {
    typedef Operands<TQ, TK, D> Op;
    constexpr int KEYS = 16 * TILES;
    const int lane = threadIdx.x & 63, col = lane & 15, g4 = lane >> 4;
    const int64_t b = blockIdx.z;
    const int hk = blockIdx.y;
    const int n = p.lengths != nullptr ? min(max(p.lengths[b], 0), p.S) : p.S;
    const int stride = (int)gridDim.x * 4 * KEYS;
    int k0 = ((int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * KEYS;
    if (k0 >= n) return;
    const TK* kb = reinterpret_cast<const TK*>(p.k) + b * p.k_b + hk * p.k_h;
    const TQ* qb = reinterpret_cast<const TQ*>(p.q) + b * p.q_b + (int64_t)hk * p.group * p.q_h;
    const float* lb = p.lse + b * p.lse_b + (int64_t)hk * p.group * p.lse_h;
    float* const w = p.w + b * p.w_b + hk * p.w_h;
    const int N = p.L * p.group;
    int last = N;  // the end of the columns that are not padding
    if constexpr (CAUSAL)
        if (p.lengths != nullptr) last = (int)min(max(n - p.q_offset, (int64_t)0), (int64_t)p.L) * p.group;
    if (last == 0) return;
    typename Op::Keys kf[TILES];
    float c[TILES], was[TILES];
    auto load = [&](int key) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) Op::keys(kf[t], kb + (int64_t)min(key + 16 * t + col, n - 1) * p.k_s, g4, p.d);
    };
    auto load_weights = [&](int key) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            c[t] = p.c;
            if constexpr (sizeof(TK) == 1) c[t] *= p.ks[b * p.ks_b + hk * p.ks_h + (min(key + 16 * t, n - 1) >> p.block_shift)];
            was[t] = w[min(key + 16 * t + col, n - 1)];
        }
    };
    typename Op::Queries qf;
    float nl[4];
    int64_t sees[4];  // the last keys of this lane's four columns
    auto column = [&](int n0) {
        float lse[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = min(n0 + 4 * g4 + e, last - 1);
            const int i = at / p.group;
            lse[e] = lb[(at - i * p.group) * p.lse_h + i];
            sees[e] = i + p.q_offset;
        }
        const int at = min(n0 + col, last - 1);
        const int i = at / p.group, h = at - i * p.group;
        // columns past the end, and rows that see no key: a query of zeros at a weight of 0
        const bool none = n0 + col >= last || lb[h * p.lse_h + i] == kNegInf;
        Op::queries(qf, qb + h * p.q_h + i * p.q_s, g4, p.d, none, p.q_and, p.q_xor);
#pragma unroll
        for (int e = 0; e < 4; ++e) nl[e] = n0 + 4 * g4 + e >= last || lse[e] == kNegInf ? kNegInf : -lse[e] * kLog2e;
    };
    load(k0);
    load_weights(k0);
    column(0);
    for (;; k0 += stride) {
        float sum[TILES] = {};
        const bool more = k0 + stride < n;
        float cc[TILES], ww[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t) cc[t] = c[t], ww[t] = was[t];
        for (int n0 = 0; n0 < last; n0 += 16) {
            if (last > 16) column(n0);
            f32x4 s[TILES];
#pragma unroll
            for (int t = 0; t < TILES; ++t) s[t] = Op::product(kf[t], qf);
            if (n0 + 16 >= last && more) {
                load(k0 + stride);
                load_weights(k0 + stride);
            }
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = fast_exp2(__builtin_fmaf(s[t][e], cc[t], nl[e]));
                    if constexpr (CAUSAL) x = k0 + 16 * t + col <= sees[e] ? x : 0.f;
                    sum[t] += x;
                }
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            const float v = sum_across_groups<16>(sum[t]);
            const int key = k0 + 16 * t + col;
            if (g4 == 0 && key < n) w[key] = ww[t] + v;
        }
        if (!more) break;
    }
}

// ---- prompts --------------------------------------------------------------------------------------------------

namespace {

constexpr int kCols = 32;  // columns of a tile: 32x32 products

// 16-bit and 8-bit keys are one operand; fp32 ones are three bf16 parts (8 bits each, exact), of whose nine products with the
// query's parts the six largest count: what is left out is below 2^-23 of |q| |k|, an fp32 sum's own rounding.
template <typename TQ, typename TK>
struct PromptTypes {
    typedef typename std::conditional<std::is_same<TQ, f16_t>::value, f16_t, bf16_t>::type E;
    typedef typename Elem<E>::vec8 V8;
    static constexpr int qparts = std::is_same<TQ, float>::value ? 3 : 1;
    static constexpr int kparts = std::is_same<TK, float>::value ? 3 : 1;
    static constexpr int tiles = kparts == 3 ? 1 : 2;  // of 32 keys per wave
    static constexpr int keys = 4 * 32 * tiles;        // per workgroup
};

// Elements x .. x + 7 of a row of d (a multiple of 16 bytes), zeros past its end.
template <typename T>
__device__ __forceinline__ Chunk<T> load8(const T* row, int x, int d) {
    Chunk<T> w = {};
    if (x < d) w.v[0] = ld16(row + x);
    if constexpr (sizeof(T) == 4) if (x + 4 < d) w.v[1] = ld16(row + x + 4);
    return w;
}

// 8 elements as the bf16 parts or the one operand that they are.
template <typename T, typename V8, int PARTS>
__device__ __forceinline__ void to_parts(const Chunk<T>& w, V8* out) {
    if constexpr (PARTS == 1) {
        out[0] = __builtin_bit_cast(V8, w.v[0]);
    } else {
        float y[8];
        unpack_chunk<T>(w, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            bf16_t t[3];
            split3(y[e], t);
#pragma unroll
            for (int i = 0; i < 3; ++i) out[i][e] = t[i];
        }
    }
}

// (query, head) of a column, columns query-major, stepping by kCols.
struct Column {
    int64_t i;
    int h;
    __device__ __forceinline__ Column(int64_t n, int group) : i(n / group), h((int)(n - n / group * group)) {}
    __device__ __forceinline__ void step(int di, int dh, int group) {
        i += di;
        h += dh;
        if (h >= group) h -= group, ++i;
    }
};

}  // namespace

// A workgroup of four waves holds 256 keys (128 in fp32) as operands and passes column tiles by, which its threads stage
// through LDS one tile ahead.  A column is a lane, so its lse is one register and the sums over columns are one
// add per score; lanes meet once, at the end.  Per wave and tile of 16-bit operands 16 MFMAs against 32 exponentials and 64 other
// VALU instructions.
template <typename TQ, typename TK, int D, bool CAUSAL>
__global__ void __launch_bounds__(256, 2) attn_weights_prompt_kernel(const WeightParams p) {
    typedef PromptTypes<TQ, TK> Types;
    typedef typename Types::E E;
    typedef typename Types::V8 V8;
    constexpr int QP = Types::qparts, KP = Types::kparts, KT = Types::tiles, KS = D / 16, DC = D / 8;
    constexpr int PER = kCols * DC / 256;  // chunks of 8 elements that a thread stages
    __shared__ __attribute__((aligned(16))) V8 stage[2][QP][kCols * DC];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    // workgroup -> (key block, part of the columns, slice); slices go round the XCDs, whose L2 then holds their queries
    const int slices = p.B * p.Hkv;
    const int slice = blockIdx.x % slices;
    const int rest = blockIdx.x / slices;
    const int part = rest % p.parts, kblock = rest / p.parts;
    const int64_t b = slice / p.Hkv;
    const int hk = slice % p.Hkv;
    const int n = p.lengths != nullptr ? min(max(p.lengths[b], 0), p.S) : p.S;
    const int kwg = kblock * Types::keys;
    if (kwg >= n) return;
    const int64_t N = (int64_t)p.L * p.group;
    int64_t first = 0, last = N;  // the block's columns
    if constexpr (CAUSAL) {
        first = min(max((int64_t)kwg - p.q_offset, (int64_t)0) * p.group, N);
        if (p.lengths != nullptr) last = min(N, max(n - p.q_offset, (int64_t)0) * p.group);
    }
    const int64_t t0 = max(first / kCols, (int64_t)part * p.part_tiles);
    const int64_t t1 = min((last + kCols - 1) / kCols, (int64_t)(part + 1) * p.part_tiles);
    if (t0 >= t1) return;  // the sum knows
    const int k0 = kwg + __builtin_amdgcn_readfirstlane(tid >> 6) * 32 * KT;

    const TK* kb = reinterpret_cast<const TK*>(p.k) + b * p.k_b + hk * p.k_h;
    V8 kf[KT][KP][KS];
    float c[KT][2];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const TK* row = kb + (int64_t)min(k0 + 32 * t + col, n - 1) * p.k_s;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int x = 16 * s + 8 * half;
            if constexpr (sizeof(TK) == 1) {
                const u32x2 w = x < p.d ? *reinterpret_cast<const u32x2*>(row + x) : u32x2{0u, 0u};
                kf[t][0][s] = codes_to_vec8<E>(w.x, w.y);
            } else {
                const Chunk<TK> w = load8(row, x, p.d);
                V8 o[KP];
                to_parts<TK, V8, KP>(w, o);
#pragma unroll
                for (int i = 0; i < KP; ++i) kf[t][i][s] = o[i];
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            c[t][u] = p.c;
            if constexpr (sizeof(TK) == 1) c[t][u] *= p.ks[b * p.ks_b + hk * p.ks_h + (min(k0 + 32 * t + 16 * u, n - 1) >> p.block_shift)];
        }
    }

    const TQ* qb = reinterpret_cast<const TQ*>(p.q) + b * p.q_b + (int64_t)hk * p.group * p.q_h;
    const float* lb = p.lse + b * p.lse_b + (int64_t)hk * p.group * p.lse_h;
    const int di = kCols / p.group, dh = kCols % p.group;
    // chunk x of row r of a tile lies at x ^ swz(r): 16 rows read one chunk each without a conflict
    auto swz = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
    Column own(t0 * kCols + col, p.group);  // this lane's column
    int64_t left = last - t0 * kCols;       // columns from the tile on
    const int r0 = tid / DC, x0 = tid % DC;  // rows r0 + k * 256 / DC of a tile
    Column src0(t0 * kCols + r0, p.group), src1(t0 * kCols + r0 + 256 / DC, p.group);
    Chunk<TQ> raw[PER];
    float lse;
    auto load = [&]() {  // the tile that src0, src1 and own stand at, and on to the next
        int64_t at[2] = {src0.i * p.q_s + src0.h * p.q_h, src1.i * p.q_s + src1.h * p.q_h};
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const bool ok = r0 + k * (256 / DC) < left;
            raw[k] = load8(qb + (ok ? at[k] : 0), 8 * x0, ok ? p.d : 0);
        }
        lse = col < left ? lb[own.h * p.lse_h + own.i] : kNegInf;
        left -= kCols;
        src0.step(di, dh, p.group);
        src1.step(di, dh, p.group);
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int r = r0 + k * (256 / DC);
            Chunk<TQ> w = raw[k];
#pragma unroll
            for (int i = 0; i < (int)(sizeof(w.v) / sizeof(w.v[0])); ++i) w.v[i] = q_bits(w.v[i], p.q_and, p.q_xor);
            V8 o[QP];
            to_parts<TQ, V8, QP>(w, o);
#pragma unroll
            for (int i = 0; i < QP; ++i) stage[buf][i][r * DC + (x0 ^ swz(r))] = o[i];
        }
    };

    float sum[KT][16] = {};
    load();
    for (int64_t t = t0; t < t1; ++t) {
        const int buf = (int)(t - t0) & 1;
        put(buf);
        const bool none = lse == kNegInf;
        const float nl = -lse * kLog2e;
        int lim = 32 * KT - 1;  // the last of the wave's keys that this column sees
        if constexpr (CAUSAL) lim = (int)min(max(own.i + p.q_offset - k0, (int64_t)-1), (int64_t)(32 * KT - 1));
        if (none) lim = -1;
        own.step(di, dh, p.group);
        if (t + 1 < t1) load();
        lds_barrier();
        // buffers alternate, and this barrier has every wave past its reads of the other one's last tile
        if (k0 < n && __ballot(lim >= 0) != 0) {
            f32x16 s[KT] = {};
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                V8 qf[QP];
#pragma unroll
                for (int i = 0; i < QP; ++i) qf[i] = stage[buf][i][col * DC + ((2 * x + half) ^ swz(col))];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < KP; ++i)
#pragma unroll
                        for (int j = 0; j < QP && i + j < 3; ++j) s[kt] = Elem<E>::mfma32(kf[kt][i][x], qf[j], s[kt]);
            }
            if (__ballot(lim < 32 * KT - 1) == 0) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sum[kt][i] += fast_exp2(__builtin_fmaf(s[kt][i], c[kt][i >> 3], nl));
            } else {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float x = fast_exp2(__builtin_fmaf(s[kt][i], c[kt][i >> 3], nl));
                        sum[kt][i] += 32 * kt + 8 * (i >> 2) + 4 * half + (i & 3) <= lim ? x : 0.f;
                    }
            }
        }
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float s = group_sum<32>(sum[kt][i]);
            v = col == i ? s : v;
        }
        const int key = k0 + 32 * kt + 8 * (col >> 2) + 4 * half + (col & 3);
        if (col < 16 && key < n) {
            if (p.parts == 1) p.w[b * p.w_b + hk * p.w_h + key] += v;
            else p.part[((int64_t)part * slices + slice) * p.S + key] = v;
        }
    }
}

// Adds the parts of a key in their order: those whose workgroup had columns.
template <bool CAUSAL>
__global__ void __launch_bounds__(256) attn_weights_sum_kernel(const WeightParams p, int keys) {
    const int key = blockIdx.x * 256 + threadIdx.x;
    const int slices = p.B * p.Hkv, slice = blockIdx.y;
    const int64_t b = slice / p.Hkv;
    const int hk = slice % p.Hkv;
    const int n = p.lengths != nullptr ? min(max(p.lengths[b], 0), p.S) : p.S;
    if (key >= n) return;
    const int64_t N = (int64_t)p.L * p.group;
    int64_t first = 0, last = N;
    if constexpr (CAUSAL) {
        first = min(max((int64_t)(key / keys * keys) - p.q_offset, (int64_t)0) * p.group, N);
        if (p.lengths != nullptr) last = min(N, max(n - p.q_offset, (int64_t)0) * p.group);
    }
    const int64_t t0 = first / kCols, t1 = (last + kCols - 1) / kCols;
    if (t0 >= t1) return;
    const int x0 = (int)(t0 / p.part_tiles), x1 = (int)((t1 - 1) / p.part_tiles);
    float v = 0.f;
    for (int x = x0; x <= x1; ++x) v += p.part[((int64_t)x * slices + slice) * p.S + key];
    p.w[b * p.w_b + hk * p.w_h + key] += v;
}

namespace {

// Parts that a prompt's columns are cut in, so that the workgroups (two fit a CU) go round a few times.
struct PromptPlan {
    int64_t key_blocks, parts, part_tiles;
    size_t bytes;
};

PromptPlan prompt_plan(const dtattn_weights_args* a, int keys, int cus) {
    PromptPlan r;
    r.key_blocks = (a->S + keys - 1) / keys;
    const int64_t group = a->Hq / a->Hkv, slices = a->B * a->Hkv;
    const int64_t tiles = (a->L * group + kCols - 1) / kCols;
    double work = (double)r.key_blocks * (double)tiles;
    if (a->causal != 0) {  // key block k sees the columns from key k * keys - q_offset on
        work = 0;
        const int64_t step = std::max<int64_t>(1, r.key_blocks / 256);  // sampled
        for (int64_t k = 0; k < r.key_blocks; k += step) {
            const int64_t from = std::min<int64_t>(std::max<int64_t>(k * keys - a->q_offset, 0), a->L);
            work += (double)step * (double)((a->L - from) * group) / kCols;
        }
    }
    work *= (double)slices;
    r.part_tiles = std::max<int64_t>(8, (int64_t)(work / (2.0 * cus * 3)) + 1);
    r.part_tiles = std::min(r.part_tiles, tiles);
    r.parts = (tiles + r.part_tiles - 1) / r.part_tiles;
    r.bytes = r.parts > 1 ? (((size_t)r.parts * slices * a->S * sizeof(float) + 255) & ~(size_t)255) : 0;
    return r;
}

bool is_prompt(const dtattn_weights_args* a) { return a->L * (a->Hq / a->Hkv) > kFewColumns; }

int prompt_keys(const dtattn_weights_args* a) { return a->k_dtype == DTATTN_FP32 ? PromptTypes<float, float>::keys : PromptTypes<bf16_t, bf16_t>::keys; }

}  // namespace

template <typename TQ, typename TK, int D>
static int launch_prompt(WeightParams p, bool causal, const PromptPlan& plan, hipStream_t stream) {
    const int64_t slices = (int64_t)p.B * p.Hkv;
    p.parts = (int32_t)plan.parts, p.part_tiles = (int32_t)plan.part_tiles, p.key_blocks = (int32_t)plan.key_blocks;
    const dim3 grid((unsigned)(slices * plan.parts * plan.key_blocks));
    if (causal) hipLaunchKernelGGL((attn_weights_prompt_kernel<TQ, TK, D, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((attn_weights_prompt_kernel<TQ, TK, D, false>), grid, dim3(256), 0, stream, p);
    const int st = check_launch("attn_weights_prompt_kernel");
    if (st != DTATTN_OK || plan.parts == 1) return st;
    const dim3 sums((unsigned)((p.S + 255) / 256), (unsigned)slices);
    const int keys = PromptTypes<TQ, TK>::keys;
    if (causal) hipLaunchKernelGGL(attn_weights_sum_kernel<true>, sums, dim3(256), 0, stream, p, keys);
    else hipLaunchKernelGGL(attn_weights_sum_kernel<false>, sums, dim3(256), 0, stream, p, keys);
    return check_launch("attn_weights_sum_kernel");
}

// per_cu: workgroups wanted per CU.  One set of columns: chunks of 32 keys; more sets load the queries again for each chunk, and take
// 64.  us at 32 keys and 6 workgroups / 64 and 4: 16 of 700 to 8191, 28 heads over 4 (codes) 13.9 / 16.1, 16x8191 bf16 32 over 8 55 / 56,
// 8 of 4000 to 8191 fp32 58 / 74; 8 of 20000 to 32768, 64 heads over 1 (codes) 32 / 25.
template <typename TQ, typename TK, int D, int TILES>
static int launch_few(const WeightParams& p, bool causal, int per_cu, hipStream_t stream) {
    const int64_t slices = (int64_t)p.B * p.Hkv, most = (p.S + 64 * TILES - 1) / (64 * TILES);
    const int64_t wanted = std::max<int64_t>(1, (int64_t)per_cu * std::max(stream_cus(stream), 1) / slices);
    const dim3 grid((unsigned)std::min(most, wanted), (unsigned)p.Hkv, (unsigned)p.B);
    if (causal) hipLaunchKernelGGL((attn_weights_kernel<TQ, TK, D, true, TILES>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((attn_weights_kernel<TQ, TK, D, false, TILES>), grid, dim3(256), 0, stream, p);
    return check_launch("attn_weights_kernel");
}

template <typename TQ, typename TK, int D>
static int launch_weights(const WeightParams& p, bool causal, const PromptPlan* plan, hipStream_t stream) {
    if (plan != nullptr) return launch_prompt<TQ, TK, D>(p, causal, *plan, stream);
    if (p.L * p.group <= 16) return launch_few<TQ, TK, D, 2>(p, causal, 6, stream);
    return launch_few<TQ, TK, D, 4>(p, causal, 4, stream);
}

template <typename TQ, typename TK>
static int dispatch_weights(const WeightParams& p, bool causal, const PromptPlan* plan, hipStream_t stream) {
    return p.d <= 64 ? launch_weights<TQ, TK, 64>(p, causal, plan, stream) : launch_weights<TQ, TK, 128>(p, causal, plan, stream);
}

}  // namespace dtattn

using namespace dtattn;

extern "C" size_t dtattn_attention_weights_workspace_size(const dtattn_weights_args* a, void* stream) {
    if (a == nullptr || a->B <= 0 || a->Hkv <= 0 || a->Hq < a->Hkv || a->L <= 0 || a->S <= 0 || !is_prompt(a)) return 0;
    const int cus = stream_cus(reinterpret_cast<hipStream_t>(stream));
    return prompt_plan(a, prompt_keys(a), cus > 0 ? cus : 256).bytes;
}

extern "C" int dtattn_attention_weights(const dtattn_weights_args* a, void* stream_) {
    const char* who = "attention_weights";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    if (a->B < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->L < 0 || a->S < 0 || a->D <= 0)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
    if (a->Hq % a->Hkv != 0) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: Hq is not a multiple of Hkv", who);
    if (a->q_dtype != DTATTN_BF16 && a->q_dtype != DTATTN_FP16 && a->q_dtype != DTATTN_FP32)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: query dtype %d not supported (bf16, fp16, fp32)", who, a->q_dtype);
    const bool codes = a->k_dtype == DTATTN_FP8_E4M3FN;
    if (!codes && a->k_dtype != a->q_dtype)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: keys are of the query's dtype or e4m3fn codes, not %d", who, a->k_dtype);
    const int64_t qe = a->q_dtype == DTATTN_FP32 ? 4 : 2, ke = codes ? 1 : qe;
    if (a->D > 128 || (a->D * ke) % 16 != 0)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: head dim %lld not supported (rows of a multiple of 16 bytes, up to 128)", who, (long long)a->D);
    if (a->S > (1 << 29) || a->L > (1 << 29) || a->B > 65535 || a->Hkv > 65535 || a->B * a->Hkv > 65535)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
    const int64_t most = (int64_t)1 << 40;
    if (a->q_offset > most || a->q_offset < -most) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: q_offset out of range", who);
    ScalePlan sp;
    const int st = plan_scale(a->scale, a->D, a->q_dtype == DTATTN_FP32 ? kSign32 : kSign16, &sp);
    if (st != DTATTN_OK) return st;
    WeightParams p = {};
    if (codes) {
        if (a->block < 16 || a->block > 256 || (a->block & (a->block - 1)) != 0 || a->S % a->block != 0)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: block %d must be a power of two from 16 to 256 that divides S", who, a->block);
        p.block_shift = __builtin_ctz((unsigned)a->block);
    }
    if (a->B == 0 || a->S == 0 || a->L == 0) return DTATTN_OK;
    if (a->weights == nullptr || a->q == nullptr || a->k == nullptr || a->lse == nullptr || (codes && a->k_scale == nullptr))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    for (int i = 0; i < 3; ++i)
        if ((a->q_stride[i] * qe) % 16 != 0 || (a->k_stride[i] * ke) % 16 != 0)
            return fail(DTATTN_ERR_UNSUPPORTED, "%s: strides must be multiples of 16 bytes", who);
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k)) & 15u)
        return fail(DTATTN_ERR_UNSUPPORTED, "%s: query and keys must be 16-byte aligned", who);
    p.w = a->weights;
    p.q = reinterpret_cast<const char*>(a->q), p.k = reinterpret_cast<const char*>(a->k);
    p.ks = a->k_scale, p.lse = a->lse, p.lengths = a->lengths;
    p.w_b = a->w_stride[0], p.w_h = a->w_stride[1];
    p.q_b = a->q_stride[0], p.q_h = a->q_stride[1], p.q_s = a->q_stride[2];
    p.k_b = a->k_stride[0], p.k_h = a->k_stride[1], p.k_s = a->k_stride[2];
    p.ks_b = a->k_scale_stride[0], p.ks_h = a->k_scale_stride[1];
    p.lse_b = a->lse_stride[0], p.lse_h = a->lse_stride[1];
    p.q_offset = a->q_offset;
    p.B = (int32_t)a->B, p.Hkv = (int32_t)a->Hkv, p.group = (int32_t)(a->Hq / a->Hkv);
    p.L = (int32_t)a->L, p.S = (int32_t)a->S, p.d = (int32_t)a->D;
    p.c = sp.scale * kLog2e;
    p.q_and = sp.q_and, p.q_xor = sp.q_xor;
    const bool causal = a->causal != 0;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    PromptPlan prompt;
    const PromptPlan* plan = nullptr;
    if (is_prompt(a)) {
        const int cus = stream_cus(stream);
        if (cus <= 0) return fail(DTATTN_ERR_DEVICE, "%s: cannot tell the stream's device", who);
        prompt = prompt_plan(a, prompt_keys(a), cus);
        if (prompt.key_blocks * prompt.parts * a->B * a->Hkv > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
        if (prompt.bytes > 0 && (a->workspace == nullptr || a->workspace_bytes < prompt.bytes))
            return fail(DTATTN_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, prompt.bytes, a->workspace_bytes);
        if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return fail(DTATTN_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
        p.part = reinterpret_cast<float*>(a->workspace);
        plan = &prompt;
    }
    if (codes) {
        if (a->q_dtype == DTATTN_BF16) return dispatch_weights<bf16_t, uint8_t>(p, causal, plan, stream);
        if (a->q_dtype == DTATTN_FP16) return dispatch_weights<f16_t, uint8_t>(p, causal, plan, stream);
        return dispatch_weights<float, uint8_t>(p, causal, plan, stream);
    }
    if (a->q_dtype == DTATTN_BF16) return dispatch_weights<bf16_t, bf16_t>(p, causal, plan, stream);
    if (a->q_dtype == DTATTN_FP16) return dispatch_weights<f16_t, f16_t>(p, causal, plan, stream);
    return dispatch_weights<float, float>(p, causal, plan, stream);
}
