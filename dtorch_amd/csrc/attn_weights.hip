// Accumulated attention weights: weights[b, hk, j] += sum over the query heads h of hk and the queries i that see key j
// of exp(scale * q[b, h, i] . k[b, hk, j] - lse[b, h, i]), lse being what the attention returned.
//
// No counterpart in the reference, which keeps no KV cache (python/dtorch/test/modules/llama.py:126-156); the weights are
// what dtattn_kv_evict chooses by.
//
// One query per sequence (decode) is bound by HBM: the keys are read once.  A prompt is bound by the matrix cores and VALU issue
// together: an exponential, an fma and an add per (query, key) pair beside its MFMAs.  Counters at 4x2048 causal bf16, 32 heads over
// 8 of 128, per wave and column tile: 16 MFMAs, 512 cycles, and 32 exponentials (two issue slots each) and 112 other VALU
// instructions on average, 773 cycles with the MFMAs' issue; the two waves of a SIMD take 1294 cycles each.  Both forms
// keep a wave's keys in registers as MFMA operands and pass the queries by, so that the sum over queries stays in registers too and
// no two waves add to one weight: the result does not depend on timing.  Measured: 16 sequences of 700 to 8191, 28 heads over 4 of
// 128, codes, one query 11.6 us (through the caches, which a decode step has just filled; loads that bypass them take 13.4); 4x2048
// causal bf16, 32 heads over 8 of 128, 96 us, not causal 138 us (990 TFLOP/s).
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
    float c;  // scale * log2(e), of either sign
    // prompts: columns go by in tiles of `rows` queries by `width` heads, the group's or a set of 32 of them
    int32_t width, rows;
    float* part;  // records of blocks that several shares meet: [B * Hkv, sets, shares + key_blocks, keys of a block]
    int32_t sets, shares;  // head sets; shares of a (sequence, kv head, head set) at most
    int32_t key_blocks;
};

namespace {

// Columns up to which the keys pass the queries by and not the other way.  us of both ways at 32 / 64 / 96 / 128 columns: 4x4000 over 1
// kv head, bf16 7.3 and 10 / 9.1 and 11 / 11.1 and 11.0 / 13.0 and 12.3; 1x8000 over 8 at 64 / 128 9.8 and 13.4 / 14.1 and 14.7.
constexpr int kFewColumns = 64;

__device__ const uint32_t kZeros[4] = {0u, 0u, 0u, 0u};

// How a wave holds one tile's 16 keys (B operand: lane & 15 is the key) and one set's 16 queries (A operand), and their product: a
// lane has queries 4 (lane / 16) .. + 3 of key lane & 15, so a sum over queries is three adds and two exchanges.
// 16-bit and 8-bit keys: 16x16x32 MFMAs on 16-bit operands; codes are exact there, and fp32 queries over codes are
// three bf16 parts.  Keys are loaded as they are, from rows that exist (and from zeros for head dims past the last), so that
// nothing stands between their loads and the next ones.
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
            f.v[i] = ld16(x < d ? row + x : reinterpret_cast<const TK*>(kZeros));
        }
    }
    // none: a query of zeros
    static __device__ __forceinline__ void queries(Queries& f, const TQ* row, int g4, int d, bool none) {
        Chunk<TQ> w[steps];
#pragma unroll
        for (int s = 0; s < steps; ++s) w[s] = load_chunk<TQ, false>(row + (dim(g4, s) < d ? dim(g4, s) : 0));
#pragma unroll
        for (int s = 0; s < steps; ++s) {
#pragma unroll
            for (int i = 0; i < (int)(sizeof(w[s].v) / sizeof(w[s].v[0])); ++i)
                w[s].v[i] = dim(g4, s) < d && !none ? w[s].v[i] : u32x4{0u, 0u, 0u, 0u};
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
        for (int s = 0; s < steps; ++s)
            f.v[s] = __builtin_bit_cast(f32x4, ld16(16 * s + 4 * g4 < d ? row + 16 * s + 4 * g4 : reinterpret_cast<const float*>(kZeros)));
    }
    static __device__ __forceinline__ void queries(Queries& f, const float* row, int g4, int d, bool none) {
        u32x4 w[steps];
#pragma unroll
        for (int s = 0; s < steps; ++s) w[s] = ld16(row + (16 * s + 4 * g4 < d ? 16 * s + 4 * g4 : 0));
#pragma unroll
        for (int s = 0; s < steps; ++s)
            f.v[s] = 16 * s + 4 * g4 < d && !none ? __builtin_bit_cast(f32x4, w[s]) : f32x4{0.f, 0.f, 0.f, 0.f};
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
        // rows that see no key may hold anything: a query of zeros.  Columns past the end are the last one again, so that an
        // infinite key is no NaN where it is none there.  Both at a weight of 0.
        const bool none = lb[h * p.lse_h + i] == kNegInf;
        Op::queries(qf, qb + h * p.q_h + i * p.q_s, g4, p.d, none);
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

constexpr int kCols = 32;       // columns of a tile: 32x32 products
// Column tiles whose time it takes to start a key block, and places that a share has at least.  us at 0 and 4 / 4 and 4 / 4 and 8 /
// 6 and 6 (causal): 4x2048 32 heads over 8, bf16 103 / 100 / 104 / 101; 1x1500 the same, fp32 71 / 67 / 67 / 69; 2x777 12 of 64, fp32
// 21 / 20 / 22 / 20; 1x777 32 over 8, bf16 22 / 20 / 20 / 21; 1x1200 8 heads, fp32 31 / 26 / 28 / 30; not causal 4x2048 141 / 144 / 145 / 146.
constexpr int kStartTiles = 4;
constexpr int kShareTiles = 4;

// 16-bit and 8-bit keys are one operand; fp32 ones are three bf16 parts (8 bits each, exact), of whose nine products with the
// query's parts the six largest count.  The second part is at most 2^-8 of a value and the third 2^-16, of either sign, so what is left
// out is at most 2^-23 of |q| |k|, what one fp32 addition rounds by (parts cut off instead of rounded: 2^-21, always of one sign).
template <typename TQ, typename TK>
struct PromptTypes {
    typedef typename std::conditional<std::is_same<TQ, f16_t>::value, f16_t, bf16_t>::type E;
    typedef typename Elem<E>::vec8 V8;
    static constexpr int qparts = std::is_same<TQ, float>::value ? 3 : 1;
    static constexpr int kparts = std::is_same<TK, float>::value ? 3 : 1;
    static constexpr int tiles = kparts == 3 ? 1 : 2;  // of 32 keys per wave
    static constexpr int keys = 4 * 32 * tiles;        // per workgroup
};

// The column tiles that the key blocks of a sequence meet, one block after another: block k meets those from first(k) to end.  Their
// list, with kStartTiles places before each block's tiles for the time that the block's start takes, is cut in equal shares, one
// per workgroup, so that all run for the same time however a causal mask cuts the blocks.
template <bool CAUSAL>
struct PromptTiles {
    const WeightParams& p;
    int keys, n, end, last;  // keys of a block and of the sequence; tiles, and queries that are not padding
    __device__ __forceinline__ PromptTiles(const WeightParams& p_, int keys_, int64_t b) : p(p_), keys(keys_) {
        n = p.lengths != nullptr ? min(max(p.lengths[b], 0), p.S) : p.S;
        last = p.L;
        if (CAUSAL && p.lengths != nullptr) last = (int)min(max(n - p.q_offset, (int64_t)0), (int64_t)p.L);
        end = (last + p.rows - 1) / p.rows;
    }
    __device__ __forceinline__ int first(int k) const {
        if constexpr (!CAUSAL) return 0;
        const int64_t query = (int64_t)k * keys - p.q_offset;
        return query >= last ? end : (int)max(query, (int64_t)0) / p.rows;
    }
    __device__ __forceinline__ int count(int k) const { return (int64_t)k * keys < n ? end - first(k) : 0; }
    // f(k0, c, pre) for 64 blocks at a time: lane's block k0 + lane has c places in the list, and those up to it pre
    template <typename F>
    __device__ __forceinline__ int scan(F f) const {
        const int lane = threadIdx.x & 63;
        int total = 0;
        for (int k0 = 0; k0 < p.key_blocks; k0 += 64) {
            int c = k0 + lane < p.key_blocks ? count(k0 + lane) : 0;
            if (c > 0) c += kStartTiles;
            const int pre = scan64(c) + total;
            f(k0, c, pre);
            total = __builtin_amdgcn_readlane(pre, 63);
        }
        return total;
    }
};

// A share's record of a key block: the sum of the two numbers is another one for each of a list's records.
__device__ __forceinline__ int64_t prompt_record(const WeightParams& p, int slice, int set, int share, int kblock) {
    return ((int64_t)slice * p.sets + set) * (p.shares + p.key_blocks) + share + kblock;
}

// V places in up to `most` shares of V / n or one more, of kShareTiles at least.
struct PromptShares {
    int n, q, rem;
    __device__ __forceinline__ PromptShares(int V, int most) {
        n = min(most, max(1, V / kShareTiles));
        q = V / n;
        rem = V - q * n;
    }
    __device__ __forceinline__ int start(int r) const { return r * q + min(r, rem); }
    __device__ __forceinline__ int of(int x) const {
        const int big = rem * (q + 1);
        return x < big ? x / (q + 1) : rem + (x - big) / q;
    }
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

}  // namespace

// A workgroup of four waves holds 256 keys (128 in fp32) as operands and passes column tiles by, which its threads stage
// through LDS one tile ahead.  A column is a lane, so its lse is one register and the sums over columns are one
// add per score; lanes meet once, at the end.  Per wave and tile of 16-bit operands 16 MFMAs against 32 exponentials and 68 to 83 other
// VALU instructions (145 on the causal border): the exponentials of one 32-key tile go under the MFMAs of the next (the last one's
// under the next column tile's), tiles on the causal border apart.  Workgroups take equal shares of the tiles, from one key block into the next, and
// as many as run at a time: parts of one block each, of even sizes, left places idle (4x2048 causal 32 heads over 8, bf16 108 us,
// equal shares 98; 1x4000 causal 28 over 4, fp16 122, shares 100).
template <typename TQ, typename TK, int D, bool CAUSAL>
__global__ void __launch_bounds__(256, D == 64 ? 3 : 2) attn_weights_prompt_kernel(const WeightParams p) {
    typedef PromptTypes<TQ, TK> Types;
    typedef typename Types::E E;
    typedef typename Types::V8 V8;
    constexpr int QP = Types::qparts, KP = Types::kparts, KT = Types::tiles, KS = D / 16, DC = D / 8;
    constexpr int PER = kCols * DC / 256, ROWS = 256 / DC;  // chunks of 8 elements that a thread stages, ROWS rows apart
    __shared__ __attribute__((aligned(16))) V8 stage[2][QP][kCols * DC];
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
    // workgroup -> (share, head set, slice): slices go round the XCDs, so an L2 loads a slice's queries and keys once
    const int slices = p.B * p.Hkv;
    const int slice = blockIdx.x % slices;
    const int set = blockIdx.x / slices % p.sets, share = blockIdx.x / slices / p.sets;
    const int64_t b = slice / p.Hkv;
    const int hk = slice % p.Hkv;
    const PromptTiles<CAUSAL> tiles(p, Types::keys, b);
    const int n = tiles.n;
    int c0 = 0, pre0 = 0;  // of the first 64 blocks
    const int all = tiles.scan([&](int k0, int c, int pre) {
        if (k0 == 0) c0 = c, pre0 = pre;
    });
    if (all == 0) return;
    const PromptShares shares(all, p.shares);
    if (share >= shares.n) return;
    const int begin = shares.start(share);
    // the block there, its tiles before the share, and the share's places from the block's first place on
    int kblock = 0, skip = 0, ahead = shares.start(share + 1);
    auto look = [&](int k0, int c, int pre) {
        const uint64_t hit = __ballot(pre > begin && pre - c <= begin);
        if (hit == 0) return;
        const int l = __builtin_ctzll(hit), place = __builtin_amdgcn_readlane(pre - c, l);
        kblock = k0 + l;
        skip = max(begin - place - kStartTiles, 0);
        ahead -= place;
    };
    if (p.key_blocks <= 64) look(0, c0, pre0);
    else tiles.scan(look);
    int t0 = tiles.first(kblock) + skip, t1 = min(tiles.first(kblock) + ahead - kStartTiles, tiles.end);
    if (t0 >= t1) return;  // the share ends before the block's first tile

    // What a thread stages of a tile: chunk x0 of columns r0, r0 + ROWS, ..., query-major (query column / width, head column % width).
    // Chunk x of column r lies at x ^ swz(r): 16 columns read one chunk each without a conflict.  Chunks past the head dim are zeros
    // from the start; columns that are none (heads past the group's, and where the width does not divide 32) are the tile's first
    // one again, so that an infinite key is no NaN where it is none there.
    auto swz = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
    const int r0 = tid / DC, x0 = tid % DC, heads = p.group - set * kCols;
    for (int i = tid; i < 2 * QP * kCols * DC; i += 256) (&stage[0][0][0])[i] = V8{};
    int srow[PER];
    const TQ* src[PER];
    const float* lse_src;
    const int crow = col / p.width < p.rows && col % p.width < heads ? col / p.width : -1;  // this lane's column (-1: none)
    {
        const TQ* qb = reinterpret_cast<const TQ*>(p.q) + b * p.q_b + ((int64_t)hk * p.group + set * kCols) * p.q_h + (int64_t)t0 * p.rows * p.q_s;
        const float* lb = p.lse + b * p.lse_b + ((int64_t)hk * p.group + set * kCols) * p.lse_h + (int64_t)t0 * p.rows;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int r = r0 + k * ROWS;
            const bool none = r / p.width >= p.rows || r % p.width >= heads;
            const int head = none ? 0 : r % p.width;
            srow[k] = 8 * x0 >= p.d ? -1 : none ? 0 : r / p.width;  // -1: nothing to stage
            src[k] = qb + (srow[k] >= 0 ? srow[k] * p.q_s + head * p.q_h + 8 * x0 : 0);
        }
        lse_src = lb + (crow >= 0 ? (int64_t)(col % p.width) * p.lse_h + crow : 0);
    }
    const int64_t step = p.rows * p.q_s;
    const int tail_rows = tiles.last % p.rows;
    const int tail = tail_rows != 0 ? tiles.end - 1 : -1;  // the tile with queries past the last
    Chunk<TQ> raw[PER];
    float lse;
    auto load = [&](int t) {  // (what is loaded is not looked at here: that would wait for it)
        const int rows = t == tail ? tail_rows : p.rows;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const TQ* at = src[k];
            if (t == tail && srow[k] >= rows) at -= srow[k] * p.q_s;  // a query that is there
            raw[k] = load8(at, 0, p.d - 8 * x0 > 0 ? p.d - 8 * x0 : p.d);
            src[k] += step;
        }
        const float* at = lse_src;
        if (t == tail && crow >= rows) at -= crow;
        lse = *at;
        lse_src += p.rows;
    };
    V8* const put_at = &stage[0][0][r0 * DC + (x0 ^ swz(r0))];
    constexpr int BUF = QP * kCols * DC;
    auto put = [&](int buf, int t) {
        // a row that sees no key (an lse of -inf) may hold anything: it counts as zeros, at a weight of 0
        if (__ballot(lse == kNegInf) != 0) {
#pragma unroll
            for (int k = 0; k < PER; ++k)
                if (__shfl(lse, r0 + k * ROWS, 64) == kNegInf) raw[k] = Chunk<TQ>{};
        }
        if (t == tail && crow >= tail_rows) lse = kNegInf;  // past the last query
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            V8 o[QP];
            to_parts<TQ, V8, QP>(raw[k], o);
            // rows ROWS apart have one swz where ROWS is a multiple of its period
            const int r = r0 + k * ROWS;
            V8* const at = ROWS % 16 == 0 ? put_at + k * ROWS * DC : &stage[0][0][r * DC + (x0 ^ swz(r))];
            if (srow[k] >= 0) {
#pragma unroll
                for (int i = 0; i < QP; ++i) at[buf * BUF + i * kCols * DC] = o[i];
            }
        }
    };
    load(t0);

    const V8* get_at[KS];
#pragma unroll
    for (int x = 0; x < KS; ++x) get_at[x] = &stage[0][0][col * DC + ((2 * x) ^ (half ^ swz(col)))];
    const TK* kb = reinterpret_cast<const TK*>(p.k) + b * p.k_b + hk * p.k_h;
    int k0 = 0;
    V8 kf[KT][KP][KS];
    float c[KT][2];
    auto load_keys = [&] {
        k0 = kblock * Types::keys + __builtin_amdgcn_readfirstlane(tid >> 6) * 32 * KT;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const TK* krow = kb + (int64_t)min(k0 + 32 * t + col, n - 1) * p.k_s;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int x = 16 * s + 8 * half;
                if constexpr (sizeof(TK) == 1) {
                    const u32x2 w = x < p.d ? *reinterpret_cast<const u32x2*>(krow + x) : u32x2{0u, 0u};
                    kf[t][0][s] = codes_to_vec8<E>(w.x, w.y);
                } else {
                    const Chunk<TK> w = load8(krow, x, p.d);
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
    };
    load_keys();

    for (;;) {  // a key block, or what of its tiles is this share's
        // every thread is past the zeros of the stage, and past the last block's tiles, before the first tile is put there
        lds_barrier();
        float sum[KT][16] = {};
        float nl;
        // Stages tile t and has the next one on its way.  Buffers alternate, and the barrier has every wave past its reads of the other
        // one's last tile.
        auto turn = [&](int buf, int t) {
            put(buf, t);
            nl = crow < 0 || lse == kNegInf ? kNegInf : -lse * kLog2e;
            if (t + 1 < t1) load(t + 1);
            lds_barrier();
        };
        V8 qf[KS];  // held for the second key tile, but for the three parts of fp32
        auto queries = [&](int buf) {
            if constexpr (QP == 1) {
#pragma unroll
                for (int x = 0; x < KS; ++x) qf[x] = get_at[x][buf * BUF];
            }
        };
        auto product = [&](int buf, int kt) {
            f32x16 s = {};
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                V8 q[QP];
#pragma unroll
                for (int j = 0; j < QP; ++j) q[j] = QP == 1 ? qf[x] : get_at[x][buf * BUF + j * kCols * DC];
#pragma unroll
                for (int i = 0; i < KP; ++i)
#pragma unroll
                    for (int j = 0; j < QP && i + j < 3; ++j) s = Elem<E>::mfma32(kf[kt][i][x], q[j], s);
            }
            return s;
        };
        auto fold = [&](const f32x16& s, int kt, float at) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[kt][i] += fast_exp2(__builtin_fmaf(s[i], c[kt][i >> 3], at));
        };
        int t = t0;
        if constexpr (CAUSAL) {
            // tiles whose first query does not see the wave's last key (an even number; a wave without keys runs through them all)
            int64_t border = t1;
            if (k0 < n) border = max(((int64_t)k0 + 32 * KT - 1 - p.q_offset + p.rows - 1) / p.rows, (int64_t)t0);
            const int t_full = (int)min(border + ((border - t0) & 1), (int64_t)t1);
            for (; t < t_full; ++t) {
                const int buf = (t - t0) & 1;
                turn(buf, t);
                // the last of the wave's keys that this column sees
                int lim = (int)min(max((int64_t)t * p.rows + p.q_offset - k0, (int64_t)-64), (int64_t)(32 * KT)) + max(crow, 0);
                if (k0 >= n || __ballot(lim >= 0) == 0) continue;
                lim -= 4 * half;
                queries(buf);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const f32x16 s = product(buf, kt);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float x = fast_exp2(__builtin_fmaf(s[i], c[kt][i >> 3], nl));
                        sum[kt][i] += 32 * kt + 8 * (i >> 2) + (i & 3) <= lim ? x : 0.f;
                    }
                }
            }
        }
        if (k0 < n) {
            // scores that wait for their exponentials: the last key tile's of the column tile before
            f32x16 wait = {};
            float wait_nl = kNegInf;
            auto full = [&](auto buffer) {
                constexpr int buf = decltype(buffer)::value;
                turn(buf, t++);
                queries(buf);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    const f32x16 s = product(buf, kt);
                    fold(wait, kt == 0 ? KT - 1 : kt - 1, kt == 0 ? wait_nl : nl);
                    wait = s;
#pragma unroll
                    for (int i = 0; i < KS; ++i) {  // a step's MFMAs, and a KS-th of the VALU instructions and exponentials
                        __builtin_amdgcn_sched_group_barrier(0x008, KP * QP == 9 ? 6 : QP, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 32 / KS, 0);
                        __builtin_amdgcn_sched_group_barrier(0x400, 16 / KS, 0);
                    }
                }
                wait_nl = nl;
            };
            while (t + 1 < t1) {
                full(std::integral_constant<int, 0>());
                // the sums stay under this tile's MFMAs: left alone they sink past the next barrier
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(sum[kt][i]));
                full(std::integral_constant<int, 1>());
            }
            if (t < t1) full(std::integral_constant<int, 0>());
            fold(wait, KT - 1, wait_nl);
        } else {
            for (; t < t1; ++t) turn((t - t0) & 1, t);
        }
        // the next block's first loads go out before this one's sums meet (its keys' in one part: three would not fit the registers)
        const int done = kblock, done_k0 = k0;
        const bool whole = p.sets == 1 && t1 - t0 == tiles.count(kblock);
        ahead -= kStartTiles + tiles.count(kblock);
        if (ahead > kStartTiles) {
            t0 = tiles.first(++kblock);
            // the loads are past t1
#pragma unroll
            for (int k = 0; k < PER; ++k) src[k] += (t0 - t1) * step;
            lse_src += (int64_t)(t0 - t1) * p.rows;
            t1 = min(t0 + ahead - kStartTiles, tiles.end);
            load(t0);
            if constexpr (QP * KP == 1) load_keys();
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            float v = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float s = group_sum<32>(sum[kt][i]);
                v = col == i ? s : v;
            }
            const int at = done_k0 + 32 * kt + 8 * (col >> 2) + 4 * half + (col & 3);
            if (col < 16 && at < n) {
                // a block whose tiles are all here is done
                if (whole) p.w[b * p.w_b + hk * p.w_h + at] += v;
                else p.part[prompt_record(p, slice, set, share, done) * Types::keys + at - done * Types::keys] = v;
            }
        }
        if (done == kblock) break;
        if constexpr (QP * KP != 1) load_keys();
    }
}

// Adds a key block's records in the order of their shares.
template <bool CAUSAL, int KEYS>
__global__ void __launch_bounds__(KEYS) attn_weights_sum_kernel(const WeightParams p) {
    const int slices = p.B * p.Hkv, slice = blockIdx.x % slices, kblock = blockIdx.x / slices, key = kblock * KEYS + threadIdx.x;
    const int64_t b = slice / p.Hkv;
    const int hk = slice % p.Hkv;
    const PromptTiles<CAUSAL> tiles(p, KEYS, b);
    int from = 0, to = 0;  // the block's tiles in the list
    const int all = tiles.scan([&](int k0, int c, int pre) {
        if (kblock - k0 < 0 || kblock - k0 >= 64) return;
        to = __builtin_amdgcn_readlane(pre, kblock - k0);
        from = to - __builtin_amdgcn_readlane(c, kblock - k0);
    });
    if (from == to || key >= tiles.n) return;
    const PromptShares shares(all, p.shares);
    // the shares with tiles of the block; one that has them all is done already
    const int first = shares.of(from + kStartTiles), last = shares.of(to - 1);
    if (p.sets == 1 && first == last) return;
    float v = 0.f;
    for (int set = 0; set < p.sets; ++set) {
        const float* record = p.part + prompt_record(p, slice, set, first, kblock) * KEYS + threadIdx.x;
#pragma unroll 8
        for (int share = first; share <= last; ++share, record += KEYS) v += *record;
    }
    p.w[b * p.w_b + hk * p.w_h + key] += v;
}

namespace {

// Shares that the tiles of a (sequence, kv head, head set) are cut in.
struct PromptPlan {
    int64_t key_blocks, sets, shares, tiles;
    int32_t width, rows;
    size_t bytes;
};

PromptPlan prompt_plan(const dtattn_weights_args* a, int keys, int cus) {
    PromptPlan r;
    r.key_blocks = (a->S + keys - 1) / keys;
    const int64_t group = a->Hq / a->Hkv, slices = a->B * a->Hkv;
    r.sets = (group + kCols - 1) / kCols;
    // a tile is whole queries (of up to 32 heads each), so that a thread's part of it is the same in every tile
    r.width = (int32_t)std::min<int64_t>(group, kCols);
    r.rows = kCols / r.width;
    r.tiles = (a->L + r.rows - 1) / r.rows;
    double work = (double)r.key_blocks * (double)r.tiles;
    if (a->causal != 0) {  // key block k sees the queries from key k * keys - q_offset on
        work = 0;
        const int64_t step = std::max<int64_t>(1, r.key_blocks / 256);  // sampled
        for (int64_t k = 0; k < r.key_blocks; k += step) {
            const int64_t from = std::min<int64_t>(std::max<int64_t>(k * keys - a->q_offset, 0), a->L);
            work += (double)step * (double)(a->L - from) / r.rows;
        }
    }
    work += (double)r.key_blocks * kStartTiles;
    // Two workgroups fit a CU, three at head dims up to 64: the shares that fill so many places, one turn or more of them, for the
    // turns that take the least time (with the price of a start for every share).  us, without places for starts, at
    // 0.8 / 0.9 / 1 / 1.2 / 2 workgroups per place: 4x2048 causal 32 heads over 8, bf16 132 / 112 / 98 / 119 / 104, not causal
    // 170 / 156 / 138 / 173 / 140; 1x4000 causal 28 over 4, fp16 112 / 102 / 100 / 118 / 103; 1x1500 causal 32 over 8, fp32
    // 76 / 75 / 72 / 91 / 80; 2x2000 causal 20 of 64 at 0.5 / 0.67 / 1 / 1.1 / 1.3: 45 / 36 / 32 / 37 / 39.
    const int64_t items = slices * r.sets, slots = (a->D <= 64 ? 3 : 2) * (int64_t)cus, least = (items + slots - 1) / slots;
    const int64_t most = std::max<int64_t>(1, (int64_t)(work / kShareTiles));
    double best = 0;
    for (int64_t turns = least; turns < least + 3; ++turns) {
        const int64_t shares = std::min(most, std::max<int64_t>(1, turns * slots / items));
        const double us = (double)((items * shares + slots - 1) / slots) * (work / shares + kStartTiles);
        if (turns == least || us < best) best = us, r.shares = shares;
    }
    r.bytes = r.shares * r.sets > 1 ? (((size_t)items * (r.shares + r.key_blocks) * keys * sizeof(float) + 255) & ~(size_t)255) : 0;
    return r;
}

bool is_prompt(const dtattn_weights_args* a) { return a->L * (a->Hq / a->Hkv) > kFewColumns; }

int prompt_keys(const dtattn_weights_args* a) { return a->k_dtype == DTATTN_FP32 ? PromptTypes<float, float>::keys : PromptTypes<bf16_t, bf16_t>::keys; }

}  // namespace

template <typename TQ, typename TK, int D>
static int launch_prompt(WeightParams p, bool causal, const PromptPlan& plan, hipStream_t stream) {
    const int64_t slices = (int64_t)p.B * p.Hkv;
    p.shares = (int32_t)plan.shares, p.sets = (int32_t)plan.sets, p.key_blocks = (int32_t)plan.key_blocks;
    p.width = plan.width, p.rows = plan.rows;
    const dim3 grid((unsigned)(slices * plan.sets * plan.shares));
    if (causal) hipLaunchKernelGGL((attn_weights_prompt_kernel<TQ, TK, D, true>), grid, dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((attn_weights_prompt_kernel<TQ, TK, D, false>), grid, dim3(256), 0, stream, p);
    const int st = check_launch("attn_weights_prompt_kernel");
    if (st != DTATTN_OK || plan.bytes == 0) return st;
    constexpr int KEYS = PromptTypes<TQ, TK>::keys;
    const dim3 sums((unsigned)(plan.key_blocks * slices));
    if (causal) hipLaunchKernelGGL((attn_weights_sum_kernel<true, KEYS>), sums, dim3(KEYS), 0, stream, p);
    else hipLaunchKernelGGL((attn_weights_sum_kernel<false, KEYS>), sums, dim3(KEYS), 0, stream, p);
    return check_launch("attn_weights_sum_kernel");
}

// per_cu: workgroups wanted per CU.  One set of columns: chunks of 32 keys; more sets load the queries again for each chunk, and take
// 64.  us (of loads that bypass the caches) at 32 keys and 6 workgroups / 64 and 4: 16 of 700 to 8191, 28 heads over 4 (codes) 13.9 / 16.1, 16x8191 bf16 32 over 8 55 / 56,
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
    if (a->S > (1 << 29) || a->L > (1 << 29) || a->B > 65535 || a->Hkv > 65535 || a->B * a->Hkv > 0x7fffffff)
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
    // the sign of a scale and a scale of 0 as they are: no product is rounded by either
    p.c = sp.q_and == 0u ? 0.f : (sp.q_xor != 0u ? -sp.scale : sp.scale) * kLog2e;
    const bool causal = a->causal != 0;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    PromptPlan prompt;
    const PromptPlan* plan = nullptr;
    if (is_prompt(a)) {
        const int cus = stream_cus(stream);
        if (cus <= 0) return fail(DTATTN_ERR_DEVICE, "%s: cannot tell the stream's device", who);
        prompt = prompt_plan(a, prompt_keys(a), cus);
        if (prompt.key_blocks * (prompt.tiles + kStartTiles) > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: too many queries and keys", who);
        if (a->B * a->Hkv * prompt.sets * prompt.shares > 0x7fffffff || a->B * a->Hkv * prompt.key_blocks > 0x7fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: grid too large", who);
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
