// Selection of the largest of some candidates by one workgroup, in ascending order of their indices: a radix select over their
// weights as unsigned numbers (11, 11 and 10 bits a round), of equal ones the first.
#pragma once
#include "fp8_cache.hpp"

namespace dtattn {

namespace {

constexpr int kSelect = 1024;

// Floats as unsigned numbers of the same order; NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (x != x) x = kNegInf;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive prefix sum over the workgroup (kSelect threads), and the total.  `lds` is not in use before the call or, until every
// thread is past a barrier, after it.
__device__ __forceinline__ int scan_all(int v, int* lds, int& total) {
    const int wave = threadIdx.x >> 6;
    const int s = scan64(v);
    if ((threadIdx.x & 63) == 63) lds[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kSelect / 64; ++i) {
        const int t = lds[i];
        before += i < wave ? t : 0;
        total += t;
    }
    return before + s - v;
}

// kept[0 .. need) = the `need` largest (fewer than cand) of weight(0 .. cand - 1), and kept[need .. need + recent) = cand, cand + 1, ...
// The candidates' weights are held PER per thread in registers (candidate PER * tid + k; PER * kSelect >= cand), or PER = 0 in
// `order`.  Called once, by kSelect threads.
template <int PER, typename Weight>
__device__ __forceinline__ void select_largest(int cand, int need, int recent, uint32_t* order, int32_t* kept, Weight weight) {
    constexpr int BINS = 2048;
    __shared__ int hist[3][BINS];  // one a round: nothing is cleared between them
    __shared__ int waves[4][kSelect / 64];
    __shared__ int found[3][2];
    const int tid = threadIdx.x, first = need;
    uint32_t mine[PER > 0 ? PER : 1];
    if constexpr (PER > 0) {
#pragma unroll
        for (int k = 0; k < PER; ++k) mine[k] = PER * tid + k < cand ? weight(PER * tid + k) : 0u;
    } else {
        for (int i = tid; i < cand; i += kSelect) order[i] = weight(i);
    }
    for (int i = tid; i < 3 * BINS; i += kSelect) (&hist[0][0])[i] = 0;
    __syncthreads();
    // The need-th largest, some bits a round: `prefix` holds the bits found so far, and `need` how many stay of those that share them
    uint32_t prefix = 0, mask = 0;
    if (need > 0) {
#pragma unroll
        for (int round = 0; round < 3; ++round) {
            const int shift = round == 0 ? 21 : round == 1 ? 10 : 0, bins = round < 2 ? 2048 : 1024;
            auto count = [&](uint32_t u) {
                if ((u & mask) == prefix) atomicAdd(&hist[round][(u >> shift) & (bins - 1)], 1);
            };
            if constexpr (PER > 0) {
#pragma unroll
                for (int k = 0; k < PER; ++k)
                    if (PER * tid + k < cand) count(mine[k]);
            } else {
                for (int i = tid; i < cand; i += kSelect) count(order[i]);
            }
            __syncthreads();
            // two bins a thread, from the largest down
            const int hi = hist[round][BINS - 1 - 2 * tid], lo = hist[round][BINS - 2 - 2 * tid];
            int total;
            const int before = scan_all(hi + lo, waves[round], total);
            if (before < need && before + hi + lo >= need) {
                const bool upper = before + hi >= need;
                found[round][0] = BINS - 1 - 2 * tid - (upper ? 0 : 1);
                found[round][1] = need - before - (upper ? 0 : hi);
            }
            __syncthreads();
            prefix |= (uint32_t)found[round][0] << shift;
            mask |= (uint32_t)(bins - 1) << shift;
            need = found[round][1];
        }
    } else {
        prefix = 0xffffffffu;  // above every weight
    }
    // those above stay, and the first `need` of those at it
    if constexpr (PER > 0) {
        int counts = 0;  // above << 16, and at it: up to 16384 of both
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (PER * tid + k < cand) counts += mine[k] > prefix ? 1 << 16 : mine[k] == prefix ? 1 : 0;
        int total;
        const int before = scan_all(counts, waves[3], total);
        int above = before >> 16, at = before & 0xffff;
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (PER * tid + k < cand) {
                const bool over = mine[k] > prefix, same = mine[k] == prefix;
                if (over || (same && at < need)) kept[above + min(at, need)] = PER * tid + k;
                above += over, at += same;
            }
    } else {
        int above = 0, at = 0;  // of the candidates before: one row of kSelect after another
        for (int i0 = 0; i0 < cand; i0 += kSelect) {
            const uint32_t u = i0 + tid < cand ? order[i0 + tid] : 0u;
            const bool over = i0 + tid < cand && u > prefix, same = i0 + tid < cand && u == prefix;
            int total;
            const int before = scan_all(((int)over << 16) + (int)same, waves[3], total);
            const int mine_at = at + (before & 0xffff);
            if (over || (same && mine_at < need)) kept[above + (before >> 16) + min(mine_at, need)] = i0 + tid;
            above += total >> 16, at += total & 0xffff;
            __syncthreads();
        }
    }
    for (int i = tid; i < recent; i += kSelect) kept[first + i] = cand + i;
}

}  // namespace

}  // namespace dtattn
