// Page tables that sequences share: fork, reserve (copy on write) and compact, on the device (rules: dtattn.h, "pages that
// sequences share").
//
// No counterpart in the reference, which keeps no KV cache (python/dtorch/test/modules/llama.py:126-156).
//
// The tables are small, so what bounds fork and a reserve of a token is their launches; compact, and a reserve that copies many pages,
// are bound by HBM (each byte read and written once): 3950 pages of 16 tokens, 8 heads and 128 dims moved, 262 MB, 58 us with the plan's 6.
// A step of 2 x 4 beams (fork and reserve) takes 13 us of the device's time in three launches, one of 32 x 4 in pages of 64 tokens 21.
// kv_fork_kernel: a workgroup holds a slice of columns of every row in LDS, so that rows may change places in place.
// kv_reserve_plan_kernel: one workgroup. The (sequence, slot) pairs that are about to be written are its items, in order; an item's
// place among those that need a page is a prefix sum, and its place among the writers of a shared page a count of equal
// entries before it, which makes the outcome independent of any order of execution.
// kv_compact_plan_kernel: one workgroup. How many pages are used, then the k-th hole and the k-th page to move, by prefix sums over the
// counts.
#include <algorithm>

#include "decode_params.hpp"
#include "fp8_cache.hpp"

namespace dtattn {

struct PagePool {
    char* data;
    int64_t page, outer, inner;  // bytes: strides of a page, and of its two other axes
    int32_t n_outer, n_inner;    // the axis of the larger stride first
    int32_t units;               // of 16 or 4 bytes, in a row
    int32_t wide;                // 16-byte units
    int32_t token_shift;         // log2 of the tokens that a row stands for
    int32_t rows_inner;          // the inner axis is that of the rows (else of the heads)
};

struct ForkParams {
    int32_t* table;
    int32_t* lengths;
    int32_t* refs;
    const int32_t* parents;
    int64_t stride;
    int32_t B, max_pages, num_pages, width;  // width: columns of a workgroup
};

struct PagesParams {
    PagePool pool[DTATTN_MAX_PAGE_POOLS];
    int32_t* table;
    const int32_t* lengths;
    int32_t* refs;
    int32_t* out;    // pages short, or in use
    int32_t* items;  // reserve: an item's page that others share, -1 of others
    int32_t* order;  // reserve: an item's place among the pages taken, -1: takes none
    int32_t* list;   // reserve: the free pages taken; compact: [0, num_pages / 2) where to, then where from
    int32_t* map;    // compact: a page's new index, of those behind the pages that stay
    int4* copies;    // reserve: a sequence's copied page: from, to, tokens
    int32_t* moves;  // compact: how many pages move
    int64_t stride;
    int32_t B, max_pages, num_pages, page_shift, n_pools;
    int32_t n_new, slots;  // slots: that a sequence's new tokens touch, at most
};

namespace {

constexpr int kForkCells = 8192;  // table slots that a workgroup holds, and sequences
constexpr int kPlan = 1024;
constexpr int kPlanItems = 4096;  // items whose shared pages LDS holds

// Exclusive prefix sum over the workgroup (kPlan threads), and the total.
__device__ __forceinline__ int scan_plan(int v, int* lds, int& total) {
    const int wave = threadIdx.x >> 6;
    const int s = scan64(v);
    __syncthreads();  // the last call's totals have been read
    if ((threadIdx.x & 63) == 63) lds[wave] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kPlan / 64; ++i) {
        const int t = lds[i];
        before += i < wave ? t : 0;
        total += t;
    }
    return before + s - v;
}

}  // namespace

__global__ void __launch_bounds__(256) kv_fork_kernel(const ForkParams p) {
    __shared__ int cells[kForkCells];
    __shared__ int children[kForkCells];
    const int tid = threadIdx.x;
    const int first = blockIdx.x * p.width, width = min(p.width, p.max_pages - first);
    auto parent = [&](int b) {
        const int q = p.parents[b];
        return q >= 0 && q < p.B ? q : -1;
    };
    for (int b = tid; b < p.B; b += 256) children[b] = 0;
    __syncthreads();
    for (int b = tid; b < p.B; b += 256) {
        const int q = parent(b);
        if (q >= 0) atomicAdd(&children[q], 1);
    }
    for (int i = tid; i < p.B * width; i += 256) cells[i] = p.table[i / width * p.stride + first + i % width];
    __syncthreads();
    for (int i = tid; i < p.B * width; i += 256) {
        const int b = i / width, page = cells[i], q = parent(b);
        const int more = children[b] - 1;
        if (more != 0 && page >= 0 && page < p.num_pages) atomicAdd(&p.refs[page], more);
        p.table[b * p.stride + first + i % width] = q >= 0 ? cells[q * width + i % width] : -1;
    }
    if (blockIdx.x != 0) return;
    __syncthreads();  // the slots have been read
    for (int b = tid; b < p.B; b += 256) cells[b] = p.lengths[b];
    __syncthreads();
    for (int b = tid; b < p.B; b += 256) {
        const int q = parent(b);
        p.lengths[b] = q >= 0 ? cells[q] : 0;
    }
}

__global__ void __launch_bounds__(kPlan) kv_reserve_plan_kernel(const PagesParams p) {
    __shared__ int waves[kPlan / 64];
    __shared__ __attribute__((aligned(16))) int held[kPlanItems];
    const int tid = threadIdx.x;
    const int64_t capacity = (int64_t)p.max_pages << p.page_shift;
    const int n = p.B * p.slots;
    const bool in_lds = n <= kPlanItems;
    int* items = in_lds ? held : p.items;
    struct Item {
        int b, slot, page, refs;  // slot: -1 outside what is written; page: -1 empty
        bool lost;                // empty though the sequence has tokens in it: they found no page
    };
    auto item = [&](int i) {
        Item r;
        r.b = i / p.slots;
        const int64_t t = min(max((int64_t)p.lengths[r.b], (int64_t)0), capacity);
        const int64_t end = min(t + p.n_new, capacity);  // positions t .. end - 1
        const int64_t s = (t >> p.page_shift) + i % p.slots;
        r.slot = t < end && s <= (end - 1) >> p.page_shift ? (int)s : -1;
        r.page = r.slot >= 0 ? p.table[r.b * p.stride + r.slot] : -1;
        if (r.page >= p.num_pages) r.page = -1;
        r.refs = r.page >= 0 ? p.refs[r.page] : 0;
        r.lost = r.slot >= 0 && r.page < 0 && i % p.slots == 0 && (t & ((1 << p.page_shift) - 1)) != 0;
        return r;
    };
    // the first counts are on their way meanwhile
    auto count_at = [&](int64_t page) { return page < p.num_pages ? p.refs[page] : 1; };
    int early[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) early[j] = count_at(4 * tid + j);
    const Item mine = tid < n ? item(tid) : Item{0, -1, -1, 0, false};  // an item that is needed again, its loads one behind another
    auto again = [&](int i) { return i < kPlan ? mine : item(i); };
    for (int i = tid; i < n; i += kPlan) {
        const Item it = again(i);
        items[i] = it.page >= 0 && it.refs > 1 ? it.page : -1;
    }
    __syncthreads();
    // who needs a page, and which one in turn
    int need = 0, lost = 0;
    for (int i0 = 0; i0 < n; i0 += kPlan) {
        const int i = i0 + tid;
        bool takes = false, gone = false;
        if (i < n) {
            const Item it = again(i);
            takes = it.slot >= 0 && it.page < 0 && !it.lost;
            gone = it.lost;
            if (it.page >= 0 && it.refs > 1) {
                int before = 0, j = 0;  // earlier items of the same page
                if (in_lds)
                    for (; j + 4 <= i; j += 4) {
                        const int4 w = *reinterpret_cast<const int4*>(&held[j]);
                        before += (w.x == it.page) + (w.y == it.page) + (w.z == it.page) + (w.w == it.page);
                    }
                for (; j < i; ++j) before += items[j] == it.page;
                takes = before < it.refs - 1;
            }
        }
        int total;
        const int k = scan_plan((int)takes | (int)gone << 16, waves, total) & 0xffff;
        if (i < n) p.order[i] = takes ? need + k : -1;
        need += total & 0xffff, lost += total >> 16;
    }
    // that many free pages, from the lowest index up
    int found = 0;
    for (int64_t p0 = 0; p0 < p.num_pages && found < need; p0 += 4 * kPlan) {
        int v[4], free = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = (p0 == 0 ? early[j] : count_at(p0 + 4 * tid + j)) <= 0;
            free += v[j];
        }
        int total;
        int k = found + scan_plan(free, waves, total);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (v[j] && k < need) p.list[k] = (int)(p0 + 4 * tid + j);
            k += v[j];
        }
        found += total;
    }
    found = min(found, need);
    if (tid == 0) *p.out = need - found + lost;
    __syncthreads();  // counts have been read, and the list is written
    for (int i = tid; i < n; i += kPlan) {
        const Item it = again(i);
        const int k = p.order[i];
        const int to = k >= 0 && k < found ? p.list[k] : -1;
        const bool shared = k >= 0 && it.page >= 0;
        if (i % p.slots == 0) {  // the slot that holds the sequence's last tokens
            const int64_t t = min(max((int64_t)p.lengths[it.b], (int64_t)0), capacity);
            p.copies[it.b] = make_int4(it.page, to, shared && to >= 0 ? (int)(t & ((1 << p.page_shift) - 1)) : 0, 0);
        }
        if (k < 0) continue;
        p.table[it.b * p.stride + it.slot] = to;
        if (shared) atomicSub(&p.refs[it.page], 1);
        if (to >= 0) p.refs[to] = 1;
    }
}

// Copies `rows` rows of n_outer x n_inner: all units of `part` of `parts` equal shares of them.
template <typename U, int THREADS>
__device__ __forceinline__ void copy_page(const PagePool& g, int64_t from, int64_t to, int n_outer, int n_inner, int part, int parts) {
    const char* src = g.data + from * g.page;
    char* dst = g.data + to * g.page;
    const int units = g.units * n_inner;  // of one outer row
    const int total = n_outer * units;    // the host keeps it below 2^31
    const int share = (total + parts - 1) / parts, end = min(total, share * (part + 1));
    constexpr int PER = 4;
    for (int i0 = share * part + (int)threadIdx.x; i0 < end; i0 += THREADS * PER) {
        int64_t off[PER];
        U v[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int i = min(i0 + k * THREADS, end - 1);
            const int o = n_outer == 1 ? 0 : i / units, r = i - o * units;
            const int in = n_inner == 1 ? 0 : r / g.units, u = r - in * g.units;
            off[k] = o * g.outer + in * g.inner + u * (int64_t)sizeof(U);
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) v[k] = __builtin_nontemporal_load(reinterpret_cast<const U*>(src + off[k]));
        // past the caches, which the next reader finds nothing in anyway after so many pages: 262 MB of moves, read and written, 63.5 us with ordinary stores, 57.9
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (i0 + k * THREADS < end) __builtin_nontemporal_store(v[k], reinterpret_cast<U*>(dst + off[k]));
    }
}

// blockIdx: sequence, pool, part of the rows.
__global__ void __launch_bounds__(256) kv_reserve_copy_kernel(const PagesParams p) {
    const int4 c = p.copies[blockIdx.x];
    if (c.z <= 0) return;
    const PagePool& g = p.pool[blockIdx.y];
    const int rows = (c.z + (1 << g.token_shift) - 1) >> g.token_shift;
    const int no = g.rows_inner ? g.n_outer : rows, ni = g.rows_inner ? rows : g.n_inner;
    if (g.wide) copy_page<u32x4, 256>(g, c.x, c.y, no, ni, blockIdx.z, gridDim.z);
    else copy_page<uint32_t, 256>(g, c.x, c.y, no, ni, blockIdx.z, gridDim.z);
}

// PER: pages a thread takes at once.  HELD: all counts are held in registers and the moves in LDS (up to PER * kPlan pages).
template <int PER, bool HELD>
__global__ void __launch_bounds__(kPlan) kv_compact_plan_kernel(const PagesParams p) {
    constexpr int MOVES = HELD ? PER * kPlan / 2 : 1;
    __shared__ int waves[kPlan / 64];
    __shared__ int lds_to[MOVES], lds_from[MOVES], lds_refs[MOVES];
    const int tid = threadIdx.x, P = p.num_pages;
    int refs[PER];
    auto load = [&](int64_t p0) {
        const int64_t first = p0 + PER * tid;
        if (PER >= 4 && first + PER <= P) {  // wide loads
            struct __attribute__((packed, aligned(4))) Four {
                int v[4];
            };
#pragma unroll
            for (int j = 0; j + 4 <= PER; j += 4) {
                const Four f = *reinterpret_cast<const Four*>(p.refs + first + j);
#pragma unroll
                for (int i = 0; i < 4; ++i) refs[j + i] = f.v[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < PER; ++j) refs[j] = first + j < P ? p.refs[first + j] : 0;
        }
    };
    int used = 0;
    for (int64_t p0 = 0; p0 < P; p0 += PER * kPlan) {
        load(p0);
        int live = 0, total;
#pragma unroll
        for (int j = 0; j < PER; ++j) live += refs[j] > 0;
        scan_plan(live, waves, total);
        used += total;
    }
    if (tid == 0) *p.out = used;
    int* to = HELD ? lds_to : p.list;
    int* from = HELD ? lds_from : p.list + (P + 1) / 2;
    int holes = 0, late = 0;
    for (int64_t p0 = 0; p0 < P; p0 += PER * kPlan) {
        if (!HELD) load(p0);
        int hole = 0, move = 0, total;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int64_t page = p0 + PER * tid + j;
            hole += page < used && refs[j] <= 0;
            move += page >= used && refs[j] > 0;
        }
        // both sums in one: a round has 2^14 pages
        const int before = scan_plan(hole | move << 16, waves, total);
        int h = holes + (before & 0xffff), m = late + (before >> 16);
        holes += total & 0xffff, late += total >> 16;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int64_t page = p0 + PER * tid + j;
            if (page < used && refs[j] <= 0) to[h++] = (int)page;
            if (page >= used && refs[j] > 0) {
                if (HELD) lds_refs[m] = refs[j];
                from[m++] = (int)page;
            } else if (page >= used && page < P) {
                p.map[page] = (int)page;
            }
        }
    }
    if (tid == 0) *p.moves = holes;  // as many as move
    __syncthreads();
    for (int i = tid; i < holes; i += kPlan) {
        const int a = from[i], b = to[i];
        p.map[a] = b;
        p.refs[b] = HELD ? lds_refs[i] : p.refs[a];
        p.refs[a] = 0;
        if (HELD) p.list[i] = b, p.list[(P + 1) / 2 + i] = a;
    }
}

// gridDim.y - 1: the table; below it: a pool's pages, part by part.
__global__ void __launch_bounds__(256) kv_compact_move_kernel(const PagesParams p, int parts) {
    if ((int)blockIdx.y == p.n_pools) {
        const int64_t n = (int64_t)p.B * p.max_pages;
        const int used = *p.out;
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
            int32_t* slot = p.table + i / p.max_pages * p.stride + i % p.max_pages;
            const int page = *slot;
            if (page >= used && page < p.num_pages) *slot = p.map[page];
        }
        return;
    }
    const PagePool& g = p.pool[blockIdx.y];
    const int32_t* to = p.list;
    const int32_t* from = p.list + (p.num_pages + 1) / 2;
    const int64_t n = (int64_t)*p.moves * parts;
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int64_t m = i / parts;
        if (g.wide) copy_page<u32x4, 256>(g, from[m], to[m], g.n_outer, g.n_inner, (int)(i % parts), parts);
        else copy_page<uint32_t, 256>(g, from[m], to[m], g.n_outer, g.n_inner, (int)(i % parts), parts);
    }
}

namespace {

// The pools as the kernels address them; `merge`: axes that follow one another in memory become one row (whole pages are copied).
int fill_pools(const dtattn_page_pool* pools, int32_t n, int64_t page_size, bool merge, const char* who, PagePool* out) {
    if (n < 1 || n > DTATTN_MAX_PAGE_POOLS)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: %d pools of pages (from 1 to %d)", who, n, DTATTN_MAX_PAGE_POOLS);
    for (int i = 0; i < n; ++i) {
        const dtattn_page_pool& a = pools[i];
        if (a.data == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: pool %d is NULL", who, i);
        if (a.heads < 1 || a.heads > (1 << 20) || a.row_bytes < 1 || a.row_bytes > (1 << 20) || a.row_tokens < 1 ||
            a.row_tokens > page_size || page_size % a.row_tokens != 0)
            return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes of pool %d", who, i);
        const int64_t rows = page_size / a.row_tokens;
        const int64_t bits = (int64_t)reinterpret_cast<uintptr_t>(a.data) | a.row_bytes | a.page_stride |
                             (a.heads > 1 ? a.head_stride : 0) | (rows > 1 ? a.row_stride : 0);
        if (bits & 3) return fail(DTATTN_ERR_UNSUPPORTED, "%s: addresses, strides and rows of pool %d must be multiples of 4 bytes", who, i);
        if (a.page_stride < 0 || a.head_stride < 0 || a.row_stride < 0) return fail(DTATTN_ERR_UNSUPPORTED, "%s: negative strides in pool %d", who, i);
        for (int j = 0; j < i; ++j)
            if (pools[j].data == a.data) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: pools %d and %d are the same memory", who, j, i);
        if (a.heads * rows * (a.row_bytes / 4) > 0x3fffffff) return fail(DTATTN_ERR_UNSUPPORTED, "%s: pages of pool %d are too large", who, i);
        PagePool& g = out[i];
        g.data = reinterpret_cast<char*>(a.data);
        g.page = a.page_stride;
        g.wide = (bits & 15) == 0;
        g.units = (int32_t)(a.row_bytes / (g.wide ? 16 : 4));
        g.token_shift = __builtin_ctzll((unsigned long long)a.row_tokens);
        g.rows_inner = rows == 1 || (a.heads > 1 && a.head_stride >= a.row_stride) || a.heads == 1;
        g.n_outer = (int32_t)(g.rows_inner ? a.heads : rows), g.n_inner = (int32_t)(g.rows_inner ? rows : a.heads);
        g.outer = g.rows_inner ? a.head_stride : a.row_stride, g.inner = g.rows_inner ? a.row_stride : a.head_stride;
        if (!merge) continue;
        const int64_t unit = g.wide ? 16 : 4;
        if (g.n_inner == 1 || g.inner == g.units * unit) g.units *= g.n_inner, g.n_inner = 1;
        if (g.n_inner == 1 && (g.n_outer == 1 || g.outer == g.units * unit)) g.units *= g.n_outer, g.n_outer = 1;
    }
    return DTATTN_OK;
}

int table_checks(int64_t B, int64_t max_pages, int64_t num_pages, int64_t stride, const char* who) {
    if (B < 0 || B > (1 << 24) || max_pages < 1 || num_pages < 1 || num_pages > (1 << 30) || max_pages > (1 << 29))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
    if (B > 1 && stride < max_pages) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: rows of the block table overlap", who);
    return DTATTN_OK;
}

int page_size_checks(int64_t page_size, int64_t max_pages, const char* who) {
    if (page_size < 16 || (page_size & (page_size - 1)) != 0 || page_size > (1 << 20))
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: page_size %lld must be a power of two >= 16", who, (long long)page_size);
    if (max_pages > ((int64_t)1 << 30) / page_size) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: too many pages a sequence", who);
    return DTATTN_OK;
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

int64_t slots_of(const dtattn_kv_reserve_args* a) { return std::min<int64_t>((a->n_new + a->page_size - 2) / a->page_size + 1, a->max_pages); }

struct ReserveSpace {
    size_t items, order, list, copies;
};
ReserveSpace reserve_space(const dtattn_kv_reserve_args* a) {
    const size_t n = (size_t)a->B * (size_t)slots_of(a);
    ReserveSpace r;
    r.items = n > (size_t)kPlanItems ? up256(4 * n) : 0;
    r.order = up256(4 * n);
    r.list = up256(4 * std::min(n, (size_t)a->num_pages));
    r.copies = up256(16 * (size_t)a->B);
    return r;
}

}  // namespace

}  // namespace dtattn

using namespace dtattn;

extern "C" int dtattn_kv_pages_fork(const dtattn_kv_fork_args* a, void* stream_) {
    const char* who = "kv_pages_fork";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    int st = table_checks(a->B, a->max_pages, a->num_pages, a->block_table_stride, who);
    if (st != DTATTN_OK) return st;
    if (a->B > kForkCells) return fail(DTATTN_ERR_UNSUPPORTED, "%s: %lld sequences (up to %d)", who, (long long)a->B, kForkCells);
    if (a->B == 0) return DTATTN_OK;
    if (a->block_table == nullptr || a->lengths == nullptr || a->page_refs == nullptr || a->parents == nullptr)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    if (a->parents == a->lengths) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: parents and lengths are the same memory", who);
    ForkParams p = {};
    p.table = a->block_table, p.lengths = a->lengths, p.refs = a->page_refs, p.parents = a->parents;
    p.stride = a->block_table_stride;
    p.B = (int32_t)a->B, p.max_pages = (int32_t)a->max_pages, p.num_pages = (int32_t)a->num_pages;
    // Slices of about 1024 slots: a slice's time is its loops over the rows.  us with 8192 and with 1024: 128 rows of 36 slots 16.6 and 4.6
    p.width = (int32_t)std::max<int64_t>(std::min<int64_t>(1024 / a->B, a->max_pages), 1);
    const int64_t grid = (a->max_pages + p.width - 1) / p.width;
    hipLaunchKernelGGL(kv_fork_kernel, dim3((unsigned)grid), dim3(256), 0, reinterpret_cast<hipStream_t>(stream_), p);
    return check_launch("kv_fork_kernel");
}

extern "C" size_t dtattn_kv_pages_reserve_workspace_size(const dtattn_kv_reserve_args* a) {
    if (a == nullptr || a->B <= 0 || a->n_new <= 0 || a->page_size <= 0 || a->max_pages <= 0 || a->num_pages <= 0 || a->n_new > (1 << 30)) return 0;
    const ReserveSpace r = reserve_space(a);
    return r.items + r.order + r.list + r.copies;
}

extern "C" int dtattn_kv_pages_reserve(const dtattn_kv_reserve_args* a, void* stream_) {
    const char* who = "kv_pages_reserve";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    int st = table_checks(a->B, a->max_pages, a->num_pages, a->block_table_stride, who);
    if (st == DTATTN_OK) st = page_size_checks(a->page_size, a->max_pages, who);
    if (st != DTATTN_OK) return st;
    if (a->n_new < 0 || a->n_new > (1 << 30)) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: bad number of new tokens", who);
    PagesParams p = {};
    st = fill_pools(a->pools, a->n_pools, a->page_size, false, who, p.pool);
    if (st != DTATTN_OK) return st;
    if (a->short_by == nullptr || a->page_refs == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    if (a->B > 0 && a->n_new > 0) {
        if (a->block_table == nullptr || a->lengths == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
        if (a->B * slots_of(a) > (1 << 28)) return fail(DTATTN_ERR_UNSUPPORTED, "%s: too many slots", who);
        const ReserveSpace r = reserve_space(a);
        const size_t need = r.items + r.order + r.list + r.copies;
        if (a->workspace == nullptr || a->workspace_bytes < need)
            return fail(DTATTN_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, need, a->workspace_bytes);
        if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return fail(DTATTN_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
        char* ws = reinterpret_cast<char*>(a->workspace);
        p.copies = reinterpret_cast<int4*>(ws);
        p.order = reinterpret_cast<int32_t*>(ws + r.copies);
        p.list = reinterpret_cast<int32_t*>(ws + r.copies + r.order);
        p.items = reinterpret_cast<int32_t*>(ws + r.copies + r.order + r.list);
    }
    p.table = a->block_table, p.lengths = a->lengths, p.refs = a->page_refs, p.out = a->short_by;
    p.stride = a->block_table_stride;
    p.B = (int32_t)(a->n_new > 0 ? a->B : 0), p.max_pages = (int32_t)a->max_pages, p.num_pages = (int32_t)a->num_pages;
    p.page_shift = __builtin_ctzll((unsigned long long)a->page_size);
    p.n_pools = a->n_pools;
    p.n_new = (int32_t)a->n_new, p.slots = (int32_t)std::max<int64_t>(slots_of(a), 1);
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    hipLaunchKernelGGL(kv_reserve_plan_kernel, dim3(1), dim3(kPlan), 0, stream, p);
    st = check_launch("kv_reserve_plan_kernel");
    if (st != DTATTN_OK || p.B == 0) return st;
    // parts of at most 4 units a thread
    int64_t most = 1;
    for (int i = 0; i < p.n_pools; ++i) most = std::max<int64_t>(most, (int64_t)p.pool[i].units * p.pool[i].n_outer * p.pool[i].n_inner);
    const unsigned parts = (unsigned)std::min<int64_t>(std::max<int64_t>(most / 1024, 1), 32);
    hipLaunchKernelGGL(kv_reserve_copy_kernel, dim3((unsigned)p.B, (unsigned)p.n_pools, parts), dim3(256), 0, stream, p);
    return check_launch("kv_reserve_copy_kernel");
}

extern "C" size_t dtattn_kv_pages_compact_workspace_size(const dtattn_kv_compact_args* a) {
    if (a == nullptr || a->num_pages <= 0) return 0;
    return 256 + up256(4 * (size_t)(a->num_pages + 1)) + up256(4 * (size_t)a->num_pages);
}

extern "C" int dtattn_kv_pages_compact(const dtattn_kv_compact_args* a, void* stream_) {
    const char* who = "kv_pages_compact";
    if (a == nullptr) return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: args is NULL", who);
    int st = table_checks(a->B, a->max_pages, a->num_pages, a->block_table_stride, who);
    if (st == DTATTN_OK) st = page_size_checks(a->page_size, a->max_pages, who);
    if (st != DTATTN_OK) return st;
    PagesParams p = {};
    st = fill_pools(a->pools, a->n_pools, a->page_size, true, who, p.pool);
    if (st != DTATTN_OK) return st;
    if ((a->B > 0 && a->block_table == nullptr) || a->page_refs == nullptr || a->used == nullptr)
        return fail(DTATTN_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    const size_t need = dtattn_kv_pages_compact_workspace_size(a);
    if (a->workspace == nullptr || a->workspace_bytes < need)
        return fail(DTATTN_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given", who, need, a->workspace_bytes);
    if ((reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0) return fail(DTATTN_ERR_WORKSPACE, "%s: workspace must be 256-byte aligned", who);
    char* ws = reinterpret_cast<char*>(a->workspace);
    p.moves = reinterpret_cast<int32_t*>(ws);
    p.list = reinterpret_cast<int32_t*>(ws + 256);
    p.map = reinterpret_cast<int32_t*>(ws + 256 + up256(4 * (size_t)(a->num_pages + 1)));
    p.table = a->block_table, p.refs = a->page_refs, p.out = a->used;
    p.stride = a->block_table_stride;
    p.B = (int32_t)a->B, p.max_pages = (int32_t)a->max_pages, p.num_pages = (int32_t)a->num_pages;
    p.n_pools = a->n_pools;
    hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
    // as few a thread as hold them; us of the launch: 512 pages with 16 a thread 6.8, with one 2.6
    if (p.num_pages <= kPlan) hipLaunchKernelGGL((kv_compact_plan_kernel<1, true>), dim3(1), dim3(kPlan), 0, stream, p);
    else if (p.num_pages <= 4 * kPlan) hipLaunchKernelGGL((kv_compact_plan_kernel<4, true>), dim3(1), dim3(kPlan), 0, stream, p);
    else if (p.num_pages <= 8 * kPlan) hipLaunchKernelGGL((kv_compact_plan_kernel<8, true>), dim3(1), dim3(kPlan), 0, stream, p);
    else if (p.num_pages <= 16 * kPlan) hipLaunchKernelGGL((kv_compact_plan_kernel<16, true>), dim3(1), dim3(kPlan), 0, stream, p);
    else hipLaunchKernelGGL((kv_compact_plan_kernel<16, false>), dim3(1), dim3(kPlan), 0, stream, p);
    st = check_launch("kv_compact_plan_kernel");
    if (st != DTATTN_OK) return st;
    int64_t most = 1;
    for (int i = 0; i < p.n_pools; ++i) most = std::max<int64_t>(most, (int64_t)p.pool[i].units * p.pool[i].n_outer * p.pool[i].n_inner);
    const int parts = (int)std::min<int64_t>(std::max<int64_t>(most / 1024, 1), 64);
    const int64_t cus = std::max(stream_cus(stream), 1);
    const int64_t grid = std::min<int64_t>(8 * cus, std::max<int64_t>((int64_t)parts * ((p.num_pages + 1) / 2), 1));
    hipLaunchKernelGGL(kv_compact_move_kernel, dim3((unsigned)grid, (unsigned)(p.n_pools + 1)), dim3(256), 0, stream, p, parts);
    return check_launch("kv_compact_move_kernel");
}
