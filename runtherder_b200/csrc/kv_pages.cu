// The paged FP8 cache: append of new keys and values, and the operations on its pages (reserve, release, fork, copy,
// compact).  The reference has no counterpart (its cache holds one sequence, include/runtherder/engine/kv_cache.h);
// the quantisation of a row is its quantize_kv_fp8 (src/kernels/quantization.cu:210-250).
//
// All bookkeeping lives on the device (page table, lengths, reference counts), so a serving step that reserves,
// appends, forks and frees can be recorded into a CUDA graph.  A page is free when its reference count is zero and
// the lowest free pages are handed out first, in the order of the request: there is no free list to keep, and the
// outcome does not depend on the timing of threads.
#include <cuda_fp8.h>

#include "paged.cuh"
#include "rh_kernels.h"

namespace rh {
namespace paged {
namespace {

// ---------------------------------------------------------------- append

struct AppendArgs {
    Layer c;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    const int* cu_seqlens;
    const int* rows;          // batch entry -> table row, or null: the same
    long long k_stride;       // elements between tokens
    long long v_stride;
    int num_tokens;
    int num_seqs;
};

// The largest |x| of a lane's eight values, as a pair of halves (NaN does not count).
__device__ __forceinline__ __nv_bfloat162 amax_pair(const uint4& x) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
    return m;
}

constexpr int kAppendWarps = 4;
constexpr int kAppendRows = 4;    // head rows per lane group and warp, all in flight at once

// A warp takes kAppendRows * 32 / (D / 8) consecutive head rows of one token (its K heads, then its V heads): eight
// rows = 2 KB of reads in flight per warp at D = 128 (the rows are requested before their place is looked up).  Bound by
// HBM for packed prompts, by latency for a decode step: 8192 tokens of 8 heads x 128 11.6 us = 4.4 TB/s of reads and writes (7.8 us at a
// copy's rate), 32 tokens 2.9 us (a launch, two dependent rounds of loads, a store).  Issue slots bound it next to HBM: two rows' maxima in a
// word, one lane's division per row and no division of indexes took it from 13.7 us.
template <int D>
__global__ void __launch_bounds__(32 * kAppendWarps, 12) append_kernel(const AppendArgs p) {
    constexpr int kLanes = D / 8;                 // lanes per head row, 16 bytes each
    constexpr int kGroups = 32 / kLanes;          // head rows a warp holds side by side
    const int lane = threadIdx.x & 31, sub = lane % kLanes, group = lane / kLanes;
    const long long index = static_cast<long long>(blockIdx.x) * kAppendWarps + (threadIdx.x >> 5);
    pdl_enter();
    if (index >= p.num_tokens) return;
    const int token = static_cast<int>(index);
    const int first = blockIdx.y * (kAppendRows * kGroups);
    const int Hkv = p.c.num_kv_heads;

    uint4 x[kAppendRows];
#pragma unroll
    for (int i = 0; i < kAppendRows; ++i) {       // the rows do not depend on where they go
        const int r = first + i * kGroups + group;
        x[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < 2 * Hkv) {
            const __nv_bfloat16* const src = r < Hkv ? p.k + token * p.k_stride + static_cast<size_t>(r) * D
                                                     : p.v + token * p.v_stride + static_cast<size_t>(r - Hkv) * D;
            x[i] = ld_stream(src + 8 * sub);
        }
    }
    if (token < p.cu_seqlens[0] || token >= p.cu_seqlens[p.num_seqs]) return;    // in front of the first sequence or behind the last: nobody's
    const int s = warp_find_last(p.cu_seqlens, p.num_seqs, token);
    const int row = p.rows != nullptr ? p.rows[s] : s;
    if (row < 0 || row >= p.c.num_rows) return;
    const int held = p.c.lens[row];
    if (held < 0 || named_before(p.rows, s, row)) return;
    const long long pos = static_cast<long long>(held) + (token - p.cu_seqlens[s]);
    const long long column = pos >> p.c.page_shift;
    if (pos < 0 || column >= p.c.pages_per_row) return;
    const int page = p.c.page_table[static_cast<size_t>(row) * p.c.pages_per_row + column];
    if (page < 0 || page >= p.c.num_pages) return;
    const int slot = static_cast<int>(pos) & ((1 << p.c.page_shift) - 1);
    // quantize_kv_fp8's arithmetic: scale = amax / 448, codes e4m3_satfinite(x * (448 / amax)).  Two rows share a word for the maximum, and
    // each of four lanes divides for one row.
    uint32_t top[kAppendRows / 2];
#pragma unroll
    for (int j = 0; j < kAppendRows / 2; ++j) {
        const __nv_bfloat162 a = amax_pair(x[2 * j]), b = amax_pair(x[2 * j + 1]);
        __nv_bfloat162 m = __hmax2(__lows2bfloat162(a, b), __highs2bfloat162(a, b));
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) m = __hmax2(m, __shfl_xor_sync(0xffffffffu, m, o));
        top[j] = *reinterpret_cast<const uint32_t*>(&m);
    }
    static_assert(kAppendRows == 4 && kLanes >= 4, "a lane per row");
    const uint32_t word = sub & 2 ? top[1] : top[0];
    const float amax = fmaxf(sub & 1 ? bf_hi(word) : bf_lo(word), 0.0f);
    const float scale = quant_scale<448>(amax), inv = quant_inv_scale<448>(amax);
#pragma unroll
    for (int i = 0; i < kAppendRows; ++i) {
        const int r = first + i * kGroups + group;
        const float by = __shfl_sync(0xffffffffu, inv, (lane & ~(kLanes - 1)) + i);
        const float2 by2 = splat2(by);
        auto four = [&](uint32_t lo, uint32_t hi) {
            return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(mul2_rn(bf2_to_f2(lo), by2), __NV_SATFINITE, __NV_E4M3)) |
                   static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(mul2_rn(bf2_to_f2(hi), by2), __NV_SATFINITE, __NV_E4M3)) << 16;
        };
        const uint2 codes = make_uint2(four(x[i].x, x[i].y), four(x[i].z, x[i].w));
        if (r < 2 * Hkv) {
            const size_t key = key_index(p.c, page, r < Hkv ? r : r - Hkv) + slot;
            st_vec8((r < Hkv ? p.c.k : p.c.v) + key * D + 8 * sub, codes);
            if (sub == i) (r < Hkv ? p.c.k_scale : p.c.v_scale)[key] = scale;
        }
    }
}

// ---------------------------------------------------------------- bookkeeping (one CTA)

constexpr int kMetaThreads = 1024;
constexpr int kMetaWarps = kMetaThreads / 32;

// Exclusive prefix sum of one value per thread over the CTA, and the total.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
    }
    __syncthreads();                          // the sums of an earlier scan have been read
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int s = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += up;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    total = warp_sums[kMetaWarps - 1];
    return incl - v + (warp > 0 ? warp_sums[warp - 1] : 0);
}

// Writes the `want` lowest pages without a reference to list[] and returns how many there were (at most `want`).
// Four counts per thread and step; stops as soon as enough are found.
__device__ int find_free(const int* ref_counts, int num_pages, int want, int* list, int* warp_sums) {
    int found = 0;
    for (int base = 0; base < num_pages && found < want; base += 4 * kMetaThreads) {
        int r[4], free_here = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int id = base + 4 * threadIdx.x + i;
            r[i] = id < num_pages ? __ldcg(ref_counts + id) : 1;     // counts that this CTA changed by atomics: past L1
            free_here += r[i] <= 0;
        }
        int total;
        int at = found + block_scan(free_here, warp_sums, total);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (r[i] <= 0) {
                if (at < want) list[at] = base + 4 * threadIdx.x + i;
                ++at;
            }
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

struct Tables {
    int* page_table;
    int* lens;
    int* ref_counts;
    int* status;
    int* scratch;
    int num_pages;
    int page_shift;
    int num_rows;
    int pages_per_row;
};

// Parts of the scratch array (rh_kv_pages_scratch_ints): the first entry that names a row, three numbers per entry,
// the list of free pages or moves, and one table row per entry.
struct Scratch {
    int* owner;     // [rows]
    int* a;         // [rows]
    int* b;         // [rows]
    int* moves;     // [0] count, then (source page, destination page, filled keys) each
    int* list;      // [pages]
    int* map;       // [pages]
    int* snapshot;  // [rows][pages_per_row]
};
__host__ __device__ inline Scratch scratch_of(int* base, int num_rows, int num_pages) {
    Scratch s;
    s.owner = base;
    s.a = s.owner + num_rows;
    s.b = s.a + num_rows;
    s.list = s.b + num_rows;
    s.map = s.list + num_pages;
    s.moves = s.map + num_pages;
    const int most = num_rows > num_pages ? num_rows : num_pages;
    s.snapshot = s.moves + 1 + 3 * most;
    return s;
}
inline size_t scratch_ints(long long num_rows, long long num_pages, long long pages_per_row) {
    const long long most = num_rows > num_pages ? num_rows : num_pages;
    return static_cast<size_t>(3 * num_rows + 2 * num_pages + 1 + 3 * most + num_rows * pages_per_row);
}

// Of the entries that name the same row the first one counts: owner[row] = that entry's index.
__device__ void first_owner(int* owner, int num_rows, const int* rows, int n) {
    for (int r = threadIdx.x; r < num_rows; r += kMetaThreads) owner[r] = INT_MAX;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kMetaThreads) {
        const int r = rows != nullptr ? rows[i] : i;
        if (r >= 0 && r < num_rows) atomicMin(&owner[r], i);
    }
    __syncthreads();
}

// Gives every named row the pages it lacks for cu_seqlens[i + 1] - cu_seqlens[i] more tokens.  advance stops a row at its first place
// without a page, so what a row lacks starts on a page's border.  Places that stay unusable all the same are counted: a partly filled
// page that is gone (a new one would pass its stale slots off as the row's tokens) and a page outside the pool.
__global__ void __launch_bounds__(kMetaThreads) reserve_kernel(const Tables t, const int* rows, const int* cu_seqlens, int n) {
    __shared__ int warp_sums[kMetaWarps];
    const Scratch s = scratch_of(t.scratch, t.num_rows, t.num_pages);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_enter();
    first_owner(s.owner, t.num_rows, rows, n);
    // pages from column a[i] to column b[i] - 1 must exist; how many of them do not: kept in snapshot[i]
    int* const missing = s.snapshot;
    for (int i = warp; i < n; i += kMetaWarps) {
        const int r = rows != nullptr ? rows[i] : i;
        const bool in_range = r >= 0 && r < t.num_rows;
        const int more = cu_seqlens[i + 1] - cu_seqlens[i];
        const int held = in_range ? t.lens[r] : -1;
        int from = 0, to = 0, lack = 0;
        if (in_range && s.owner[r] == i && held >= 0 && more > 0) {
            const long long first = (static_cast<long long>(held) + (1 << t.page_shift) - 1) >> t.page_shift;
            from = static_cast<int>(first < t.pages_per_row ? first : t.pages_per_row);      // (a length may be anything)
            const long long need = (static_cast<long long>(held) + more + (1 << t.page_shift) - 1) >> t.page_shift;
            to = static_cast<int>(need < t.pages_per_row ? need : t.pages_per_row);
            if (need > t.pages_per_row && lane == 0) atomicAdd(&t.status[0], static_cast<int>(need - t.pages_per_row));
            int unusable = 0;
            for (int j = (held >> t.page_shift) + lane; j < to; j += 32) {
                const int page = t.page_table[static_cast<size_t>(r) * t.pages_per_row + j];
                if (page < 0 && j >= from) ++lack;
                else unusable += page < 0 || page >= t.num_pages;
            }
            lack = __reduce_add_sync(0xffffffffu, lack);
            unusable = __reduce_add_sync(0xffffffffu, unusable);
            if (unusable > 0 && lane == 0) atomicAdd(&t.status[0], unusable);
        } else if (lane == 0 && (!in_range || s.owner[r] != i)) {
            atomicAdd(&t.status[1], 1);
        }
        if (lane == 0) {
            s.a[i] = from;
            s.b[i] = to;
            missing[i] = lack;
        }
    }
    __syncthreads();
    int asked = 0;
    for (int base = 0; base < n; base += kMetaThreads) {      // missing[] -> offsets into the list of free pages
        const int i = base + threadIdx.x;
        int total;
        const int at = asked + block_scan(i < n ? missing[i] : 0, warp_sums, total);
        if (i < n) missing[i] = at;
        asked += total;
    }
    __syncthreads();
    if (asked == 0) return;
    const int found = find_free(t.ref_counts, t.num_pages, asked < t.num_pages ? asked : t.num_pages, s.list, warp_sums);
    if (threadIdx.x == 0 && found < asked) atomicAdd(&t.status[0], asked - found);
    for (int i = warp; i < n; i += kMetaWarps) {
        const int r = rows != nullptr ? rows[i] : i;
        int at = missing[i];
        for (int base = s.a[i]; base < s.b[i]; base += 32) {
            const int j = base + lane;
            int* const place = t.page_table + static_cast<size_t>(r) * t.pages_per_row + j;
            const bool lacks = j < s.b[i] && *place < 0;
            const unsigned m = __ballot_sync(0xffffffffu, lacks);
            const int mine = at + __popc(m & ((1u << lane) - 1u));
            if (lacks && mine < found) {
                *place = s.list[mine];
                t.ref_counts[s.list[mine]] = 1;
            }
            at += __popc(m);
        }
    }
}

// Drops every page of the named rows; lens[row] = new_len.  A page is exchanged out of its place before its count goes
// down, so a row that is named twice is released once.
__global__ void __launch_bounds__(256) release_kernel(const Tables t, const int* rows, int new_len) {
    pdl_enter();
    const int r = rows != nullptr ? rows[blockIdx.x] : static_cast<int>(blockIdx.x);
    if (r < 0 || r >= t.num_rows) {
        if (threadIdx.x == 0) atomicAdd(&t.status[1], 1);
        return;
    }
    for (int j = threadIdx.x; j < t.pages_per_row; j += blockDim.x) {
        const int page = atomicExch(&t.page_table[static_cast<size_t>(r) * t.pages_per_row + j], -1);
        if (page >= 0 && page < t.num_pages) atomicSub(&t.ref_counts[page], 1);
    }
    if (threadIdx.x == 0) t.lens[r] = new_len;
}

// lens += the new tokens, up to the row's first place without a page: the tokens from there on were not stored, and the next reserve
// asks for that place again.  (Counting them in would leave the place empty for good, and the row's later tokens of that page with it.)
__global__ void __launch_bounds__(256) advance_kernel(const Tables t, const int* rows, const int* cu_seqlens, int n) {
    pdl_enter();
    const int i = (blockIdx.x * blockDim.x + threadIdx.x) / 32;      // a warp per entry
    if (i >= n) return;
    const int r = rows != nullptr ? rows[i] : i;
    if (named_before(rows, i, r) || r < 0 || r >= t.num_rows) return;
    const int held = t.lens[r], more = cu_seqlens[i + 1] - cu_seqlens[i], lane = threadIdx.x & 31;
    if (held < 0 || more <= 0) return;
    const long long room = static_cast<long long>(t.pages_per_row) << t.page_shift, all = static_cast<long long>(held) + more;
    int end = static_cast<int>(all < room ? all : room);
    for (int base = held >> t.page_shift; static_cast<long long>(base) << t.page_shift < end; base += 32) {
        const int j = base + lane;
        bool missing = false;
        if (static_cast<long long>(j) << t.page_shift < end) {
            const int page = t.page_table[static_cast<size_t>(r) * t.pages_per_row + j];
            missing = page < 0 || page >= t.num_pages;
        }
        const unsigned m = __ballot_sync(0xffffffffu, missing);
        if (m != 0u) {
            end = (base + __ffs(m) - 1) << t.page_shift;
            break;
        }
    }
    if (lane == 0 && end > held) t.lens[r] = end;
}

// Bookkeeping is one CTA's work: its steps depend on one another and their data are a few kilobytes, so it is bound by the
// latency of some ten rounds of loads and barriers (a fork of 8 children 9.5 us with its copies, 13 us for the bookkeeping
// of 64 children with 31 shared pages each; a reserve in which nothing is lacking 3.3 us, an advance of 32 rows 1.5).  The search for
// free pages starts at page 0 and takes 4096 pages a step: a reserve of 32 rows that each need a page, 95 % of the pool used, 5.0 us
// with 1500 pages, 8.8 with 20 000, 46 with 200 000.
//
// children[i] becomes a second owner of parents[i]'s whole pages and of a page of its own for the keys behind them.
// All parents are read before any child is written (a beam step permutes rows), and the pages of the children's old
// contents are dropped last, so no page that is copied from in this call is handed out in it.
__global__ void __launch_bounds__(kMetaThreads) fork_kernel(const Tables t, const int* parents, const int* children, int n) {
    __shared__ int warp_sums[kMetaWarps];
    const Scratch s = scratch_of(t.scratch, t.num_rows, t.num_pages);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_enter();
    first_owner(s.owner, t.num_rows, children, n);
    // a[i]: tokens of the new child, -2: the entry does not count, -1: its parent is idle
    for (int i = warp; i < n; i += kMetaWarps) {
        const int par = parents[i], child = children[i];
        int held = -2;
        if (par >= 0 && par < t.num_rows && child >= 0 && child < t.num_rows && s.owner[child] == i) {
            if (par != child) held = max(-1, t.lens[par]);
        } else if (lane == 0) {
            atomicAdd(&t.status[1], 1);
        }
        if (held > 0) {
            const int full = min(held >> t.page_shift, t.pages_per_row);
            for (int j = lane; j < full; j += 32) {
                const int page = t.page_table[static_cast<size_t>(par) * t.pages_per_row + j];
                const bool real = page >= 0 && page < t.num_pages;
                s.snapshot[static_cast<size_t>(i) * t.pages_per_row + j] = real ? page : -1;
                if (real) atomicAdd(&t.ref_counts[page], 1);
            }
        }
        if (lane == 0) {
            int tail = -1;                             // b[i]: the page that holds the keys behind the whole pages
            const int column = held >> t.page_shift;
            if (held > 0 && (held & ((1 << t.page_shift) - 1)) != 0 && column < t.pages_per_row) {
                tail = t.page_table[static_cast<size_t>(par) * t.pages_per_row + column];
                if (tail >= t.num_pages) tail = -1;
            }
            s.a[i] = held;
            s.b[i] = tail;
        }
    }
    __syncthreads();
    // destinations, in the order of the entries
    int asked = 0;
    for (int base = 0; base < n; base += kMetaThreads) {
        const int i = base + threadIdx.x;
        const bool wants = i < n && s.b[i] >= 0;
        int total;
        const int at = asked + block_scan(wants ? 1 : 0, warp_sums, total);
        if (wants) {
            int* const move = s.moves + 1 + 3 * at;
            move[0] = s.b[i];
            move[2] = s.a[i] & ((1 << t.page_shift) - 1);
            s.b[i] = at;
        }
        asked += total;
    }
    __syncthreads();
    const int found = asked > 0 ? find_free(t.ref_counts, t.num_pages, asked < t.num_pages ? asked : t.num_pages, s.list, warp_sums) : 0;
    for (int k = threadIdx.x; k < found; k += kMetaThreads) {
        s.moves[1 + 3 * k + 1] = s.list[k];
        t.ref_counts[s.list[k]] = 1;
    }
    if (threadIdx.x == 0) {
        s.moves[0] = found;
        if (found < asked) atomicAdd(&t.status[0], asked - found);
    }
    __syncthreads();
    // the children's old pages go, their new ones come
    for (int i = warp; i < n; i += kMetaWarps) {
        int held = s.a[i];
        if (held == -2) continue;
        const int child = children[i];
        int* const row = t.page_table + static_cast<size_t>(child) * t.pages_per_row;
        const int full = held > 0 ? min(held >> t.page_shift, t.pages_per_row) : 0;
        const int tail = s.b[i];                       // rank of the tail's destination, -1: none
        const int fresh = tail >= 0 && tail < found ? s.list[tail] : -1;
        for (int j = lane; j < t.pages_per_row; j += 32) {
            const int old = row[j];
            if (old >= 0 && old < t.num_pages) atomicSub(&t.ref_counts[old], 1);
            row[j] = j < full ? s.snapshot[static_cast<size_t>(i) * t.pages_per_row + j] : (j == full ? fresh : -1);
        }
        if (held > 0 && fresh < 0) held = full << t.page_shift;      // no page for the tail: the whole pages alone
        if (lane == 0) t.lens[child] = held;
    }
}

// The moves that pack the used pages to the front: the k-th used page at or above the number of used pages goes to the
// k-th unused page below it.  Sources and destinations are disjoint, so the copies need no order.
__global__ void __launch_bounds__(kMetaThreads) compact_plan_kernel(const Tables t) {
    __shared__ int warp_sums[kMetaWarps];
    const Scratch s = scratch_of(t.scratch, t.num_rows, t.num_pages);
    pdl_enter();
    int used = 0;
    for (int base = 0; base < t.num_pages; base += kMetaThreads) {
        const int id = base + threadIdx.x;
        int total;
        (void)block_scan(id < t.num_pages && t.ref_counts[id] > 0 ? 1 : 0, warp_sums, total);
        used += total;
    }
    int holes = 0, sources = 0;
    for (int base = 0; base < t.num_pages; base += kMetaThreads) {
        const int id = base + threadIdx.x;
        const bool live = id < t.num_pages && t.ref_counts[id] > 0;
        const bool hole = id < used && !live, source = live && id >= used;
        int total_h, total_s;
        const int at_h = holes + block_scan(hole ? 1 : 0, warp_sums, total_h);
        const int at_s = sources + block_scan(source ? 1 : 0, warp_sums, total_s);
        if (hole) s.moves[1 + 3 * at_h + 1] = id;
        if (source) {
            s.moves[1 + 3 * at_s] = id;
            s.moves[1 + 3 * at_s + 2] = 1 << t.page_shift;
        }
        if (id < t.num_pages) s.map[id] = id;
        holes += total_h;
        sources += total_s;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < sources; k += kMetaThreads) {
        const int src = s.moves[1 + 3 * k], dst = s.moves[1 + 3 * k + 1];
        s.map[src] = dst;
        t.ref_counts[dst] = t.ref_counts[src];
        t.ref_counts[src] = 0;
    }
    if (threadIdx.x == 0) s.moves[0] = sources;
}

// ---------------------------------------------------------------- moving pages

struct MoveArgs {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    const int* src;        // explicit lists (stride 1), or
    const int* dst;
    int count;             // their length; negative: the moves of scratch, with their count and fills
    const int* moves;
    const int* map;        // compact: where every page went
    int* page_table;
    int* status;
    int table_entries;
    int num_layers;
    int num_pages;
    int page_shift;
    int num_kv_heads;
    int head_dim;
};

constexpr int kMoveThreads = 256;
constexpr int kMoveVecs = 4;                                       // 16-byte pieces per thread and step
constexpr int kMoveChunk = kMoveThreads * kMoveVecs;               // pieces per work item: 16 KB

// Work items: (move, layer, K or V, 16 KB piece of the block).  Bound by HBM: every byte is read and written once; a
// thread has four 16-byte loads in flight, eight CTAs share an SM.  A compaction's CTAs also rewrite the page table.
// Measured: 64 children of a row with a filled part of a 64-key page, 28 layers x 8 heads x 128 (416 MB read and written), 74 us with the
// fork kernel in front = 5.6 TB/s; 1500 pages compacted 59 us; 4 pages copied 3.1 us.
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const MoveArgs p) {
    pdl_enter();
    const int n = p.count >= 0 ? p.count : p.moves[0];
    const int ps = 1 << p.page_shift;
    const int vecs_per_key = p.head_dim >> 4;
    const int chunks = (p.num_kv_heads * ps * vecs_per_key + kMoveChunk - 1) / kMoveChunk;
    const long long items = static_cast<long long>(n) * p.num_layers * 2 * chunks;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        int chunk, slab, layer, m;
        if (items <= INT_MAX) {                                    // (a 64-bit division is a call)
            const unsigned rest = static_cast<unsigned>(item) / static_cast<unsigned>(chunks), block = rest >> 1;
            chunk = static_cast<int>(static_cast<unsigned>(item) - rest * static_cast<unsigned>(chunks));
            slab = static_cast<int>(rest & 1u);
            m = static_cast<int>(block / static_cast<unsigned>(p.num_layers));
            layer = static_cast<int>(block - static_cast<unsigned>(m) * static_cast<unsigned>(p.num_layers));
        } else {
            const long long rest = item / chunks, block = rest >> 1;
            chunk = static_cast<int>(item - rest * chunks);
            slab = static_cast<int>(rest & 1);
            m = static_cast<int>(block / p.num_layers);
            layer = static_cast<int>(block - static_cast<long long>(m) * p.num_layers);
        }
        int src, dst, fill = ps;
        if (p.count >= 0) {
            src = p.src[m];
            dst = p.dst[m];
        } else {
            src = p.moves[1 + 3 * m];
            dst = p.moves[1 + 3 * m + 1];
            fill = p.moves[1 + 3 * m + 2];
        }
        if (src < 0 || src >= p.num_pages || dst < 0 || dst >= p.num_pages) {
            if (layer == 0 && slab == 0 && chunk == 0 && threadIdx.x == 0) atomicAdd(&p.status[1], 1);
            continue;
        }
        if (src == dst) continue;
        const size_t keys_per_page = static_cast<size_t>(p.num_kv_heads) << p.page_shift;
        const size_t from = (static_cast<size_t>(layer) * p.num_pages + src) * keys_per_page;
        const size_t to = (static_cast<size_t>(layer) * p.num_pages + dst) * keys_per_page;
        uint4* const codes = reinterpret_cast<uint4*>(slab ? p.v : p.k);
        float* const scale = slab ? p.v_scale : p.k_scale;
        const int per_head = fill * vecs_per_key;                  // 16-byte pieces of a head that are in use
        const int total = p.num_kv_heads * per_head;
        const int begin = chunk * kMoveChunk;
        if (begin >= total) continue;
        uint4 held[kMoveVecs] = {};
        size_t at[kMoveVecs];
#pragma unroll
        for (int i = 0; i < kMoveVecs; ++i) {
            const int e = begin + i * kMoveThreads + threadIdx.x;
            at[i] = 0;
            if (e < total) {
                int off = e;
                if (fill != ps) {
                    const int head = static_cast<int>(static_cast<unsigned>(e) / static_cast<unsigned>(per_head));
                    off = head * ps * vecs_per_key + (e - head * per_head);
                }
                at[i] = static_cast<size_t>(off);
                held[i] = ld_stream(codes + from * vecs_per_key + at[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < kMoveVecs; ++i)
            if (begin + i * kMoveThreads + static_cast<int>(threadIdx.x) < total) st_vec(codes + to * vecs_per_key + at[i], held[i]);
        if (chunk == 0) {
            for (int e = threadIdx.x; e < static_cast<int>(keys_per_page); e += kMoveThreads)
                if ((e & (ps - 1)) < fill) scale[to + e] = scale[from + e];
        }
    }
    if (p.map != nullptr) {
        for (int e = blockIdx.x * kMoveThreads + threadIdx.x; e < p.table_entries; e += gridDim.x * kMoveThreads) {
            const int page = p.page_table[e];
            if (page >= 0 && page < p.num_pages) {
                const int now = p.map[page];
                if (now != page) p.page_table[e] = now;
            }
        }
    }
}

Tables tables_of(const rh_kv_pages* c) {
    Tables t;
    t.page_table = c->page_table;
    t.lens = c->lens;
    t.ref_counts = c->ref_counts;
    t.status = c->status;
    t.scratch = c->scratch;
    t.num_pages = c->num_pages;
    t.page_shift = 31 - __builtin_clz(static_cast<unsigned>(c->page_size));
    t.num_rows = c->num_rows;
    t.pages_per_row = c->pages_per_row;
    return t;
}

MoveArgs move_args(const rh_kv_pages* c) {
    MoveArgs a = {};
    a.k = c->k;
    a.v = c->v;
    a.k_scale = c->k_scale;
    a.v_scale = c->v_scale;
    a.page_table = c->page_table;
    a.status = c->status;
    a.num_layers = c->num_layers;
    a.num_pages = c->num_pages;
    a.page_shift = 31 - __builtin_clz(static_cast<unsigned>(c->page_size));
    a.num_kv_heads = c->num_kv_heads;
    a.head_dim = c->head_dim;
    return a;
}

// CTAs for at most `moves` moves: one per item up to eight per SM.
int launch_moves(const MoveArgs& a, long long moves, cudaStream_t stream, const char* fn) {
    const long long pieces = static_cast<long long>(a.num_kv_heads) * (1 << a.page_shift) * (a.head_dim >> 4);
    const long long items = moves * a.num_layers * 2 * ((pieces + kMoveChunk - 1) / kMoveChunk);
    const long long most = 8LL * host::num_sms();
    const unsigned grid = static_cast<unsigned>(items < 1 ? 1 : (items < most ? items : most));
    host::launch<move_kernel>(dim3(grid), dim3(kMoveThreads), 0, stream, a);
    return host::check_launch(fn);
}

}  // namespace
}  // namespace paged

namespace host {

int check_pages(const rh_kv_pages* c, const char* fn) {
    RH_REQUIRE(c != nullptr, RH_ERR_INVALID_ARG, "%s: null cache", fn);
    RH_REQUIRE(c->k && c->v && c->k_scale && c->v_scale && c->page_table && c->lens && c->ref_counts && c->status && c->scratch,
               RH_ERR_INVALID_ARG, "%s: the cache holds a null pointer", fn);
    RH_REQUIRE(c->num_layers >= 1 && c->num_pages >= 1 && c->num_kv_heads >= 1 && c->num_rows >= 1 && c->pages_per_row >= 1, RH_ERR_INVALID_ARG,
               "%s: num_layers, num_pages, num_kv_heads, num_rows and pages_per_row must be >= 1", fn);
    RH_REQUIRE(c->page_size >= paged::kMinPage && c->page_size <= paged::kMaxPage && (c->page_size & (c->page_size - 1)) == 0,
               RH_ERR_UNSUPPORTED_DIM, "%s: page_size must be a power of two in 16..256", fn);
    RH_REQUIRE(c->head_dim == 64 || c->head_dim == 128, RH_ERR_UNSUPPORTED_DIM, "%s: head_dim must be 64 or 128", fn);
    // (rows: the scratch's list of moves, three ints each, and a thread index of 32 per row stay within 32 bits)
    RH_REQUIRE(c->num_pages <= (1 << 24) && c->num_rows <= (1 << 24) && c->num_kv_heads <= 1024 && c->num_layers <= 4096, RH_ERR_UNSUPPORTED_DIM,
               "%s: at most 2^24 pages, 2^24 rows, 1024 kv heads and 4096 layers", fn);
    RH_REQUIRE(static_cast<long long>(c->num_rows) * c->pages_per_row <= INT_MAX / 2 && static_cast<long long>(c->pages_per_row) * c->page_size <= INT_MAX / 2,
               RH_ERR_UNSUPPORTED_DIM, "%s: num_rows * pages_per_row and pages_per_row * page_size must stay below 2^30", fn);
    RH_REQUIRE(static_cast<long long>(c->num_pages) * c->num_kv_heads * c->page_size <= INT_MAX, RH_ERR_UNSUPPORTED_DIM,
               "%s: num_pages * num_kv_heads * page_size must stay below 2^31", fn);
    RH_REQUIRE(aligned16(c->k) && aligned16(c->v) && aligned16(c->k_scale) && aligned16(c->v_scale), RH_ERR_MISALIGNED,
               "%s: k, v, k_scale and v_scale must be 16-byte aligned", fn);
    return RH_OK;
}

int paged_layer(const rh_kv_pages* c, int layer, const char* fn, paged::Layer* out) {
    if (const int e = check_pages(c, fn)) return e;
    RH_REQUIRE(layer >= 0 && layer < c->num_layers, RH_ERR_INVALID_ARG, "%s: layer %d out of range (0..%d)", fn, layer, c->num_layers - 1);
    const size_t keys = static_cast<size_t>(c->num_pages) * c->num_kv_heads * c->page_size;
    out->k = c->k + static_cast<size_t>(layer) * keys * c->head_dim;
    out->v = c->v + static_cast<size_t>(layer) * keys * c->head_dim;
    out->k_scale = c->k_scale + static_cast<size_t>(layer) * keys;
    out->v_scale = c->v_scale + static_cast<size_t>(layer) * keys;
    out->page_table = c->page_table;
    out->lens = c->lens;
    out->num_pages = c->num_pages;
    out->page_shift = 31 - __builtin_clz(static_cast<unsigned>(c->page_size));
    out->num_kv_heads = c->num_kv_heads;
    out->num_rows = c->num_rows;
    out->pages_per_row = c->pages_per_row;
    return RH_OK;
}

}  // namespace host
}  // namespace rh

using namespace rh;

extern "C" size_t rh_kv_pages_scratch_ints(int num_rows, int num_pages, int pages_per_row) {
    if (num_rows < 1 || num_pages < 1 || pages_per_row < 1) return 0;
    return paged::scratch_ints(num_rows, num_pages, pages_per_row);
}

extern "C" int rh_kv_append_paged_fp8(const rh_kv_pages* cache, int layer, const void* k, const void* v, long long k_stride, long long v_stride,
                                      const int* rows_or_null, const int* cu_seqlens, int num_tokens, int num_seqs, void* stream) {
    const char* const fn = "rh_kv_append_paged_fp8";
    paged::AppendArgs a;
    if (const int e = host::paged_layer(cache, layer, fn, &a.c)) return e;
    RH_REQUIRE(k && v && cu_seqlens, RH_ERR_INVALID_ARG, "%s: null pointer", fn);
    RH_REQUIRE(num_tokens >= 1 && num_seqs >= 1, RH_ERR_INVALID_ARG, "%s: num_tokens and num_seqs must be >= 1", fn);
    RH_REQUIRE(rows_or_null != nullptr || num_seqs <= cache->num_rows, RH_ERR_INVALID_ARG, "%s: more sequences than table rows", fn);
    const long long width = static_cast<long long>(cache->num_kv_heads) * cache->head_dim;
    RH_REQUIRE(k_stride >= width && v_stride >= width, RH_ERR_INVALID_ARG, "%s: a token stride is below num_kv_heads * head_dim", fn);
    RH_REQUIRE(host::aligned16(k) && host::aligned16(v) && k_stride % 8 == 0 && v_stride % 8 == 0, RH_ERR_MISALIGNED,
               "%s: k and v must be 16-byte aligned and their token strides multiples of 8", fn);
    a.k = static_cast<const __nv_bfloat16*>(k);
    a.v = static_cast<const __nv_bfloat16*>(v);
    a.cu_seqlens = cu_seqlens;
    a.rows = rows_or_null;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.num_tokens = num_tokens;
    a.num_seqs = num_seqs;
    const int rows_per_warp = paged::kAppendRows * 32 / (cache->head_dim / 8);
    const dim3 grid((static_cast<unsigned>(num_tokens) + paged::kAppendWarps - 1) / paged::kAppendWarps,
                    static_cast<unsigned>((2 * cache->num_kv_heads + rows_per_warp - 1) / rows_per_warp)), block(32 * paged::kAppendWarps);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (cache->head_dim == 128) host::launch<paged::append_kernel<128>>(grid, block, 0, s, a);
    else host::launch<paged::append_kernel<64>>(grid, block, 0, s, a);
    return host::check_launch(fn);
}

extern "C" int rh_kv_pages_reserve(const rh_kv_pages* cache, const int* rows_or_null, const int* cu_seqlens, int num_seqs, void* stream) {
    const char* const fn = "rh_kv_pages_reserve";
    if (const int e = host::check_pages(cache, fn)) return e;
    RH_REQUIRE(cu_seqlens != nullptr, RH_ERR_INVALID_ARG, "%s: null pointer", fn);
    RH_REQUIRE(num_seqs >= 1 && num_seqs <= cache->num_rows, RH_ERR_INVALID_ARG, "%s: num_seqs must be in 1..num_rows", fn);
    host::launch<paged::reserve_kernel>(dim3(1), dim3(paged::kMetaThreads), 0, static_cast<cudaStream_t>(stream), paged::tables_of(cache),
                                        rows_or_null, cu_seqlens, num_seqs);
    return host::check_launch(fn);
}

extern "C" int rh_kv_pages_release(const rh_kv_pages* cache, const int* rows_or_null, int num_rows, int new_len, void* stream) {
    const char* const fn = "rh_kv_pages_release";
    if (const int e = host::check_pages(cache, fn)) return e;
    RH_REQUIRE(num_rows >= 1 && num_rows <= cache->num_rows, RH_ERR_INVALID_ARG, "%s: num_rows must be in 1..the cache's rows", fn);
    RH_REQUIRE(new_len == 0 || new_len == -1, RH_ERR_INVALID_ARG, "%s: new_len must be 0 (an empty sequence) or -1 (idle)", fn);
    host::launch<paged::release_kernel>(dim3(static_cast<unsigned>(num_rows)), dim3(256), 0, static_cast<cudaStream_t>(stream), paged::tables_of(cache),
                                        rows_or_null, new_len);
    return host::check_launch(fn);
}

extern "C" int rh_kv_pages_advance(const rh_kv_pages* cache, const int* rows_or_null, const int* cu_seqlens, int num_seqs, void* stream) {
    const char* const fn = "rh_kv_pages_advance";
    if (const int e = host::check_pages(cache, fn)) return e;
    RH_REQUIRE(cu_seqlens != nullptr, RH_ERR_INVALID_ARG, "%s: null pointer", fn);
    RH_REQUIRE(num_seqs >= 1 && num_seqs <= cache->num_rows, RH_ERR_INVALID_ARG, "%s: num_seqs must be in 1..num_rows", fn);
    host::launch<paged::advance_kernel>(dim3(static_cast<unsigned>((num_seqs + 7) / 8)), dim3(256), 0, static_cast<cudaStream_t>(stream),
                                        paged::tables_of(cache), rows_or_null, cu_seqlens, num_seqs);
    return host::check_launch(fn);
}

extern "C" int rh_kv_pages_fork(const rh_kv_pages* cache, const int* parents, const int* children, int count, void* stream) {
    const char* const fn = "rh_kv_pages_fork";
    if (const int e = host::check_pages(cache, fn)) return e;
    RH_REQUIRE(parents && children, RH_ERR_INVALID_ARG, "%s: null pointer", fn);
    RH_REQUIRE(count >= 1 && count <= cache->num_rows, RH_ERR_INVALID_ARG, "%s: count must be in 1..num_rows", fn);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    host::launch<paged::fork_kernel>(dim3(1), dim3(paged::kMetaThreads), 0, s, paged::tables_of(cache), parents, children, count);
    if (const int e = host::check_launch(fn)) return e;
    paged::MoveArgs a = paged::move_args(cache);
    a.count = -1;
    a.moves = paged::scratch_of(cache->scratch, cache->num_rows, cache->num_pages).moves;
    return paged::launch_moves(a, count, s, fn);
}

extern "C" int rh_kv_pages_copy(const rh_kv_pages* cache, const int* src, const int* dst, int count, void* stream) {
    const char* const fn = "rh_kv_pages_copy";
    if (const int e = host::check_pages(cache, fn)) return e;
    RH_REQUIRE(src && dst, RH_ERR_INVALID_ARG, "%s: null pointer", fn);
    RH_REQUIRE(count >= 1 && count <= cache->num_pages, RH_ERR_INVALID_ARG, "%s: count must be in 1..num_pages", fn);
    paged::MoveArgs a = paged::move_args(cache);
    a.src = src;
    a.dst = dst;
    a.count = count;
    return paged::launch_moves(a, count, static_cast<cudaStream_t>(stream), fn);
}

extern "C" int rh_kv_pages_compact(const rh_kv_pages* cache, void* stream) {
    const char* const fn = "rh_kv_pages_compact";
    if (const int e = host::check_pages(cache, fn)) return e;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    host::launch<paged::compact_plan_kernel>(dim3(1), dim3(paged::kMetaThreads), 0, s, paged::tables_of(cache));
    if (const int e = host::check_launch(fn)) return e;
    const paged::Scratch parts = paged::scratch_of(cache->scratch, cache->num_rows, cache->num_pages);
    paged::MoveArgs a = paged::move_args(cache);
    a.count = -1;
    a.moves = parts.moves;
    a.map = parts.map;
    a.table_entries = cache->num_rows * cache->pages_per_row;
    return paged::launch_moves(a, cache->num_pages, s, fn);
}
