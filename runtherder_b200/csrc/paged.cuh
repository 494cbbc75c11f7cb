// What the kernels on the paged FP8 cache share: the layout of a layer's pool, the search of a packed batch for the
// sequence of a token, and the check of a cache description at the C boundary.
//
// Layout.  k and v are [layers][pages][kv heads][page size][head_dim] E4M3 codes, the scales [layers][pages][kv heads]
// [page size] fp32.  The keys of one head lie next to one another within a page (the one-sequence cache of the
// reference, include/runtherder/engine/kv_cache.h:18-22, puts the heads of a token next to one another): an attention
// CTA works on one kv head, so a page is then one run of page size x head_dim bytes for it, fetched by a single bulk
// copy, and its scales are another.
#pragma once
#include <climits>

#include "rh_common.cuh"

namespace rh {
namespace paged {

constexpr int kMinPage = 16, kMaxPage = 256;

// One layer of the pool and the tables, as kernels take them.
struct Layer {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    const int* page_table;   // [rows][pages_per_row]
    const int* lens;         // [rows]: tokens held, negative: idle
    int num_pages;
    int page_shift;          // log2(page size)
    int num_kv_heads;
    int num_rows;
    int pages_per_row;
};

// First key of (page, head) in units of keys: codes at this * head_dim bytes, scales at this * 4 bytes.
__device__ __forceinline__ size_t key_index(const Layer& c, int page, int head) {
    return (static_cast<size_t>(page) * c.num_kv_heads + head) << c.page_shift;
}

// The last s in 0..n-1 with first[s] <= t (0 when there is none), found by the whole warp 32 ways at a time;
// first[] is a non-decreasing list of n entries.  Empty sequences share their start with their successor, so the
// last one is the one that holds t.
__device__ __forceinline__ int warp_find_last(const int* first, int n, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, count = n;
    while (count > 1) {
        const int step = (count + 31) >> 5;
        const int at = lo + lane * step;
        const bool below = lane * step < count && first[at] <= t;
        const unsigned hits = __ballot_sync(0xffffffffu, below);
        const int last = hits ? 31 - __clz(hits) : 0;
        const int next = lo + last * step;
        count = min(step, lo + count - next);
        lo = next;
        if (step == 1) break;
    }
    return lo;
}

// Whether an entry in front of entry s names the same row (rows == null: never), found by the whole warp.  Of entries that
// name a row twice the first counts.
__device__ __forceinline__ bool named_before(const int* rows, int s, int row) {
    if (rows == nullptr) return false;
    bool found = false;
    for (int i = threadIdx.x & 31; i < s; i += 32) found |= rows[i] == row;
    return __any_sync(0xffffffffu, found);
}

}  // namespace paged

namespace host {

// Checks a cache description, all of its arrays whatever the call uses, and reports through fail().
int check_pages(const rh_kv_pages* c, const char* fn);
// The same plus the layer index; fills `out` with that layer.
int paged_layer(const rh_kv_pages* c, int layer, const char* fn, paged::Layer* out);

}  // namespace host
}  // namespace rh
