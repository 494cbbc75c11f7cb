// What the attention kernels on the paged cache share: the arguments of a decode step, the layout of its scratch, and
// the constants of the softmax states they exchange.
//
// A state of a query row over some of its keys is (m, l, acc[D]) with out = acc / l over those keys; m is a log2-domain
// exponent to which l and acc are relative, so states over disjoint keys add up as 2^(m - M) (l, acc).
#pragma once
#include <climits>

#include "paged.cuh"
#include "rh_pipeline.cuh"

namespace rh {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMInit = -1.0e30f;    // m before any key (finite: differences stay defined)
constexpr float kLgFloor = -100.0f;   // floor of log2(V scale): a zero scale must not give -inf - -inf
constexpr int kMaxSeqs = 4096;        // sequences of a decode call
constexpr int kOwnCols = 8;           // query heads of a segment of own keys
constexpr int kPrefixCols = 8;        // query rows of a prefix segment
constexpr int kHeaderInts = 4;        // {shared keys, own tiles per head, -, -}, then the first tile of every sequence
constexpr int kSharedAlign = 256;     // the prefix is cut down to a multiple of this (the largest page), the rest is own

// Bounded wait of a whole warp on an mbarrier phase: polls without the suspend-time hint (a hinted wait wakes late), the
// lanes meet again behind it.  Returns false, for all lanes, when the phase never completed.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int where, int* error_word, int tries = 1 << 20) {
    const uint32_t addr = pipe::smem_u32(bar);
    for (int i = 0; i < tries; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(addr), "r"(parity)
            : "memory");
        if (__all_sync(0xffffffffu, ok != 0)) return true;
    }
    if (error_word != nullptr) atomicCAS(error_word, 0, (where << 8) | 1);
    return false;
}

struct DecodeArgs {
    Layer c;
    __nv_bfloat16* out;
    const __nv_bfloat16* q;
    long long q_stride;        // elements between sequences
    const int* rows;
    const int* shared_pages;   // null: nothing is shared
    const int* shared_len;
    int* header;
    float* own_states;
    float* prefix_states;
    float* block_ml;           // [splits][rows][2] and [splits][rows][D], where the tensor-memory kernel takes the prefix
    float* block_acc;
    int* error_word;
    int num_seqs;
    int group;                 // query heads per kv head
    int head_chunks;
    int own_cols;
    int prefix_chunks;         // 0: nothing is shared, or the tensor-memory kernel takes it
    int block_splits;
    float scale_log2e;

    __device__ __forceinline__ int shared_keys() const {
        if (shared_len == nullptr) return 0;
        const int room = c.pages_per_row << c.page_shift;
        const int n = min(*shared_len, room);
        return n < kSharedAlign ? 0 : n - n % kSharedAlign;
    }
};

// States of `cols` query rows: m [cols], l [cols], then acc [cols][dim] from a 16-byte boundary on.
__host__ __device__ constexpr int acc_offset(int cols) { return (2 * cols + 3) / 4 * 4; }
__host__ __device__ constexpr long long state_floats(int cols, int dim) { return acc_offset(cols) + static_cast<long long>(cols) * dim; }

// Warps of the grid that get tiles: a tile each at least.  (Two or four tiles each where there are few leave fewer states to
// join, but the chain of a warp's tiles is what a small call waits for: 64 x 100 keys 12.6 us with one, 14.9 with two, 18.3 with
// four; 8 x 300 keys 10.6, 12.3, 13.0; 1 x 8196 keys 14.0, 15.8, 14.2.)
__device__ __forceinline__ long long warps_in_use(long long total, long long warps) { return total < 1 ? 1 : (total < warps ? total : warps); }

// The line of `total` tiles dealt to `warps` warps: warp w takes tiles line_start(w) .. line_start(w + 1) - 1, so tile t is that of the last
// w with floor(total w / warps) <= t.  The short division wants both sides in 32 bits: the tiles of a call may be more (4096 entries that
// name one long row), with t still small.
__host__ __device__ inline long long line_start(long long total, long long warps, long long w) { return total * w / warps; }
__host__ __device__ inline long long line_warp(long long total, long long warps, long long t) {
    const unsigned long long n = static_cast<unsigned long long>(t + 1) * static_cast<unsigned long long>(warps) - 1, by = static_cast<unsigned long long>(total);
    return (n | by) >> 32 == 0 ? static_cast<long long>(static_cast<unsigned>(n) / static_cast<unsigned>(by)) : static_cast<long long>(n / by);
}

inline int decode_ctas() { return 4 * host::num_sms(); }

// Query rows per kv head (entries x group) from which the tensor-memory kernel takes the prefix.  Whole calls with 8192 shared and
// 100 own keys, 32/8 heads, mma.sync / tcgen05: 16 rows 18.4 / 22.5 us, 24 rows 23.9 / 22.5, 40 rows 31.7 / 22.8, 64 rows 45 / 28.
constexpr int kBlockRows = 17;
int prefix_splits(int num_seqs, int num_kv_heads, int group);

struct DecodeScratch {
    size_t own, prefix, block_ml, block_acc, floats;
};
inline DecodeScratch decode_scratch(int num_seqs, int num_q_heads, int num_kv_heads, int dim) {
    const int group = num_q_heads / num_kv_heads, chunks = (group + kOwnCols - 1) / kOwnCols;
    const int cols = group < kOwnCols ? group : kOwnCols;
    const size_t warps = static_cast<size_t>(decode_ctas()) * 4;
    DecodeScratch s = {};
    s.own = (static_cast<size_t>(kHeaderInts + num_seqs + 1) + 3) / 4 * 4;
    s.prefix = s.own + (static_cast<size_t>(num_seqs) * num_kv_heads * chunks + warps) * static_cast<size_t>(state_floats(cols, dim));
    s.block_ml = s.block_acc = s.floats = s.prefix;
    if (num_seqs == 1) return s;
    const size_t rows = static_cast<size_t>(num_seqs) * group;
    if (rows < kBlockRows) {
        const size_t segs = static_cast<size_t>(num_kv_heads) * ((rows + kPrefixCols - 1) / kPrefixCols);
        s.floats = s.prefix + (segs + warps) * static_cast<size_t>(state_floats(kPrefixCols, dim));
    } else {
        const size_t states = static_cast<size_t>(prefix_splits(num_seqs, num_kv_heads, group)) * num_seqs * num_q_heads;
        s.block_acc = (s.prefix + 3) / 4 * 4;
        s.block_ml = s.block_acc + states * dim;
        s.floats = s.block_ml + states * 2;
    }
    return s;
}

}  // namespace paged
}  // namespace rh
