// Attention of many query rows over the paged FP8 cache on the 5th-generation tensor cores:
//
//   prefill   causal attention of a packed batch's new tokens: token i of an entry whose row holds n tokens sees the
//             keys 0 .. n + i of that row (its own prompt so far, and the history in front of it)
//   prefix    the shared keys of a decode step: every entry of the batch is one token, all see the same keys
//
// The reference's counterpart is flash_prefill_bf16 (include/runtherder/kernels/flash_prefill.cuh:27-40), one sequence
// in a contiguous cache.  As in flash_prefill_ws.cu a CTA carries one or two blocks of 128 query rows of one kv head (the
// group's heads x consecutive tokens), walks key tiles of 64, keeps S and O in tensor memory, and splits the work by role:
//
//   S[128 x 64] = Q K^T      E4M3 x E4M3 (tcgen05 kind::f8f6f4), operands in shared memory
//   O[128 x D] += W V        f16 (kind::f16): W = 2^(S c ks - m) in tensor memory, V = code x V scale in shared memory
//
//   softmax warps (8 per block)   scores -> weights; two rows x sixteen keys per thread
//   product warps                 one warp issues S = Q K^T (of both blocks in turn), one per block O += W V
//   conversion warps (4)          raw E4M3 V tiles -> f16 operand tiles, scales folded in; a tile's constants for the softmax
//   copy warp                     fetches K tiles (tensor-map copies, swizzled as the product wants them), V tiles (bulk
//                                 copies) and scales page by page into four stages
//
// What is different from there, and why.
// (1) K codes are operands as they lie in the cache: q is split into two E4M3 parts, q = hi + lo, and S = hi K^T + lo K^T.
//     bf16 has 8 significant bits, E4M3 4: with the row scaled so that its largest |q| is in 128..256, every element
//     above 2^-9 of it is exact, smaller ones are off by at most 2^-16 of it.  Two E4M3 products take the time of one f16
//     product, and nothing has to convert K: clock stamps of the f16 form (0.80 ms on 8192 tokens, 32/8 heads of 128) had
//     every product waiting for the converted K tile, and both row blocks in step behind it.
// (2) The V scale is folded into the f16 V operand instead of riding in the exponent: no per-key additions and multiplications
//     in the softmax.  That is two roundings of 2^-11, the scale's (common to a key's row of V) and the product's; flash_prefill_ws.cu
//     has neither.  f16 holds vs * 448 only for vs in 2^-22 .. 2^-1 (with a common factor of 2^8); a tile with a scale outside
//     keeps the exponent form, and both add up in one O: beside a key of scale vs > 1/2 the others' weights are taken relative to a
//     maximum up to 2^8 vs higher, and f16 loses what is below 2^-32 of that.
// (3) The running maximum may lag the true one by up to 2^8, so that O is rescaled a handful of times per row instead of on most
//     tiles.  Weights carry a factor of 2^7: they stay below 2^15, and what f16 loses of small ones is below 2^-32 of the largest
//     (unshifted it was 2^-25: over 8192 keys that may be 2^-12 of the output, over 128k keys 2^-8, all of it missing from the
//     numerator and present in the denominator).  Each weight is rounded to f16 once, 2^-11; the denominator sums the unrounded
//     fp32 weights, so a row that one key dominates is off by up to 2^-11 (its largest weight is seldom a power of two; in
//     flash_prefill_ws.cu it is exactly 1): an eighth of the bf16 store's 2^-8, like every other rounding here.
// (4) Rows carry their own last visible key, pages may be missing, and places that no row may see may hold anything: the
//     tiles that reach past some row's last key (and only those) replace NaN codes of V by zero and mark the key, so that
//     exactly the rows that see it get NaN.
//
// Measured (B200, 32/8 heads of 128).  Six ragged prompts of 8192 tokens together 228 us = 634 TFLOP/s; one prompt of 8192 tokens 610 - 665
// us = 825 - 900 TFLOP/s, by how long the power cap leaves the clock up (flash_prefill_ws.cu on a contiguous cache: 718 us); the 32768
// shared keys of 128 sequences about 85 us.
// A tile of 64 keys takes two row blocks 1.3 us and costs 1152 cycles of products (tensor pipe 30 - 39 % busy) and 1024 of
// exponentials; issue slots are 53 % busy.  What bounds it is the chain of a tile through a softmax warp (scores from tensor memory,
// maximum, exponentials, weights to tensor memory, the product that frees them).  Tried without gain: 128-key tiles (765 us), the next
// tile's scores loaded early (650 us, spills), exponentials partly as polynomials or left out altogether (no change), the two
// blocks' softmax phases made exclusive (607 - 660 us), two one-block CTAs per SM (737 us).  A CTA costs 9.2 us besides its tiles: 4.2 to
// fetch and split q, 2.7 to store its rows, 1.0 to find its tokens; ragged prompts with seven CTAs per SM lose a third of their
// time to that.  CTAs that fetch further work by cluster launch control, with its first tiles on the way, took ragged prompts to 217 - 223
// us, but short ones from 13.4 to 14.4 and one long one with 16-key pages from 680 to 702: not kept.
#include <cuda.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <cmath>
#include <type_traits>

#include "flash_prefill_roles.cuh"
#include "flash_prefill_tc.cuh"
#include "paged_prefill.cuh"
#include "rh_kernels.h"

namespace rh {
namespace paged {
namespace {

using namespace tc;
using ws::group_or;

// Bounded wait on an mbarrier phase that also ends when another thread of the CTA has given up (ws::wait_phase's contract):
// the common case, a phase that is complete or completes within a few polls, is a loop of two instructions.
// (Called by whole warps.)  kBackoffNs: pause after sixteen polls, for roles that are ahead (every poll goes through the shared-memory pipe).
template <int kBackoffNs = 0>
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* gave_up, int where, int* error_word) {
    const uint32_t addr = pipe::smem_u32(bar);
    for (int i = 0; i < ws::kTries / 16; ++i) {
        uint32_t left;
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .u32 n;\n\tmov.u32 n, 16;\n"
            "again%=:\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "@p bra done%=;\n\t"
            "sub.u32 n, n, 1;\n\t"
            "setp.ne.u32 p, n, 0;\n\t"
            "@p bra again%=;\n"
            "done%=:\n\t"
            "mov.u32 %0, n;\n\t}"
            : "=r"(left)
            : "r"(addr), "r"(parity)
            : "memory");
        // The lanes of a warp may see the phase complete on different polls: they meet again here, before instructions that
        // want the whole warp.
        if (__all_sync(0xffffffffu, left != 0)) return true;
        if (__any_sync(0xffffffffu, *gave_up != 0)) return false;
        if constexpr (kBackoffNs > 0) __nanosleep(kBackoffNs);
    }
    *gave_up = 1;
    if (error_word != nullptr) atomicCAS(error_word, 0, (where << 8) | 1);
    return false;
}

constexpr int kVBuffers = 3;             // f16 V operand tiles
constexpr int kStages = 4;               // tiles (K and V codes, scales) in flight or in use
constexpr int kCstRing = 4;              // a tile's constants: read until its weights are out, at most two tiles after they were written
constexpr int kFoldShift = 8;            // V operand = code * vs * 2^8
constexpr float kFoldLow = 2.384185791015625e-07f;    // 2^-22
constexpr float kFoldHigh = 0.5f;
constexpr float kLag = 8.0f;             // how far (log2) the running maximum may lie below the true one
constexpr float kShift = 7.0f;           // weights are 2^7 * weight, at most 2^15: f16 holds them down to 2^-31 of the row's largest

struct BlockArgs {
    Layer c;
    __nv_bfloat16* out;
    const __nv_bfloat16* q;
    const int* rows;
    const int* cu_seqlens;     // prefill
    const int* shared_pages;   // prefix
    const int* shared_len;
    float* state_ml;           // [splits][num_rows of out][2], [..][D]; null: the rows are finished here
    float* state_acc;
    int* error_word;
    long long q_stride;
    long long out_rows;
    int num_tokens;            // prefix: the batch's entries
    int num_seqs;
    int num_q_heads;
    int group;
    int heads_per_cta;
    int tokens_per_block;
    int slot_mul;              // ceil(2^16 / tokens_per_block): exact for the 128 rows of a block
    int head_chunks;
    float scale_log2e;
};

// What a CTA works on: its tokens (indexes into q, and how many exist from the first on), the keys in front of them and the keys that
// any of its rows sees, and where they lie.
struct Job {
    const int* pages;
    int token0, tokens, held, total_keys, work;
};

// Per block: S complete, O += W V complete and W ready, each for even and for odd tiles, and S read (where S has one buffer).
// "W ready" is two because a warp may finish tile i + 1 (whose scores only wait for everyone to have READ those of tile i) while another
// one still rescales O for tile i, and its arrival must not count for tile i.
enum BlockBar { kBarQK = 0, kBarPV = 2, kBarSRead = 4, kBarWReady = 5 };

template <int D, int kBlocks>
struct Geo {
    static constexpr int kSoftmaxWarps = 8 * kBlocks;
    static constexpr int kIssuerWarp0 = kSoftmaxWarps;
    static constexpr int kConvWarp0 = kSoftmaxWarps + 1 + kBlocks;          // one warp for S, one per block for O (24 warps: 80 registers each)
    static constexpr int kConvThreads = 128;
    static constexpr int kCopyWarp = kConvWarp0 + kConvThreads / 32;
    static constexpr int kThreads = 32 * (kCopyWarp + 1);
    // One row block of a shared prefix is held to 96 registers a thread (as for a block of 640), so that its 480 threads leave
    // a CTA of the decode kernel, which works on the sequences' own keys at the same time, room on the SM: 32 sequences
    // with 32768 shared keys and one of their own 60.6 -> 51.0 us, 12 with 8192 and 600 31.2 -> 30.3 us.
    static constexpr int kBoundThreads = kBlocks == 1 ? 640 : kThreads;
    static constexpr int kPieces = kKeys * (D / 16);                        // 16-byte pieces of a raw tile
    static constexpr int kPerConv = kPieces / kConvThreads;
    static constexpr int kTmem = kTmemCols * kBlocks;
    // A block's 256 columns.  D = 128: S 64, O 128, W (f16 pairs) 32, lo part of Q (four codes each) 32.  D = 64: S twice, O 64,
    // W_i over the columns of S_i; no warp waits for the others to have read S, nor for the last product to have read W.  One prompt of
    // 8192 tokens, heads of 64: 513 us as for 128, 480 - 490 so; 700 tokens behind 12000 keys 140 / 137.  Heads of 128 have the
    // columns for it only with lo in shared memory, which their products fill first: six ragged prompts 228 / 233 us.
    static constexpr bool kTwoS = D == 64;
    static constexpr int kOCol = kTwoS ? 2 * kKeys : kKeys, kWCol = kTwoS ? 0 : kOCol + D, kQCol = kWCol + kKeys / 2;
    static constexpr int kSStep = kTwoS ? kKeys : 0;                        // from S (and W) of an even tile to that of an odd one
    static_assert((kTwoS ? kOCol + D : kQCol + D / 4) <= kTmemCols, "tensor memory of a block");
    static constexpr int kDimBlocks = D / 64;                               // of the V operand
    static constexpr int kQPart = kRows * D;                                // q hi (or lo) of a block: rows of D bytes
    static constexpr int kTileBytes = kDimBlocks * kKeys * 128;             // an f16 V operand tile
    static constexpr int kRawBytes = kKeys * D;
    static constexpr int kScaleAt = 2 * kRawBytes;                          // a stage: K codes, V codes, K scales, V scales (1 KB aligned)
    static constexpr int kStageBytes = 2 * kRawBytes + 1024;
    static constexpr int kCstFloats = 3 * kKeys + 4;                        // K scales; where V scales ride in the exponent: log2, inverse; flags
    static constexpr int kSQ = 0;
    static constexpr int kSK = kSQ + kBlocks * 2 * kQPart;                  // (a block's 128 rows of hi, then of lo; at the end its rows of out)
    static constexpr int kSV = kSK + kStages * kStageBytes;
    static constexpr int kSRow = kSV + kVBuffers * kTileBytes;                    // per block: the rows' factors
    static constexpr int kSCst = kSRow + kBlocks * kRows * 4;           // [kCstRing]
    static constexpr int kSPoison = kSCst + kCstRing * kCstFloats * 4;      // per V buffer and key: 0, or NaN
    static constexpr int kSBar = kSPoison + kVBuffers * kKeys * 4;
    static constexpr int kSmemBytes = kSBar + 512 + 1024;
    static constexpr int kBarsPerBlock = 7;
    static constexpr int kBarVReady = kBarsPerBlock * kBlocks;
    static constexpr int kBarVEmpty = kBarVReady + kVBuffers;
    static constexpr int kBarFull = kBarVEmpty + kVBuffers;
    static constexpr int kBarEmpty = kBarFull + kStages;
    static constexpr int kBarCst = kBarEmpty + kStages;
    static constexpr int kBarConv = kBarCst + kCstRing;
    static constexpr int kNumBars = kBarConv + 1;
    static constexpr int kJobAt = 8 * kNumBars + 4 * (4 + kStages);         // what the CTA works on, from the warp that looks it up
    static_assert(kJobAt % 8 == 0 && kJobAt + static_cast<int>(sizeof(Job)) <= 512, "barrier area");
    // arrivals per phase
    __device__ static constexpr uint32_t bar_count(int i) {
        if (i < kBarVReady) {
            const int of = i % kBarsPerBlock;
            // S: the product's completion, and the product warp for the rest that the tile needs; O: the completion; then the softmax warps
            return of < kBarPV ? 2 : of < kBarSRead ? 1 : 8;
        }
        if (i < kBarVEmpty) return kConvThreads;
        if (i < kBarFull) return kBlocks;
        if (i < kBarEmpty) return 1 + 32;                       // the bulk copies' bytes, and the copy warp's lanes for their scales
        if (i < kBarCst) return 1 + kConvThreads / 32;          // the S products, the conversion warps
        if (i < kBarConv) return kKeys / 32;
        return kConvThreads;
    }
    static_assert(kSK % 1024 == 0 && kStageBytes % 1024 == 0 && kSV % 1024 == 0 && kTileBytes % 1024 == 0, "operand tiles are 1 KB aligned");
};
enum TileFlag { kSlow = 16 };            // flags: bits 0..3 = sixteen-key groups that exist, 16 = V scales ride in the exponent

// Shared-memory descriptor of an E4M3 operand with rows of D bytes (K-major): 128-byte swizzle for D = 128, 64-byte for 64.
template <int D>
__device__ __forceinline__ uint64_t code_desc(uint32_t addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(1) << 16;
    d |= static_cast<uint64_t>((8 * D) >> 4) << 32;                         // eight rows
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(D == 128 ? 2 : 4) << 61;
    return d;
}
// byte offset of 16-byte piece `piece` of row `row` in such an operand
template <int D>
__device__ __forceinline__ int code_at(int row, int piece) {
    return D == 128 ? row * 128 + ((piece ^ (row & 7)) << 4) : row * 64 + ((piece ^ ((row >> 1) & 3)) << 4);
}
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// the same product with the rows (A) in tensor memory: lane = row, four codes per 32-bit column
__device__ __forceinline__ void umma_f8_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
        : "memory");
}
// rows y .. of a [rows][D] byte array into shared memory, swizzled by the map; x is always 0
__device__ __forceinline__ void tensor_load(void* dst, const CUtensorMap* map, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(pipe::smem_u32(dst)),
                 "l"(map), "r"(0), "r"(y), "r"(pipe::smem_u32(bar))
                 : "memory");
}
// A value twice in a register pair, kept as one 64-bit operand: built from two floats at every use, a pair costs two moves
// (a fifth of the softmax loop's instructions were these).
__device__ __forceinline__ unsigned long long both(float v) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float2 fma2_both(float2 a, unsigned long long b, unsigned long long c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rd;\n\tmov.b64 ra, {%2, %3};\n\tfma.rn.f32x2 rd, ra, %4, %5;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "l"(b), "l"(c));
    return d;
}
// true in one lane of the (whole) warp
__device__ __forceinline__ bool elect_one() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}
// Whether a V scale is outside what the f16 operand holds.  (A NaN is not: it makes the operand NaN.)
__device__ __forceinline__ bool outside_fold(float vs) { return vs != 0.0f && vs == vs && !(vs >= kFoldLow && vs <= kFoldHigh); }
// Two bf16 times a power of two -> E4M3 codes hi and lo: hi is the value cut after four significant bits, which E4M3 holds,
// lo the four that are left.
__device__ __forceinline__ void split_e4m3x2(uint32_t w, float down, uint32_t& hi, uint32_t& lo) {
    const uint32_t top = w & 0xfff0fff0u;
    const float2 x = mul2_rn(bf2_to_f2(w), splat2(down)), h = mul2_rn(bf2_to_f2(top), splat2(down));
    hi = __nv_cvt_float2_to_fp8x2(h, __NV_SATFINITE, __NV_E4M3);
    lo = __nv_cvt_float2_to_fp8x2(add2_rn(x, neg2(h)), __NV_SATFINITE, __NV_E4M3);
}
// The tokens of an entry that the call has (offsets may name more: the grid has CTAs for the call's).
__device__ __forceinline__ int entry_tokens(const BlockArgs& p, int s) { return max(0, min(p.cu_seqlens[s + 1], p.num_tokens) - p.cu_seqlens[s]); }
// The keys that a row holds, at most what its table has places for (a length may be anything); negative: idle.
__device__ __forceinline__ int keys_held(const BlockArgs& p, int row) { return min(p.c.lens[row], p.c.pages_per_row << p.c.page_shift); }
// The batch entry and the token tile of CTA `index` (of all token tiles of all entries); false: there is none.
// Tiles are numbered from the one with the most keys down, so the long ones start first: depth = keys in units of a
// tile's tokens, and for at most 32 entries the number of tiles beyond a depth is one warp sum.
__device__ __forceinline__ bool find_tile(const BlockArgs& p, int index, int tile_tokens, int& seq, int& tile) {
    const int lane = threadIdx.x & 31;
    if (p.num_seqs <= 32) {
        int n = 0, behind = 0;
        if (lane < p.num_seqs) {
            n = (entry_tokens(p, lane) + tile_tokens - 1) / tile_tokens;
            const int row = p.rows != nullptr ? p.rows[lane] : lane;
            if (row >= 0 && row < p.c.num_rows) behind = max(0, keys_held(p, row)) / tile_tokens;
        }
        // the largest depth d such that the tiles of depth > d are at most `index`; tile t of an entry has depth behind + t + 1
        const int deepest = __reduce_max_sync(0xffffffffu, n > 0 ? behind + n : 0);
        int lo = 0, hi = deepest;                 // tiles deeper than lo: > index (or lo = 0); than hi: <= index
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            const int deeper = __reduce_add_sync(0xffffffffu, min(n, max(0, behind + n - mid)));
            if (deeper <= index) hi = mid;
            else lo = mid + 1;
        }
        const int deeper = __reduce_add_sync(0xffffffffu, min(n, max(0, behind + n - lo)));
        // among the tiles of depth lo, the (index - deeper)-th entry that has one
        const bool here = n > 0 && lo > behind && lo <= behind + n;
        const unsigned who = __ballot_sync(0xffffffffu, here);
        const int want = index - deeper;
        if (want >= __popc(who)) return false;
        seq = __fns(who, 0, want + 1);
        tile = __shfl_sync(0xffffffffu, lo - behind - 1, seq);
        return true;
    }
    int before = 0;
    for (int base = 0; base < p.num_seqs; base += 32) {
        const int s = base + lane;
        const int n = s < p.num_seqs ? (entry_tokens(p, s) + tile_tokens - 1) / tile_tokens : 0;
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, before + incl > index);
        if (hit != 0u) {
            const int at = __ffs(hit) - 1;
            seq = base + at;
            const int inside = index - before - __shfl_sync(0xffffffffu, incl - n, at);
            tile = __shfl_sync(0xffffffffu, n, at) - 1 - inside;
            return true;
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    return false;
}

// grid (kv heads x head chunks, token tiles, key ranges)
template <int D, int kBlocks, bool kPrefix>
__global__ void __launch_bounds__(kPrefix ? Geo<D, kBlocks>::kBoundThreads : Geo<D, kBlocks>::kThreads, 1) paged_blocks_kernel(const BlockArgs p, const __grid_constant__ CUtensorMap k_map) {
    using G = Geo<D, kBlocks>;
    extern __shared__ unsigned char raw_smem[];
    const uint32_t base = (pipe::smem_u32(raw_smem) + 1023u) & ~1023u;
    unsigned char* const sm = raw_smem + (base - pipe::smem_u32(raw_smem));
    uint64_t* const bars = reinterpret_cast<uint64_t*>(sm + G::kSBar);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(sm + G::kSBar + 8 * G::kNumBars);
    volatile int* const gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* const least = reinterpret_cast<int*>(tmem_slot + 2);            // prefix: the CTA's least last visible key
    int* const stage_groups = reinterpret_cast<int*>(tmem_slot + 4);     // [kStages] sixteen-key groups that were fetched

    // (through a shuffle, so that the compiler knows the warp's number and what follows from it to be uniform: the product
    // warps' descriptors then live in uniform registers)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if constexpr (kPrefix) {
        if (*p.shared_len < kSharedAlign) {      // nothing is shared: no state is written, and none is read
            pdl_trigger();
            pdl_wait();
            return;
        }
    }
    const int kvh = blockIdx.x / p.head_chunks;
    const int chunk = blockIdx.x - kvh * p.head_chunks;

    if (warp == 1) {
        for (int i = lane; i < G::kNumBars; i += 32) pipe::mbar_init(&bars[i], G::bar_count(i));
        if (lane == 0) {
            *gave_up = 0;
            *least = INT_MAX;
        }
        pipe::mbar_init_fence();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pipe::smem_u32(tmem_slot)), "r"(G::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // ---- what this CTA works on.  The prefix kernel follows a kernel of the same call whose results it does not need, and
    //      which has seen its own predecessors complete before this one may start: it waits at its end instead. ----
    if constexpr (!kPrefix) pdl_wait();
    pdl_trigger();
    Job* const job = reinterpret_cast<Job*>(sm + G::kSBar + G::kJobAt);
    const int tile_tokens = kBlocks * p.tokens_per_block;
    if (warp == 2) {                 // (one warp: 24 of them waiting for the same loads and warp sums took twice as long)
        Job j = {};
        if constexpr (kPrefix) {
            const int room = p.c.pages_per_row << p.c.page_shift;
            const int n = min(*p.shared_len, room);
            j.total_keys = n < kSharedAlign ? 0 : n - n % kSharedAlign;
            j.token0 = blockIdx.y * tile_tokens;
            j.tokens = p.num_tokens - j.token0;
            j.pages = p.shared_pages;
            j.work = 1;
        } else {
            int seq = 0, tile = 0;
            if (find_tile(p, blockIdx.y, tile_tokens, seq, tile)) {
                const int first = p.cu_seqlens[seq], n = entry_tokens(p, seq);
                const int row = p.rows != nullptr ? p.rows[seq] : seq;
                j.token0 = first + tile * tile_tokens;
                j.tokens = n - tile * tile_tokens;
                j.work = first >= 0 && j.tokens > 0;
                const int behind = row >= 0 && row < p.c.num_rows ? keys_held(p, row) : -1;
                if (behind >= 0) {
                    const long long room = static_cast<long long>(p.c.pages_per_row) << p.c.page_shift;
                    j.held = behind + tile * tile_tokens;
                    const long long seen = static_cast<long long>(j.held) + min(j.tokens, tile_tokens);
                    j.total_keys = static_cast<int>(seen < room ? seen : room);
                    j.pages = p.c.page_table + static_cast<size_t>(row) * p.c.pages_per_row;
                }
            }
        }
        if (lane == 0) *job = j;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const int token0 = job->token0, tokens = job->tokens, held = job->held, total_keys = __shfl_sync(0xffffffffu, job->total_keys, 0);
    const bool work = __shfl_sync(0xffffffffu, job->work, 0) != 0;
    const int* const pages = job->pages;

    const int all_tiles = (total_keys + kKeys - 1) / kKeys;
    const int j0 = static_cast<int>(static_cast<long long>(all_tiles) * blockIdx.z / gridDim.z);
    const int n_tiles = work ? static_cast<int>(static_cast<long long>(all_tiles) * (blockIdx.z + 1) / gridDim.z) - j0 : 0;

    const int blk = warp < G::kSoftmaxWarps ? warp >> 3 : (warp > G::kIssuerWarp0 && warp < G::kConvWarp0 ? warp - G::kIssuerWarp0 - 1 : 0);
    const int wb = warp & 7;
    const int block_tok = blk * p.tokens_per_block;          // first token of the block, counted from token0
    uint64_t* const bb = bars + blk * G::kBarsPerBlock;
    const uint32_t tmem_s = tmem + blk * kTmemCols, tmem_o = tmem_s + G::kOCol, tmem_w = tmem_s + G::kWCol, tmem_q = tmem_s + G::kQCol;
    const int q_off = G::kSQ + blk * 2 * G::kQPart;

    // a row of a block: its head slot and token (counted from token0); whether it exists; the last key it sees
    auto row_at = [&](int row, int& tok, int& head) {
        const int slot = (row * p.slot_mul) >> 16;           // row / tokens_per_block
        tok = block_tok + (row - slot * p.tokens_per_block);
        const int hg = chunk * p.heads_per_cta + slot;
        head = kvh * p.group + hg;
        return work && slot < p.heads_per_cta && hg < p.group && tok < tokens;
    };
    auto last_key = [&](int tok) {
        if constexpr (kPrefix) {
            const int b = token0 + tok;
            const int row = p.rows != nullptr ? p.rows[b] : b;
            if (row < 0 || row >= p.c.num_rows) return -1;
            return max(-1, p.c.lens[row]);
        } else {
            return held + tok;
        }
    };
    // the least last visible key of the CTA's rows: tiles beyond it hold keys that a row must not see
    if constexpr (kPrefix) {
        if (tid < min(tokens, tile_tokens)) atomicMin(least, last_key(tid));
        __syncthreads();
    }
    const int seen_by_all = kPrefix ? *least : held;

    // ---- Q (softmax warps): bf16 -> two E4M3 parts, hi in shared memory, lo (D = 128) in tensor memory (products whose rows come from
    //      there read a third of the shared memory: its port is what this kernel fills first).  A row is scaled by a power of
    //      two so that its largest |q| lies in 2^7 .. 2^8; its scores take that back.  D / 16 lanes read a row together; lo
    //      goes through shared memory, because a tensor-memory store wants a row per thread. ----
    float* const row_factor = reinterpret_cast<float*>(sm + G::kSRow) + blk * kRows;
    if (warp < G::kSoftmaxWarps && n_tiles > 0) {
        constexpr int kLanes = D / 16, kRowsAtOnce = 32 / kLanes, kSteps = 16 / kRowsAtOnce;     // a warp takes 16 rows
        const int sub = lane % kLanes, row0 = 16 * wb + lane / kLanes;      // a lane takes 8 values of each half of its rows
        uint4 w[kSteps][2];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            int tok, head;
            w[i][0] = w[i][1] = make_uint4(0u, 0u, 0u, 0u);
            if (row_at(row0 + i * kRowsAtOnce, tok, head)) {
                const uint4* const src = reinterpret_cast<const uint4*>(p.q + (token0 + tok) * p.q_stride + static_cast<long long>(head) * D) + sub;
                w[i][0] = src[0];
                w[i][1] = src[kLanes];
            }
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int row = row0 + i * kRowsAtOnce;
            uint32_t top = 0u;
#pragma unroll
            for (int h = 0; h < 2; ++h) top = amax_acc_bf16x2(amax_acc_bf16x2(amax_acc_bf16x2(amax_acc_bf16x2(top, w[i][h].x), w[i][h].y), w[i][h].z), w[i][h].w);
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) top = max_nan_bf16x2(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float lo_max = bf_lo(top), hi_max = bf_hi(top), amax = fmaxf(lo_max, hi_max);
            int e = ((__float_as_int(amax) >> 23) & 0xff) - 127;
            e = amax > 0.0f ? max(-100, e) - 7 : 0;
            float down = __int_as_float((127 - e) << 23);
            // A row that holds an infinity or a NaN has NaN among its lo codes (an infinity less itself), hence in every score; its
            // factor stays a number, so that keys it must not see, at -inf, remain weightless and a row that sees none stays empty.
            const bool finite = lo_max <= 3.4e38f && hi_max <= 3.4e38f;
            // (a normal number at least: a masked score times zero would be NaN, and whatever is that small changes no weight)
            if (sub == 0) row_factor[row] = finite ? fmaxf(fabsf(p.scale_log2e) * __int_as_float((127 + e) << 23), FLT_MIN) : 1.0f;
            if (p.scale_log2e < 0.0f) down = -down;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t h0, l0, h1, l1, h2, l2, h3, l3;
                split_e4m3x2(w[i][h].x, down, h0, l0);
                split_e4m3x2(w[i][h].y, down, h1, l1);
                split_e4m3x2(w[i][h].z, down, h2, l2);
                split_e4m3x2(w[i][h].w, down, h3, l3);
                unsigned char* const at = sm + q_off + code_at<D>(row, (sub + h * kLanes) >> 1) + 8 * (sub & 1);
                *reinterpret_cast<uint2*>(at) = make_uint2((h0 & 0xffffu) | (h1 << 16), (h2 & 0xffffu) | (h3 << 16));
                *reinterpret_cast<uint2*>(at + G::kQPart) = make_uint2((l0 & 0xffffu) | (l1 << 16), (l2 & 0xffffu) | (l3 << 16));
            }
        }
        fence_async_smem();
        if constexpr (!G::kTwoS) {
            named_sync(4 + blk, 256);
            constexpr int kPieces = D / 32;                      // 16-byte pieces of half a row
            const int row = 32 * (wb & 3) + lane, part = wb >> 2;
            uint32_t lo[4 * kPieces];
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(sm + q_off + G::kQPart + code_at<D>(row, kPieces * part + i));
                lo[4 * i] = v.x; lo[4 * i + 1] = v.y; lo[4 * i + 2] = v.z; lo[4 * i + 3] = v.w;
            }
            tmem_st_words<4 * kPieces>(tmem_q + (static_cast<uint32_t>(32 * (wb & 3)) << 16) + part * (4 * kPieces), lo);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    if (warp < G::kConvWarp0) named_sync(3, 32 * G::kConvWarp0);
    tc_fence_after();

    if (warp < G::kSoftmaxWarps) {
        // =============================== softmax ===============================
        const int c2 = lane & 3;
        const int row_a = 32 * (wb & 3) + 16 * (wb >> 2) + (lane >> 2), row_b = row_a + 8;
        const uint32_t my_lanes16 = static_cast<uint32_t>(32 * (wb & 3) + 16 * (wb >> 2)) << 16;
        int tok_a, tok_b, head_a, head_b;
        const bool valid_a = row_at(row_a, tok_a, head_a), valid_b = row_at(row_b, tok_b, head_b);
        const int qpos_a = valid_a ? last_key(tok_a) : INT_MAX, qpos_b = valid_b ? last_key(tok_b) : INT_MAX;
        const float c_a = n_tiles > 0 ? row_factor[row_a] : 0.0f, c_b = n_tiles > 0 ? row_factor[row_b] : 0.0f;
        float m_a = kMInit, m_b = kMInit, l_a = 0.0f, l_b = 0.0f;
        const float* const cst0 = reinterpret_cast<const float*>(sm + G::kSCst);
        // One tile.  The plain form (kAny false) is for tiles that every row sees whole and whose V
        // scales are in the operand; kAny serves every tile.  Returns false when a wait gave up.
        auto weigh = [&](auto any, int i, const float* cst, int flags) -> bool {
            constexpr bool kAny = decltype(any)::value;
            const int key0 = (j0 + i) * kKeys;
            const bool slow = kAny && (flags & kSlow) != 0;
            uint32_t sr[32];
            tmem_ld_frag_x8(sr, tmem_s + (i & 1) * G::kSStep + my_lanes16);
            if constexpr (!G::kTwoS) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) pipe::mbar_arrive(&bb[kBarSRead]);    // S may be overwritten by the next product
            }
            // pair 2 g: row a, keys 8 g + 2 c2 + {0, 1}; pair 2 g + 1: the same keys of row b.  (The constants lie in the
            // order of the weights: four for g = 2 a, 2 a + 1 at 16 a + 4 c2.)
            float2 sv[16];
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const float4 kk = *reinterpret_cast<const float4*>(cst + 16 * a + 4 * c2);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int g = 2 * a + h;
                    const float2 k2 = h ? make_float2(kk.z, kk.w) : make_float2(kk.x, kk.y);
                    sv[2 * g] = mul2_rn(make_float2(__uint_as_float(sr[4 * g]), __uint_as_float(sr[4 * g + 1])), k2);
                    sv[2 * g + 1] = mul2_rn(make_float2(__uint_as_float(sr[4 * g + 2]), __uint_as_float(sr[4 * g + 3])), k2);
                }
            }
            float f_a = c_a, f_b = c_b;
            if constexpr (kAny) {
                if (slow) {                                  // the V scales ride in the exponent on this tile
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const float4 lg = *reinterpret_cast<const float4*>(cst + kKeys + 16 * a + 4 * c2);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int g = 2 * a + h;
                            const float x = h ? lg.z : lg.x, y = h ? lg.w : lg.y;
                            sv[2 * g] = make_float2(fmaf(sv[2 * g].x, c_a, x), fmaf(sv[2 * g].y, c_a, y));
                            sv[2 * g + 1] = make_float2(fmaf(sv[2 * g + 1].x, c_b, x), fmaf(sv[2 * g + 1].y, c_b, y));
                        }
                    }
                    f_a = f_b = 1.0f;
                }
                if (key0 + kKeys - 1 > seen_by_all || (flags & 15) != 15) {
                    if (!wait_bar(&bars[G::kBarVReady + i % kVBuffers], (i / kVBuffers) & 1, gave_up, __LINE__, p.error_word)) return false;   // marks of bad V rows
                    const float* const poison = reinterpret_cast<const float*>(sm + G::kSPoison) + (i % kVBuffers) * kKeys + 2 * c2;
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        const int key = key0 + 8 * g + 2 * c2;
                        const float2 bad = *reinterpret_cast<const float2*>(poison + 8 * g);
                        const bool gone = ((flags >> (g >> 1)) & 1) == 0;
                        sv[2 * g].x = gone || key > qpos_a ? -INFINITY : sv[2 * g].x + bad.x;
                        sv[2 * g].y = gone || key + 1 > qpos_a ? -INFINITY : sv[2 * g].y + bad.y;
                        sv[2 * g + 1].x = gone || key > qpos_b ? -INFINITY : sv[2 * g + 1].x + bad.x;
                        sv[2 * g + 1].y = gone || key + 1 > qpos_b ? -INFINITY : sv[2 * g + 1].y + bad.y;
                    }
                }
            }
            float mx_a = fmaxf(sv[0].x, sv[0].y), mx_b = fmaxf(sv[1].x, sv[1].y);
#pragma unroll
            for (int g = 1; g < 8; ++g) {
                mx_a = fmaxf(mx_a, fmaxf(sv[2 * g].x, sv[2 * g].y));
                mx_b = fmaxf(mx_b, fmaxf(sv[2 * g + 1].x, sv[2 * g + 1].y));
            }
            mx_a *= f_a;
            mx_b *= f_b;
            // The maximum of the four threads of a row is only needed when one of them has left the old one too far behind.
            const bool moved = __any_sync(0xffffffffu, mx_a > m_a + kLag || mx_b > m_b + kLag);
            float corr_a = 1.0f, corr_b = 1.0f;
            if (moved) {                                     // every row of the warp follows its maximum
                mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1));
                mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1));
                mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
                mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
                const float mn_a = fmaxf(m_a, mx_a), mn_b = fmaxf(m_b, mx_b);
                corr_a = ex2f(m_a - mn_a);
                corr_b = ex2f(m_b - mn_b);
                m_a = mn_a;
                m_b = mn_b;
                l_a *= corr_a;
                l_b *= corr_b;
            }
            const unsigned long long f2_a = both(f_a), f2_b = both(f_b), neg_a = both(kShift - m_a), neg_b = both(kShift - m_b);
            float2 sum_a = make_float2(0.0f, 0.0f), sum_b = make_float2(0.0f, 0.0f);
            // word 4 (g / 2) + g % 2: row a, keys 8 g + 2 c2 + {0, 1}; + 2: row b.  In tensor memory that is pair 8 (g / 2) +
            // 2 c2 + g % 2 of the row, so V's rows are laid out in that order.
            uint32_t wv[16];
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                const float2 xa = fma2_both(sv[2 * g], f2_a, neg_a), xb = fma2_both(sv[2 * g + 1], f2_b, neg_b);
                const float2 ea = make_float2(ex2f(xa.x), ex2f(xa.y)), eb = make_float2(ex2f(xb.x), ex2f(xb.y));
                if (kAny && slow) {
                    const float2 rv = *reinterpret_cast<const float2*>(cst + 2 * kKeys + 16 * (g >> 1) + 4 * c2 + 2 * (g & 1));
                    sum_a = make_float2(sum_a.x + (ea.x == 0.0f ? 0.0f : ea.x * rv.x), sum_a.y + (ea.y == 0.0f ? 0.0f : ea.y * rv.y));
                    sum_b = make_float2(sum_b.x + (eb.x == 0.0f ? 0.0f : eb.x * rv.x), sum_b.y + (eb.y == 0.0f ? 0.0f : eb.y * rv.y));
                } else {
                    sum_a = add2_rn(ea, sum_a);
                    sum_b = add2_rn(eb, sum_b);
                }
                wv[4 * (g >> 1) + (g & 1)] = pack_f16x2(ea.x, ea.y);
                wv[4 * (g >> 1) + 2 + (g & 1)] = pack_f16x2(eb.x, eb.y);
            }
            l_a += sum_a.x + sum_a.y;
            l_b += sum_b.x + sum_b.y;
            // W and O are free once O += W_{i-1} V_{i-1} is complete, a tile's work ago.  (Of two buffers of W this one is.)
            if (i > 0 && (!G::kTwoS || moved)) {
                if (!wait_bar(&bb[kBarPV + ((i - 1) & 1)], ((i - 1) >> 1) & 1, gave_up, __LINE__, p.error_word)) return false;
                tc_fence_after();
            }
            tmem_st_frag_x4(tmem_w + (i & 1) * G::kSStep + my_lanes16, wv);
            if (moved && i > 0) {
                const float2 ca = splat2(corr_a), cb2 = splat2(corr_b);
#pragma unroll 1
                for (int cb = 0; cb < D; cb += 64) {
                    uint32_t ov[32];
                    tmem_ld_frag_x8(ov, tmem_o + my_lanes16 + cb);
#pragma unroll
                    for (int g = 0; g < 8; ++g) {
                        const float2 oa = mul2_rn(make_float2(__uint_as_float(ov[4 * g]), __uint_as_float(ov[4 * g + 1])), ca);
                        const float2 ob = mul2_rn(make_float2(__uint_as_float(ov[4 * g + 2]), __uint_as_float(ov[4 * g + 3])), cb2);
                        ov[4 * g] = __float_as_uint(oa.x);
                        ov[4 * g + 1] = __float_as_uint(oa.y);
                        ov[4 * g + 2] = __float_as_uint(ob.x);
                        ov[4 * g + 3] = __float_as_uint(ob.y);
                    }
                    tmem_st_frag_x8(tmem_o + my_lanes16 + cb, ov);
                }
            }
            return true;
        };
        bool ok = true;
        for (int i = 0; i < n_tiles; ++i) {
            ok = wait_bar(&bb[kBarQK + (i & 1)], (i >> 1) & 1, gave_up, __LINE__, p.error_word);
            if (!ok) break;
            tc_fence_after();
            const float* const cst = cst0 + (i & (kCstRing - 1)) * G::kCstFloats;
            const int flags = reinterpret_cast<const int*>(cst)[3 * kKeys];
            if (flags == 15 && (j0 + i) * kKeys + kKeys - 1 <= seen_by_all) ok = weigh(std::false_type{}, i, cst, flags);
            else ok = weigh(std::true_type{}, i, cst, flags);
            if (!ok) break;
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) pipe::mbar_arrive(&bb[kBarWReady + (i & 1)]);
        }
        // ---- epilogue: finished rows, or their states ----
        if (ok && n_tiles > 0)
            ok = wait_bar(&bb[kBarPV + ((n_tiles - 1) & 1)], ((n_tiles - 1) >> 1) & 1, gave_up, __LINE__, p.error_word);
        if (ok && work) {
            tc_fence_after();
            l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
            l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
            l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
            l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
            const bool states = p.state_ml != nullptr;
            const float unfold = 1.0f / static_cast<float>(1 << kFoldShift);
            const float f_a = states ? unfold : unfold / l_a, f_b = states ? unfold : unfold / l_b;
            const bool none_a = l_a == 0.0f, none_b = l_b == 0.0f;     // a row that saw nothing is zero, whatever stale values met its zero weights
            const long long split = static_cast<long long>(blockIdx.z) * p.out_rows;
            const long long at_a = split + (valid_a ? static_cast<long long>(token0 + tok_a) * p.num_q_heads + head_a : 0);
            const long long at_b = split + (valid_b ? static_cast<long long>(token0 + tok_b) * p.num_q_heads + head_b : 0);
            if (states && c2 == 0) {
                if (valid_a) *reinterpret_cast<float2*>(p.state_ml + 2 * at_a) = make_float2(m_a - kShift, l_a);
                if (valid_b) *reinterpret_cast<float2*>(p.state_ml + 2 * at_b) = make_float2(m_b - kShift, l_b);
            }
            // Finished rows go through shared memory (where the block's Q was) so that whole rows are stored: 16-byte pieces,
            // their places swizzled by the row.
            unsigned char* const row_a_at = sm + q_off + row_a * (2 * D);
            unsigned char* const row_b_at = sm + q_off + row_b * (2 * D);
#pragma unroll 1
            for (int cb = 0; cb < D; cb += 64) {
                uint32_t ov[32];
                if (n_tiles > 0) {
                    tmem_ld_frag_x8(ov, tmem_o + my_lanes16 + cb);
                } else {
#pragma unroll
                    for (int g = 0; g < 32; ++g) ov[g] = 0u;
                }
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const float2 va = none_a ? make_float2(0.0f, 0.0f) : make_float2(__uint_as_float(ov[4 * g]) * f_a, __uint_as_float(ov[4 * g + 1]) * f_a);
                    const float2 vb = none_b ? make_float2(0.0f, 0.0f) : make_float2(__uint_as_float(ov[4 * g + 2]) * f_b, __uint_as_float(ov[4 * g + 3]) * f_b);
                    if (states) {
                        const int d = cb + 8 * g + 2 * c2;
                        if (valid_a) *reinterpret_cast<float2*>(p.state_acc + at_a * D + d) = va;
                        if (valid_b) *reinterpret_cast<float2*>(p.state_acc + at_b * D + d) = vb;
                    } else {
                        const int piece = cb / 8 + g;
                        *reinterpret_cast<uint32_t*>(row_a_at + ((piece ^ (row_a & 7)) << 4) + 4 * c2) = pack_bf16x2(va.x, va.y);
                        *reinterpret_cast<uint32_t*>(row_b_at + ((piece ^ (row_b & 7)) << 4) + 4 * c2) = pack_bf16x2(vb.x, vb.y);
                    }
                }
            }
        }
        if (p.state_ml == nullptr) {
            const bool all = !group_or(4 + blk, 256, !ok);       // (whoever gave up comes here too)
            if (all && work) {
                constexpr int kLanes = D / 8, kRowsAtOnce = 32 / kLanes;
                const int sub = lane % kLanes;
#pragma unroll 4
                for (int i = 0; i < 16 / kRowsAtOnce; ++i) {
                    const int row = 16 * wb + i * kRowsAtOnce + lane / kLanes;
                    int tok, head;
                    if (row_at(row, tok, head))
                        st_vec(p.out + (static_cast<long long>(token0 + tok) * p.num_q_heads + head) * D + 8 * sub,
                               *reinterpret_cast<const uint4*>(sm + q_off + row * (2 * D) + ((sub ^ (row & 7)) << 4)));
                }
            }
        }
    } else if (warp < G::kConvWarp0) {
        // =============================== products of row block `blk` ===============================
        constexpr uint32_t kIdescQK = instr_desc(kKeys, false);        // E4M3 operands have format number 0, as f16 has in its kind
        constexpr uint32_t kIdescPV = instr_desc(D, true);
        const uint64_t q_tile = code_desc<D>(base + G::kSQ), k_tile = code_desc<D>(base + G::kSK), v_tile = smem_desc(base + G::kSV, kKeys * 128);
        // Whole warps walk the loops and one elected thread issues: loop counters, descriptors and tensor-memory addresses are
        // then in uniform registers, where the instructions want them (in a branch of one thread each product costs about 130
        // cycles of moves: 24 products a tile).  The two chains, S_{i+1} once S_i is read and O += W_i V_i once W_i is
        // stored, are separate warps' so that neither waits for the other.
        bool ok = true;
        if (warp == G::kIssuerWarp0) {
            for (int i = 0; i < n_tiles; ++i) {
                const int stage = i % kStages;
                const uint64_t kd = k_tile + static_cast<uint64_t>(stage * (G::kStageBytes >> 4));
                ok = wait_bar(&bars[G::kBarFull + stage], (i / kStages) & 1, gave_up, __LINE__, p.error_word);
#pragma unroll
                for (int g = 0; g < kBlocks; ++g) {
                    uint64_t* const of = bars + g * G::kBarsPerBlock;
                    // S_i goes where S_{i-1} was, once that is read; of two buffers where S_{i-2} and W_{i-2} were, once O += W_{i-2} V_{i-2} is complete
                    if constexpr (G::kTwoS) {
                        if (ok && i > 1) ok = wait_bar(&of[kBarPV + (i & 1)], ((i >> 1) - 1) & 1, gave_up, __LINE__, p.error_word);
                    } else {
                        if (ok && i > 0) ok = wait_bar(&of[kBarSRead], (i - 1) & 1, gave_up, __LINE__, p.error_word);
                    }
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t q_hi = q_tile + static_cast<uint64_t>(g * 2 * (G::kQPart >> 4));
                    const uint32_t d = tmem + g * kTmemCols + (i & 1) * G::kSStep, q_lo = tmem + g * kTmemCols + G::kQCol;
                    if (elect_one()) {
#pragma unroll
                        for (int s = 0; s < D / 32; ++s) umma_f8(d, q_hi + 2 * s, kd + 2 * s, kIdescQK, s > 0);
#pragma unroll
                        for (int s = 0; s < D / 32; ++s) {
                            if constexpr (G::kTwoS) umma_f8(d, q_hi + (G::kQPart >> 4) + 2 * s, kd + 2 * s, kIdescQK, true);
                            else umma_f8_ts(d, q_lo + 8 * s, kd + 2 * s, kIdescQK, true);
                        }
                        umma_commit(&of[kBarQK + (i & 1)]);
                        if (g == kBlocks - 1) umma_commit(&bars[G::kBarEmpty + stage]);        // K_i is free once these products are done
                    }
                    __syncwarp();
                }
                if (!ok) break;
                ok = wait_bar(&bars[G::kBarCst + (i & (kCstRing - 1))], (i / kCstRing) & 1, gave_up, __LINE__, p.error_word);
#pragma unroll
                for (int g = 0; g < kBlocks; ++g)
                    if (ok && lane == 0) pipe::mbar_arrive(&bars[g * G::kBarsPerBlock + kBarQK + (i & 1)]);      // the tile's constants are there
                if (!ok) break;
            }
        } else {
            for (int i = 0; i < n_tiles; ++i) {
                const int buf = i % kVBuffers;
                ok = wait_bar(&bars[G::kBarVReady + buf], (i / kVBuffers) & 1, gave_up, __LINE__, p.error_word) &&
                     wait_bar(&bb[kBarWReady + (i & 1)], (i >> 1) & 1, gave_up, __LINE__, p.error_word);
                if (!ok) break;
                tc_fence_after();
                const uint64_t vd = v_tile + static_cast<uint64_t>(buf * (G::kTileBytes >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int s = 0; s < kKeys / 16; ++s)
                        umma_f16_ts(tmem_o, tmem_w + (i & 1) * G::kSStep + s * 8, vd + s * (2048 >> 4), kIdescPV, i > 0 || s > 0);
                    umma_commit(&bb[kBarPV + (i & 1)]);
                    umma_commit(&bars[G::kBarVEmpty + buf]);
                }
                __syncwarp();
            }
        }
    } else if (warp < G::kCopyWarp) {
        // =============================== conversion of V ===============================
        constexpr int kPerRow = D / 16;
        const int t = tid - 32 * G::kConvWarp0;
        float* const poison = reinterpret_cast<float*>(sm + G::kSPoison);
        int met = 0;                                         // meetings of the conversion warps so far
        auto meet = [&]() {                                  // bounded, unlike a named barrier: a thread that gave up does not come
            pipe::mbar_arrive(&bars[G::kBarConv]);
            return wait_bar(&bars[G::kBarConv], met++ & 1, gave_up, __LINE__, p.error_word);
        };
        bool ok = true;
        for (int i = 0; i < n_tiles && ok; ++i) {
            const int buf = i % kVBuffers, stage = i % kStages, key0 = (j0 + i) * kKeys;
            const unsigned char* const raw = sm + G::kSK + stage * G::kStageBytes + G::kRawBytes;
            const float* const raw_vs = reinterpret_cast<const float*>(sm + G::kSK + stage * G::kStageBytes + G::kScaleAt) + kKeys;
            ok = wait_bar<50>(&bars[G::kBarFull + stage], (i / kStages) & 1, gave_up, __LINE__, p.error_word);
            if (i >= kVBuffers)      // the operand buffer is free once every block's O += W V that read it is complete
                ok = ok && wait_bar<50>(&bars[G::kBarVEmpty + buf], ((i / kVBuffers) - 1) & 1, gave_up, __LINE__, p.error_word);
            if (!ok) break;
            const int groups = stage_groups[stage];
            const bool edge = key0 + kKeys - 1 > seen_by_all || groups != 15;      // uniform
            if (edge) {          // rows that hold a NaN code, or have no finite scale: zero, and marked for the scores
                if (t < kKeys) poison[buf * kKeys + t] = raw_vs[t] <= 3.0e38f ? 0.0f : NAN;
                if (!meet()) { ok = false; break; }
#pragma unroll
                for (int n = 0; n < G::kPerConv; ++n) {
                    const int c = t + G::kConvThreads * n;
                    const uint4 w = *reinterpret_cast<const uint4*>(raw + c * 16);
                    const uint32_t hit = (((w.x & 0x7f7f7f7fu) + 0x01010101u) | ((w.y & 0x7f7f7f7fu) + 0x01010101u) |
                                          ((w.z & 0x7f7f7f7fu) + 0x01010101u) | ((w.w & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u;
                    if (hit != 0u) poison[buf * kKeys + c / kPerRow] = NAN;
                }
                if (!meet()) { ok = false; break; }
            }
            auto counts = [&](int k) { return key0 + k < total_keys && ((groups >> (k >> 4)) & 1) && outside_fold(raw_vs[k]); };
            const bool slow = __any_sync(0xffffffffu, counts(lane) || counts(lane + 32));
            if (t < kKeys) {
                // the tile's constants, in the order of the weights (key 16 a + 8 h + 2 c + e lies at 16 a + 4 c + 2 h + e).  The slot's
                // last reader was tile i - 4, which the softmax has left: O += W V of tile i - 3 is complete.
                float* const cst = reinterpret_cast<float*>(sm + G::kSCst) + (i & (kCstRing - 1)) * G::kCstFloats;
                const int place = ws::key_of_k_row(t);
                cst[place] = raw_vs[t - kKeys];                                     // (the K scales lie in front of the V scales)
                if (slow) {
                    const float vs = raw_vs[t];
                    const float lg = fmaxf(lg2f(vs), kLgFloor) + static_cast<float>(kFoldShift);
                    cst[kKeys + place] = lg + vs * 0.0f;                            // (the maximum loses a NaN scale: it is added back)
                    cst[2 * kKeys + place] = ex2f(-lg);
                }
                if (t == 0) reinterpret_cast<int*>(cst)[3 * kKeys] = groups | (slow ? kSlow : 0);
                __syncwarp();
                if (lane == 0) pipe::mbar_arrive(&bars[G::kBarCst + (i & (kCstRing - 1))]);
            }
            // E4M3 -> f16 operand rows: [dim block of 64][row][128 bytes, swizzled].  Consecutive threads take consecutive
            // pieces of the raw tile; the upper half of a row's pieces stores its second half first, so that the eight
            // threads of a row write eight different 16-byte columns.
            unsigned char* const v_dst = sm + G::kSV + buf * G::kTileBytes;
#pragma unroll
            for (int n = 0; n < G::kPerConv; ++n) {
                const int c = t + G::kConvThreads * n;
                const int key = c / kPerRow, ch = c % kPerRow;
                uint4 w = *reinterpret_cast<const uint4*>(raw + c * 16);
                float vs = slow ? 1.0f : raw_vs[key] * static_cast<float>(1 << kFoldShift);
                if (edge && (poison[buf * kKeys + key] != 0.0f || key0 + key >= total_keys || !((groups >> (key >> 4)) & 1))) {
                    w = make_uint4(0u, 0u, 0u, 0u);
                    vs = 0.0f;
                }
                const __half2 f = __float2half2_rn(vs);
                uint32_t h[8];
                e4m3x4_to_f16x2x2(w.x, h[0], h[1]);
                e4m3x4_to_f16x2x2(w.y, h[2], h[3]);
                e4m3x4_to_f16x2x2(w.z, h[4], h[5]);
                e4m3x4_to_f16x2x2(w.w, h[6], h[7]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&h[e]), f);
                    h[e] = *reinterpret_cast<const uint32_t*>(&x);
                }
                // key 16 a + 8 h + 2 c + e becomes row 16 a + 4 c + 2 h + e: the order in which the weights lie
                const int row = ws::key_of_k_row(key);
                unsigned char* const dst = v_dst + (ch >> 2) * (kKeys * 128) + swz128(row, 2 * (ch & 3));
                const uintptr_t one = reinterpret_cast<uintptr_t>(dst), other = one ^ 16;
                const bool second = (ch >> 2) & 1;
                const uint4 h0 = make_uint4(h[0], h[1], h[2], h[3]), h1 = make_uint4(h[4], h[5], h[6], h[7]);
                *reinterpret_cast<uint4*>(second ? other : one) = second ? h1 : h0;
                *reinterpret_cast<uint4*>(second ? one : other) = second ? h0 : h1;
            }
            fence_async_smem();
            pipe::mbar_arrive(&bars[G::kBarVReady + buf]);
            __syncwarp();
            if (lane == 0) pipe::mbar_arrive(&bars[G::kBarEmpty + stage]);
        }
    } else {
        // =============================== copies ===============================
        // A tile is one run of keys per page: lane r looks up run r's page, one elected lane issues a run's two copies.  The
        // scales (256 bytes each of K and V) come by ordinary asynchronous copies, 16 bytes per lane.
        const int shift = p.c.page_shift;
        const int run_shift = shift < 6 ? shift : 6, run_keys = 1 << run_shift, runs = kKeys >> run_shift;
        const int my_key = lane < runs ? lane << run_shift : 0;      // first key of this lane's run
        const int scale_key = 4 * (lane & 15);                       // the four keys whose scales this lane copies
        const float* const scales = lane < 16 ? p.c.k_scale : p.c.v_scale;
        auto page_of = [&](int i) {
            const int key = (j0 + i) * kKeys + my_key;
            int id = -1;
            if (lane < runs && i < n_tiles && key < total_keys && (key >> shift) < p.c.pages_per_row) id = pages[key >> shift];
            return id >= 0 && id < p.c.num_pages ? id : -1;
        };
        int id = page_of(0), next = page_of(1);
        int issued = 0;
        auto copy_tile = [&](int i) {
            const int stage = i % kStages, after = page_of(i + 2);
            const unsigned have = __ballot_sync(0xffffffffu, id >= 0);               // the runs of the tile that exist
            if (i >= kStages && !wait_bar<50>(&bars[G::kBarEmpty + stage], ((i / kStages) - 1) & 1, gave_up, __LINE__, p.error_word)) return false;
            unsigned char* const dst = sm + G::kSK + stage * G::kStageBytes;
            uint64_t* const full = &bars[G::kBarFull + stage];
            if (elect_one()) {
                int groups = 0;
                for (int r = 0; r < runs; ++r)
                    if ((have >> r) & 1) groups |= ((1 << (run_keys >> 4)) - 1) << (r * (run_keys >> 4));
                stage_groups[stage] = groups;
                pipe::mbar_expect_tx(full, static_cast<uint32_t>((__popc(have) << run_shift) * 2 * D));
            }
            __syncwarp();
            const int in_page = ((j0 + i) * kKeys) & ((1 << shift) - 1) & ~(run_keys - 1);     // (0 for pages of at most a tile)
            for (int r = 0; r < runs; ++r) {
                const int page = __shfl_sync(0xffffffffu, id, r);
                if (page >= 0 && elect_one()) {
                    const size_t key = key_index(p.c, page, kvh) + in_page;
                    const int at = (r << run_shift) * D;
                    tensor_load(dst + at, &k_map, static_cast<int>(key), full);
                    pipe::bulk_load(dst + G::kRawBytes + at, p.c.v + key * D, static_cast<uint32_t>(D << run_shift), full);
                }
                __syncwarp();
            }
            const int page = __shfl_sync(0xffffffffu, id, scale_key >> run_shift);
            const size_t key = page >= 0 ? key_index(p.c, page, kvh) + in_page + (scale_key & (run_keys - 1)) : 0;
            cp16_zfill(pipe::smem_u32(dst + G::kScaleAt + (lane >> 4) * (kKeys * 4) + scale_key * 4), scales + key, page >= 0);
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(pipe::smem_u32(full)) : "memory");
            issued = i + 1;
            id = next;
            next = after;
            return true;
        };
        bool ok = true;
        for (int i = 0; i < n_tiles && ok; ++i) ok = copy_tile(i);
        if (!ok)        // somebody gave up: let the copies on their way land (bounded again) before the CTA ends
            for (int i = max(0, issued - kStages); i < issued; ++i)
                for (int tries = 0; tries < (1 << 12) && !pipe::mbar_try_wait(&bars[G::kBarFull + i % kStages], (i / kStages) & 1); ++tries) {}
        cp_async_wait<0>();
    }

    // ---- common exit ----
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::kTmem) : "memory");
    }
    if constexpr (kPrefix) pdl_wait();       // its completion then stands for that of the kernel in front of it too
}

// Joins the states of a row's key ranges: out = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i.
template <int D>
__global__ void __launch_bounds__(256) join_ranges_kernel(__nv_bfloat16* out, const float* ml, const float* acc, const int* cu_seqlens, int num_seqs,
                                                          long long rows, int num_q_heads, int splits) {
    constexpr int kLanes = D / 4;
    pdl_enter();
    const long long row = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / kLanes;
    const int j = threadIdx.x % kLanes;
    if (row >= rows) return;
    const long long token = row / num_q_heads;
    if (token < cu_seqlens[0] || token >= cu_seqlens[num_seqs]) return;       // padding is left as it was
    float m = kMInit, l = 0.0f;
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
        const long long at = i * rows + row;
        const float2 s = *reinterpret_cast<const float2*>(ml + 2 * at);
        const float4 x = *reinterpret_cast<const float4*>(acc + at * D + 4 * j);
        const float n = fmaxf(m, s.x), f = ex2f(m - n), g = ex2f(s.x - n);
        l = l * f + s.y * g;
        a.x = a.x * f + x.x * g;
        a.y = a.y * f + x.y * g;
        a.z = a.z * f + x.z * g;
        a.w = a.w * f + x.w * g;
        m = n;
    }
    uint2 w = make_uint2(0u, 0u);
    if (l != 0.0f) {
        const float inv = 1.0f / l;
        w.x = pack_bf16x2(a.x * inv, a.y * inv);
        w.y = pack_bf16x2(a.z * inv, a.w * inv);
    }
    st_vec8(out + row * D + 4 * j, w);
}

// Query heads of a group are dealt evenly over row blocks of at most four; a block takes as many tokens as fit.
void deal_heads(int group, BlockArgs& a) {
    a.group = group;
    a.head_chunks = (group + 3) / 4;
    a.heads_per_cta = (group + a.head_chunks - 1) / a.head_chunks;
    a.tokens_per_block = kRows / a.heads_per_cta;
    a.slot_mul = (65536 + a.tokens_per_block - 1) / a.tokens_per_block;
}

// The K codes of a layer as rows of head_dim bytes, copied in boxes of one run of keys, swizzled as the products read them.
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int make_k_map(const Layer& c, int head_dim, const char* fn, CUtensorMap* map) {
    static const EncodeTiled encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            f = nullptr;
        }
        return reinterpret_cast<EncodeTiled>(f);
    }();
    RH_REQUIRE(encode != nullptr, RH_ERR_CUDA, "%s: the driver has no cuTensorMapEncodeTiled", fn);
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(head_dim), (static_cast<cuuint64_t>(c.num_pages) * c.num_kv_heads) << c.page_shift};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(head_dim)};
    const int page = 1 << c.page_shift;
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(head_dim), static_cast<cuuint32_t>(page < kKeys ? page : kKeys)}, steps[2] = {1, 1};
    const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, c.k, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    RH_REQUIRE(r == CUDA_SUCCESS, RH_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", fn, static_cast<int>(r));
    return RH_OK;
}

template <int D, int kBlocks, bool kPrefix>
int launch_blocks_as(const BlockArgs& a, unsigned tiles, unsigned splits, cudaStream_t stream, const char* fn) {
    using G = Geo<D, kBlocks>;
    const dim3 grid(static_cast<unsigned>(a.c.num_kv_heads * a.head_chunks), tiles, splits);
    CUtensorMap map;
    if (const int e = make_k_map(a.c, D, fn, &map)) return e;
    (void)host::setup<&paged_blocks_kernel<D, kBlocks, kPrefix>, G::kThreads, G::kSmemBytes>();
    host::launch<paged_blocks_kernel<D, kBlocks, kPrefix>>(grid, dim3(G::kThreads), static_cast<size_t>(G::kSmemBytes), stream, a, map);
    return host::check_launch(fn);
}

// Token tiles a packed batch has at most: every sequence may end inside a tile.
long long most_tiles(long long num_tokens, int num_seqs, int tile_tokens) {
    const long long n = num_tokens / tile_tokens + num_seqs;
    return n < num_tokens ? n : num_tokens;
}

// Time of a call in units of one key tile of a CTA: waves x (tiles per CTA + what a CTA costs besides).  Two row blocks
// share a converted tile and cost about 1.5 times one block's.
double cost(long long ctas, long long tiles, int splits, int blocks) {
    const long long waves = (ctas * splits + host::num_sms() - 1) / host::num_sms();
    const double per = static_cast<double>((tiles + splits - 1) / splits) * (blocks == 2 ? 1.5 : 1.0) + 4.0;
    return static_cast<double>(waves) * per;
}

}  // namespace

int prefix_splits(int num_seqs, int num_kv_heads, int group) {
    BlockArgs a = {};
    deal_heads(group, a);
    const int blocks = num_seqs > a.tokens_per_block ? 2 : 1;
    const long long ctas = static_cast<long long>(num_kv_heads) * a.head_chunks * ((num_seqs + blocks * a.tokens_per_block - 1) / (blocks * a.tokens_per_block));
    // All CTAs take equally long: the fewest waves that fill the SMs to nine tenths (every further range costs a state
    // per query row, written and read back).
    int best = 1;
    double best_fill = 0.0;
    for (int waves = 1; waves <= 4; ++waves) {
        const long long slots = static_cast<long long>(waves) * host::num_sms(), n = slots / ctas;
        if (n < 1 || n > 64) continue;
        const double fill = static_cast<double>(n * ctas) / static_cast<double>(slots);
        if (fill > best_fill + 0.05) {
            best_fill = fill;
            best = static_cast<int>(n);
        }
        if (fill >= 0.9) break;
    }
    return best;
}

int launch_prefix(const DecodeArgs& d, int head_dim, cudaStream_t stream, const char* fn) {
    BlockArgs a = {};
    a.c = d.c;
    a.q = d.q;
    a.rows = d.rows;
    a.shared_pages = d.shared_pages;
    a.shared_len = d.shared_len;
    a.state_ml = d.block_ml;
    a.state_acc = d.block_acc;
    a.error_word = d.error_word;
    a.q_stride = d.q_stride;
    a.num_q_heads = d.c.num_kv_heads * d.group;
    a.out_rows = static_cast<long long>(d.num_seqs) * a.num_q_heads;
    a.num_tokens = d.num_seqs;
    a.num_seqs = d.num_seqs;
    a.scale_log2e = d.scale_log2e;
    deal_heads(d.group, a);
    const int blocks = d.num_seqs > a.tokens_per_block ? 2 : 1;
    const unsigned tiles = static_cast<unsigned>((d.num_seqs + blocks * a.tokens_per_block - 1) / (blocks * a.tokens_per_block));
    const unsigned splits = static_cast<unsigned>(d.block_splits);
    if (head_dim == 128)
        return blocks == 2 ? launch_blocks_as<128, 2, true>(a, tiles, splits, stream, fn) : launch_blocks_as<128, 1, true>(a, tiles, splits, stream, fn);
    return blocks == 2 ? launch_blocks_as<64, 2, true>(a, tiles, splits, stream, fn) : launch_blocks_as<64, 1, true>(a, tiles, splits, stream, fn);
}

}  // namespace paged
}  // namespace rh

using namespace rh;

extern "C" int rh_flash_prefill_packed_splits(int num_tokens, int num_seqs, int max_keys, int num_q_heads, int num_kv_heads, int head_dim) {
    if (num_tokens < 1 || num_seqs < 1 || max_keys < 1 || num_q_heads < 1 || num_kv_heads < 1 || num_q_heads % num_kv_heads != 0) return 1;
    paged::BlockArgs a = {};
    paged::deal_heads(num_q_heads / num_kv_heads, a);
    const long long heads = static_cast<long long>(num_kv_heads) * a.head_chunks;
    const long long tiles = (max_keys + tc::kKeys - 1) / tc::kKeys;
    const long long one = heads * paged::most_tiles(num_tokens, num_seqs, a.tokens_per_block);
    if (one > 2LL * host::num_sms()) return 1;
    const int blocks = one > host::num_sms() ? 2 : 1;
    const long long ctas = blocks == 2 ? heads * paged::most_tiles(num_tokens, num_seqs, 2 * a.tokens_per_block) : one;
    int best = 1;
    double least = paged::cost(ctas, tiles, 1, blocks);
    for (int s = 2; s <= 32 && s * 8 <= tiles; ++s) {          // at least eight tiles a range: the join costs about four
        const double c = paged::cost(ctas, tiles, s, blocks) + 4.0;
        if (c < 0.95 * least) {
            least = c;
            best = s;
        }
    }
    (void)head_dim;      // (one ratio of a CTA's time to a tile's serves both sizes of head)
    return best;
}

extern "C" size_t rh_flash_prefill_packed_scratch_floats(int num_tokens, int num_q_heads, int head_dim, int num_splits) {
    if (num_tokens < 1 || num_q_heads < 1 || head_dim < 1 || num_splits < 2) return 0;
    return static_cast<size_t>(num_splits) * static_cast<size_t>(num_tokens) * static_cast<size_t>(num_q_heads) * static_cast<size_t>(head_dim + 2) + 4;
}

extern "C" int rh_flash_prefill_packed_bf16(void* out, const void* q, long long q_stride, const rh_kv_pages* cache, int layer, const int* rows_or_null,
                                            const int* cu_seqlens, int num_tokens, int num_seqs, int num_q_heads, float scale, float* partial_or_null,
                                            int num_splits, void* stream) {
    const char* const fn = "rh_flash_prefill_packed_bf16";
    paged::BlockArgs a = {};
    if (const int e = host::paged_layer(cache, layer, fn, &a.c)) return e;
    RH_REQUIRE(out && q && cu_seqlens, RH_ERR_INVALID_ARG, "%s: null pointer", fn);
    RH_REQUIRE(num_tokens >= 1 && num_seqs >= 1, RH_ERR_INVALID_ARG, "%s: num_tokens and num_seqs must be >= 1", fn);
    RH_REQUIRE(rows_or_null != nullptr || num_seqs <= cache->num_rows, RH_ERR_INVALID_ARG, "%s: more sequences than table rows", fn);
    RH_REQUIRE(num_q_heads >= 1 && num_q_heads % cache->num_kv_heads == 0, RH_ERR_INVALID_ARG, "%s: num_q_heads must be a multiple of num_kv_heads", fn);
    RH_REQUIRE(num_q_heads <= 1024, RH_ERR_UNSUPPORTED_DIM, "%s: at most 1024 query heads", fn);
    RH_REQUIRE(std::isfinite(scale * paged::kLog2e), RH_ERR_INVALID_ARG, "%s: scale must be finite (and so must scale * log2 e)", fn);
    RH_REQUIRE(num_splits >= 1 && num_splits <= 64, RH_ERR_INVALID_ARG, "%s: num_splits must be in 1..64", fn);
    RH_REQUIRE(num_splits == 1 || partial_or_null != nullptr, RH_ERR_INVALID_ARG, "%s: splits need scratch", fn);
    RH_REQUIRE(q_stride >= static_cast<long long>(num_q_heads) * cache->head_dim, RH_ERR_INVALID_ARG, "%s: q_stride is below num_q_heads * head_dim", fn);
    RH_REQUIRE(host::aligned16(q) && q_stride % 8 == 0 && host::aligned16(partial_or_null), RH_ERR_MISALIGNED,
               "%s: q and partial must be 16-byte aligned, q_stride a multiple of 8", fn);
    RH_REQUIRE(host::aligned16(out), RH_ERR_MISALIGNED, "%s: out must be 16-byte aligned", fn);
    a.out = static_cast<__nv_bfloat16*>(out);
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.rows = rows_or_null;
    a.cu_seqlens = cu_seqlens;
    a.error_word = host::device_error_word();
    a.q_stride = q_stride;
    a.num_q_heads = num_q_heads;
    a.out_rows = static_cast<long long>(num_tokens) * num_q_heads;
    a.num_tokens = num_tokens;
    a.num_seqs = num_seqs;
    a.scale_log2e = scale * paged::kLog2e;
    paged::deal_heads(num_q_heads / cache->num_kv_heads, a);
    if (num_splits > 1) {
        a.state_acc = partial_or_null;
        a.state_ml = partial_or_null + static_cast<size_t>(num_splits) * a.out_rows * cache->head_dim;
    }
    const long long heads = static_cast<long long>(cache->num_kv_heads) * a.head_chunks;
    // Two row blocks per CTA once one-block CTAs are more than the SMs: a tile is converted once for twice the rows, one and a half
    // times a block's time.  One / two blocks: 128 tokens 9.8 / 13.1 us, 511 16.4 / 20.4; 1000 31.7 / 29.7, six prompts of 2048
    // together 53.8 / 40.6, 700 tokens behind 2000 keys 90.8 / 62.8.  (Just above the border a short prompt without history, whose second
    // wave would have few keys, loses: 600 tokens 18.8 / 21.8.)
    const int blocks = heads * paged::most_tiles(num_tokens, num_seqs, a.tokens_per_block) * num_splits > host::num_sms() ? 2 : 1;
    const long long tiles = paged::most_tiles(num_tokens, num_seqs, blocks * a.tokens_per_block);
    RH_REQUIRE(tiles <= 65535, RH_ERR_UNSUPPORTED_DIM, "%s: too many token tiles in one call (%lld)", fn, tiles);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned y = static_cast<unsigned>(tiles), z = static_cast<unsigned>(num_splits);
    int e;
    if (cache->head_dim == 128)
        e = blocks == 2 ? paged::launch_blocks_as<128, 2, false>(a, y, z, s, fn) : paged::launch_blocks_as<128, 1, false>(a, y, z, s, fn);
    else
        e = blocks == 2 ? paged::launch_blocks_as<64, 2, false>(a, y, z, s, fn) : paged::launch_blocks_as<64, 1, false>(a, y, z, s, fn);
    if (e != RH_OK || num_splits == 1) return e;
    const long long threads = a.out_rows * (cache->head_dim / 4);
    const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
    if (cache->head_dim == 128)
        host::launch<paged::join_ranges_kernel<128>>(grid, dim3(256), 0, s, a.out, a.state_ml, a.state_acc, cu_seqlens, num_seqs, a.out_rows, num_q_heads, num_splits);
    else
        host::launch<paged::join_ranges_kernel<64>>(grid, dim3(256), 0, s, a.out, a.state_ml, a.state_acc, cu_seqlens, num_seqs, a.out_rows, num_q_heads, num_splits);
    return host::check_launch(fn);
}
