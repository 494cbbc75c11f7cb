// Attention of many query rows over the paged FP8 cache on the 5th-generation tensor cores:
//
//   prefill   causal attention of a packed batch's new tokens: token i of an entry whose row holds n tokens sees the
//             keys 0 .. n + i of that row (its own prompt so far, and the history in front of it)
//   prefix    the shared keys of a decode step: every entry of the batch is one token, all see the same keys
//
// The reference's counterpart is flash_prefill_bf16 (include/runtherder/kernels/flash_prefill.cuh:27-40), one sequence
// in a contiguous cache.  Geometry and roles are those of flash_prefill_ws.cu: a CTA carries one or two blocks of 128
// query rows of one kv head (the group's heads x consecutive tokens), walks key tiles of 64, S and O in tensor memory
//
//   S[128 x 64] = Q K^T      (f16: bf16 queries, E4M3 keys: both exact in f16)          tcgen05.mma, operands in shared memory
//   O[128 x D] += W V        W = 2^(S ks - m) as f16 in tensor memory
//
//   softmax warps (8 per block)   scores -> weights; two rows x sixteen keys per thread
//   product warp (1 per block)    issues the products
//   conversion warps              raw E4M3 tiles -> f16 operand tiles
//   copy warp                     fetches raw tiles page by page with bulk copies, two tiles ahead
//
// What is different from there, and why.  (1) The arithmetic per score bounds the kernel, so the V scale is folded into
// the f16 V operand (one rounding of 2^-11, like a weight's) instead of riding in the exponent: no per-key additions
// and multiplications in the softmax.  f16 holds vs * 448 only for vs in 2^-22 .. 2^-1 (with a common factor of 2^8);
// a tile with a scale outside keeps the exponent form, and both forms add up in one accumulator.  (2) The running
// maximum may lag the true one by up to 2^8: weights stay below 2^8, exact enough in f16, sums are fp32, and O is
// rescaled a handful of times per row instead of on most tiles.  (3) Rows carry their own last visible key, pages may be
// missing, and places that no row may see may hold anything: the tiles that reach past some row's last key (and only
// those) replace NaN codes by zero and mark the key, so that exactly the rows that see it get NaN.
#include <cuda_fp16.h>

#include <cmath>

#include "flash_prefill_roles.cuh"
#include "flash_prefill_tc.cuh"
#include "paged_prefill.cuh"
#include "rh_kernels.h"

namespace rh {
namespace paged {
namespace {

using namespace tc;
using ws::group_or;
using ws::kLazyNs;
using ws::wait_phase;

constexpr int kRawStages = 2;
constexpr int kCstRing = 4;              // constants of a tile are read while those of the next two are written
constexpr int kFoldShift = 8;            // V operand = code * vs * 2^8
constexpr float kFoldLow = 2.384185791015625e-07f;    // 2^-22
constexpr float kFoldHigh = 0.5f;
constexpr float kLag = 8.0f;             // how far (log2) the running maximum may lie below the true one

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
    int head_chunks;
    float scale_log2e;
};

template <int D, int kBlocks>
struct Geo {
    static constexpr int kSoftmaxWarps = 8 * kBlocks;
    static constexpr int kIssuerWarp0 = kSoftmaxWarps;
    static constexpr int kConvWarp0 = kSoftmaxWarps + kBlocks;
    static constexpr int kConvWarps = kBlocks == 1 ? 3 : 4;
    static constexpr int kConvThreads = 32 * kConvWarps;
    static constexpr int kCopyWarp = kConvWarp0 + kConvWarps;
    static constexpr int kThreads = 32 * (kCopyWarp + 1);
    static constexpr int kPieces = kKeys * (D / 16);                        // 16-byte pieces of a raw tile
    static constexpr int kPerConv = (kPieces + kConvThreads - 1) / kConvThreads;
    static constexpr int kTmem = kTmemCols * kBlocks;
    static constexpr int kDimBlocks = D / 64;
    static constexpr int kQBytes = kDimBlocks * kRows * 128;
    static constexpr int kTileBytes = kDimBlocks * kKeys * 128;             // an f16 operand tile
    static constexpr int kRawBytes = kKeys * D;
    static constexpr int kStageBytes = 2 * kRawBytes + 2 * kKeys * 4;       // raw K, raw V, K scales, V scales
    static constexpr int kSQ = 0;
    static constexpr int kSK = kSQ + kBlocks * kQBytes;
    static constexpr int kSV = kSK + 2 * kTileBytes;
    static constexpr int kSRaw = kSV + 2 * kTileBytes;
    static constexpr int kCstFloats = 3 * kKeys + 4;                        // ksl, lgv, rvs, {flags}
    static constexpr int kSCst = kSRaw + kRawStages * kStageBytes;
    static constexpr int kSRow = kSCst + kCstRing * kCstFloats * 4;         // row maxima of |q| (two halves), later the rows' q factors
    static constexpr int kSPoison = kSRow + kBlocks * 2 * kRows * 4;
    static constexpr int kSBar = kSPoison + kKeys * 4;
    static constexpr int kSmemBytes = kSBar + 256 + 1024;
    static constexpr int kBarsPerBlock = 6;
    static constexpr int kBarKReady = kBarsPerBlock * kBlocks;
    static constexpr int kBarVReady = kBarKReady + 2;
    static constexpr int kBarRawFull = kBarVReady + 2;
    static constexpr int kBarRawEmpty = kBarRawFull + kRawStages;
    static constexpr int kNumBars = kBarRawEmpty + kRawStages;
    static_assert(8 * kNumBars + 32 <= 256, "barrier area");
};
enum BlockBar { kBarQK = 0, kBarPV = 2, kBarSRead = 4, kBarWReady = 5 };
enum TileFlag { kSlow = 16 };            // flags: bits 0..3 = sixteen-key groups that exist, 16 = V scales ride in the exponent

// the row of the K operand tile that holds key `key` of the tile (the inverse of ws::key_of_k_row)
__device__ __forceinline__ int k_row_of_key(int key) { return (key & 48) | ((key & 2) << 2) | ((key & 12) >> 1) | (key & 1); }

// The batch entry and the token tile of CTA `index` (of all token tiles of all entries); false: there is none.
// Tiles are numbered from the one with the most keys down, so the long ones start first: depth = keys in units of a
// tile's tokens, and for at most 32 entries the number of tiles beyond a depth is one warp sum.
__device__ __forceinline__ bool find_tile(const BlockArgs& p, int index, int tile_tokens, int& seq, int& tile) {
    const int lane = threadIdx.x & 31;
    if (p.num_seqs <= 32) {
        int n = 0, behind = 0;
        if (lane < p.num_seqs) {
            n = (max(0, p.cu_seqlens[lane + 1] - p.cu_seqlens[lane]) + tile_tokens - 1) / tile_tokens;
            const int row = p.rows != nullptr ? p.rows[lane] : lane;
            if (row >= 0 && row < p.c.num_rows) behind = max(0, p.c.lens[row]) / tile_tokens;
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
        const int n = s < p.num_seqs ? (max(0, p.cu_seqlens[s + 1] - p.cu_seqlens[s]) + tile_tokens - 1) / tile_tokens : 0;
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
__global__ void __launch_bounds__(Geo<D, kBlocks>::kThreads, 1) paged_blocks_kernel(const BlockArgs p) {
    using G = Geo<D, kBlocks>;
    extern __shared__ unsigned char raw_smem[];
    const uint32_t base = (pipe::smem_u32(raw_smem) + 1023u) & ~1023u;
    unsigned char* const sm = raw_smem + (base - pipe::smem_u32(raw_smem));
    uint64_t* const bars = reinterpret_cast<uint64_t*>(sm + G::kSBar);
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(sm + G::kSBar + 8 * G::kNumBars);
    volatile int* const gave_up = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* const raw_groups = reinterpret_cast<int*>(tmem_slot + 2);       // [kRawStages] sixteen-key groups that were fetched
    int* const least = raw_groups + kRawStages;                          // the CTA's least last visible key

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.x / p.head_chunks;
    const int chunk = blockIdx.x - kvh * p.head_chunks;

    if (tid == 0) {
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            uint64_t* const bb = bars + g * G::kBarsPerBlock;
            pipe::mbar_init(&bb[kBarQK], 1);
            pipe::mbar_init(&bb[kBarQK + 1], 1);
            pipe::mbar_init(&bb[kBarPV], 1);
            pipe::mbar_init(&bb[kBarPV + 1], 1);
            pipe::mbar_init(&bb[kBarSRead], 8);
            pipe::mbar_init(&bb[kBarWReady], 8);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            pipe::mbar_init(&bars[G::kBarKReady + i], G::kConvThreads);
            pipe::mbar_init(&bars[G::kBarVReady + i], G::kConvThreads);
        }
#pragma unroll
        for (int i = 0; i < kRawStages; ++i) {
            pipe::mbar_init(&bars[G::kBarRawFull + i], 1);
            pipe::mbar_init(&bars[G::kBarRawEmpty + i], G::kConvThreads);
        }
        *gave_up = 0;
        *least = INT_MAX;
        pipe::mbar_init_fence();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pipe::smem_u32(tmem_slot)), "r"(G::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // ---- what this CTA works on.  The prefix kernel follows a kernel of the same call whose results it does not need, and
    //      which has seen its own predecessors complete before this one may start: it waits at its end instead. ----
    if constexpr (!kPrefix) pdl_wait();
    pdl_trigger();
    int token0, tokens;              // the CTA's tokens: indexes into q, and how many exist from there on
    int held, total_keys;            // keys in front of the CTA's first token; keys that any of its rows sees
    const int* pages = nullptr;
    const int tile_tokens = kBlocks * p.tokens_per_block;
    bool work = true;
    if constexpr (kPrefix) {
        const int room = p.c.pages_per_row << p.c.page_shift;
        const int n = min(*p.shared_len, room);
        total_keys = n < kSharedAlign ? 0 : n - n % kSharedAlign;
        token0 = blockIdx.y * tile_tokens;
        tokens = p.num_tokens - token0;
        held = 0;
        pages = p.shared_pages;
    } else {
        int seq = 0, tile = 0;
        work = find_tile(p, blockIdx.y, tile_tokens, seq, tile);
        token0 = tokens = held = total_keys = 0;
        if (work) {
            const int first = p.cu_seqlens[seq], n = min(p.cu_seqlens[seq + 1], p.num_tokens) - first;
            const int row = p.rows != nullptr ? p.rows[seq] : seq;
            token0 = first + tile * tile_tokens;
            tokens = n - tile * tile_tokens;
            work = first >= 0 && tokens > 0;
            if (row >= 0 && row < p.c.num_rows && p.c.lens[row] >= 0) {
                const long long room = static_cast<long long>(p.c.pages_per_row) << p.c.page_shift;
                held = p.c.lens[row] + tile * tile_tokens;
                const long long seen = static_cast<long long>(held) + min(tokens, tile_tokens);
                total_keys = static_cast<int>(seen < room ? seen : room);
                pages = p.c.page_table + static_cast<size_t>(row) * p.c.pages_per_row;
            }
        }
    }
    const int all_tiles = (total_keys + kKeys - 1) / kKeys;
    const int j0 = static_cast<int>(static_cast<long long>(all_tiles) * blockIdx.z / gridDim.z);
    const int n_tiles = work ? static_cast<int>(static_cast<long long>(all_tiles) * (blockIdx.z + 1) / gridDim.z) - j0 : 0;

    const int blk = warp < G::kSoftmaxWarps ? warp >> 3 : (warp < G::kConvWarp0 ? warp - G::kIssuerWarp0 : 0);
    const int wb = warp & 7;
    const int block_tok = blk * p.tokens_per_block;          // first token of the block, counted from token0
    uint64_t* const bb = bars + blk * G::kBarsPerBlock;
    const uint32_t tmem_s = tmem + blk * kTmemCols, tmem_o = tmem_s + kKeys, tmem_w = tmem_o + kD;
    const int q_off = G::kSQ + blk * G::kQBytes;

    // a row of a block: its head slot and token (counted from token0); whether it exists; the last key it sees
    auto row_at = [&](int row, int& tok, int& head) {
        const int slot = row / p.tokens_per_block;
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

    // ---- Q (softmax warps): bf16 -> f16 into shared memory.  A row whose largest |q| f16 does not hold well is scaled by
    //      a power of two, which its scores take back (rare; `scaled` is uniform over the block's warps). ----
    bool scaled = false;
    float* const row_amax = reinterpret_cast<float*>(sm + G::kSRow) + blk * 2 * kRows;
    if (warp < G::kSoftmaxWarps && n_tiles > 0) {
        constexpr int kHalf = D / 16;                        // 16-byte pieces per thread: half a row
        const int row = 32 * (wb & 3) + lane, part = wb >> 2;
        int tok, head;
        const bool valid = row_at(row, tok, head);
        const uint4* const src = reinterpret_cast<const uint4*>(p.q + (valid ? (token0 + tok) * p.q_stride + static_cast<long long>(head) * D : 0)) + kHalf * part;
        uint4 w[kHalf];
        uint32_t amax2 = 0u;
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
            w[i] = make_uint4(0u, 0u, 0u, 0u);
            if (valid) w[i] = src[i];
            amax2 = amax_acc_bf16x2(amax_acc_bf16x2(amax_acc_bf16x2(amax_acc_bf16x2(amax2, w[i].x), w[i].y), w[i].z), w[i].w);
        }
        row_amax[part * kRows + row] = fmaxf(bf_lo(amax2), bf_hi(amax2));
        named_sync(4 + blk, 256);
        const float amax = fmaxf(row_amax[row], row_amax[kRows + row]);
        const bool odd = amax > 0.0f && !(amax >= 0.015625f && amax < 32768.0f);     // outside 2^-6 .. 2^15
        scaled = group_or(4 + blk, 256, odd);                // (also: everyone has read row_amax)
        float down = 1.0f;
        if (scaled) {
            int e = ((__float_as_int(amax) >> 23) & 0xff) - 127;
            e = odd ? max(-100, min(100, e)) : 0;
            down = __int_as_float((127 - e) << 23);
            if (part == 0) row_amax[row] = __int_as_float((127 + e) << 23);
        }
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
            uint4 h;
            h.x = pack_f16x2(bf_lo(w[i].x) * down, bf_hi(w[i].x) * down);
            h.y = pack_f16x2(bf_lo(w[i].y) * down, bf_hi(w[i].y) * down);
            h.z = pack_f16x2(bf_lo(w[i].z) * down, bf_hi(w[i].z) * down);
            h.w = pack_f16x2(bf_lo(w[i].w) * down, bf_hi(w[i].w) * down);
            const int piece = kHalf * part + i;
            *reinterpret_cast<uint4*>(sm + q_off + (piece >> 3) * (kRows * 128) + swz128(row, piece & 7)) = h;
        }
        fence_async_smem();
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
        const int qpos_min = min(qpos_a, qpos_b);
        const float up_a = scaled ? row_amax[row_a] : 1.0f, up_b = scaled ? row_amax[row_b] : 1.0f;
        float m_a = kMInit, m_b = kMInit, l_a = 0.0f, l_b = 0.0f;
        bool ok = true;
        for (int i = 0; i < n_tiles && ok; ++i) {
            ok = wait_phase(&bb[kBarQK + (i & 1)], (i >> 1) & 1, gave_up, __LINE__, p.error_word);
            if (!ok) break;
            tc_fence_after();
            uint32_t sr[32];
            tmem_ld_frag_x8(sr, tmem_s + my_lanes16);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) pipe::mbar_arrive(&bb[kBarSRead]);

            const float* const cst = reinterpret_cast<const float*>(sm + G::kSCst) + (i & (kCstRing - 1)) * G::kCstFloats;
            const int flags = reinterpret_cast<const int*>(cst)[3 * kKeys];
            const int key0 = (j0 + i) * kKeys;
            // pair 2 (2 a + h): row a, keys 16 a + 4 c2 + 2 h + {0, 1}; pair 2 (2 a + h) + 1: the same keys of row b
            float2 sv[16];
            if (scaled) {
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    sr[4 * g] = __float_as_uint(__uint_as_float(sr[4 * g]) * up_a);
                    sr[4 * g + 1] = __float_as_uint(__uint_as_float(sr[4 * g + 1]) * up_a);
                    sr[4 * g + 2] = __float_as_uint(__uint_as_float(sr[4 * g + 2]) * up_b);
                    sr[4 * g + 3] = __float_as_uint(__uint_as_float(sr[4 * g + 3]) * up_b);
                }
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const float4 kk = *reinterpret_cast<const float4*>(cst + 16 * a + 4 * c2);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = 4 * (2 * a + h);
                    const float2 k2 = h ? make_float2(kk.z, kk.w) : make_float2(kk.x, kk.y);
                    sv[r / 2] = mul2_rn(make_float2(__uint_as_float(sr[r]), __uint_as_float(sr[r + 1])), k2);
                    sv[r / 2 + 1] = mul2_rn(make_float2(__uint_as_float(sr[r + 2]), __uint_as_float(sr[r + 3])), k2);
                }
            }
            if (flags & kSlow) {                             // the V scales ride in the exponent on this tile
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const float4 lg = *reinterpret_cast<const float4*>(cst + kKeys + 16 * a + 4 * c2);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float x = h ? lg.z : lg.x, y = h ? lg.w : lg.y;
                        const int g = 2 * a + h;
                        sv[2 * g].x += x; sv[2 * g].y += y;
                        sv[2 * g + 1].x += x; sv[2 * g + 1].y += y;
                    }
                }
            }
            if (key0 + kKeys - 1 > qpos_min || (flags & 15) != 15) {
#pragma unroll
                for (int g = 0; g < 8; ++g) {
                    const int key = key0 + 16 * (g >> 1) + 4 * c2 + 2 * (g & 1);
                    const bool gone = ((flags >> (g >> 1)) & 1) == 0;
                    if (gone || key > qpos_a) sv[2 * g].x = -INFINITY;
                    if (gone || key + 1 > qpos_a) sv[2 * g].y = -INFINITY;
                    if (gone || key > qpos_b) sv[2 * g + 1].x = -INFINITY;
                    if (gone || key + 1 > qpos_b) sv[2 * g + 1].y = -INFINITY;
                }
            }
            float mx_a = fmaxf(sv[0].x, sv[0].y), mx_b = fmaxf(sv[1].x, sv[1].y);
#pragma unroll
            for (int g = 1; g < 8; ++g) {
                mx_a = fmaxf(mx_a, fmaxf(sv[2 * g].x, sv[2 * g].y));
                mx_b = fmaxf(mx_b, fmaxf(sv[2 * g + 1].x, sv[2 * g + 1].y));
            }
            mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 1));
            mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 1));
            mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, 2));
            mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, 2));
            const bool moved = __any_sync(0xffffffffu, mx_a > m_a + kLag || mx_b > m_b + kLag);
            float corr_a = 1.0f, corr_b = 1.0f;
            if (moved) {                                     // every row of the warp follows its maximum
                const float mn_a = fmaxf(m_a, mx_a), mn_b = fmaxf(m_b, mx_b);
                corr_a = ex2f(m_a - mn_a);
                corr_b = ex2f(m_b - mn_b);
                m_a = mn_a;
                m_b = mn_b;
                l_a *= corr_a;
                l_b *= corr_b;
            }
            const float2 neg_a = splat2(-m_a), neg_b = splat2(-m_b);
            float2 sum_a = make_float2(0.0f, 0.0f), sum_b = make_float2(0.0f, 0.0f);
            uint32_t wv[16];                 // word 4 a + h: row a, keys 16 a + 4 c2 + 2 h + {0, 1}; 4 a + 2 + h: row b
            if (flags & kSlow) {
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const float4 rv = *reinterpret_cast<const float4*>(cst + 2 * kKeys + 16 * a + 4 * c2);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int g = 2 * a + h;
                        const float2 r2 = h ? make_float2(rv.z, rv.w) : make_float2(rv.x, rv.y);
                        const float2 xa = add2_rn(sv[2 * g], neg_a), xb = add2_rn(sv[2 * g + 1], neg_b);
                        const float2 ea = make_float2(ex2f(xa.x), ex2f(xa.y)), eb = make_float2(ex2f(xb.x), ex2f(xb.y));
                        sum_a = fma2_rn(ea, r2, sum_a);
                        sum_b = fma2_rn(eb, r2, sum_b);
                        wv[4 * a + h] = pack_f16x2(ea.x, ea.y);
                        wv[4 * a + 2 + h] = pack_f16x2(eb.x, eb.y);
                    }
                }
            } else {
#pragma unroll
                for (int a = 0; a < 4; ++a) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int g = 2 * a + h;
                        const float2 xa = add2_rn(sv[2 * g], neg_a), xb = add2_rn(sv[2 * g + 1], neg_b);
                        const float2 ea = make_float2(ex2f(xa.x), ex2f(xa.y)), eb = make_float2(ex2f(xb.x), ex2f(xb.y));
                        sum_a = add2_rn(ea, sum_a);
                        sum_b = add2_rn(eb, sum_b);
                        wv[4 * a + h] = pack_f16x2(ea.x, ea.y);
                        wv[4 * a + 2 + h] = pack_f16x2(eb.x, eb.y);
                    }
                }
            }
            l_a += sum_a.x + sum_a.y;
            l_b += sum_b.x + sum_b.y;
            // W buffer i % 2 is free: O += W_{i-2} V_{i-2} was issued before S_i by the same thread, and the commit that
            // completed S_i's barrier covers it.  O may be touched once O += W_{i-1} V_{i-1} has completed; that wait may be
            // skipped on other tiles because no later product completes before this warp has signalled "W ready" for it.
            const bool rescale = moved && i > 0;
            if (rescale) {
                ok = wait_phase(&bb[kBarPV + ((i - 1) & 1)], ((i - 1) >> 1) & 1, gave_up, __LINE__, p.error_word);
                if (!ok) break;
                tc_fence_after();
            }
            tmem_st_frag_x4(tmem_w + (i & 1) * (kKeys / 2) + my_lanes16, wv);
            if (rescale) {
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
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) pipe::mbar_arrive(&bb[kBarWReady]);
        }
        // ---- epilogue: finished rows, or their states ----
        if (ok && n_tiles > 0)
            ok = wait_phase(&bb[kBarPV + ((n_tiles - 1) & 1)], ((n_tiles - 1) >> 1) & 1, gave_up, __LINE__, p.error_word);
        if (ok && work) {
            tc_fence_after();
            l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
            l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
            l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
            l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);
            const long long at_a = valid_a ? static_cast<long long>(token0 + tok_a) * p.num_q_heads + head_a : 0;
            const long long at_b = valid_b ? static_cast<long long>(token0 + tok_b) * p.num_q_heads + head_b : 0;
            const bool states = p.state_ml != nullptr;
            const float unfold = 1.0f / static_cast<float>(1 << kFoldShift);
            const float f_a = states ? unfold : (l_a == 0.0f ? 0.0f : unfold / l_a), f_b = states ? unfold : (l_b == 0.0f ? 0.0f : unfold / l_b);
            const long long split = static_cast<long long>(blockIdx.z) * p.out_rows;
            if (states && c2 == 0) {
                if (valid_a) *reinterpret_cast<float2*>(p.state_ml + 2 * (split + at_a)) = make_float2(m_a, l_a);
                if (valid_b) *reinterpret_cast<float2*>(p.state_ml + 2 * (split + at_b)) = make_float2(m_b, l_b);
            }
#pragma unroll 1
            for (int cb = 0; cb < D; cb += 32) {
                uint32_t ov[16];
                if (n_tiles > 0) {
                    tmem_ld_frag_x4(ov, tmem_o + my_lanes16 + cb);
                } else {
#pragma unroll
                    for (int g = 0; g < 16; ++g) ov[g] = 0u;
                }
                // a row that saw nothing is zero, whatever stale values met its zero weights
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float2 va = l_a == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(__uint_as_float(ov[4 * g]) * f_a, __uint_as_float(ov[4 * g + 1]) * f_a);
                    const float2 vb = l_b == 0.0f ? make_float2(0.0f, 0.0f) : make_float2(__uint_as_float(ov[4 * g + 2]) * f_b, __uint_as_float(ov[4 * g + 3]) * f_b);
                    const int d = cb + 8 * g + 2 * c2;
                    if (states) {
                        if (valid_a) *reinterpret_cast<float2*>(p.state_acc + (split + at_a) * D + d) = va;
                        if (valid_b) *reinterpret_cast<float2*>(p.state_acc + (split + at_b) * D + d) = vb;
                    } else {
                        if (valid_a) *reinterpret_cast<uint32_t*>(p.out + at_a * D + d) = pack_bf16x2(va.x, va.y);
                        if (valid_b) *reinterpret_cast<uint32_t*>(p.out + at_b * D + d) = pack_bf16x2(vb.x, vb.y);
                    }
                }
            }
        }
    } else if (warp < G::kConvWarp0) {
        // =============================== products of row block `blk` ===============================
        constexpr uint32_t kIdescQK = instr_desc(kKeys, false);
        constexpr uint32_t kIdescPV = instr_desc(D, true);
        auto issue_qk = [&](int t) {
            tc_fence_after();
            if (lane == 0) {
                const uint32_t k_base = base + G::kSK + (t & 1) * G::kTileBytes;
#pragma unroll
                for (int d = 0; d < G::kDimBlocks; ++d)
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        umma_f16(tmem_s, smem_desc(base + q_off + d * (kRows * 128) + s * 32, 16), smem_desc(k_base + d * (kKeys * 128) + s * 32, 16),
                                 kIdescQK, d > 0 || s > 0);
                umma_commit(&bb[kBarQK + (t & 1)]);
            }
            __syncwarp();
        };
        bool ok = n_tiles > 0 && wait_phase<kLazyNs>(&bars[G::kBarKReady], 0, gave_up, __LINE__, p.error_word);
        if (ok) issue_qk(0);
        for (int i = 0; i < n_tiles && ok; ++i) {
            if (i + 1 < n_tiles) {
                ok = wait_phase<kLazyNs>(&bb[kBarSRead], i & 1, gave_up, __LINE__, p.error_word) &&
                     wait_phase<kLazyNs>(&bars[G::kBarKReady + ((i + 1) & 1)], ((i + 1) >> 1) & 1, gave_up, __LINE__, p.error_word);
                if (!ok) break;
                issue_qk(i + 1);
            }
            ok = wait_phase<kLazyNs>(&bb[kBarWReady], i & 1, gave_up, __LINE__, p.error_word) &&
                 wait_phase<kLazyNs>(&bars[G::kBarVReady + (i & 1)], (i >> 1) & 1, gave_up, __LINE__, p.error_word);
            if (!ok) break;
            tc_fence_after();
            if (lane == 0) {
                const uint32_t v_base = base + G::kSV + (i & 1) * G::kTileBytes;
#pragma unroll
                for (int s = 0; s < kKeys / 16; ++s)
                    umma_f16_ts(tmem_o, tmem_w + (i & 1) * (kKeys / 2) + s * 8, smem_desc(v_base + s * 2048, kKeys * 128), kIdescPV, i > 0 || s > 0);
                umma_commit(&bb[kBarPV + (i & 1)]);
            }
            __syncwarp();
        }
    } else if (warp < G::kCopyWarp) {
        // =============================== conversion ===============================
        constexpr int kPerRow = D / 16;
        const int t = tid - 32 * G::kConvWarp0;
        // the least last visible key of the CTA's rows: tiles beyond it may hold keys that a row must not see
        if constexpr (kPrefix) {
            int mine = INT_MAX;
            for (int tok = t; tok < min(tokens, tile_tokens); tok += G::kConvThreads) mine = min(mine, last_key(tok));
            mine = __reduce_min_sync(0xffffffffu, mine);
            if (lane == 0) atomicMin(least, mine);
            named_sync(1, G::kConvThreads);
        }
        const int seen_by_all = kPrefix ? *least : held;
        auto wait_blocks = [&](int which, int buf, uint32_t parity, int where) {
            bool all = true;
#pragma unroll
            for (int g = 0; g < kBlocks; ++g)
                all = all && wait_phase<kLazyNs>(&bars[g * G::kBarsPerBlock + which + buf], parity, gave_up, where, p.error_word);
            return all;
        };
        int* const poison = reinterpret_cast<int*>(sm + G::kSPoison);
        bool ok = true;
        for (int i = 0; i < n_tiles && ok; ++i) {
            const int buf = i & 1, stage = i % kRawStages;
            const uint32_t freed = ((i - 2) >> 1) & 1;
            const unsigned char* const raw = sm + G::kSRaw + stage * G::kStageBytes;
            const float* const raw_ks = reinterpret_cast<const float*>(raw + 2 * G::kRawBytes);
            const float* const raw_vs = raw_ks + kKeys;
            const int key0 = (j0 + i) * kKeys;
            if (i >= 2) ok = wait_blocks(kBarQK, buf, freed, __LINE__);
            ok = ok && wait_phase<kLazyNs>(&bars[G::kBarRawFull + stage], (i / kRawStages) & 1, gave_up, __LINE__, p.error_word);
            if (group_or(1, G::kConvThreads, !ok)) { ok = false; break; }
            const int groups = raw_groups[stage];
            const bool edge = key0 + kKeys - 1 > seen_by_all || groups != 15;      // uniform
            if (edge) {          // keys whose V row holds a NaN code or has no finite scale: their scores become NaN, their row zero
                if (t < kKeys) poison[t] = !(raw_vs[t] <= 3.0e38f);
                named_sync(1, G::kConvThreads);
#pragma unroll
                for (int n = 0; n < G::kPerConv; ++n) {
                    const int c = t + G::kConvThreads * n;
                    if (c < G::kPieces) {
                        const uint4 w = *reinterpret_cast<const uint4*>(raw + G::kRawBytes + c * 16);
                        const uint32_t hit = (((w.x & 0x7f7f7f7fu) + 0x01010101u) | ((w.y & 0x7f7f7f7fu) + 0x01010101u) |
                                              ((w.z & 0x7f7f7f7fu) + 0x01010101u) | ((w.w & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u;
                        if (hit != 0u) poison[c / kPerRow] = 1;
                    }
                }
                named_sync(1, G::kConvThreads);
            }
            // whether some V scale is outside what the f16 operand holds (of the keys that count)
            bool outside = false;
            if (t < kKeys && key0 + t < total_keys && ((groups >> (t >> 4)) & 1) && !(edge && poison[t])) {
                const float vs = raw_vs[t];
                outside = vs != 0.0f && !(vs >= kFoldLow && vs <= kFoldHigh) && vs == vs;
            }
            const bool slow = group_or(1, G::kConvThreads, outside);
            if (t < kKeys) {
                float* const cst = reinterpret_cast<float*>(sm + G::kSCst) + (i & (kCstRing - 1)) * G::kCstFloats;
                const bool none = (edge && poison[t]) || (slow && raw_vs[t] != raw_vs[t]);      // (the exponent form would lose a NaN scale)
                cst[t] = none ? NAN : raw_ks[t] * p.scale_log2e;
                if (slow) {
                    const float lg = fmaxf(lg2f(raw_vs[t]), kLgFloor) + static_cast<float>(kFoldShift);
                    cst[kKeys + t] = lg;
                    cst[2 * kKeys + t] = ex2f(-lg);
                }
                if (t == 0) reinterpret_cast<int*>(cst)[3 * kKeys] = groups | (slow ? kSlow : 0);
            }
            // E4M3 -> f16 operand rows: [dim block of 64][row][128 bytes, swizzled].  Consecutive threads take consecutive
            // pieces of the raw tile; the upper half of a row's pieces stores its second half first, so that the eight
            // threads of a row write eight different 16-byte columns.
            unsigned char* const k_dst = sm + G::kSK + buf * G::kTileBytes;
            unsigned char* const v_dst = sm + G::kSV + buf * G::kTileBytes;
            auto place = [&](unsigned char* tile, int row, int ch, const uint4& h0, const uint4& h1) {
                unsigned char* const dst = tile + (ch >> 2) * (kKeys * 128) + swz128(row, 2 * (ch & 3));
                const uintptr_t other = reinterpret_cast<uintptr_t>(dst) ^ 16;
                const bool second = (ch >> 2) & 1;
                *reinterpret_cast<uint4*>(second ? other : reinterpret_cast<uintptr_t>(dst)) = second ? h1 : h0;
                *reinterpret_cast<uint4*>(second ? reinterpret_cast<uintptr_t>(dst) : other) = second ? h0 : h1;
            };
#pragma unroll
            for (int n = 0; n < G::kPerConv; ++n) {
                const int c = t + G::kConvThreads * n;
                if (c < G::kPieces) {
                    const uint4 w = *reinterpret_cast<const uint4*>(raw + c * 16);
                    uint4 h0, h1;
                    e4m3x4_to_f16x2x2(w.x, h0.x, h0.y);
                    e4m3x4_to_f16x2x2(w.y, h0.z, h0.w);
                    e4m3x4_to_f16x2x2(w.z, h1.x, h1.y);
                    e4m3x4_to_f16x2x2(w.w, h1.z, h1.w);
                    place(k_dst, k_row_of_key(c / kPerRow), c % kPerRow, h0, h1);
                }
            }
            fence_async_smem();
            pipe::mbar_arrive(&bars[G::kBarKReady + buf]);
            // V of the tile, once O += W_{i-2} V_{i-2} is complete
            if (i >= 2) ok = wait_blocks(kBarPV, buf, freed, __LINE__);
            if (group_or(1, G::kConvThreads, !ok)) { ok = false; break; }
#pragma unroll
            for (int n = 0; n < G::kPerConv; ++n) {
                const int c = t + G::kConvThreads * n;
                if (c < G::kPieces) {
                    const int key = c / kPerRow;
                    uint4 w = *reinterpret_cast<const uint4*>(raw + G::kRawBytes + c * 16);
                    float vs = slow ? 1.0f : raw_vs[key] * static_cast<float>(1 << kFoldShift);
                    if (edge && (poison[key] || key0 + key >= total_keys || !((groups >> (key >> 4)) & 1))) {
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
                    place(v_dst, key, c % kPerRow, make_uint4(h[0], h[1], h[2], h[3]), make_uint4(h[4], h[5], h[6], h[7]));
                }
            }
            fence_async_smem();
            pipe::mbar_arrive(&bars[G::kBarVReady + buf]);
            pipe::mbar_arrive(&bars[G::kBarRawEmpty + stage]);
        }
    } else {
        // =============================== copies ===============================
        // A tile is one run per page and array: lane (array, run) of K codes, V codes, K scales, V scales.
        const int shift = p.c.page_shift;
        const int run_keys = shift < 6 ? 1 << shift : kKeys, runs = kKeys / run_keys;
        const int array = lane / runs, run = lane - array * runs;
        auto page_of = [&](int i) {
            const int key = (j0 + i) * kKeys + run * run_keys;
            int id = -1;
            if (lane < 4 * runs && i < n_tiles && key < total_keys && (key >> shift) < p.c.pages_per_row) id = pages[key >> shift];
            return id >= 0 && id < p.c.num_pages ? id : -1;
        };
        const int per_key = array < 2 ? D : 4;
        const uint32_t bytes = static_cast<uint32_t>(run_keys * per_key);
        const unsigned char* const src0 = array == 0 ? p.c.k : array == 1 ? p.c.v : array == 2 ? reinterpret_cast<const unsigned char*>(p.c.k_scale)
                                                                                               : reinterpret_cast<const unsigned char*>(p.c.v_scale);
        const int dst0 = (array < 2 ? array * G::kRawBytes : 2 * G::kRawBytes + (array - 2) * kKeys * 4) + run * static_cast<int>(bytes);
        int next = page_of(0);
        int issued = 0;
        bool ok = true;
        for (int i = 0; i < n_tiles; ++i) {
            const int id = next;
            next = page_of(i + 1);
            const int stage = i % kRawStages;
            if (i >= kRawStages) ok = wait_phase<kLazyNs>(&bars[G::kBarRawEmpty + stage], ((i / kRawStages) - 1) & 1, gave_up, __LINE__, p.error_word);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            const unsigned have = __ballot_sync(0xffffffffu, id >= 0);      // bits 0 .. runs-1: the runs of the tile that exist
            int groups = 0;
            for (int r = 0; r < runs; ++r)
                if ((have >> r) & 1) groups |= ((1 << (run_keys / 16)) - 1) << (r * (run_keys / 16));
            if (lane == 0) {
                raw_groups[stage] = groups;
                pipe::mbar_expect_tx(&bars[G::kBarRawFull + stage], static_cast<uint32_t>(__popc(have & ((1u << runs) - 1u)) * run_keys * (2 * D + 8)));
            }
            __syncwarp();
            if (id >= 0) {
                const size_t key = key_index(p.c, id, kvh) + (((j0 + i) * kKeys + run * run_keys) & ((1 << shift) - 1));
                pipe::bulk_load(sm + G::kSRaw + stage * G::kStageBytes + dst0, src0 + key * per_key, bytes, &bars[G::kBarRawFull + stage]);
            }
            issued = i + 1;
        }
        if (!ok)        // somebody gave up: let the copies on their way land (bounded again) before the CTA ends
            for (int i = max(0, issued - kRawStages); i < issued; ++i) {
                for (int tries = 0; tries < (1 << 12) && !pipe::mbar_try_wait(&bars[G::kBarRawFull + i % kRawStages], (i / kRawStages) & 1); ++tries) {}
            }
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
}

template <int D, int kBlocks, bool kPrefix>
int launch_blocks_as(const BlockArgs& a, unsigned tiles, unsigned splits, cudaStream_t stream, const char* fn) {
    using G = Geo<D, kBlocks>;
    const dim3 grid(static_cast<unsigned>(a.c.num_kv_heads * a.head_chunks), tiles, splits);
    (void)host::setup<&paged_blocks_kernel<D, kBlocks, kPrefix>, G::kThreads, G::kSmemBytes>();
    host::launch<paged_blocks_kernel<D, kBlocks, kPrefix>>(grid, dim3(G::kThreads), static_cast<size_t>(G::kSmemBytes), stream, a);
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
    (void)head_dim;
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
    RH_REQUIRE(num_splits >= 1 && num_splits <= 64, RH_ERR_INVALID_ARG, "%s: num_splits must be in 1..64", fn);
    RH_REQUIRE(num_splits == 1 || partial_or_null != nullptr, RH_ERR_INVALID_ARG, "%s: splits need scratch", fn);
    RH_REQUIRE(q_stride >= static_cast<long long>(num_q_heads) * cache->head_dim, RH_ERR_INVALID_ARG, "%s: q_stride is below num_q_heads * head_dim", fn);
    RH_REQUIRE(host::aligned16(q) && q_stride % 8 == 0 && host::aligned16(partial_or_null), RH_ERR_MISALIGNED,
               "%s: q and partial must be 16-byte aligned, q_stride a multiple of 8", fn);
    RH_REQUIRE((reinterpret_cast<uintptr_t>(out) & 7u) == 0, RH_ERR_MISALIGNED, "%s: out must be 8-byte aligned", fn);
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
    // two row blocks per CTA once one-block CTAs are more than the SMs: a tile is converted once for twice the rows
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
