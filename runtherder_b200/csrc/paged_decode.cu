// Attention of one new token per sequence over the paged FP8 cache, for a batch that may share a prefix.
//
//   out[b, h] = sum_j softmax_j(scale * q[b, h] . K_j) V_j    over keys j = 0 .. lens[row of b]
//
// The first `shared` keys lie in the same pages for every sequence: they are read once and multiplied with the
// queries of all sequences; the keys behind them are each sequence's own.  Both parts leave (m, l, acc) states in the
// caller's scratch which a second kernel joins.  The reference decodes one sequence (flash_decode_split_bf16,
// include/runtherder/kernels/flash_decode.cuh:27-62; flash_decode.cu here).
//
// Work.  A segment is (sequence, kv head, up to 8 query heads) for own keys and (kv head, 8 of the batch's query rows)
// for the prefix, cut into tiles of 16 keys.  All tiles of all segments form one line that is dealt out evenly to all
// warps of the grid, so neither ragged lengths nor few long sequences leave SMs idle; a warp that crosses from one
// segment into the next writes one state for each.  Segment s and warp w meet at most once and both only grow along
// the line, so s + w is a slot that no other pair uses.
//
// A tile.  The rows are tensor-core operands as they lie: S^T[16 keys x 8 cols] = K q^T and O^T[16 dims x 8 cols] +=
// V^T W^T with mma.sync.m16n8k16 (f16, fp32 accumulation; E4M3 converts to f16 exactly), columns being query heads.
// A decode step has 1 to 8 rows per kv head and sequence, far below a tcgen05 tile, and the op is bound by HBM: 264
// bytes per key and kv head.  Scales never touch the operands: the K scale multiplies the fp32 score, the V scale
// rides in the exponent of the weight (its log2 is added to the score), the denominator takes it out again.  A tile's
// K codes and V codes are one run of memory each in this cache's layout: one lane fetches them with two bulk copies into the
// warp's own ring, a tile ahead, the scales come by one asynchronous copy per lane; there is no barrier among warps.
//
// Measured (B200, 32/8 heads of 128): 8 x 32768 keys 68 us = 5.3 TB/s, 64 x 2000 keys 38.8 us = 3.8 TB/s, of 6.5 for a copy; a
// lone sequence of 8196 keys (24/8 heads) 14 us out of L2, 17 us with 28 caches in turn (flash_decode.cu, which joins four warps in a CTA before it
// writes a state, 9.3 - 9.8 us so; 65536 keys 35 us in either).  The decode kernel alone on 64 x 2000 keys takes 34 us (DRAM 56 % busy, issue slots
// 46 %, 385 instructions per tile): a warp's tile is a chain of some 2000 cycles (wait, products, exponentials, transposes, products),
// sixteen warps of 128 registers fill an SM (twenty of 96 spill: 64 x 2000 keys 44.9 us), and the E4M3 conversions alone are 8 us at one per
// cycle and SM.  What a small call waits for is latency:
// some 3 us to find its tiles and look up pages, the chain, and 4 us for the joining kernel.
#include <cuda_fp16.h>

#include <cmath>

#include "flash_prefill_tc.cuh"
#include "paged.cuh"
#include "paged_attention.cuh"
#include "paged_prefill.cuh"
#include "rh_kernels.h"
#include "rh_pipeline.cuh"

namespace rh {
namespace paged {
namespace {

using tc::e4m3x4_to_f16x2x2;
using tc::ex2f;
using tc::lg2f;
using tc::pack_f16x2;

constexpr int kDecWarps = 4;
constexpr int kDecThreads = 32 * kDecWarps;
constexpr int kTile = 16;              // keys per tile
static_assert(kPrefixCols == 8 && kOwnCols == 8, "a segment has the eight columns of a product");
constexpr int kStages = 2;             // tiles in a warp's ring (with three, 8 x 32768 keys take 72.5 us instead of 68: sixteen warps per SM have enough on the way)
static_assert((kStages & (kStages - 1)) == 0, "counters wrap");
constexpr int kDecCtas = 4;            // CTAs per SM
constexpr float kLag = 8.0f;           // how far (log2) the running maximum may lie below the true one
// Weights enter the second product as 2^7 * weight (at most 2^15), rounded to f16 once: 2^-11 each, an eighth of the bf16 store's rounding, and
// below 2^-32 of the row's largest lost.  (flash_decode.cu enters two f16 parts of each.)
constexpr float kShift = 7.0f;

// D(16x8, fp32) += A(16x16, f16, row) * B(16x8, f16, col)
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8x8 transpose of 16-bit elements across the warp
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// 4-byte asynchronous copy; arrives on `bar` (which counts every lane) once it has landed
__device__ __forceinline__ void cp4_arrive(void* dst, const void* src, uint64_t* bar) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(pipe::smem_u32(dst)), "l"(src) : "memory");
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(pipe::smem_u32(bar)) : "memory");
}

template <int D>
struct Ring {
    static constexpr int kCodes = kTile * D;                         // bytes of K (or V) codes of a tile
    static constexpr int kStageBytes = 2 * kCodes + 2 * kTile * 4;   // K, V, K scales, V scales
    static constexpr int kWarpBytes = kStages * kStageBytes;
    static constexpr int kBarOffset = kDecWarps * kWarpBytes;
    static constexpr int kTableOffset = kBarOffset + kDecWarps * kStages * 8;   // first tile of every sequence follows
};

// One warp's way through `tiles` tiles of a segment: keys key0 .. key0 + 16 tiles - 1 of the list `pages`, of which the
// first `limit` exist; eight columns (query rows).  Called by whole warps.
template <int D>
struct Walk {
    using R = Ring<D>;
    static constexpr int kKWords = D / 16;    // 32-bit words of a K row per lane = k-steps of the first product
    static constexpr int kVWords = D / 32;
    static constexpr int kMB = D / 16;        // 16-dim blocks of the second product

    const DecodeArgs& p;
    unsigned char* ring;
    uint64_t* full;
    uint32_t& turn;           // tiles this warp has taken from its ring so far: stage and parity of the next
    int lane, r, c;

    float o[kMB][4];
    float m[2], l[2];         // of columns 2c and 2c + 1; l: this lane's part

    __device__ __forceinline__ Walk(const DecodeArgs& p_, unsigned char* ring_, uint64_t* full_, uint32_t& turn_)
        : p(p_), ring(ring_), full(full_), turn(turn_) {
        lane = threadIdx.x & 31;
        r = lane >> 2;
        c = lane & 3;
    }

    // col_row(col): offset of a column's query row, -1: none; col_limit(col): keys that the column sees.
    // Returns false when a wait gave up.
    template <typename ColRow, typename ColLimit>
    __device__ __forceinline__ bool run(const int* pages, int columns, int key0, int tiles, int limit, int kvh, ColRow col_row, ColLimit col_limit) {
        const int shift = p.c.page_shift, per_page = shift - 4;
        // where the next 32 tiles lie, one per lane, in units of tiles from the start of the layer; -1 where there is no page
        auto places = [&](int first) {
            const int key = key0 + (first + lane) * kTile;
            int id = -1;
            if (first + lane < tiles && (key >> shift) < columns) id = pages[key >> shift];
            return id >= 0 && id < p.c.num_pages ? ((id * p.c.num_kv_heads + kvh) << per_page) + ((key >> 4) & ((1 << per_page) - 1)) : -1;
        };
        int here = places(0), ahead = places(32);
        uint32_t live = 0;                      // bit i % 32: tile i has a page
        uint32_t put = turn;                    // the stage that is filled next
        auto issue = [&](int i) {               // a tile without a page takes its turn without bytes
            const int at = __shfl_sync(0xffffffffu, here, i & 31);
            if ((i & 31) == 31) {
                here = ahead;
                ahead = places(i + 33);
            }
            const uint32_t stage = put++ % kStages;
            uint64_t* const bar = full + stage;
            unsigned char* const dst = ring + stage * R::kStageBytes;
            const bool there = at >= 0;
            live = there ? live | (1u << (i & 31)) : live & ~(1u << (i & 31));
            const size_t tile = there ? static_cast<size_t>(at) : 0;
            if (lane == 0) {
                if (there) {
                    pipe::mbar_expect_tx(bar, 2 * R::kCodes);
                    pipe::bulk_load(dst, p.c.k + tile * R::kCodes, R::kCodes, bar);
                    pipe::bulk_load(dst + R::kCodes, p.c.v + tile * R::kCodes, R::kCodes, bar);
                } else {
                    pipe::mbar_arrive(bar);
                }
            }
            // the scales: one per lane (K, then V), by ordinary asynchronous copies that arrive on the same barrier
            cp4_arrive(dst + 2 * R::kCodes + lane * 4, (lane < kTile ? p.c.k_scale : p.c.v_scale) + tile * kTile + (lane & (kTile - 1)), bar);
        };
        __syncwarp();                           // the ring's last readers are done
#pragma unroll 1
        for (int i = 0; i < min(kStages - 1, tiles); ++i) issue(i);

        // ---- q as the B operand: column r, dims 64 ch + 16 c + 0..15, scaled by a power of two into (-2, 2) (exact; f16 then
        //      holds any bf16 row) ----
        uint32_t qb[kKWords][2];
        float factor[2];
        int see[2];                             // keys that the columns 2c and 2c + 1 see
        {
            const long long row = col_row(r);
            uint4 raw[D / 32];
#pragma unroll
            for (int ch = 0; ch < D / 64; ++ch) {
                raw[2 * ch] = raw[2 * ch + 1] = make_uint4(0u, 0u, 0u, 0u);
                if (row >= 0) {
                    const uint4* const src = reinterpret_cast<const uint4*>(p.q + row + 64 * ch + 16 * c);
                    raw[2 * ch] = src[0];
                    raw[2 * ch + 1] = src[1];
                }
            }
            const int sees = min(limit, col_limit(r));
            see[0] = __shfl_sync(0xffffffffu, sees, 8 * c);
            see[1] = __shfl_sync(0xffffffffu, sees, 8 * c + 4);
            uint32_t amax2 = 0u;
#pragma unroll
            for (int v = 0; v < D / 32; ++v) amax2 = amax_acc_bf16x2(amax_acc_bf16x2(amax_acc_bf16x2(amax_acc_bf16x2(amax2, raw[v].x), raw[v].y), raw[v].z), raw[v].w);
            float amax = fmaxf(bf_lo(amax2), bf_hi(amax2));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            int e = ((__float_as_int(amax) >> 23) & 0xff) - 127;
            e = amax > 0.0f ? max(-100, min(126, e)) : 0;
            const float down = __int_as_float((127 - e) << 23);
            const float mine = p.scale_log2e * __int_as_float((127 + e) << 23);
            factor[0] = __shfl_sync(0xffffffffu, mine, 8 * c);
            factor[1] = __shfl_sync(0xffffffffu, mine, 8 * c + 4);
#pragma unroll
            for (int s = 0; s < kKWords; ++s) {
                const uint4& w = raw[s >> 1];
                const uint32_t lo = s & 1 ? w.z : w.x, hi = s & 1 ? w.w : w.y;
                qb[s][0] = pack_f16x2(bf_lo(lo) * down, bf_hi(lo) * down);
                qb[s][1] = pack_f16x2(bf_lo(hi) * down, bf_hi(hi) * down);
            }
        }
        // tiles that every column sees whole
        const int everyone = __reduce_min_sync(0xffffffffu, min(see[0], see[1]));
        const int plain = max(0, min(tiles, (everyone - key0) >> 4));

#pragma unroll
        for (int b = 0; b < kMB; ++b) o[b][0] = o[b][1] = o[b][2] = o[b][3] = 0.0f;
        m[0] = m[1] = kMInit;
        l[0] = l[1] = 0.0f;

        bool ok = true;
#pragma unroll 1
        for (int i = 0; i < tiles; ++i) {
            __syncwarp();                              // the stage that is filled next has been read by every lane
            if (i + kStages - 1 < tiles) issue(i + kStages - 1);
            const uint32_t stage = turn % kStages;
            ok = warp_wait(full + stage, (turn / kStages) & 1, __LINE__, p.error_word);
            if (!ok) {                                 // gave up: let the copies on their way land (bounded again), then leave
                for (int k = 1; k < kStages && i + k < tiles; ++k) {
                    const uint32_t t = turn + k;
                    (void)warp_wait(full + t % kStages, (t / kStages) & 1, __LINE__, p.error_word, 1 << 12);
                }
                break;
            }
            ++turn;
            if ((live >> (i & 31)) & 1u) {
                if (i < plain) fold<false>(ring + stage * R::kStageBytes, key0 + i * kTile, qb, factor, see);
                else fold<true>(ring + stage * R::kStageBytes, key0 + i * kTile, qb, factor, see);
            }
        }
        return ok;
    }

    // kPartial: some column must not see some of the tile's keys.
    template <bool kPartial>
    __device__ __forceinline__ void fold(const unsigned char* st, int kb, const uint32_t (&qb)[kKWords][2], const float (&factor)[2], const int (&see)[2]) {
        const int key_a = 4 * (r >> 1) + (r & 1);      // tile-local keys of rows r and r + 8 of the first product: key_a, key_a + 2
        // ---- S^T = K q^T ----
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f}, t[4] = {0.0f, 0.0f, 0.0f, 0.0f};      // two chains
#pragma unroll
        for (int ch = 0; ch < D / 64; ++ch) {
            const uint4 ka = *reinterpret_cast<const uint4*>(st + key_a * D + 64 * ch + 16 * c);
            const uint4 kc = *reinterpret_cast<const uint4*>(st + (key_a + 2) * D + 64 * ch + 16 * c);
            const uint32_t aw[4] = {ka.x, ka.y, ka.z, ka.w}, bw[4] = {kc.x, kc.y, kc.z, kc.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t a0, a1, a2, a3;
                e4m3x4_to_f16x2x2(aw[k], a0, a2);
                e4m3x4_to_f16x2x2(bw[k], a1, a3);
                mma16816(k & 1 ? t : s, a0, a1, a2, a3, qb[4 * ch + k][0], qb[4 * ch + k][1]);
            }
        }
        uint32_t vw[4][kVWords];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned char* const src = st + R::kCodes + (4 * c + i) * D + r * (D / 8);
            if constexpr (D == 128) {
                const uint4 v = *reinterpret_cast<const uint4*>(src);
                vw[i][0] = v.x; vw[i][1] = v.y; vw[i][2] = v.z; vw[i][3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(src);
                vw[i][0] = v.x; vw[i][1] = v.y;
            }
        }
        const float* const sc = reinterpret_cast<const float*>(st + 2 * R::kCodes) + key_a;
        const float ks_a = sc[0], ks_b = sc[2], vs_a = sc[kTile], vs_b = sc[kTile + 2];
        const float lg_a = fmaxf(lg2f(vs_a), kLgFloor), lg_b = fmaxf(lg2f(vs_b), kLgFloor);
        const float rv_a = ex2f(-lg_a - kShift), rv_b = ex2f(-lg_b - kShift);
        float add_a = fmaf(vs_a, 0.0f, lg_a), add_b = fmaf(vs_b, 0.0f, lg_b);        // (the maximum loses a NaN scale: it is added back)
        if constexpr (kPartial) {
            // A column must not see some of these keys, whose V codes may be anything: a NaN code times weight zero would
            // be NaN.  NaN codes become zero here, and the score of such a key NaN for the columns that do see it.
            unsigned bad[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bool nan = false;
#pragma unroll
                for (int w = 0; w < kVWords; ++w) {
                    const uint32_t hit = ((vw[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                    nan |= hit != 0u;
                    if (hit != 0u) vw[i][w] = 0u;
                }
                bad[i] = __ballot_sync(0xffffffffu, nan);
            }
            const unsigned lanes = 0x11111111u << (r >> 1);      // the lanes that hold key_a's and key_b's V rows
            if (((r & 1) ? bad[1] : bad[0]) & lanes) add_a = NAN;
            if (((r & 1) ? bad[3] : bad[2]) & lanes) add_b = NAN;
        }
        // log2-domain scores with the V scale in the exponent: rows a, b x columns 2c, 2c + 1
        float x0 = fmaf(s[0] + t[0], ks_a * factor[0], add_a), x1 = fmaf(s[1] + t[1], ks_a * factor[1], add_a);
        float x2 = fmaf(s[2] + t[2], ks_b * factor[0], add_b), x3 = fmaf(s[3] + t[3], ks_b * factor[1], add_b);
        if constexpr (kPartial) {
            if (kb + key_a >= see[0]) x0 = -INFINITY;
            if (kb + key_a >= see[1]) x1 = -INFINITY;
            if (kb + key_a + 2 >= see[0]) x2 = -INFINITY;
            if (kb + key_a + 2 >= see[1]) x3 = -INFINITY;
        }
        // The maximum may lag the true one by up to 2^kLag, so the eight rows need not agree on it on most tiles.
        float t0 = fmaxf(x0, x2), t1 = fmaxf(x1, x3);
        if (__any_sync(0xffffffffu, t0 > m[0] + kLag || t1 > m[1] + kLag)) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, off));
                t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, off));
            }
            const float n0 = fmaxf(m[0], t0), n1 = fmaxf(m[1], t1);
            const float f0 = ex2f(m[0] - n0), f1 = ex2f(m[1] - n1);
            l[0] *= f0;
            l[1] *= f1;
#pragma unroll
            for (int b = 0; b < kMB; ++b) {
                o[b][0] *= f0; o[b][1] *= f1;
                o[b][2] *= f0; o[b][3] *= f1;
            }
            m[0] = n0;
            m[1] = n1;
        }
        const float s0 = m[0] - kShift, s1 = m[1] - kShift;
        const float w0 = ex2f(x0 - s0), w1 = ex2f(x1 - s1), w2 = ex2f(x2 - s0), w3 = ex2f(x3 - s1);
        if constexpr (kPartial) {       // a masked key adds nothing to the denominator even where its stale V scale is no number
            l[0] += (w0 == 0.0f ? 0.0f : w0 * rv_a) + (w2 == 0.0f ? 0.0f : w2 * rv_b);
            l[1] += (w1 == 0.0f ? 0.0f : w1 * rv_a) + (w3 == 0.0f ? 0.0f : w3 * rv_b);
        } else {
            l[0] = fmaf(w2, rv_b, fmaf(w0, rv_a, l[0]));
            l[1] = fmaf(w3, rv_b, fmaf(w1, rv_a, l[1]));
        }
        const uint32_t b0 = transpose8x8(pack_f16x2(w0, w1)), b1 = transpose8x8(pack_f16x2(w2, w3));
        // ---- O^T += V^T W^T: bytes of keys 4c .. 4c + 3 transposed into key pairs ----
#pragma unroll
        for (int w = 0; w < kVWords; ++w) {
            const uint32_t t01 = __byte_perm(vw[0][w], vw[1][w], 0x5140), t23 = __byte_perm(vw[2][w], vw[3][w], 0x5140);
            const uint32_t u01 = __byte_perm(vw[0][w], vw[1][w], 0x7362), u23 = __byte_perm(vw[2][w], vw[3][w], 0x7362);
            uint32_t a0, a1, a2, a3;
            e4m3x4_to_f16x2x2(t01, a0, a1);
            e4m3x4_to_f16x2x2(t23, a2, a3);
            mma16816(o[2 * w], a0, a1, a2, a3, b0, b1);
            e4m3x4_to_f16x2x2(u01, a0, a1);
            e4m3x4_to_f16x2x2(u23, a2, a3);
            mma16816(o[2 * w + 1], a0, a1, a2, a3, b0, b1);
        }
    }

    // The state of the columns < live to `slot`: m [cols], l [cols], acc [cols][D] (cols: the slot's columns)
    __device__ __forceinline__ void store(float* slot, int cols, int used) {
        const float unshift = ex2f(-kShift);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float sum = l[e];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            const int col = 2 * c + e;
            if (col < used) {
                if (r == 0) {
                    slot[col] = m[e];
                    slot[cols + col] = sum;
                }
                float4* const dst = reinterpret_cast<float4*>(slot + acc_offset(cols) + col * D + r * (D / 8));
#pragma unroll
                for (int q = 0; q < kMB / 2; ++q)
                    dst[q] = make_float4(o[2 * q][e] * unshift, o[2 * q][2 + e] * unshift, o[2 * q + 1][e] * unshift, o[2 * q + 1][2 + e] * unshift);
            }
        }
    }
};

// The keys that a batch entry's row holds for it with its new token, within its table; 0: idle or unknown.
__device__ __forceinline__ int keys_of(const DecodeArgs& p, int b) {
    const int row = p.rows != nullptr ? p.rows[b] : b;
    if (row < 0 || row >= p.c.num_rows) return 0;
    const int held = p.c.lens[row];
    if (held < 0) return 0;
    const int room = p.c.pages_per_row << p.c.page_shift;
    return held < room ? held + 1 : room;
}

template <int D>
__global__ void __launch_bounds__(kDecThreads, kDecCtas) decode_kernel(const DecodeArgs p) {
    using R = Ring<D>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int warp_sum[kDecWarps];
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + R::kBarOffset);
    int* const first_tile = reinterpret_cast<int*>(smem + R::kTableOffset);     // [num_seqs + 1], in tiles of one kv head
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < kDecWarps * kStages) pipe::mbar_init(bars + threadIdx.x, 1 + 32);      // the codes' bytes, and every lane's scale
    pipe::mbar_init_fence();

    pdl_wait();
    pdl_trigger();
    const int shared_keys = p.shared_keys();
    // ---- the line of tiles: prefix segments first, then every sequence's own keys ----
    int running = 0;
    for (int base = 0; base < p.num_seqs; base += kDecThreads) {
        const int b = base + threadIdx.x;
        const int own = b < p.num_seqs ? max(0, keys_of(p, b) - shared_keys) : 0;
        const int mine = (own + kTile - 1) / kTile;
        int incl = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, off);
            if (lane >= off) incl += up;
        }
        __syncthreads();
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        int before = running, all = 0;
#pragma unroll
        for (int w = 0; w < kDecWarps; ++w) {
            before += w < warp ? warp_sum[w] : 0;
            all += warp_sum[w];
        }
        if (b < p.num_seqs) first_tile[b] = before + incl - mine;
        running += all;
    }
    if (threadIdx.x == 0) first_tile[p.num_seqs] = running;
    __syncthreads();
    const int heads = p.c.num_kv_heads * p.head_chunks;                  // own segments per sequence
    const int prefix_segs = p.prefix_chunks * p.c.num_kv_heads;          // none when another kernel takes the prefix
    const int prefix_tiles = shared_keys / kTile;
    const long long prefix_total = static_cast<long long>(prefix_segs) * prefix_tiles;
    const long long total = prefix_total + static_cast<long long>(running) * heads;
    const long long warps = warps_in_use(total, static_cast<long long>(gridDim.x) * kDecWarps);
    if (blockIdx.x == 0) {           // what the joining kernel needs to find the states
        if (threadIdx.x == 0) {
            p.header[0] = shared_keys;
            p.header[1] = running;
        }
        for (int b = threadIdx.x; b <= p.num_seqs; b += kDecThreads) p.header[kHeaderInts + b] = first_tile[b];
    }
    const long long w = static_cast<long long>(blockIdx.x) * kDecWarps + warp;
    if (w >= warps) return;
    long long t = line_start(total, warps, w);
    const long long end = line_start(total, warps, w + 1);

    unsigned char* const ring = smem + warp * R::kWarpBytes;
    uint64_t* const full = bars + warp * kStages;
    uint32_t turn = 0;
    bool ok = true;
    while (t < end && ok) {
        if (t < prefix_total) {
            const int seg = static_cast<int>(t / prefix_tiles), at = static_cast<int>(t - static_cast<long long>(seg) * prefix_tiles);
            const int tiles = static_cast<int>(min(end - t, static_cast<long long>(prefix_tiles - at)));
            const int kvh = seg / p.prefix_chunks, row0 = (seg - kvh * p.prefix_chunks) * kPrefixCols;
            const int rows = p.num_seqs * p.group;
            Walk<D> walk(p, ring, full, turn);
            ok = walk.run(p.shared_pages, p.c.pages_per_row, at * kTile, tiles, shared_keys, kvh,
                          [&](int col) -> long long {
                              const int row = row0 + col;
                              if (row >= rows) return -1;
                              const int b = row / p.group;
                              return b * p.q_stride + static_cast<long long>(kvh * p.group + (row - b * p.group)) * D;
                          },
                          [&](int col) { return row0 + col < rows ? keys_of(p, (row0 + col) / p.group) : INT_MAX; });
            walk.store(p.prefix_states + (seg + w) * state_floats(kPrefixCols, D), kPrefixCols, min(kPrefixCols, rows - row0));
            t += tiles;
        } else {
            const long long u = t - prefix_total;
            const int at_all = static_cast<int>(u / heads);              // the sequence whose tiles of all heads hold u
            int lo = 0, hi = p.num_seqs;                                 // last b with first_tile[b] <= at_all
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (first_tile[mid] <= at_all) lo = mid;
                else hi = mid;
            }
            const int b = lo, n = first_tile[b + 1] - first_tile[b];
            const long long inside = u - static_cast<long long>(first_tile[b]) * heads;
            const int head = static_cast<int>(inside / n), at = static_cast<int>(inside - static_cast<long long>(head) * n);
            const int tiles = static_cast<int>(min(end - t, static_cast<long long>(n - at)));
            const int kvh = head / p.head_chunks, h0 = (head - kvh * p.head_chunks) * kOwnCols;
            const int row = p.rows != nullptr ? p.rows[b] : b;
            const int live = min(p.own_cols, p.group - h0);
            const int keys = keys_of(p, b);
            Walk<D> walk(p, ring, full, turn);
            ok = walk.run(p.c.page_table + static_cast<size_t>(row) * p.c.pages_per_row, p.c.pages_per_row, shared_keys + at * kTile, tiles, keys, kvh,
                          [&](int col) -> long long { return col < live ? b * p.q_stride + static_cast<long long>(kvh * p.group + h0 + col) * D : -1; },
                          [&](int) { return keys; });
            walk.store(p.own_states + (static_cast<long long>(b) * heads + head + w) * state_floats(p.own_cols, D), p.own_cols, live);
            t += tiles;
        }
    }
}

// Joins the states of a query row: M = max m_i, out = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i, zero where nothing
// was seen.  kRowThreads threads share a row: D / 4 lanes hold four dims each, the groups of lanes take the states in
// turn.  A lone sequence has as many states as warps worked on it (hundreds) and few rows: a CTA of 1024 threads takes a row.
// A large batch has thousands of rows of a few states: a group each.  In between 256 threads.  Whole calls with 1024 / 256 / D / 4
// threads: 1 x 8196 keys, 24 rows, 14 / 20 / 46 us; 4 x 2000, 128 rows, 13.8 / 15.3 / 20; 12 x 2000, 384 rows, 22 / 17.7 / 24; 32 x 2000,
// 1024 rows, 42 / 28.3 / 30.7; 64 x 2000, 2048 rows, 72 / 43 / 40.  Bound by latency: two rounds of dependent loads (where the states
// lie, the states).
template <int D, int kRowThreads, int kThreads>
__global__ void __launch_bounds__(kThreads) join_kernel(const DecodeArgs p, int decode_warps) {
    constexpr int kVecs = D / 4, kGroups = kRowThreads / kVecs, kRows = kThreads / kRowThreads;
    __shared__ float4 s_acc[kRows][kGroups][kVecs];
    __shared__ float s_m[kRows][kGroups], s_l[kRows][kGroups];
    const int slot_row = threadIdx.x / kRowThreads, tid = threadIdx.x % kRowThreads;
    const int g = tid / kVecs, j = tid % kVecs;
    const int num_q = p.c.num_kv_heads * p.group;
    const int rows = p.num_seqs * num_q;
    const int out_row = min(static_cast<int>(blockIdx.x) * kRows + slot_row, rows - 1);      // (the last CTA repeats its last row)
    const int b = out_row / num_q, qh = out_row - b * num_q;
    const int kvh = qh / p.group, hg = qh - kvh * p.group;
    pdl_enter();

    float m = kMInit, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto take = [&](float mi, float li, const float4& a) {
        const float n = fmaxf(m, mi);
        const float f = ex2f(m - n), fi = ex2f(mi - n);
        l = l * f + li * fi;
        acc.x = acc.x * f + a.x * fi;
        acc.y = acc.y * f + a.y * fi;
        acc.z = acc.z * f + a.z * fi;
        acc.w = acc.w * f + a.w * fi;
        m = n;
    };
    const int shared_keys = p.header[0], own_tiles = p.header[1], first = p.header[kHeaderInts + b], after = p.header[kHeaderInts + b + 1];
    const int heads = p.c.num_kv_heads * p.head_chunks;
    const int prefix_tiles = shared_keys / kTile;
    const long long prefix_total = static_cast<long long>(p.prefix_chunks * p.c.num_kv_heads) * prefix_tiles;
    const long long total = prefix_total + static_cast<long long>(own_tiles) * heads;
    const long long warps = warps_in_use(total, decode_warps);
    auto warp_of = [&](long long t) { return line_warp(total, warps, t); };      // the warp that worked on tile t
    auto take_slots = [&](const float* base, long long from, int count, int cols, int col) {
        const long long size = state_floats(cols, D);
        const float* s = base + (from + g) * size;
#pragma unroll 4
        for (int i = g; i < count; i += kGroups, s += kGroups * size)
            take(s[col], s[cols + col], *reinterpret_cast<const float4*>(s + acc_offset(cols) + col * D + 4 * j));
    };
    if (prefix_total > 0) {
        const int row = b * p.group + hg;
        const long long seg = static_cast<long long>(kvh) * p.prefix_chunks + row / kPrefixCols;
        const long long t0 = seg * prefix_tiles, w0 = warp_of(t0);
        take_slots(p.prefix_states, seg + w0, static_cast<int>(warp_of(t0 + prefix_tiles - 1) - w0) + 1, kPrefixCols, row % kPrefixCols);
    }
    if (after > first) {
        const int n = after - first, head = kvh * p.head_chunks + hg / kOwnCols;
        const long long seg = static_cast<long long>(b) * heads + head;
        const long long t0 = prefix_total + static_cast<long long>(first) * heads + static_cast<long long>(head) * n, w0 = warp_of(t0);
        take_slots(p.own_states, seg + w0, static_cast<int>(warp_of(t0 + n - 1) - w0) + 1, p.own_cols, hg % kOwnCols);
    }
    if (p.block_splits > 0 && shared_keys > 0) {      // the prefix as the tensor-memory kernel left it
#pragma unroll 4
        for (int i = g; i < p.block_splits; i += kGroups) {
            const long long at = static_cast<long long>(i) * rows + out_row;
            const float2 ml = *reinterpret_cast<const float2*>(p.block_ml + 2 * at);
            take(ml.x, ml.y, *reinterpret_cast<const float4*>(p.block_acc + at * D + 4 * j));
        }
    }
    if constexpr (kGroups > 1) {
        s_acc[slot_row][g][j] = acc;
        if (j == 0) {
            s_m[slot_row][g] = m;
            s_l[slot_row][g] = l;
        }
        __syncthreads();
        if (g != 0) return;
        float top = kMInit;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) top = fmaxf(top, s_m[slot_row][i]);
        l = 0.0f;
        acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int i = 0; i < kGroups; ++i) {
            const float f = ex2f(s_m[slot_row][i] - top);
            const float4 a = s_acc[slot_row][i][j];
            l = fmaf(s_l[slot_row][i], f, l);
            acc.x = fmaf(a.x, f, acc.x);
            acc.y = fmaf(a.y, f, acc.y);
            acc.z = fmaf(a.z, f, acc.z);
            acc.w = fmaf(a.w, f, acc.w);
        }
    }
    uint2 w = make_uint2(0u, 0u);         // no key seen: zero
    if (l != 0.0f) {
        const float inv = 1.0f / l;
        w.x = pack_bf16x2(acc.x * inv, acc.y * inv);
        w.y = pack_bf16x2(acc.z * inv, acc.w * inv);
    }
    st_vec8(p.out + static_cast<long long>(out_row) * D + 4 * j, w);
}

template <int D>
int launch_decode(const DecodeArgs& a, cudaStream_t stream, const char* fn) {
    constexpr int kBase = Ring<D>::kTableOffset;
    const size_t need = static_cast<size_t>(kBase) + 4 * static_cast<size_t>(a.num_seqs + 1);
    (void)host::setup<&decode_kernel<D>, kDecThreads, static_cast<size_t>(kBase) + 4 * (kMaxSeqs + 1)>();
    const int ctas = decode_ctas();
    host::launch<decode_kernel<D>>(dim3(static_cast<unsigned>(ctas)), dim3(kDecThreads), need, stream, a);
    return host::check_launch(fn);
}

template <int D, int kRowThreads, int kThreads>
void launch_join_as(const DecodeArgs& a, int rows, cudaStream_t stream) {
    constexpr int kRows = kThreads / kRowThreads;
    host::launch<join_kernel<D, kRowThreads, kThreads>>(dim3(static_cast<unsigned>((rows + kRows - 1) / kRows)), dim3(kThreads), 0, stream, a,
                                                        decode_ctas() * kDecWarps);
}
template <int D>
int launch_join(const DecodeArgs& a, cudaStream_t stream, const char* fn) {
    const int rows = a.num_seqs * a.c.num_kv_heads * a.group;
    if (rows <= host::num_sms()) launch_join_as<D, 1024, 1024>(a, rows, stream);
    else if (rows <= 8 * host::num_sms()) launch_join_as<D, 256, 256>(a, rows, stream);
    else launch_join_as<D, D / 4, 256>(a, rows, stream);
    return host::check_launch(fn);
}

}  // namespace
}  // namespace paged
}  // namespace rh

using namespace rh;

extern "C" size_t rh_flash_decode_paged_scratch_floats(int num_seqs, int num_q_heads, int num_kv_heads, int head_dim) {
    if (num_seqs < 1 || num_q_heads < 1 || num_kv_heads < 1 || head_dim < 1 || num_q_heads % num_kv_heads != 0) return 0;
    return paged::decode_scratch(num_seqs, num_q_heads, num_kv_heads, head_dim).floats;
}

extern "C" int rh_flash_decode_paged_bf16(void* out, const void* q, long long q_stride, const rh_kv_pages* cache, int layer, const int* rows_or_null,
                                          int num_seqs, int num_q_heads, float scale, float* partial, const int* shared_pages_or_null,
                                          const int* shared_len_or_null, void* stream) {
    const char* const fn = "rh_flash_decode_paged_bf16";
    paged::DecodeArgs a = {};
    if (const int e = host::paged_layer(cache, layer, fn, &a.c)) return e;
    RH_REQUIRE(out && q && partial, RH_ERR_INVALID_ARG, "%s: null pointer", fn);
    RH_REQUIRE((shared_pages_or_null == nullptr) == (shared_len_or_null == nullptr), RH_ERR_INVALID_ARG,
               "%s: shared_pages and shared_len go together", fn);
    RH_REQUIRE(num_seqs >= 1 && num_seqs <= paged::kMaxSeqs, RH_ERR_INVALID_ARG, "%s: num_seqs must be in 1..%d", fn, paged::kMaxSeqs);
    RH_REQUIRE(rows_or_null != nullptr || num_seqs <= cache->num_rows, RH_ERR_INVALID_ARG, "%s: more sequences than table rows", fn);
    RH_REQUIRE(static_cast<long long>(num_seqs) * cache->pages_per_row * (cache->page_size / paged::kTile) <= INT_MAX, RH_ERR_UNSUPPORTED_DIM,
               "%s: num_seqs * pages_per_row * page_size must stay below 2^35", fn);
    RH_REQUIRE(num_q_heads >= 1 && num_q_heads % cache->num_kv_heads == 0, RH_ERR_INVALID_ARG, "%s: num_q_heads must be a multiple of num_kv_heads", fn);
    RH_REQUIRE(num_q_heads <= 1024, RH_ERR_UNSUPPORTED_DIM, "%s: at most 1024 query heads", fn);
    RH_REQUIRE(std::isfinite(scale * paged::kLog2e), RH_ERR_INVALID_ARG, "%s: scale must be finite (and so must scale * log2 e)", fn);
    RH_REQUIRE(q_stride >= static_cast<long long>(num_q_heads) * cache->head_dim, RH_ERR_INVALID_ARG, "%s: q_stride is below num_q_heads * head_dim", fn);
    RH_REQUIRE(host::aligned16(q) && q_stride % 8 == 0 && host::aligned16(partial), RH_ERR_MISALIGNED,
               "%s: q and partial must be 16-byte aligned, q_stride a multiple of 8", fn);
    RH_REQUIRE((reinterpret_cast<uintptr_t>(out) & 7u) == 0, RH_ERR_MISALIGNED, "%s: out must be 8-byte aligned", fn);
    a.out = static_cast<__nv_bfloat16*>(out);
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.q_stride = q_stride;
    a.rows = rows_or_null;
    // one sequence has nobody to share with: its prefix is its own
    a.shared_pages = num_seqs > 1 ? shared_pages_or_null : nullptr;
    a.shared_len = num_seqs > 1 ? shared_len_or_null : nullptr;
    a.num_seqs = num_seqs;
    a.group = num_q_heads / cache->num_kv_heads;
    a.head_chunks = (a.group + paged::kOwnCols - 1) / paged::kOwnCols;
    a.own_cols = a.group < paged::kOwnCols ? a.group : paged::kOwnCols;
    a.scale_log2e = scale * paged::kLog2e;
    a.error_word = host::device_error_word();
    const paged::DecodeScratch parts = paged::decode_scratch(num_seqs, num_q_heads, cache->num_kv_heads, cache->head_dim);
    a.header = reinterpret_cast<int*>(partial);
    a.own_states = partial + parts.own;
    a.prefix_states = partial + parts.prefix;
    a.block_ml = partial + parts.block_ml;
    a.block_acc = partial + parts.block_acc;
    if (a.shared_pages != nullptr) {
        if (num_seqs * a.group < paged::kBlockRows) a.prefix_chunks = (num_seqs * a.group + paged::kPrefixCols - 1) / paged::kPrefixCols;
        else a.block_splits = paged::prefix_splits(num_seqs, cache->num_kv_heads, a.group);
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (const int e = cache->head_dim == 128 ? paged::launch_decode<128>(a, s, fn) : paged::launch_decode<64>(a, s, fn)) return e;
    if (a.block_splits > 0)
        if (const int e = paged::launch_prefix(a, cache->head_dim, s, fn)) return e;
    return cache->head_dim == 128 ? paged::launch_join<128>(a, s, fn) : paged::launch_join<64>(a, s, fn);
}

extern "C" int rh_selfcheck_decode_line(long long tiles, long long warps, long long tile, long long* warp_host, long long* first_host) {
    const char* const fn = "rh_selfcheck_decode_line";
    RH_REQUIRE(warp_host && first_host, RH_ERR_INVALID_ARG, "%s: null pointer", fn);
    RH_REQUIRE(tiles >= 1 && tiles <= (1LL << 42) && warps >= 1 && warps <= (1 << 16) && tile >= 0 && tile < tiles, RH_ERR_INVALID_ARG,
               "%s: tiles must be in 1..2^42, warps in 1..2^16, tile in 0..tiles - 1", fn);
    *warp_host = paged::line_warp(tiles, warps, tile);
    *first_host = paged::line_start(tiles, warps, *warp_host);
    return RH_OK;
}
