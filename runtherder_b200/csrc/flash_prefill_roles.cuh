// Helpers of the prefill kernels whose warps take roles: the bounded wait that one thread's giving up ends for the
// whole CTA, a barrier with a vote, and the order in which K rows become operand rows.
#pragma once
#include "flash_prefill_tc.cuh"

namespace rh {
namespace ws {

constexpr int kTries = 1 << 20;
constexpr int kLazyNs = 100;      // pause between polls of the product and conversion warps

// Bounded wait that also ends when another thread of the CTA has given up.  kBackoffNs > 0 sleeps between
// tries: for the roles whose reaction time is not on the critical path (a poll is a shared-memory access and
// an issue slot taken from the softmax warps).
template <int kBackoffNs = 0>
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, volatile int* gave_up, int where, int* error_word,
                                           int tries = kTries, int* tries_used = nullptr) {
    const uint32_t addr = pipe::smem_u32(bar);
    for (int i = 0; i < tries; ++i) {       // a try blocks for a while in hardware before it reports failure
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(addr), "r"(parity)
            : "memory");
        if (ok != 0) return true;
        if ((i & 15) == 15 && *gave_up != 0) {                 // looked at now and then: a poll is a shared-memory access
            if (tries_used != nullptr) *tries_used = i + 1;
            return false;
        }
        if constexpr (kBackoffNs > 0) __nanosleep(kBackoffNs);
    }
    *gave_up = 1;
    if (error_word != nullptr) atomicCAS(error_word, 0, (where << 8) | 1);
    if (tries_used != nullptr) *tries_used = tries;
    return false;
}

// Barrier among the `count` threads that use named barrier `id`, returning the OR of their predicates.
__device__ __forceinline__ bool group_or(int id, int count, bool pred) {
    uint32_t out;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %3, 0;\n\t"
        "bar.red.or.pred p, %1, %2, q;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(out)
        : "r"(id), "r"(count), "r"(static_cast<uint32_t>(pred))
        : "memory");
    return out != 0;
}

// the key whose K row becomes row r of the K operand tile (S column 16a + 8h + 2c + e holds key 16a + 4c + 2h + e)
__device__ __forceinline__ int key_of_k_row(int r) { return (r & 48) | ((r & 6) << 1) | ((r & 8) >> 2) | (r & 1); }

}  // namespace ws
}  // namespace rh
