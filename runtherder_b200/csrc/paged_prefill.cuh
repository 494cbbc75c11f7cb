// Launchers of the tensor-memory attention kernel on the paged cache (paged_prefill.cu).
#pragma once
#include "paged_attention.cuh"

namespace rh {
namespace paged {

// Prefix part of a decode step: all query rows over the shared keys, dealt to a.block_splits key ranges whose states
// go to a.block_ml / a.block_acc.
int launch_prefix(const DecodeArgs& a, int head_dim, cudaStream_t stream, const char* fn);
// Key ranges that launch_prefix should be given for this batch on this device.
int prefix_splits(int num_seqs, int num_kv_heads, int group);

}  // namespace paged
}  // namespace rh
