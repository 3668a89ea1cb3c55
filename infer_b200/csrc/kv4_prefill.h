// Launch of the many-row attention kernel (kv4_prefill.cu).
#pragma once

#include "kv4_attention.cuh"

namespace fth {
namespace kv4 {

int PrefillGrid();                          // blocks of threads; two arrival counters each
int64_t PrefillPartialFloats(int head_dim); // room for partial results
int LaunchPrefill(const AttentionParams& p, int head_dim, int dtype, cudaStream_t s);

}  // namespace kv4
}  // namespace fth
