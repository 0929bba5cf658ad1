// Log probabilities of given tokens from logits (logprobs.cu): linked into libwf_bitnet.so and libwf_seq.so.
#pragma once
#include "common.cuh"

namespace wf {

constexpr int LP_TOP_MAX = 64;     // alternatives a row

// logits [n, V] of dtype 0 f32, 1 bf16, 2 f16, rows ld elements apart; tokens [n]; logprob, entropy [n]; top_logprob, top_id [n, k] (null for k = 0)
int launch_token_logprobs(const void* logits, int dtype, int n, int V, long long ld, const int32_t* tokens, int k, float temperature, float* logprob, float* entropy,
                          float* top_logprob, int32_t* top_id, cudaStream_t s);

}  // namespace wf
