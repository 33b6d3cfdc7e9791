// Launchers of the token log probabilities over fp32 logits, for the model handle (logprobs.cu;
// gpt2q.h gpt2q_logprobs states the definitions). Device pointers; temperature 1.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace gpt2q {

cudaError_t launch_logprobs(const float* logits, int ld, int rows, int vocab, const int32_t* targets, int top, float* lp,
                            float* entropy, float* stats, int32_t* top_ids, float* top_lp, cudaStream_t st);
// in place: the logits become their gradient; targets / d_lp or d_ent may be null
cudaError_t launch_logprobs_grad(float* logits, int ld, int rows, int vocab, const int32_t* targets, const float* stats,
                                 const float* d_lp, const float* d_ent, cudaStream_t st);

}  // namespace gpt2q
