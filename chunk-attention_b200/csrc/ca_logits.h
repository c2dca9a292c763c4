// Log probabilities from logits (ca_logits.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ca {

struct LogProbsParams {
    const void* logits;      // [n_rows, vocab]
    int64_t row_stride;
    int n_rows, vocab, splits;
    const int32_t* tokens;   // [n_tokens]
    const int32_t* rows;     // null: token i belongs to row i
    int n_tokens, top;
    float* log_probs;
    float* entropy;
    float* top_log_probs;    // [n_rows, top]
    int32_t* top_ids;
    float2* lse;             // [n_rows]: maximum, log of the sum relative to it
};
int log_probs_splits(int n_rows, int vocab);  // CTAs of a row (a cluster)
cudaError_t launch_log_probs(const LogProbsParams& p, int dtype, cudaStream_t stream);

}  // namespace ca
