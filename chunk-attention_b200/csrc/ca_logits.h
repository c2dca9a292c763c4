// Log probabilities from logits (ca_logits.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace ca {

constexpr int LOG_PROBS_HITS = 512;
struct LogProbsPart {  // what a stretch of a row gives
    float m, l, a;     // reference (log2 units), sum, sum of y 2^y
    float limit;       // threshold of the best
    int n_hits;        // notes of vectors that reached it
};
struct LogProbsParams {
    const void* logits;      // [n_rows, vocab]
    int64_t row_stride;
    int n_rows, vocab;
    int splits;              // CTAs of a row's cluster; 0: stretches
    int turns;               // of a row, when stretches are handed out: `each` turns to a CTA, one more to the first `more`
    int64_t each;
    int more;
    const int32_t* tokens;   // [n_tokens]
    const int32_t* rows;     // null: token i belongs to row i
    int n_tokens, top;
    float* log_probs;
    float* entropy;
    float* top_log_probs;    // [n_rows, top]
    int32_t* top_ids;
    LogProbsPart* parts;     // [n_rows + log_probs_ctas()], when stretches are handed out
    uint32_t* hits;          // [n_rows + log_probs_ctas()][hits_room]: their notes, where the best are asked for
    int hits_room;
    double2* lse;            // [n_rows]: a reference, log of the sum relative to it
    bool tokens_here;        // the rows' CTAs look the tokens up, else a kernel behind them does
#if defined(__CUDACC__)
    __device__ __forceinline__ int64_t begin(int b) const { return b * each + min(b, more); }
    __device__ __forceinline__ int owner(int64_t turn) const {
        const int64_t big = more * (each + 1);
        return turn < big ? (int)(turn / (each + 1)) : more + (int)((turn - big) / each);
    }
#endif
};
int log_probs_splits(int n_rows, int vocab, int esize);
int log_probs_ctas();        // that share all rows
int log_probs_hits_room(int vocab, int esize);
void log_probs_shape(LogProbsParams& p, int esize);  // splits and turns, from n_rows and vocab
cudaError_t read_log_probs_status(int* status, cudaStream_t stream);  // 0, or STATUS_* of the first wait that ran out
cudaError_t launch_log_probs(const LogProbsParams& p, int dtype, cudaStream_t stream);

}  // namespace ca
