// logprobs.cuh — log probabilities of tokens, entropy, top alternatives.
#pragma once

#include "brew_common.cuh"

namespace brew {

struct LogprobsParams {
    const float* logits;   // [rows][ld]
    int64_t ld;
    int vocab, rows;
    const int32_t* tokens;
    float *logprob, *entropy;
    int top;               // <= BREW_MAX_TOP
    int32_t* top_ids;      // [rows][top]
    float* top_logprobs;
};

int logprobs_launch(const LogprobsParams& p, cudaStream_t s);

}  // namespace brew
