// logprobs.cuh — log probabilities of given tokens, entropy and top alternatives.
#pragma once

#include "common.cuh"

namespace sg {

struct LogprobsArgs {
    const void *logits;
    uint64_t ld;  // elements between rows
    uint32_t rows, vocab, top;
    const int32_t *tokens;
    float *logprob, *entropy;
    int32_t *rank, *top_ids;
    float *top_logprobs;
};

constexpr uint32_t LP_TOP_MAX = SG_LOGPROBS_TOP_MAX;

sg_status logprobs_launch(const LogprobsArgs &a, int32_t type, int sms, cudaStream_t s, cudaError_t *err);

}  // namespace sg
