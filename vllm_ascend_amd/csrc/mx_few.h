// The MXFP4 experts of a few tokens in two launches (mx_few.hip)
#pragma once

#include "gmm_mx.h"

namespace moe355 {

struct MxFew {
    const void* x;           // [tokens, K] of the dtype, or codes [tokens, K / 2]
    const uint8_t* x_scale;  // of codes
    bool quantised;
    const int32_t* ids;      // [tokens, top_k]; one outside [0, E) counts for nothing
    const uint16_t* probs;
    const uint16_t* residual;
    int top_k;
    int64_t* expert_tokens;
};
bool mx_few_takes(int64_t tokens, int top_k, int64_t hidden, int64_t intermediate, int num_experts);
// up: to hidden rows in the order of the pairs, which down reads; down.out: the result [tokens, N]
int mx_few(const MxArgs& up, const MxArgs& down, const MxFew& f, int dtype, int64_t tokens, hipStream_t st);

}  // namespace moe355
