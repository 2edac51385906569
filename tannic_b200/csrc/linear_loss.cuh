// The cross entropy of a linear layer for a few tokens: interface between the dispatcher (linear_loss.cu) and the streaming
// kernels (linear_loss_few.cu).
#pragma once

#include "common.cuh"

namespace tnb {

struct FewTokens {
    int dtype = 0;                         // TN_FLOAT16, TN_BFLOAT16 or TN_FLOAT32
    int64_t tokens = 0, hidden = 0, vocab = 0;
    const void* h = nullptr;               // [tokens, hidden], rows h_pitch elements apart
    int64_t h_pitch = 0;
    const void* w = nullptr;               // [vocab, hidden], rows w_pitch elements apart
    int64_t w_pitch = 0;
    const void* targets = nullptr;         // int64 (wide) or int32
    int wide = 0;
    int64_t ignore = 0;
    // loss: maximum and sum of exponentials of every group of logits, [few_loss_parts][tokens], and the targets' logits
    float2* parts = nullptr;
    float* target_logit = nullptr;
    // gradient
    const float* grad = nullptr;
    const float* lse = nullptr;
    float* sums = nullptr;                 // [few_grad_blocks][tokens][hidden], may be null (no dhidden wanted)
    void* dhidden = nullptr;
    void* dweight = nullptr;               // dense, may be null
};

bool few_loss_fits(int64_t tokens, int64_t hidden);
int64_t few_loss_parts();
tn_status few_loss(const FewTokens& p, cudaStream_t stream);

bool few_grad_fits(int64_t tokens, int64_t hidden);
int64_t few_grad_blocks(int64_t vocab);
tn_status few_grad(const FewTokens& p, cudaStream_t stream);

}  // namespace tnb
