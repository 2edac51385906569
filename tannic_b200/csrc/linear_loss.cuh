// The cross entropy of a linear layer for a few tokens: interface between the dispatcher (linear_loss.cu), the streaming
// kernels (linear_loss_few.cu), the gradient of a few tokens of 16 bits (linear_loss_half.cu) and the float32 tiles (linear_loss_f32.cu).
#pragma once

#include "common.cuh"

namespace tnb {

// Two elements as one packed instruction each, rounded like the single ones.
__device__ __forceinline__ uint64_t pair_bits(float2 v) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ float2 pair_of(uint64_t r) {
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(x)), "l"(pair_bits(y)));
    return pair_of(r);
}
__device__ __forceinline__ float2 mul2(float2 x, float2 y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(x)), "l"(pair_bits(y)));
    return pair_of(r);
}
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair_bits(x)), "l"(pair_bits(y)), "l"(pair_bits(z)));
    return pair_of(r);
}

struct FewTokens {
    int dtype = 0;                         // TN_FLOAT16, TN_BFLOAT16 or TN_FLOAT32
    int64_t tokens = 0, hidden = 0, vocab = 0;
    int sms = 1;                           // that the persistent kernels may use
    const void* h = nullptr;               // [tokens, hidden], rows h_pitch elements apart
    int64_t h_pitch = 0;
    const void* w = nullptr;               // [vocab, hidden], rows w_pitch elements apart
    int64_t w_pitch = 0;
    const void* targets = nullptr;         // int64 (wide) or int32
    int wide = 0;
    int64_t ignore = 0;
    // loss: maximum and sum of exponentials of every group of logits, [groups][tokens], and the targets' logits
    float2* parts = nullptr;               // (few_loss: few_loss_parts() groups, f32_loss: f32_loss_parts())
    float* target_logit = nullptr;
    // gradient
    const float* grad = nullptr;
    const float* lse = nullptr;
    float* sums = nullptr;                 // [blocks or shares][tokens][hidden], null where no dhidden is wanted
    void* dhidden = nullptr;
    void* dweight = nullptr;               // dense, may be null
};

bool few_loss_fits(int dtype, int64_t tokens, int64_t hidden);
int64_t few_loss_parts(const FewTokens& p);
tn_status few_loss(const FewTokens& p, cudaStream_t stream);

// d is scaled by kTop over the largest |grad|, and what is formed from it scaled back.
constexpr float kTop = 16384.0f;  // float16 ends at 65504
__device__ __forceinline__ float unscale(float v, float largest) { return v * (1.0f / kTop) * largest; }

// 16 bits, up to sixteen tokens
bool half_grad_fits(const FewTokens& p);
int64_t half_grad_blocks(const FewTokens& p);
tn_status half_grad(const FewTokens& p, cudaStream_t stream);

// float32, up to four tokens
bool few_grad_fits(const FewTokens& p);
int64_t few_grad_blocks(const FewTokens& p);
tn_status few_grad(const FewTokens& p, cudaStream_t stream);
// dhidden from `n` blocks' sums
tn_status few_dhidden(const FewTokens& p, int64_t n, cudaStream_t stream);

// float32, up to 64 tokens (gradient: 32). `h`: workspace of f32_row_floats, `d`: of f32_d_floats.
bool f32_fits(int dtype, int64_t tokens, int64_t hidden, bool gradient);
int64_t f32_loss_parts(int64_t tokens, int64_t vocab);
size_t f32_row_floats(int64_t tokens, int64_t hidden);
size_t f32_d_floats(int64_t tokens, int64_t vocab);
int64_t f32_grad_shares(int64_t hidden, int64_t vocab);
tn_status f32_loss(const FewTokens& p, float* h, cudaStream_t stream);
tn_status f32_grad(const FewTokens& p, float* h, float* d, cudaStream_t stream);

}  // namespace tnb
