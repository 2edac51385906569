// The cross entropy of a linear layer and its gradient for up to 64 tokens of float32, on the FP32 pipe.
//
// The tensor cores take float32 as three bfloat16 parts: W would be read (4 bytes an element), written as parts (6) and read again (6, for
// each product), and a tile of 128 rows would be mostly empty. With N tokens the products are 2 N operations per element of W and pass, so
// up to about 64 of them the FP32 pipe keeps up with what the parts would cost (32 tokens, 4096 x 32768: loss 596 us with parts).
// All three products are tiles in shared memory, filled by cp.async several steps ahead; two neighbouring elements go through one
// packed multiply-add. What a thread reads from shared memory has to serve many of them: in the first two a thread holds 16 tokens
// and all lanes of a warp the same ones, so that a token's values are one broadcast for the warp (with 1 x 8 sums a thread, neighbouring
// lanes on neighbouring tokens, shared memory was the bound and 16 tokens over 4096 x 32768 took 330 us).
//
//   logits  [tokens] x [128 or 256 vocabulary rows], K = hidden. Epilogue: maximum and sum of exponentials per token and warp, or d.
//   dh      [tokens] x [256 columns], K = a share of the vocabulary; the shares' sums are added in order afterwards.
//   dW      [128 vocabulary rows] x [128 columns], K = tokens: bound by writing dW.
#include <algorithm>

#include "linear_loss.cuh"

namespace tnb {
namespace {

constexpr int kThreads = 256;
constexpr int kCols = 128;       // of a tile of dW
constexpr int kTokens = 16;      // of a thread
constexpr int kStep = 32;        // of K
constexpr int kPitch = kStep + 4;   // floats of a tile's row along K: 16-byte aligned, eight neighbouring rows in different banks
constexpr int kWide = kCols + 4;    // floats of a tile's row along the columns
constexpr int kStages = 4;

__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
    uint64_t a, b, c, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(x.x), "f"(x.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(y.x), "f"(y.y));
    asm("mov.b64 %0, {%1, %2};" : "=l"(c) : "f"(z.x), "f"(z.y));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}

__device__ __forceinline__ int64_t target_of(const FewTokens& p, int64_t n) {
    return p.wide ? static_cast<const int64_t*>(p.targets)[n] : static_cast<int64_t>(static_cast<const int32_t*>(p.targets)[n]);
}

// Four floats into shared memory, of which the first `valid` are read and the others are zero. ALIGNED: one 16-byte copy.
template <bool ALIGNED>
__device__ __forceinline__ void copy4(float* to, const float* from, int valid) {
    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    valid = max(0, min(4, valid));
    if constexpr (ALIGNED) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(4 * valid) : "memory");
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * j), "l"(j < valid ? from + j : from), "r"(j < valid ? 4 : 0) : "memory");
    }
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until the oldest of kStages - 1 groups has arrived
__device__ __forceinline__ void wait_oldest() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory"); }

// The tokens as the products read them: [rows][padded], zero where there is no token, no target (that is for the gradient) or no column.
__global__ void __launch_bounds__(256) few_rows_kernel(const FewTokens p, int rows, int64_t padded, int drop_ignored, float* __restrict__ out) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows * padded; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t n = i / padded, c = i - n * padded;
        const bool in = n < p.tokens && c < p.hidden && !(drop_ignored && target_of(p, n) == p.ignore);
        out[i] = in ? static_cast<const float*>(p.h)[n * p.h_pitch + c] : 0.0f;
    }
}

// Lane i ends up with the sum (or maximum) of value i >> 1 over all lanes.
template <bool MAX>
__device__ __forceinline__ float lane_reduce(float (&v)[kTokens], int lane) {
    auto two = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
    int o = 16;
#pragma unroll
    for (int n = kTokens / 2; n >= 1; n /= 2, o /= 2) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const bool up = lane & o;
            const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
            v[i] = two(keep, __shfl_xor_sync(0xFFFFFFFFu, give, o));
        }
    }
    return two(v[0], __shfl_xor_sync(0xFFFFFFFFu, v[0], 1));
}

// TM: tokens of the tile (16, 32 or 64), sixteen to a group of warps; a warp has WIDTH vocabulary rows a lane, 32 apart.
template <int TM> constexpr int kGroupWarps = 8 / (TM / kTokens);
template <int TM> constexpr int kWidth = TM == 16 ? 1 : 2;
template <int TM> constexpr int kLogitCols = kGroupWarps<TM> * 32 * kWidth<TM>;

// h: [TM][padded]. D: write d into `d` ([TM][d_pitch]), else the warps' statistics.
template <int TM, bool ALIGNED, bool D>
__global__ void __launch_bounds__(kThreads) logits_kernel(const FewTokens p, const float* __restrict__ h, int64_t padded, float* __restrict__ d, int64_t d_pitch) {
    constexpr int COLS = kLogitCols<TM>, W = kWidth<TM>;
    extern __shared__ __align__(16) float smem[];  // [kStages][(TM + COLS)][kPitch]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n0 = warp / kGroupWarps<TM> * kTokens, part = warp % kGroupWarps<TM>;
    const int64_t v0 = static_cast<int64_t>(blockIdx.x) * COLS;
    const int steps = static_cast<int>((p.hidden + kStep - 1) / kStep);
    auto fill = [&](int step) {
        if (step < steps) {
            float* a = smem + (step % kStages) * (TM + COLS) * kPitch;
            float* b = a + TM * kPitch;
            const int64_t k0 = static_cast<int64_t>(step) * kStep;
            for (int i = threadIdx.x; i < TM * (kStep / 4); i += kThreads) {
                const int r = i / (kStep / 4), c = i % (kStep / 4) * 4;
                const int valid = static_cast<int>(min(int64_t(4), padded - k0 - c));
                copy4<true>(a + r * kPitch + c, h + r * padded + (valid > 0 ? k0 + c : 0), valid);
            }
#pragma unroll
            for (int i = threadIdx.x; i < COLS * (kStep / 4); i += kThreads) {
                const int r = i / (kStep / 4), c = i % (kStep / 4) * 4;
                const int valid = v0 + r < p.vocab ? static_cast<int>(min(int64_t(4), p.hidden - k0 - c)) : 0;
                copy4<ALIGNED>(b + r * kPitch + c, static_cast<const float*>(p.w) + (valid > 0 ? (v0 + r) * p.w_pitch + k0 + c : 0), valid);
            }
        }
        commit();
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) fill(s);
    float2 acc[kTokens][W];  // even and odd elements of K
#pragma unroll
    for (int i = 0; i < kTokens; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) acc[i][j] = make_float2(0.0f, 0.0f);
    for (int step = 0; step < steps; ++step) {
        wait_oldest();
        __syncthreads();  // this step's tile is there for everyone, and the last step's is read
        fill(step + kStages - 1);
        const float* a = smem + (step % kStages) * (TM + COLS) * kPitch;
        const float* b = a + TM * kPitch + (part * 32 * W + lane) * kPitch;
        a += n0 * kPitch;
#pragma unroll
        for (int k = 0; k < kStep; k += 4) {
            float4 y[W];
#pragma unroll
            for (int j = 0; j < W; ++j) y[j] = *reinterpret_cast<const float4*>(b + 32 * j * kPitch + k);
#pragma unroll
            for (int i = 0; i < kTokens; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(a + i * kPitch + k);
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    acc[i][j] = fma2(make_float2(x.x, x.y), make_float2(y[j].x, y[j].y), acc[i][j]);
                    acc[i][j] = fma2(make_float2(x.z, x.w), make_float2(y[j].z, y[j].w), acc[i][j]);
                }
            }
        }
    }
    const int64_t v = v0 + part * 32 * W + lane;  // and 32 further
    if constexpr (D) {
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const int n = n0 + i;
            const int64_t target = n < p.tokens ? target_of(p, n) : -1;
            const bool counts = n < p.tokens && target != p.ignore;
            const float lse = counts ? p.lse[n] : 0.0f;
            const float grad = !counts ? 0.0f : target < 0 || target >= p.vocab ? NAN : p.grad[n];
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float x = acc[i][j].x + acc[i][j].y - lse;
                if (v + 32 * j < d_pitch) d[n * d_pitch + v + 32 * j] = counts && v + 32 * j < p.vocab ? (v + 32 * j == target ? expm1f(x) : __expf(x)) * grad : 0.0f;
            }
        }
    } else {
        float top[kTokens], sum[kTokens];
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const int n = n0 + i;
            const int64_t target = n < p.tokens ? target_of(p, n) : -1;
            top[i] = -INFINITY;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const bool in = v + 32 * j < p.vocab;
                acc[i][j].x = in ? acc[i][j].x + acc[i][j].y : -INFINITY;
                top[i] = fmaxf(top[i], acc[i][j].x);
                if (in && v + 32 * j == target) p.target_logit[n] = acc[i][j].x;
            }
        }
        const float m = lane_reduce<true>(top, lane);  // of token lane / 2
#pragma unroll
        for (int i = 0; i < kTokens; ++i) {
            const float mi = __shfl_sync(0xFFFFFFFFu, m, 2 * i), base = mi == -INFINITY ? 0.0f : mi;
            sum[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < W; ++j) sum[i] += __expf(acc[i][j].x - base);
        }
        const float s = lane_reduce<false>(sum, lane);
        const int n = n0 + (lane >> 1);
        if ((lane & 1) == 0 && n < p.tokens) p.parts[(static_cast<int64_t>(blockIdx.x) * kGroupWarps<TM> + part) * p.tokens + n] = make_float2(m, s);
    }
}

// dh's sums over the vocabulary rows [blockIdx.y * share, + share): sixteen tokens and 4 columns a thread, 256 columns a block. With fewer than 64
// tokens the warps that are left share K (kShares of them), each with sums of its own.
constexpr int kHiddenCols = 256, kHiddenWide = kHiddenCols + 4, kHiddenStages = 3;
template <int TM> constexpr int kShares = 4 / (TM / kTokens);

template <int TM, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) dhidden_kernel(const FewTokens p, const float* __restrict__ d, int64_t d_pitch, int64_t share) {
    extern __shared__ __align__(16) float smem[];  // [kHiddenStages] of [TM][kPitch] and [kStep][kHiddenWide]
    constexpr int TILE = TM * kPitch + kStep * kHiddenWide, S = kShares<TM>, MINE = kStep / S;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int half = warp & 1, turn = (warp >> 1) % S, n0 = (warp >> 1) / S * kTokens;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kHiddenCols, first = blockIdx.y * share, last = min(p.vocab, first + share);
    const int steps = last > first ? static_cast<int>((last - first + kStep - 1) / kStep) : 0;
    auto fill = [&](int step) {
        if (step < steps) {
            float* a = smem + (step % kHiddenStages) * TILE;
            float* b = a + TM * kPitch;
            const int64_t k0 = first + static_cast<int64_t>(step) * kStep;
            for (int i = threadIdx.x; i < TM * (kStep / 4); i += kThreads) {
                const int r = i / (kStep / 4), c = i % (kStep / 4) * 4;
                const int valid = static_cast<int>(min(int64_t(4), last - k0 - c));
                copy4<true>(a + r * kPitch + c, d + r * d_pitch + (valid > 0 ? k0 + c : 0), valid);
            }
#pragma unroll
            for (int i = threadIdx.x; i < kStep * (kHiddenCols / 4); i += kThreads) {
                const int r = i / (kHiddenCols / 4), c = i % (kHiddenCols / 4) * 4;
                const int valid = k0 + r < last ? static_cast<int>(min(int64_t(4), p.hidden - c0 - c)) : 0;
                copy4<ALIGNED>(b + r * kHiddenWide + c, static_cast<const float*>(p.w) + (valid > 0 ? (k0 + r) * p.w_pitch + c0 + c : 0), valid);
            }
        }
        commit();
    };
#pragma unroll
    for (int s = 0; s < kHiddenStages - 1; ++s) fill(s);
    float2 acc[kTokens][2];
#pragma unroll
    for (int i = 0; i < kTokens; ++i) acc[i][0] = acc[i][1] = make_float2(0.0f, 0.0f);
    for (int step = 0; step < steps; ++step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kHiddenStages - 2) : "memory");
        __syncthreads();
        fill(step + kHiddenStages - 1);
        const float* a = smem + (step % kHiddenStages) * TILE + n0 * kPitch + turn * MINE;
        const float* b = smem + (step % kHiddenStages) * TILE + TM * kPitch + turn * MINE * kHiddenWide + half * 128 + 4 * lane;
#pragma unroll 2
        for (int k = 0; k < MINE; k += 4) {
            float4 y[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) y[q] = *reinterpret_cast<const float4*>(b + (k + q) * kHiddenWide);
#pragma unroll
            for (int i = 0; i < kTokens; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(a + i * kPitch + k);
                const float s[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    acc[i][0] = fma2(make_float2(s[q], s[q]), make_float2(y[q].x, y[q].y), acc[i][0]);
                    acc[i][1] = fma2(make_float2(s[q], s[q]), make_float2(y[q].z, y[q].w), acc[i][1]);
                }
            }
        }
    }
    const int64_t c = c0 + half * 128 + 4 * lane;
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
        const int64_t n = n0 + i;
        if (n < p.tokens) {
            float* to = p.sums + ((blockIdx.y * S + turn) * p.tokens + n) * p.hidden + c;
            if (c < p.hidden) to[0] = acc[i][0].x;
            if (c + 1 < p.hidden) to[1] = acc[i][0].y;
            if (c + 2 < p.hidden) to[2] = acc[i][1].x;
            if (c + 3 < p.hidden) to[3] = acc[i][1].y;
        }
    }
}

// dW: a tile of 128 x 128, K = the tokens, all of them in shared memory at once.
template <int TM, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) dweight_kernel(const FewTokens p, const float* __restrict__ h, int64_t padded, const float* __restrict__ d, int64_t d_pitch) {
    extern __shared__ __align__(16) float smem[];  // [TM][kWide] of d and of h
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kCols;
    float* a = smem;
    float* b = smem + TM * kWide;
    for (int i = threadIdx.x; i < TM * (kCols / 4); i += kThreads) {
        const int r = i / (kCols / 4), c = i % (kCols / 4) * 4;
        const int valid = static_cast<int>(min(int64_t(4), padded - c0 - c));
        copy4<true>(b + r * kWide + c, h + r * padded + (valid > 0 ? c0 + c : 0), valid);
    }
    // the columns of h stay, the rows of d come by
    for (int64_t v0 = static_cast<int64_t>(blockIdx.y) * kCols; v0 < p.vocab; v0 += static_cast<int64_t>(gridDim.y) * kCols) {
        __syncthreads();  // the last rows of d are read
        for (int i = threadIdx.x; i < TM * (kCols / 4); i += kThreads) {
            const int r = i / (kCols / 4), c = i % (kCols / 4) * 4;
            const int valid = static_cast<int>(min(int64_t(4), d_pitch - v0 - c));
            copy4<true>(a + r * kWide + c, d + r * d_pitch + (valid > 0 ? v0 + c : 0), valid);
        }
        commit();
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        float2 acc[8][4];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = make_float2(0.0f, 0.0f);
#pragma unroll 4
        for (int k = 0; k < TM; ++k) {
            const float4 x0 = *reinterpret_cast<const float4*>(a + k * kWide + 4 * ty), x1 = *reinterpret_cast<const float4*>(a + k * kWide + 4 * ty + 64);
            const float4 y0 = *reinterpret_cast<const float4*>(b + k * kWide + 4 * tx), y1 = *reinterpret_cast<const float4*>(b + k * kWide + 4 * tx + 64);
            const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 both = make_float2(x[i], x[i]);
                acc[i][0] = fma2(both, make_float2(y0.x, y0.y), acc[i][0]);
                acc[i][1] = fma2(both, make_float2(y0.z, y0.w), acc[i][1]);
                acc[i][2] = fma2(both, make_float2(y1.x, y1.y), acc[i][2]);
                acc[i][3] = fma2(both, make_float2(y1.z, y1.w), acc[i][3]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t v = v0 + 4 * ty + 64 * (i / 4) + i % 4;
            if (v < p.vocab) {
                float* to = static_cast<float*>(p.dweight) + v * p.hidden;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int64_t c = c0 + 4 * tx + 64 * q;
                    const float4 out = make_float4(acc[i][2 * q].x, acc[i][2 * q].y, acc[i][2 * q + 1].x, acc[i][2 * q + 1].y);
                    if (ALIGNED) {
                        if (c < p.hidden) *reinterpret_cast<float4*>(to + c) = out;
                    } else {
                        if (c < p.hidden) to[c] = out.x;
                        if (c + 1 < p.hidden) to[c + 1] = out.y;
                        if (c + 2 < p.hidden) to[c + 2] = out.z;
                        if (c + 3 < p.hidden) to[c + 3] = out.w;
                    }
                }
            }
        }
    }
}

// ------------------------------------------------------------------ host ---------------
int token_rows(int64_t tokens) { return tokens <= 16 ? 16 : tokens <= 32 ? 32 : 64; }
int64_t padded_of(int64_t n) { return (n + 3) & ~int64_t(3); }
bool aligned(const FewTokens& p) {
    return p.hidden % 4 == 0 && p.w_pitch % 4 == 0 && ((reinterpret_cast<uintptr_t>(p.w) | reinterpret_cast<uintptr_t>(p.dweight)) & 15) == 0;
}

// Vocabulary rows of a block of dh: about two blocks to every SM, each with at least eight steps.
int64_t vocabulary_share(int64_t hidden, int64_t vocab) {
    const int64_t blocks = std::max<int64_t>(1, std::min((int64_t)sm_count() * 2 / ceil_div(hidden, kHiddenCols), vocab / (8 * kStep)));
    return ceil_div(ceil_div(vocab, blocks), kStep) * kStep;
}

template <typename K>
tn_status allow(K kernel, size_t smem, int& last) {
    int dev = 0;
    TN_CUDA(cudaGetDevice(&dev));
    if (last == dev) return TN_SUCCESS;
    TN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    last = dev;
    return TN_SUCCESS;
}

tn_status prepare_rows(const FewTokens& p, float* h, bool drop_ignored, cudaStream_t stream) {
    const int rows = token_rows(p.tokens);
    const int64_t padded = padded_of(p.hidden);
    few_rows_kernel<<<(unsigned)std::min<int64_t>(ceil_div(rows * padded, 256), (int64_t)sm_count() * 4), 256, 0, stream>>>(p, rows, padded, drop_ignored, h);
    return after_launch("few_rows_kernel");
}

template <int TM, bool ALIGNED, bool D>
tn_status logits(const FewTokens& p, const float* h, float* d, int64_t d_pitch, cudaStream_t stream) {
    static thread_local int device = -1;
    const size_t smem = sizeof(float) * kStages * (TM + kLogitCols<TM>) * kPitch;
    TN_TRY(allow(logits_kernel<TM, ALIGNED, D>, smem, device));
    logits_kernel<TM, ALIGNED, D><<<(unsigned)ceil_div(p.vocab, kLogitCols<TM>), kThreads, smem, stream>>>(p, h, padded_of(p.hidden), d, d_pitch);
    return after_launch("logits_kernel");
}

template <int TM, bool ALIGNED>
tn_status gradient(const FewTokens& p, const float* h, float* d, int64_t d_pitch, cudaStream_t stream) {
    TN_TRY((logits<TM, ALIGNED, true>(p, h, d, d_pitch, stream)));
    const int64_t across = ceil_div(p.hidden, kCols);
    if (p.sums) {
        static thread_local int device = -1;
        const size_t smem = sizeof(float) * kHiddenStages * (TM * kPitch + kStep * kHiddenWide);
        TN_TRY(allow(dhidden_kernel<TM, ALIGNED>, smem, device));
        const int64_t share = vocabulary_share(p.hidden, p.vocab);
        dhidden_kernel<TM, ALIGNED><<<dim3((unsigned)ceil_div(p.hidden, kHiddenCols), (unsigned)ceil_div(p.vocab, share)), kThreads, smem, stream>>>(p, d, d_pitch, share);
        TN_TRY(after_launch("dhidden_kernel"));
        TN_TRY(few_dhidden(p, f32_grad_shares(p.tokens, p.hidden, p.vocab), stream));
    }
    if (p.dweight) {
        static thread_local int device = -1;
        const size_t smem = sizeof(float) * 2 * TM * kWide;
        TN_TRY(allow(dweight_kernel<TM, ALIGNED>, smem, device));
        const int64_t rows = std::min(ceil_div(p.vocab, kCols), std::max<int64_t>(1, (int64_t)sm_count() * 4 / across));
        dweight_kernel<TM, ALIGNED><<<dim3((unsigned)across, (unsigned)rows), kThreads, smem, stream>>>(p, h, padded_of(p.hidden), d, d_pitch);
        TN_TRY(after_launch("dweight_kernel"));
    }
    return TN_SUCCESS;
}

}  // namespace

// Up to 64 tokens; grid extents within their limits.
bool f32_fits(int dtype, int64_t tokens, int64_t hidden) { return dtype == TN_FLOAT32 && tokens <= 64 && hidden <= int64_t(1) << 20; }
int64_t f32_loss_parts(int64_t tokens, int64_t vocab) {
    switch (token_rows(tokens)) {
        case 16: return ceil_div(vocab, kLogitCols<16>) * kGroupWarps<16>;
        case 32: return ceil_div(vocab, kLogitCols<32>) * kGroupWarps<32>;
        default: return ceil_div(vocab, kLogitCols<64>) * kGroupWarps<64>;
    }
}
size_t f32_row_floats(int64_t tokens, int64_t hidden) { return (size_t)token_rows(tokens) * padded_of(hidden); }
size_t f32_d_floats(int64_t tokens, int64_t vocab) { return (size_t)token_rows(tokens) * padded_of(vocab); }
int64_t f32_grad_shares(int64_t tokens, int64_t hidden, int64_t vocab) {
    return ceil_div(vocab, vocabulary_share(hidden, vocab)) * (64 / token_rows(tokens));
}

tn_status f32_loss(const FewTokens& p, float* h, cudaStream_t stream) {
    TN_TRY(prepare_rows(p, h, false, stream));
    const bool a = aligned(p);
    switch (token_rows(p.tokens)) {
        case 16: return a ? logits<16, true, false>(p, h, nullptr, 0, stream) : logits<16, false, false>(p, h, nullptr, 0, stream);
        case 32: return a ? logits<32, true, false>(p, h, nullptr, 0, stream) : logits<32, false, false>(p, h, nullptr, 0, stream);
        default: return a ? logits<64, true, false>(p, h, nullptr, 0, stream) : logits<64, false, false>(p, h, nullptr, 0, stream);
    }
}

tn_status f32_grad(const FewTokens& p, float* h, float* d, cudaStream_t stream) {
    TN_TRY(prepare_rows(p, h, true, stream));
    const bool a = aligned(p);
    const int64_t pitch = padded_of(p.vocab);
    switch (token_rows(p.tokens)) {
        case 16: return a ? gradient<16, true>(p, h, d, pitch, stream) : gradient<16, false>(p, h, d, pitch, stream);
        case 32: return a ? gradient<32, true>(p, h, d, pitch, stream) : gradient<32, false>(p, h, d, pitch, stream);
        default: return a ? gradient<64, true>(p, h, d, pitch, stream) : gradient<64, false>(p, h, d, pitch, stream);
    }
}

}  // namespace tnb
