// The cross entropy of a linear layer and its gradient for up to 64 tokens of float32.
//
// The large path writes float32 weights out as three bfloat16 parts first: 4 bytes an element read, 6 written, and 6 read again for each
// product, which for a few tokens is most of the time (16 tokens over 4096 x 32768: loss 594 us, here 177).
// Here W stays as it is. Its tiles come into shared memory by cp.async, several steps ahead, and a warp splits its fragments in registers:
// x = hi + lo, both tf32 (11 significand bits each, rounded to nearest), a b = hi hi + hi lo + lo hi; what is left out is below
// 2^-22 of the product and of either sign. The products run as mma.sync m16n8k8: tcgen05 takes its operands from shared memory, where
// the parts would have to be written back, and its 128-row tile would be mostly empty; the bound is W's way through shared memory.
// The tensor cores cut off below an accumulator's last place, so every step of 32 starts from zero and is added in float32.
//
//   logits  [tokens] x [64 or 128 vocabulary rows], K = hidden. Epilogue: maximum and sum of exponentials per token and warp, or d.
//   dh      [tokens] x [256 columns], K = a share of the vocabulary; the shares' sums are added in order afterwards.
//   dW      [128 vocabulary rows] x [128 columns], K = tokens: bound by writing dW.
#include <algorithm>

#include "linear_loss.cuh"

namespace tnb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kCols = 128;       // of a tile of dW
constexpr int kStep = 32;        // of K
constexpr int kPitch = kStep + 4;   // floats of a tile's row along K: rows g and columns t of a fragment lie in banks 4 g + t
constexpr int kWide = kCols + 8;    // floats of a tile's row along the columns: rows t and columns g in banks 8 t + g

// A fragment's element as two tf32.
struct Split { uint32_t hi, lo; };
__device__ __forceinline__ Split split(float x) {
    Split s;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(s.hi) : "f"(x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(s.lo) : "f"(x - __uint_as_float(s.hi)));
    return s;
}
// c += a b for 16 x 8 x 8: lane (g = lane / 4, t = lane % 4) holds a at rows g, g + 8 and columns t, t + 4 (row first), b at rows t, t + 4 of
// column g, c at rows g, g + 8 (row last) and columns 2 t, 2 t + 1.
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
struct FragmentA { uint32_t hi[4], lo[4]; };
struct FragmentB { uint32_t hi[2], lo[2]; };
// element(row, k) and element(k, column)
template <typename F>
__device__ __forceinline__ FragmentA fragment_a(F&& element, int g, int t) {
    FragmentA f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const Split s = split(element(g + 8 * (q & 1), t + 4 * (q >> 1)));
        f.hi[q] = s.hi;
        f.lo[q] = s.lo;
    }
    return f;
}
template <typename F>
__device__ __forceinline__ FragmentB fragment_b(F&& element, int g, int t) {
    FragmentB f;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const Split s = split(element(t + 4 * q, g));
        f.hi[q] = s.hi;
        f.lo[q] = s.lo;
    }
    return f;
}
__device__ __forceinline__ void mma3(float (&c)[4], const FragmentA& a, const FragmentB& b) {
    mma(c, a.lo, b.hi);
    mma(c, a.hi, b.lo);
    mma(c, a.hi, b.hi);
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
// The tokens as the products read them: [rows][padded], zero where there is no token, no target (that is for the gradient) or no column; behind
// them their hi and lo, which every warp of the logits would otherwise work out for itself.
__global__ void __launch_bounds__(256) few_rows_kernel(const FewTokens p, int rows, int64_t padded, int drop_ignored, float* __restrict__ out) {
    chain_go();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < rows * padded; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t n = i / padded, c = i - n * padded;
        const bool in = n < p.tokens && c < p.hidden && !(drop_ignored && target_of(p, n) == p.ignore);
        const float x = in ? static_cast<const float*>(p.h)[n * p.h_pitch + c] : 0.0f;
        const Split s = split(x);
        out[i] = x;
        out[i + rows * padded] = __uint_as_float(s.hi);
        out[i + 2 * rows * padded] = __uint_as_float(s.lo);
    }
}

// TM: tokens of the tile (16, 32 or 64). A warp has all of them and NT fragments of eight vocabulary rows. The thread block's two halves
// take the two halves of K, each with its own stages: with one block to an SM, and few blocks where the vocabulary is small, the time is that
// of the steps one after the other (64 tokens over 16903 x 2104: 116 us, with eight warps a block and all of K 210).
constexpr int kMostFragments = 2;
constexpr int columns_of(int fragments) { return kWarps * 8 * fragments; }
constexpr int kLogitThreads = 2 * kThreads;
// Steps in shared memory. Five fit for the smallest tile and serve whole copies (16 tokens over 8192 x 4096: 93 us, with three 105); element by
// element the way to the first step is longer than they save (4005 x 1033: 46 us against 55), and the larger tiles, of which four would fit,
// do not gain.
template <int TM, bool ALIGNED> constexpr int kLogitStages = TM == 16 && ALIGNED ? 5 : 3;

// h: hi and lo of the tokens, [2][TM][padded]. D: write d into `d` ([TM][d_pitch]), else the warps' statistics.
template <int TM, int NT, bool ALIGNED, bool D>
__global__ void __launch_bounds__(kLogitThreads) logits_kernel(const FewTokens p, const float* h, int64_t padded, float* d, int64_t d_pitch) {
    constexpr int COLS = columns_of(NT), MT = TM / 16, STAGE = (2 * TM + COLS) * kPitch, STAGES = kLogitStages<TM, ALIGNED>;
    extern __shared__ __align__(16) float smem[];  // [2][STAGES][2 TM + COLS][kPitch]
    const int half = threadIdx.x / kThreads, tid = threadIdx.x % kThreads;
    const int lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int64_t v0 = static_cast<int64_t>(blockIdx.x) * COLS;
    const int all = static_cast<int>((p.hidden + kStep - 1) / kStep), first_step = half * ((all + 1) / 2), steps = half ? all - first_step : (all + 1) / 2;
    float* const stages = smem + half * STAGES * STAGE;
    auto fill = [&](int step) {
        if (step < steps) {
            float* a = stages + (step % STAGES) * STAGE;
            float* b = a + 2 * TM * kPitch;
            const int64_t k0 = static_cast<int64_t>(first_step + step) * kStep;
            for (int i = tid; i < 2 * TM * (kStep / 4); i += kThreads) {
                const int r = i / (kStep / 4), c = i % (kStep / 4) * 4;
                const int valid = static_cast<int>(min(int64_t(4), padded - k0 - c));
                copy4<true>(a + r * kPitch + c, h + r * padded + (valid > 0 ? k0 + c : 0), valid);
            }
#pragma unroll
            for (int i = tid; i < COLS * (kStep / 4); i += kThreads) {
                const int r = i / (kStep / 4), c = i % (kStep / 4) * 4;
                const int valid = v0 + r < p.vocab ? static_cast<int>(min(int64_t(4), p.hidden - k0 - c)) : 0;
                copy4<ALIGNED>(b + r * kPitch + c, static_cast<const float*>(p.w) + (valid > 0 ? (v0 + r) * p.w_pitch + k0 + c : 0), valid);
            }
        }
        commit();
    };
    auto half_barrier = [&] { asm volatile("bar.sync %0, %1;" ::"r"(half + 1), "n"(kThreads) : "memory"); };
    chain_wait();
    chain_go();
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) fill(s);
    float sum[MT][NT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[i][j][q] = 0.0f;
    for (int step = 0; step < steps; ++step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        half_barrier();  // this step's tile is there for everyone, and the last step's is read
        fill(step + STAGES - 1);
        const float* a = stages + (step % STAGES) * STAGE;
        const float* b = a + (2 * TM + warp * 8 * NT) * kPitch;
        float part[MT][NT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) part[i][j][q] = 0.0f;
#pragma unroll
        for (int k = 0; k < kStep; k += 8) {
            FragmentB y[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) y[j] = fragment_b([&](int kk, int c) { return b[(8 * j + c) * kPitch + k + kk]; }, g, t);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                FragmentA x;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float* at = a + (16 * i + g + 8 * (q & 1)) * kPitch + k + t + 4 * (q >> 1);
                    x.hi[q] = __float_as_uint(at[0]);
                    x.lo[q] = __float_as_uint(at[TM * kPitch]);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) mma3(part[i][j], x, y[j]);
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) sum[i][j][q] += part[i][j][q];
    }
    // the second half's sums, through its own stages
    asm volatile("cp.async.wait_all;" ::: "memory");
    half_barrier();
    float* const other = smem + STAGES * STAGE + tid;
    if (half == 1) {
#pragma unroll
        for (int i = 0; i < MT * NT * 4; ++i) other[i * kThreads] = sum[i / (NT * 4)][i / 4 % NT][i % 4];
    }
    __syncthreads();
    if (half == 1) return;
#pragma unroll
    for (int i = 0; i < MT * NT * 4; ++i) sum[i / (NT * 4)][i / 4 % NT][i % 4] += other[i * kThreads];
    // lane (g, t) holds tokens 16 i + g and + 8, vocabulary rows 8 j + 2 t and + 1 of its warp's
    const int64_t first = v0 + warp * 8 * NT + 2 * t;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int up = 0; up < 2; ++up) {
            const int n = 16 * i + g + 8 * up;
            const int64_t target = n < p.tokens ? target_of(p, n) : -1;
            if constexpr (D) {
                const bool counts = n < p.tokens && target != p.ignore;
                const float lse = counts ? p.lse[n] : 0.0f;
                const float grad = !counts ? 0.0f : target < 0 || target >= p.vocab ? NAN : p.grad[n];
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int64_t v = first + 8 * j + q;
                        const float x = sum[i][j][2 * up + q] - lse;
                        if (v < d_pitch) d[n * d_pitch + v] = counts && v < p.vocab ? (v == target ? expm1f(x) : expf(x)) * grad : 0.0f;
                    }
            } else {
                float m = -INFINITY, s = 0.0f, x[NT][2];
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int64_t v = first + 8 * j + q;
                        x[j][q] = v < p.vocab ? sum[i][j][2 * up + q] : -INFINITY;
                        m = fmaxf(m, x[j][q]);
                        if (v == target && v < p.vocab) p.target_logit[n] = x[j][q];
                    }
                m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
                const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int j = 0; j < NT; ++j) s += __expf(x[j][0] - base) + __expf(x[j][1] - base);
                s += __shfl_xor_sync(0xFFFFFFFFu, s, 1);
                s += __shfl_xor_sync(0xFFFFFFFFu, s, 2);
                if (t == 0 && n < p.tokens) p.parts[(static_cast<int64_t>(blockIdx.x) * kWarps + warp) * p.tokens + n] = make_float2(m, s);
            }
        }
}

// dh's sums over the vocabulary rows [blockIdx.y * share, + share): 256 columns a block, 32 a warp.
constexpr int kHiddenCols = 256, kHiddenWide = kHiddenCols + 8, kHiddenStages = 3;

template <int TM, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) dhidden_kernel(const FewTokens p, const float* d, int64_t d_pitch, int64_t share) {
    extern __shared__ __align__(16) float smem[];  // [kHiddenStages] of [TM][kPitch] and [kStep][kHiddenWide]
    constexpr int TILE = TM * kPitch + kStep * kHiddenWide, MT = TM / 16, NT = kHiddenCols / kWarps / 8;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
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
    chain_wait();
    chain_go();
#pragma unroll
    for (int s = 0; s < kHiddenStages - 1; ++s) fill(s);
    float sum[MT][NT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[i][j][q] = 0.0f;
    for (int step = 0; step < steps; ++step) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kHiddenStages - 2) : "memory");
        __syncthreads();
        fill(step + kHiddenStages - 1);
        const float* a = smem + (step % kHiddenStages) * TILE;
        const float* b = a + TM * kPitch + warp * 8 * NT;
#pragma unroll
        for (int i = 0; i < MT; ++i) {  // sixteen tokens at a time: their step from zero takes 16 registers
            float part[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) part[j][q] = 0.0f;
#pragma unroll
            for (int k = 0; k < kStep; k += 8) {
                const FragmentA x = fragment_a([&](int r, int kk) { return a[(16 * i + r) * kPitch + k + kk]; }, g, t);
#pragma unroll
                for (int j = 0; j < NT; ++j) mma3(part[j], x, fragment_b([&](int kk, int c) { return b[(k + kk) * kHiddenWide + 8 * j + c]; }, g, t));
            }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) sum[i][j][q] += part[j][q];
        }
    }
    const int64_t column = c0 + warp * 8 * NT + 2 * t;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t n = 16 * i + g + 8 * (q >> 1);
            if (n < p.tokens) {
                float* to = p.sums + (blockIdx.y * p.tokens + n) * p.hidden;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int64_t c = column + 8 * j + (q & 1);
                    if (c < p.hidden) to[c] = sum[i][j][q];
                }
            }
        }
}

// dW: a tile of 128 x 128, K = the tokens, all of them in shared memory at once; a warp has 32 vocabulary rows and 64 columns.
template <int TM, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) dweight_kernel(const FewTokens p, const float* h, int64_t padded, const float* d, int64_t d_pitch) {
    extern __shared__ __align__(16) float smem[];  // [TM][kWide] of d and of h
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int row = warp / 2 * 32, column = warp % 2 * 64;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * kCols;
    float* a = smem;
    float* b = smem + TM * kWide;
    chain_wait();
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
        float sum[2][8][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) sum[i][j][q] = 0.0f;
#pragma unroll 2
        for (int k = 0; k < TM; k += 8) {
            FragmentA x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) x[i] = fragment_a([&](int r, int kk) { return a[(k + kk) * kWide + row + 16 * i + r]; }, g, t);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const FragmentB y = fragment_b([&](int kk, int c) { return b[(k + kk) * kWide + column + 8 * j + c]; }, g, t);
#pragma unroll
                for (int i = 0; i < 2; ++i) mma3(sum[i][j], x[i], y);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int up = 0; up < 2; ++up) {
                const int64_t v = v0 + row + 16 * i + g + 8 * up;
                if (v < p.vocab) {
                    float* to = static_cast<float*>(p.dweight) + v * p.hidden;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int64_t c = c0 + column + 8 * j + 2 * t;
                        if (ALIGNED) {
                            if (c < p.hidden) *reinterpret_cast<float2*>(to + c) = make_float2(sum[i][j][2 * up], sum[i][j][2 * up + 1]);
                        } else {
                            if (c < p.hidden) to[c] = sum[i][j][2 * up];
                            if (c + 1 < p.hidden) to[c + 1] = sum[i][j][2 * up + 1];
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
    TN_CUDA(launch_chained(false, few_rows_kernel, (unsigned)std::min<int64_t>(ceil_div(rows * padded, 256), (int64_t)sm_count() * 4), 256, 0, stream, 1, p, rows,
                           padded, drop_ignored, h));
    return after_launch("few_rows_kernel");
}

// One fragment a warp where two would leave half of the SMs idle: 64 tokens over 8192 x 4096 140 us, with two 195. The smaller tiles have too
// little to do for their loads of the tokens then (32 tokens there: 150 us against 135).
int fragments(int tile, int64_t vocab) { return tile == 64 && 2 * ceil_div(vocab, columns_of(kMostFragments)) <= sm_count() ? 1 : kMostFragments; }

template <int TM, int NT, bool ALIGNED, bool D>
tn_status logits_of(const FewTokens& p, const float* h, float* d, int64_t d_pitch, cudaStream_t stream) {
    static thread_local int device = -1;
    constexpr size_t smem = sizeof(float) * 2 * kLogitStages<TM, ALIGNED> * (2 * TM + columns_of(NT)) * kPitch;
    static_assert(smem <= 227 * 1024, "does not fit");
    TN_TRY(allow(logits_kernel<TM, NT, ALIGNED, D>, smem, device));
    TN_CUDA(launch_chained(true, logits_kernel<TM, NT, ALIGNED, D>, (unsigned)ceil_div(p.vocab, columns_of(NT)), kLogitThreads, smem, stream, 1, p,
                           h + TM * padded_of(p.hidden), padded_of(p.hidden), d, d_pitch));
    return after_launch("logits_kernel");
}
template <int TM, bool ALIGNED, bool D>
tn_status logits(const FewTokens& p, const float* h, float* d, int64_t d_pitch, cudaStream_t stream) {
    if constexpr (TM == 64) {
        if (fragments(TM, p.vocab) == 1) return logits_of<TM, 1, ALIGNED, D>(p, h, d, d_pitch, stream);
    }
    return logits_of<TM, kMostFragments, ALIGNED, D>(p, h, d, d_pitch, stream);
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
        TN_CUDA(launch_chained(true, dhidden_kernel<TM, ALIGNED>, dim3((unsigned)ceil_div(p.hidden, kHiddenCols), (unsigned)ceil_div(p.vocab, share)), kThreads, smem, stream,
                               1, p, d, d_pitch, share));
        TN_TRY(after_launch("dhidden_kernel"));
        TN_TRY(few_dhidden(p, f32_grad_shares(p.hidden, p.vocab), stream));
    }
    if (p.dweight) {
        static thread_local int device = -1;
        const size_t smem = sizeof(float) * 2 * TM * kWide;
        TN_TRY(allow(dweight_kernel<TM, ALIGNED>, smem, device));
        const int64_t rows = std::min(ceil_div(p.vocab, kCols), std::max<int64_t>(1, (int64_t)sm_count() * 4 / across));
        TN_CUDA(launch_chained(true, dweight_kernel<TM, ALIGNED>, dim3((unsigned)across, (unsigned)rows), kThreads, smem, stream, 1, p, h, padded_of(p.hidden), d, d_pitch));
        TN_TRY(after_launch("dweight_kernel"));
    }
    return TN_SUCCESS;
}

}  // namespace

// The loss up to 64 tokens and the gradient up to 32, where the large path's bfloat16 parts, written out first, have cost more than they gain;
// grid extents within their limits.
bool f32_fits(int dtype, int64_t tokens, int64_t hidden, bool gradient) {
    return dtype == TN_FLOAT32 && tokens <= (gradient ? 32 : 64) && hidden <= int64_t(1) << 20;
}
int64_t f32_loss_parts(int64_t tokens, int64_t vocab) { return ceil_div(vocab, columns_of(fragments(token_rows(tokens), vocab))) * kWarps; }
size_t f32_row_floats(int64_t tokens, int64_t hidden) { return 3 * (size_t)token_rows(tokens) * padded_of(hidden); }
size_t f32_d_floats(int64_t tokens, int64_t vocab) { return (size_t)token_rows(tokens) * padded_of(vocab); }
int64_t f32_grad_shares(int64_t hidden, int64_t vocab) { return ceil_div(vocab, vocabulary_share(hidden, vocab)); }

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
        default: return a ? gradient<32, true>(p, h, d, pitch, stream) : gradient<32, false>(p, h, d, pitch, stream);
    }
}

}  // namespace tnb
