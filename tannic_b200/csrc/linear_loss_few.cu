// The cross entropy of a linear layer for one token (float32: up to four) and its gradient for up to four of float32.
//
// With so few rows the products are all weights: the bound is reading W once (and writing dW once), and a tensor-core tile of 128
// rows would be empty. float32 operands gain most, which would otherwise be written out as three bfloat16 parts first.
// One token over 131072 x 4096 bfloat16: 171 us, 6.3 TB/s.
//
//   loss       A warp takes four vocabulary rows at a time and forms their products with all tokens in float32; the tokens lie in
//              shared memory and every value read from there serves four rows.
//   gradient   lse is known, so one pass over W does everything: a thread block keeps a few rows of W in shared memory, forms their
//              logits (a thread holds eight columns of the tokens and of their gradient's sums in registers), d from them, and
//              then both dh += d W and dW = d^T h before the next rows take their place. W is read once. Each block writes its
//              sums of dh; a second kernel adds them in order.
#include <algorithm>

#include "linear_loss.cuh"

namespace tnb {
namespace {

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Pack {
    T v[VEC];
};

// V sums over the 32 lanes at once (V a power of two up to 32): afterwards lane i holds the sum number i >> (5 - log2 V). Each step
// halves the values a lane carries instead of passing all of them on.
template <int V>
__device__ __forceinline__ float lane_sums(float (&v)[V], int lane) {
    int o = 16;
#pragma unroll
    for (int n = V / 2; n >= 1; n /= 2, o /= 2) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const bool up = lane & o;
            const float give = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
            v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
        }
    }
    for (; o >= 1; o /= 2) v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
    return v[0];
}
template <int V> constexpr int kLog2 = V == 1 ? 0 : 1 + kLog2<V / 2>;
template <> constexpr int kLog2<1> = 0;

__device__ __forceinline__ int64_t target_of(const FewTokens& p, int64_t n) {
    return p.wide ? static_cast<const int64_t*>(p.targets)[n] : static_cast<int64_t>(static_cast<const int32_t*>(p.targets)[n]);
}

constexpr int kLossThreads = 512;
constexpr int kRows = 4;  // vocabulary rows of a warp at a time

// NT: tokens, rounded up to a power of two.
template <typename T, int VEC, int NT>
__global__ void __launch_bounds__(kLossThreads, 1) few_loss_kernel(const FewTokens p, int64_t padded) {
    extern __shared__ __align__(16) float hid[];  // [NT][padded], zeros behind a row's end and in the rows without a token
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    chain_go();
    for (int64_t i = threadIdx.x; i < NT * padded; i += kLossThreads) {
        const int64_t n = i / padded, c = i - n * padded;
        hid[i] = n < p.tokens && c < p.hidden ? to_compute<float>(static_cast<const T*>(p.h)[n * p.h_pitch + c]) : 0.0f;
    }
    __syncthreads();
    const int warps = gridDim.x * (kLossThreads / 32), me = blockIdx.x * (kLossThreads / 32) + warp;
    constexpr int V = kRows * NT, SHIFT = 5 - kLog2<V>;
    const int index = lane >> SHIFT, row_in = index / NT, token = index % NT;
    const bool speaks = (lane & ((1 << SHIFT) - 1)) == 0 && token < p.tokens;
    const int64_t target = token < p.tokens ? target_of(p, token) : -1;
    float m = -INFINITY, s = 0.0f;
    for (int64_t v0 = static_cast<int64_t>(me) * kRows; v0 < p.vocab; v0 += static_cast<int64_t>(warps) * kRows) {
        float2 acc[kRows][NT];
        const T* w[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            w[r] = static_cast<const T*>(p.w) + min(v0 + r, p.vocab - 1) * p.w_pitch;  // a row behind the last is not used
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[r][n] = make_float2(0.0f, 0.0f);
        }
        if constexpr (VEC > 1) {
#pragma unroll 2
            for (int c = lane * VEC; c < p.hidden; c += 32 * VEC) {
                Pack<T, VEC> x[kRows];
#pragma unroll
                for (int r = 0; r < kRows; ++r) x[r] = *reinterpret_cast<const Pack<T, VEC>*>(w[r] + c);
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float2 q = *reinterpret_cast<const float2*>(hid + n * padded + c + j);
#pragma unroll
                        for (int r = 0; r < kRows; ++r) acc[r][n] = fma2(make_float2(to_compute<float>(x[r].v[j]), to_compute<float>(x[r].v[j + 1])), q, acc[r][n]);
                    }
                }
            }
        } else {
            // elements 32 apart, two at a time
#pragma unroll 2
            for (int c = lane; c < p.hidden; c += 64) {
                const bool second = c + 32 < p.hidden;
                float2 x[kRows];
#pragma unroll
                for (int r = 0; r < kRows; ++r) x[r] = make_float2(to_compute<float>(w[r][c]), second ? to_compute<float>(w[r][c + 32]) : 0.0f);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float2 q = make_float2(hid[n * padded + c], second ? hid[n * padded + c + 32] : 0.0f);
#pragma unroll
                    for (int r = 0; r < kRows; ++r) acc[r][n] = fma2(x[r], q, acc[r][n]);
                }
            }
        }
        float sums[V];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n) sums[r * NT + n] = acc[r][n].x + acc[r][n].y;
        const float logit = lane_sums<V>(sums, lane);
        const int64_t v = v0 + row_in;
        if (v < p.vocab) {
            const float now = fmaxf(m, logit), base = now == -INFINITY ? 0.0f : now;
            s = s * __expf(m - base) + __expf(logit - base);
            m = now;
            if (speaks && v == target) p.target_logit[token] = logit;
        }
    }
    // the lanes of one token (different rows) join: the row's bits are the top ones of the lane
#pragma unroll
    for (int o = 16; o >= 32 / kRows; o >>= 1) {
        const float om = __shfl_xor_sync(0xFFFFFFFFu, m, o), os = __shfl_xor_sync(0xFFFFFFFFu, s, o);
        const float now = fmaxf(m, om), base = now == -INFINITY ? 0.0f : now;
        s = s * __expf(m - base) + os * __expf(om - base);
        m = now;
    }
    if (speaks && row_in == 0) p.parts[static_cast<int64_t>(me) * p.tokens + token] = make_float2(m, s);
}

constexpr int kGradThreads = 512;
constexpr int E = 8;  // columns of a thread

constexpr int kGradRows = 4;
constexpr int kDepth = 3;  // batches of rows in shared memory: two in use, one on its way

// One barrier a batch: between two of them a warp forms its part of the next batch's logits and does everything else of this
// batch's, so that the chain logits - exponential - products of one batch runs under the other's.
template <int VEC, int NT>
__global__ void __launch_bounds__(kGradThreads, 1) few_grad_kernel(const FewTokens p) {
    constexpr int ITEMS = E / VEC, R = kGradRows, V = R * NT, SHIFT = 5 - kLog2<V>, WARPS = kGradThreads / 32;
    constexpr bool RING = VEC > 1;  // else the rows are read from memory twice, the second time from L1 or L2
    using P = Pack<float, VEC>;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float part[2][WARPS][32];
    __shared__ __align__(16) float dvals[WARPS][32];
    const int t = threadIdx.x, threads = blockDim.x, lane = t & 31, warp = t >> 5;
    P* ring = reinterpret_cast<P*>(smem) + t;  // [kDepth][R][ITEMS][threads]
    const int vecs = static_cast<int>(p.hidden / VEC);
    auto inside = [&](int i) { return i * threads + t < vecs; };
    if (p.sums) chain_go();

    // the tokens' columns of this thread; a token without a target is nothing, whatever it holds
    float2 h[NT][E / 2], dh[NT][E / 2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const bool counts = n < p.tokens && target_of(p, n) != p.ignore;
        float x[E];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                x[i * VEC + j] = counts && inside(i) ? static_cast<const float*>(p.h)[n * p.h_pitch + static_cast<int64_t>(i * threads + t) * VEC + j] : 0.0f;
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
            h[n][k] = make_float2(x[2 * k], x[2 * k + 1]);
            dh[n][k] = make_float2(0.0f, 0.0f);
        }
    }
    // what this lane's (row, token) needs
    const int index = lane >> SHIFT, row_in = index / NT, token = index % NT;
    bool counts = token < p.tokens;
    const int64_t target = counts ? target_of(p, token) : 0;
    counts = counts && target != p.ignore;
    const float lse = counts ? p.lse[token] : 0.0f;
    const float grad = !counts ? 0.0f : target < 0 || target >= p.vocab ? NAN : p.grad[token];
    // absent warps add nothing; columns behind the row's end are zero and stay so
    for (int i = t; i < 2 * WARPS * 32; i += threads) (&part[0][0][0])[i] = 0.0f;
    if constexpr (RING) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (!inside(i))
                for (int k = 0; k < kDepth * R; ++k)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) ring[(k * ITEMS + i) * threads].v[j] = 0.0f;
    }
    __syncthreads();

    const int64_t step = static_cast<int64_t>(gridDim.x) * R;
    // rows behind the last one are read as the last one; their d is zero and nothing is written for them
    auto row_at = [&](int64_t v) { return reinterpret_cast<const P*>(static_cast<const float*>(p.w) + min(v, p.vocab - 1) * p.w_pitch) + t; };
    auto fetch = [&](int64_t v0, int s) {
        if constexpr (RING) {
            if (v0 < p.vocab) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const P* from = row_at(v0 + r);
#pragma unroll
                    for (int i = 0; i < ITEMS; ++i)
                        if (inside(i)) {
                            const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(ring + ((s * R + r) * ITEMS + i) * threads));
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from + i * threads) : "memory");
                        }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    };
    // this thread's columns of row r of the batch at v0, in slot s
    auto row = [&](int64_t v0, int s, int r, float2 (&x)[E / 2]) {
        P q[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if constexpr (RING) {
                q[i] = ring[((s * R + r) * ITEMS + i) * threads];
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) q[i].v[j] = 0.0f;
                if (inside(i)) q[i] = row_at(v0 + r)[i * threads];
            }
        }
#pragma unroll
        for (int k = 0; k < E / 2; ++k)
            x[k] = make_float2(q[2 * k / VEC].v[2 * k % VEC], q[(2 * k + 1) / VEC].v[(2 * k + 1) % VEC]);
    };
    auto logits = [&](int64_t v0, int s, int to) {
        float dots[V];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float2 x[E / 2];
            row(v0, s, r, x);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int k = 0; k < E / 2; ++k) sum = fma2(x[k], h[n][k], sum);
                dots[r * NT + n] = sum.x + sum.y;
            }
        }
        part[to][warp][lane] = lane_sums<V>(dots, lane);
    };

    int64_t v0 = static_cast<int64_t>(blockIdx.x) * R;
    fetch(v0, 0);
    fetch(v0 + step, 1);
    if constexpr (RING) asm volatile("cp.async.wait_group 1;" ::: "memory");
    if (v0 < p.vocab) logits(v0, 0, 0);
    __syncthreads();
    int slot = 0, parity = 0;
    float* out_row = static_cast<float*>(p.dweight) + v0 * p.hidden;
    for (; v0 < p.vocab; v0 += step, parity ^= 1, out_row += step * p.hidden) {
        // a thread reads what it copied itself, and the slot that is filled now is the one that it read last
        const int next = slot == kDepth - 1 ? 0 : slot + 1, after = next == kDepth - 1 ? 0 : next + 1;
        fetch(v0 + 2 * step, after);
        if constexpr (RING) asm volatile("cp.async.wait_group 1;" ::: "memory");
        // the other parity's sums were read before the last barrier
        if (v0 + step < p.vocab) logits(v0 + step, next, parity ^ 1);
        float even = 0.0f, odd = 0.0f;
#pragma unroll
        for (int k = 0; k < WARPS; k += 2) {
            even += part[parity][k][lane];
            odd += part[parity][k + 1][lane];
        }
        const float x_lse = even + odd - lse;
        const int64_t v = v0 + row_in;
        float d = 0.0f;
        if (counts && v < p.vocab) d = (v == target ? expm1f(x_lse) : expf(x_lse)) * grad;
        // every warp keeps the batch's d for itself, in the order (row, token)
        __syncwarp();
        if ((lane & ((1 << SHIFT) - 1)) == 0) dvals[warp][index] = d;
        __syncwarp();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float dr[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n) dr[n] = dvals[warp][r * NT + n];
            float2 x[E / 2], out[E / 2];
            row(v0, slot, r, x);
#pragma unroll
            for (int k = 0; k < E / 2; ++k) out[k] = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float2 both = make_float2(dr[n], dr[n]);
#pragma unroll
                for (int k = 0; k < E / 2; ++k) {
                    dh[n][k] = fma2(both, x[k], dh[n][k]);
                    out[k] = fma2(both, h[n][k], out[k]);
                }
            }
            if (p.dweight && v0 + r < p.vocab) {
                P* to = reinterpret_cast<P*>(out_row + r * p.hidden) + t;
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    P q;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int e = i * VEC + j;
                        q.v[j] = e % 2 ? out[e / 2].y : out[e / 2].x;
                    }
                    if (inside(i)) to[i * threads] = q;
                }
            }
        }
        slot = next;
        __syncthreads();
    }
    if (p.sums) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n < p.tokens) {
                float* to = p.sums + (static_cast<int64_t>(blockIdx.x) * p.tokens + n) * p.hidden;
#pragma unroll
                for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int e = i * VEC + j;
                        if (inside(i)) to[static_cast<int64_t>(i * threads + t) * VEC + j] = e % 2 ? dh[n][e / 2].y : dh[n][e / 2].x;
                    }
            }
        }
    }
}

// dh: the blocks' sums added in an order that depends on their number only; COLS columns per block, 1024 / COLS threads a column. Tokens
// without a target get zero.
template <typename T, int COLS>
__global__ void __launch_bounds__(1024) few_dhidden_kernel(const FewTokens p, int blocks) {
    __shared__ float part[32][COLS + 1];
    chain_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t n_all = p.tokens * p.hidden, c = static_cast<int64_t>(blockIdx.x) * COLS + lane % COLS;
    float sum = 0.0f;
    if (c < n_all) {
#pragma unroll 5
        for (int b = threadIdx.x / COLS; b < blocks; b += 1024 / COLS) sum += p.sums[static_cast<int64_t>(b) * n_all + c];
    }
#pragma unroll
    for (int o = COLS; o < 32; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane < COLS) part[warp][lane] = sum;
    __syncthreads();
    if (warp >= COLS) return;
    sum = part[lane][warp];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const int64_t out = static_cast<int64_t>(blockIdx.x) * COLS + warp;
    if (lane == 0 && out < n_all) {
        const bool counts = target_of(p, out / p.hidden) != p.ignore;
        static_cast<T*>(p.dhidden)[out] = from_compute<T, float>(counts ? sum : 0.0f);
    }
}

// ------------------------------------------------------------------ host ---------------
bool fits16(const void* p, int64_t pitch_bytes) { return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(pitch_bytes)) & 15) == 0; }

template <typename K>
tn_status allow(K kernel, int& last) {
    int device = 0;
    TN_CUDA(cudaGetDevice(&device));
    return allow_shared_memory(kernel, device, last);
}

template <typename T, int VEC, int NT>
tn_status loss_one(const FewTokens& p, cudaStream_t stream) {
    static thread_local int device = -1;
    const int64_t padded = (p.hidden + 7) & ~int64_t(7);
    const size_t smem = sizeof(float) * NT * (size_t)padded;
    TN_TRY(allow(few_loss_kernel<T, VEC, NT>, device));
    TN_CUDA(launch_chained(false, few_loss_kernel<T, VEC, NT>, (unsigned)p.sms, kLossThreads, smem, stream, 1, p, padded));
    return after_launch("few_loss_kernel");
}
template <typename T, int VEC>
tn_status loss_tokens(const FewTokens& p, cudaStream_t stream) {
    if constexpr (sizeof(T) == 4) {
        if (p.tokens > 1) return p.tokens <= 2 ? loss_one<T, VEC, 2>(p, stream) : loss_one<T, VEC, 4>(p, stream);
    }
    return loss_one<T, VEC, 1>(p, stream);
}
template <typename T>
tn_status loss_typed(const FewTokens& p, cudaStream_t stream) {
    constexpr int VEC = 16 / sizeof(T);
    const bool wide = p.hidden % VEC == 0 && fits16(p.w, p.w_pitch * (int64_t)sizeof(T));
    return wide ? loss_tokens<T, VEC>(p, stream) : loss_tokens<T, 1>(p, stream);
}

template <typename T>
tn_status dhidden_typed(const FewTokens& p, int64_t n, cudaStream_t stream) {
    const bool many = p.tokens * p.hidden >= 32 * (int64_t)sm_count();
    TN_CUDA(launch_chained(true, many ? few_dhidden_kernel<T, 32> : few_dhidden_kernel<T, 8>, (unsigned)ceil_div(p.tokens * p.hidden, many ? 32 : 8), 1024, 0,
                           stream, 1, p, (int)n));
    return after_launch("few_dhidden_kernel");
}

template <int VEC, int NT>
tn_status grad_one(const FewTokens& p, cudaStream_t stream) {
    static thread_local int device = -1;
    const int threads = (int)(ceil_div(ceil_div(p.hidden / VEC, E / VEC), 32) * 32);
    const size_t smem = VEC > 1 ? sizeof(float) * E * kGradRows * kDepth * (size_t)threads : 0;
    TN_TRY(allow(few_grad_kernel<VEC, NT>, device));
    const int64_t blocks = few_grad_blocks(p);
    TN_CUDA(launch_chained(false, few_grad_kernel<VEC, NT>, (unsigned)blocks, threads, smem, stream, 1, p));
    TN_TRY(after_launch("few_grad_kernel"));
    return p.dhidden ? few_dhidden(p, blocks, stream) : TN_SUCCESS;
}
template <int VEC>
tn_status grad_tokens(const FewTokens& p, cudaStream_t stream) {
    if (p.tokens <= 1) return grad_one<VEC, 1>(p, stream);
    if (p.tokens <= 2) return grad_one<VEC, 2>(p, stream);
    return grad_one<VEC, 4>(p, stream);
}
}  // namespace

// As many columns as shared memory takes beside the tokens. One token of 16 bits: from two on the tensor cores are faster, empty rows and
// all (four tokens over 32768 x 4096: 59 us against 98); float32 up to four, where its own tiles begin to be (eight: 164 us here).
bool few_loss_fits(int dtype, int64_t tokens, int64_t hidden) {
    const int64_t nt = tokens <= 1 ? 1 : tokens <= 2 ? 2 : 4;
    return tokens <= (dtype == TN_FLOAT32 ? 4 : 1) && nt * (hidden + 8) * 4 <= 200 * 1024;
}
int64_t few_loss_parts(const FewTokens& p) { return (int64_t)p.sms * (kLossThreads / 32); }

tn_status few_loss(const FewTokens& p, cudaStream_t stream) {
    switch (p.dtype) {
        case TN_FLOAT16: return loss_typed<__half>(p, stream);
        case TN_BFLOAT16: return loss_typed<__nv_bfloat16>(p, stream);
        default: return loss_typed<float>(p, stream);
    }
}

tn_status few_dhidden(const FewTokens& p, int64_t n, cudaStream_t stream) {
    switch (p.dtype) {
        case TN_FLOAT16: return dhidden_typed<__half>(p, n, stream);
        case TN_BFLOAT16: return dhidden_typed<__nv_bfloat16>(p, n, stream);
        default: return dhidden_typed<float>(p, n, stream);
    }
}

// Four tokens with eight columns in each of 512 threads.
bool few_grad_fits(const FewTokens& p) { return p.dtype == TN_FLOAT32 && p.tokens <= 4 && p.hidden <= kGradThreads * E; }
int64_t few_grad_blocks(const FewTokens& p) { return std::min<int64_t>(p.sms, ceil_div(p.vocab, kGradRows)); }

tn_status few_grad(const FewTokens& p, cudaStream_t stream) {
    const bool wide = p.hidden % 4 == 0 && fits16(p.w, p.w_pitch * 4) && fits16(p.dweight, 0);
    return wide ? grad_tokens<4>(p, stream) : grad_tokens<1>(p, stream);
}

}  // namespace tnb
