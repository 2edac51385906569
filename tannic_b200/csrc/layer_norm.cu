// Layer normalisation over the last axis, forward and backward.
//
//   mu = mean(x)   r = 1 / sqrt(mean((x - mu)^2) + eps)   y = (x - mu) r w + b
//   z = (x - mu) r,  g = dy w:   dx = r (g - mean(g) - z mean(g z)),  dw = sum_rows dy z,  db = sum_rows dy
//
// Both passes are bound by HBM: the forward pass has to move x once in and y once out, the backward
// pass x and dy in and dx out, so a row is read once into registers (as it is stored: 16 bytes of a
// 16-bit type cost four registers) and everything else happens there. The mean is subtracted before
// the squares are summed (no E[x^2] - mu^2 cancellation); sums are float32 (float64 for float64).
//
// A row belongs to a warp while its lanes can hold it (32 elements each, 24 for 768 columns), beyond that to a thread block of
// up to 512 threads: few threads with many elements each keep the shuffles down. What is in flight must not depend
// on registers then, so the rows come through a ring in shared memory (cp.async, 16 bytes): a thread copies the
// vectors that it reads itself, two rows ahead, and waits for nobody else's. Rows that are not
// aligned to 16 bytes (VEC = 1) come as the 16-byte chunks that cover them, and a thread takes its elements from there one by
// one; rows longer than 16384 elements are read again from L2 by a looping kernel.
//
// The parameters' gradients are sums over all rows. The thread blocks of the backward kernel are
// resident for the whole pass and walk the rows with the grid's stride; a thread sees the same columns
// in every row, so it keeps its columns' two sums in registers, the warps of a block add theirs up in shared memory, and the
// block writes ONE partial row at its end. A second kernel adds the partial rows (a few hundred) in a fixed order: no
// atomics, the same bits on every run.
#include <algorithm>

#include "common.cuh"

namespace tnb {
namespace {

struct NormArgs {
    const void* x;
    const void* dy;       // backward only
    const void* weight;   // may be null
    const void* bias;     // may be null
    void* y;              // y, or dx
    void* mean;           // float32 (float64 for float64 rows); the forward pass may leave them out
    void* rstd;
    void* partial;        // backward: [blocks][2][cols]
    int64_t rows, x_pitch, dy_pitch;
    int cols;
    double eps;
};

template <typename T> struct stat_of { using type = float; };
template <> struct stat_of<double> { using type = double; };

// VEC consecutive elements moved by loads of up to 16 bytes.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Pack {
    T v[VEC];
};

template <typename S>
__device__ __forceinline__ S warp_sum(S v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Sum over a group of TPR threads. `slot` is the shared memory of this reduction ([TPR / 32] values); two
// consecutive reductions use different slots, so one barrier each is enough: a slot is written
// again only after a barrier that every reader of its old contents has passed.
template <typename S, int TPR>
__device__ __forceinline__ S group_sum(S v, S* slot) {
    v = warp_sum(v);
    if constexpr (TPR > 32) {
        if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < TPR / 32; ++w) v += slot[w];
    }
    return v;
}

// Two elements at a time: float32 as one packed instruction (the add, mul and fma of f32x2, rounded like the single ones), which
// halves the arithmetic of kernels that are as near to the issue limit as to HBM's.
template <typename S> struct Two { S a, b; };
template <typename S> __device__ __forceinline__ Two<S> both(S v) { return {v, v}; }
__device__ __forceinline__ uint64_t bits(Two<float> v) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.a), "f"(v.b));
    return r;
}
__device__ __forceinline__ Two<float> pair_of(uint64_t r) {
    Two<float> v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.a), "=f"(v.b) : "l"(r));
    return v;
}
__device__ __forceinline__ Two<float> add(Two<float> x, Two<float> y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(x)), "l"(bits(y)));
    return pair_of(r);
}
__device__ __forceinline__ Two<float> mul(Two<float> x, Two<float> y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(x)), "l"(bits(y)));
    return pair_of(r);
}
__device__ __forceinline__ Two<float> fma(Two<float> x, Two<float> y, Two<float> z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(x)), "l"(bits(y)), "l"(bits(z)));
    return pair_of(r);
}
__device__ __forceinline__ Two<double> add(Two<double> x, Two<double> y) { return {x.a + y.a, x.b + y.b}; }
__device__ __forceinline__ Two<double> mul(Two<double> x, Two<double> y) { return {x.a * y.a, x.b * y.b}; }
__device__ __forceinline__ Two<double> fma(Two<double> x, Two<double> y, Two<double> z) { return {::fma(x.a, y.a, z.a), ::fma(x.b, y.b, z.b)}; }

// Elements 2k and 2k + 1 of a thread's ITEMS vectors.
template <typename S, typename T, int VEC, int N>
__device__ __forceinline__ Two<S> two_of(const Pack<T, VEC> (&p)[N], int k) {
    return {to_compute<S>(p[2 * k / VEC].v[2 * k % VEC]), to_compute<S>(p[(2 * k + 1) / VEC].v[(2 * k + 1) % VEC])};
}

constexpr int kMost = 512;       // threads of a block that holds one row
constexpr int kRowWarps = 4;     // warps of a block whose warps hold a row each

// Sums of NV values over the threads that share a row: the warp, or (BLOCK) the thread block. `slots`: shared memory, NV values for each
// warp. Two consecutive reductions use different slots, so one barrier each is enough: a slot is written again only
// after a barrier that every reader of its old contents has passed.
template <typename S, int NV, bool BLOCK>
__device__ __forceinline__ void row_sums(S (&v)[NV], S* slots) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] += __shfl_xor_sync(0xFFFFFFFFu, v[k], o);
    }
    if constexpr (BLOCK) {
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int k = 0; k < NV; ++k) slots[(threadIdx.x >> 5) * NV + k] = v[k];
        }
        __syncthreads();
        static_assert(kMost <= 512, "sixteen warps");
        const int w = threadIdx.x & 15;
#pragma unroll
        for (int k = 0; k < NV; ++k) v[k] = w < static_cast<int>(blockDim.x >> 5) ? slots[w * NV + k] : S(0);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) {
#pragma unroll
            for (int k = 0; k < NV; ++k) v[k] += __shfl_xor_sync(0xFFFFFFFFu, v[k], o);
        }
    }
}

__device__ __forceinline__ float inverse_root(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inverse_root(double v) { return 1.0 / sqrt(v); }

// Where a thread stands: lane `t` of the `threads` that share row `first`, then every `step`-th.
template <bool BLOCK>
struct Place {
    int threads, t;
    int64_t first, step;
    __device__ __forceinline__ Place() {
        if constexpr (BLOCK) {
            threads = blockDim.x;
            t = threadIdx.x;
            first = blockIdx.x;
            step = gridDim.x;
        } else {
            threads = 32;
            t = threadIdx.x & 31;
            first = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
            step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
        }
    }
};

// N operands' rows on their way into shared memory, DEPTH slots of them. Aligned rows lie there as vectors, [slot][operand][item][thread], and
// a thread copies and reads its own. Others (VEC = 1) lie as in memory, at the same offset from a 16-byte boundary, in a
// window per warp or block, and the threads that share a row meet after the wait.
template <typename T, int VEC, int ITEMS, int N, int DEPTH, bool BLOCK>
struct Ring {
    static constexpr bool kVectors = VEC > 1;
    using V = Pack<T, VEC>;
    uint8_t* mine;
    int pitch;            // threads of the block, or bytes of a window
    int slot = 0;
    __host__ __device__ static int window_bytes(int cols) { return (cols * static_cast<int>(sizeof(T)) + 30) & ~15; }
    __host__ static size_t bytes(int cols, int threads) {
        return kVectors ? sizeof(V) * ITEMS * N * DEPTH * static_cast<size_t>(threads) : static_cast<size_t>(window_bytes(cols)) * N * DEPTH * (BLOCK ? 1 : threads / 32);
    }
    __device__ __forceinline__ Ring(uint8_t* smem, int cols) {
        if constexpr (kVectors) {
            mine = smem + threadIdx.x * sizeof(V);
            pitch = blockDim.x;
        } else {
            pitch = window_bytes(cols);
            mine = smem + (BLOCK ? 0 : static_cast<int>(threadIdx.x >> 5) * N * DEPTH * pitch);
        }
    }
    __device__ __forceinline__ V* vector(int s, int operand, int item) const { return reinterpret_cast<V*>(mine) + ((s * N + operand) * ITEMS + item) * pitch; }
    __device__ __forceinline__ static void copy16(const void* to, const void* from, int bytes) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from), "r"(bytes) : "memory");
    }
    // The row at `row` into slot s; `lowest` is the operand's first byte. Nothing before it and nothing behind the row is read.
    __device__ __forceinline__ void fetch(int s, int operand, const T* row, const void* lowest, int cols, int t, int threads) const {
        if constexpr (kVectors) {
            const V* from = reinterpret_cast<const V*>(row) + t;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (i * threads + t < cols / VEC) copy16(vector(s, operand, i), from + i * threads, 16);
        } else {
            const uintptr_t begin = reinterpret_cast<uintptr_t>(row), end = begin + cols * sizeof(T), first = begin & ~uintptr_t(15);
            uint8_t* window = mine + (s * N + operand) * pitch;
            for (uintptr_t at = first + 16 * t; at < end; at += 16 * threads) {
                if (at >= reinterpret_cast<uintptr_t>(lowest)) {
                    copy16(window + (at - first), reinterpret_cast<const void*>(at), static_cast<int>(min(uintptr_t(16), end - at)));
                } else {
                    // the chunk begins before the tensor does
                    for (uintptr_t e = begin; e < min(at + 16, end); e += sizeof(T)) *reinterpret_cast<T*>(window + (e - first)) = *reinterpret_cast<const T*>(e);
                }
            }
        }
    }
    __device__ __forceinline__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    // until the oldest of DEPTH groups has arrived
    __device__ __forceinline__ static void wait() {
        asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
        if constexpr (!kVectors) meet();
    }
    __device__ __forceinline__ static void meet() {
        if constexpr (BLOCK) __syncthreads();
        else __syncwarp();
    }
    // vector `item` of thread t from the current slot
    __device__ __forceinline__ V read(int operand, const T* row, int item, int t, int threads) const {
        if constexpr (kVectors) {
            return *vector(slot, operand, item);
        } else {
            V v;
            v.v[0] = reinterpret_cast<const T*>(mine + (slot * N + operand) * pitch + (reinterpret_cast<uintptr_t>(row) & 15))[item * threads + t];
            return v;
        }
    }
    __device__ __forceinline__ int last() const { return slot == 0 ? DEPTH - 1 : slot - 1; }
    __device__ __forceinline__ void next() { slot = slot + 1 == DEPTH ? 0 : slot + 1; }
};

// First byte of an operand whose rows are `pitch` elements apart.
template <typename T>
__device__ __forceinline__ const void* lowest_byte(const void* base, int64_t pitch, int64_t rows) {
    return pitch < 0 ? static_cast<const T*>(base) + (rows - 1) * pitch : static_cast<const T*>(base);
}

template <typename T, typename P, int VEC, int ITEMS, int DEPTH, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? kMost : 32 * kRowWarps, 1) norm_forward(const NormArgs a) {
    using S = typename stat_of<T>::type;
    constexpr int E = VEC * ITEMS;
    __shared__ S slots[2][BLOCK ? kMost / 32 : 1];
    extern __shared__ __align__(16) uint8_t dynamic[];
    const Place<BLOCK> at;
    Ring<T, VEC, ITEMS, 1, DEPTH, BLOCK> ring(dynamic, a.cols);
    const int vecs = a.cols / VEC;
    const S share = S(1) / static_cast<S>(a.cols);
    const void* lowest = lowest_byte<T>(a.x, a.x_pitch, a.rows);
    auto inside = [&](int i) { return i * at.threads + at.t < vecs; };
    auto row_at = [&](int64_t r) { return static_cast<const T*>(a.x) + r * a.x_pitch; };
    auto fetch = [&](int64_t r, int slot) {
        if (r < a.rows) ring.fetch(slot, 0, row_at(r), lowest, a.cols, at.t, at.threads);
        ring.commit();
    };
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) fetch(at.first + d * at.step, d);
    // the parameters of this thread's columns, read once for all rows
    Pack<P, VEC> w[ITEMS], b[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            w[i].v[j] = from_compute<P, S>(S(1));
            b[i].v[j] = from_compute<P, S>(S(0));
        }
        if (inside(i) && a.weight) w[i] = static_cast<const Pack<P, VEC>*>(a.weight)[i * at.threads + at.t];
        if (inside(i) && a.bias) b[i] = static_cast<const Pack<P, VEC>*>(a.bias)[i * at.threads + at.t];
    }
    for (int64_t row = at.first; row < a.rows; row += at.step) {
        // the slot before this row's is the one that was read last, before the shuffles of its sums
        fetch(row + (DEPTH - 1) * at.step, ring.last());
        ring.wait();
        Pack<T, VEC> p[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) p[i].v[j] = T(0.0f);
            if (inside(i)) p[i] = ring.read(0, row_at(row), i, at.t, at.threads);
        }
        Two<S> v[E / 2], pair = both(S(0));
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
            v[k] = two_of<S>(p, k);
            pair = add(pair, v[k]);
        }
        S sum[1] = {pair.a + pair.b};
        row_sums<S, 1, BLOCK>(sum, slots[0]);
        const S mean = sum[0] * share;
        pair = both(S(0));
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
            v[k] = add(v[k], both(-mean));
            // what lies behind the row's end is not mean away from it
            if (!inside(2 * k / VEC)) v[k].a = S(0);
            if (!inside((2 * k + 1) / VEC)) v[k].b = S(0);
            pair = fma(v[k], v[k], pair);
        }
        sum[0] = pair.a + pair.b;
        row_sums<S, 1, BLOCK>(sum, slots[1]);
        const S rstd = inverse_root(sum[0] * share + static_cast<S>(a.eps));
        if (at.t == 0) {
            if (a.mean) static_cast<S*>(a.mean)[row] = mean;
            if (a.rstd) static_cast<S*>(a.rstd)[row] = rstd;
        }
        Pack<T, VEC>* y = reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.y) + row * a.cols);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
            const Two<S> r = fma(mul(v[k], both(rstd)), two_of<S>(w, k), two_of<S>(b, k));
            p[2 * k / VEC].v[2 * k % VEC] = from_compute<T, S>(r.a);
            p[(2 * k + 1) / VEC].v[(2 * k + 1) % VEC] = from_compute<T, S>(r.b);
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (inside(i)) y[i * at.threads + at.t] = p[i];
        ring.next();
    }
}

// KEEP: x - mean and g stay in registers between the two halves of the work; else they are formed again (32 elements in each of 512 threads leave
// no room; 24 of 16 bits in a lane leave room for half as many warps, 57 us against 55 at 50432 x 768). A vector that is
// read again is the thread's own, so that needs no barrier.
template <typename T, typename P, int VEC, int ITEMS, int DEPTH, bool BLOCK, bool KEEP>
__global__ void __launch_bounds__(BLOCK ? kMost : 32 * kRowWarps, 1) norm_backward(const NormArgs a) {
    using S = typename stat_of<T>::type;
    static_assert(KEEP || VEC > 1, "a window is not read again after the sums without a barrier");
    constexpr int E = VEC * ITEMS;
    __shared__ S slots[2][BLOCK ? kMost / 32 * 2 : 1];
    extern __shared__ __align__(16) uint8_t dynamic[];
    const Place<BLOCK> at;
    Ring<T, VEC, ITEMS, 2, DEPTH, BLOCK> ring(dynamic, a.cols);
    const int vecs = a.cols / VEC;
    const S share = S(1) / static_cast<S>(a.cols);
    Two<S> dw[E / 2], db[E / 2];
#pragma unroll
    for (int k = 0; k < E / 2; ++k) dw[k] = db[k] = both(S(0));
    auto inside = [&](int i) { return i * at.threads + at.t < vecs; };
    auto weight_at = [&](int i) {
        Pack<P, VEC> p;
        if (a.weight) {
            p = static_cast<const Pack<P, VEC>*>(a.weight)[i * at.threads + at.t];
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) p.v[j] = from_compute<P, S>(S(1));
        }
        return p;
    };
    const void *lowest_x = lowest_byte<T>(a.x, a.x_pitch, a.rows), *lowest_dy = lowest_byte<T>(a.dy, a.dy_pitch, a.rows);
    auto x_at = [&](int64_t r) { return static_cast<const T*>(a.x) + r * a.x_pitch; };
    auto dy_at = [&](int64_t r) { return static_cast<const T*>(a.dy) + r * a.dy_pitch; };
    auto fetch = [&](int64_t r, int slot) {
        if (r < a.rows) {
            ring.fetch(slot, 0, x_at(r), lowest_x, a.cols, at.t, at.threads);
            ring.fetch(slot, 1, dy_at(r), lowest_dy, a.cols, at.t, at.threads);
        }
        ring.commit();
    };
    // The work goes G vectors at a time, an even number of elements.
    constexpr int G = VEC > 1 ? 1 : 2, PAIRS = G * VEC / 2;
    auto weights = [&](int i0, Pack<P, VEC> (&p)[G]) {
#pragma unroll
        for (int i = 0; i < G; ++i) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) p[i].v[j] = P(0.0f);
            if (inside(i0 + i)) p[i] = weight_at(i0 + i);
        }
    };
    constexpr bool WEIGHTS = E <= 24;  // the weight stays in registers, as float32
    Two<S> w[WEIGHTS ? E / 2 : 1];
    if constexpr (WEIGHTS) {
#pragma unroll
        for (int i0 = 0; i0 < ITEMS; i0 += G) {
            Pack<P, VEC> p[G];
            weights(i0, p);
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) w[i0 * VEC / 2 + k] = two_of<S>(p, k);
        }
    }
    S mean = 0, rstd = 0;
    auto statistics = [&](int64_t r) {
        if (r < a.rows) {
            mean = static_cast<const S*>(a.mean)[r];
            rstd = static_cast<const S*>(a.rstd)[r];
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) fetch(at.first + d * at.step, d);
    statistics(at.first);
    int parity = 0;
    for (int64_t row = at.first; row < a.rows; row += at.step, parity ^= 1) {
        fetch(row + (DEPTH - 1) * at.step, ring.last());
        const S mu = mean, rs = rstd;
        statistics(row + at.step);
        ring.wait();
        auto read = [&](int i0, Pack<T, VEC> (&px)[G], Pack<T, VEC> (&pd)[G]) {
#pragma unroll
            for (int i = 0; i < G; ++i) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) px[i].v[j] = pd[i].v[j] = T(0.0f);  // behind the row's end: no gradient
                if (inside(i0 + i)) {
                    px[i] = ring.read(0, x_at(row), i0 + i, at.t, at.threads);
                    pd[i] = ring.read(1, dy_at(row), i0 + i, at.t, at.threads);
                }
            }
        };
        Two<S> c[KEEP ? E / 2 : 1], g[KEEP ? E / 2 : 1];  // x - mean and dy * weight
        Two<S> sum_g = both(S(0)), sum_gc = both(S(0));
#pragma unroll
        for (int i0 = 0; i0 < ITEMS; i0 += G) {
            Pack<T, VEC> px[G], pd[G];
            Pack<P, VEC> pw[G];
            read(i0, px, pd);
            if constexpr (!WEIGHTS) weights(i0, pw);
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) {
                const int at_k = i0 * VEC / 2 + k;
                const Two<S> d = two_of<S>(pd, k), cc = add(two_of<S>(px, k), both(-mu));
                const Two<S> gg = mul(d, WEIGHTS ? w[WEIGHTS ? at_k : 0] : two_of<S>(pw, k));
                if constexpr (KEEP) {
                    c[at_k] = cc;
                    g[at_k] = gg;
                }
                sum_g = add(sum_g, gg);
                sum_gc = fma(gg, cc, sum_gc);
                dw[at_k] = fma(mul(cc, both(rs)), d, dw[at_k]);
                db[at_k] = add(db[at_k], d);
            }
        }
        S sums[2] = {sum_g.a + sum_g.b, (sum_gc.a + sum_gc.b) * rs};
        row_sums<S, 2, BLOCK>(sums, slots[parity]);
        // dx = r (g - mean(g)) - (x - mean) r^2 mean(g z)
        const Two<S> by_g = both(rs), by_c = both(-rs * rs * (sums[1] * share)), shift = both(-rs * (sums[0] * share));
        Pack<T, VEC>* dx = reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.y) + row * a.cols);
#pragma unroll
        for (int i0 = 0; i0 < ITEMS; i0 += G) {
            Pack<T, VEC> px[G], pd[G];
            Pack<P, VEC> pw[G];
            if constexpr (!KEEP) {
                read(i0, px, pd);
                if constexpr (!WEIGHTS) weights(i0, pw);
            }
#pragma unroll
            for (int k = 0; k < PAIRS; ++k) {
                const int at_k = i0 * VEC / 2 + k;
                Two<S> cc, gg;
                if constexpr (KEEP) {
                    cc = c[at_k];
                    gg = g[at_k];
                } else {
                    cc = add(two_of<S>(px, k), both(-mu));
                    gg = mul(two_of<S>(pd, k), WEIGHTS ? w[WEIGHTS ? at_k : 0] : two_of<S>(pw, k));
                }
                const Two<S> r = fma(cc, by_c, fma(gg, by_g, shift));
                px[2 * k / VEC].v[2 * k % VEC] = from_compute<T, S>(r.a);
                px[(2 * k + 1) / VEC].v[(2 * k + 1) % VEC] = from_compute<T, S>(r.b);
            }
#pragma unroll
            for (int i = 0; i < G; ++i)
                if (inside(i0 + i)) dx[(i0 + i) * at.threads + at.t] = px[i];
        }
        ring.next();
    }
    if (a.partial == nullptr) return;  // uniform: no parameter gradients wanted
    chain_go();
    S* mine = static_cast<S*>(a.partial) + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
    S* all = BLOCK ? mine : reinterpret_cast<S*>(dynamic);
    // a block that holds one row has its sums; the warps of the others add theirs up one after the other, where the ring was
    for (int k = 0; k < (BLOCK ? 1 : static_cast<int>(blockDim.x >> 5)); ++k) {
        if (!BLOCK) __syncthreads();
        if (BLOCK || static_cast<int>(threadIdx.x >> 5) == k) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (inside(i)) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const int c = (i * at.threads + at.t) * VEC + j, e = i * VEC + j;
                        const S one = e % 2 ? dw[e / 2].b : dw[e / 2].a, two = e % 2 ? db[e / 2].b : db[e / 2].a;
                        all[c] = k ? all[c] + one : one;
                        all[a.cols + c] = k ? all[a.cols + c] + two : two;
                    }
                }
        }
    }
    if (!BLOCK) {
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * a.cols; c += blockDim.x) mine[c] = all[c];
    }
}

// Rows longer than the registers of 512 threads hold: the row is read three times, from L2 after the first.
constexpr int kLong = 1024;

template <typename T, typename P>
__global__ void __launch_bounds__(kLong) norm_forward_long(const NormArgs a) {
    using S = typename stat_of<T>::type;
    __shared__ S slots[2][kLong / 32];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_pitch;
        S sum = 0;
        for (int c = threadIdx.x; c < a.cols; c += kLong) sum += to_compute<S>(x[c]);
        const S mean = group_sum<S, kLong>(sum, slots[0]) / static_cast<S>(a.cols);
        S square = 0;
        for (int c = threadIdx.x; c < a.cols; c += kLong) {
            const S d = to_compute<S>(x[c]) - mean;
            square += d * d;
        }
        const S rstd = S(1) / sqrt(group_sum<S, kLong>(square, slots[1]) / static_cast<S>(a.cols) + static_cast<S>(a.eps));
        if (threadIdx.x == 0) {
            if (a.mean) static_cast<S*>(a.mean)[row] = mean;
            if (a.rstd) static_cast<S*>(a.rstd)[row] = rstd;
        }
        T* y = static_cast<T*>(a.y) + row * a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kLong) {
            S v = (to_compute<S>(x[c]) - mean) * rstd;
            if (a.weight) v *= to_compute<S>(static_cast<const P*>(a.weight)[c]);
            if (a.bias) v += to_compute<S>(static_cast<const P*>(a.bias)[c]);
            y[c] = from_compute<T, S>(v);
        }
    }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kLong) norm_backward_long(const NormArgs a) {
    using S = typename stat_of<T>::type;
    __shared__ S slots[2][kLong / 32];
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_pitch;
        const T* dy = static_cast<const T*>(a.dy) + row * a.dy_pitch;
        const S mean = static_cast<const S*>(a.mean)[row], rstd = static_cast<const S*>(a.rstd)[row];
        S sum_g = 0, sum_gz = 0;
        for (int c = threadIdx.x; c < a.cols; c += kLong) {
            const S z = (to_compute<S>(x[c]) - mean) * rstd;
            S g = to_compute<S>(dy[c]);
            if (a.weight) g *= to_compute<S>(static_cast<const P*>(a.weight)[c]);
            sum_g += g;
            sum_gz += g * z;
        }
        const S mean_g = group_sum<S, kLong>(sum_g, slots[0]) / static_cast<S>(a.cols);
        const S mean_gz = group_sum<S, kLong>(sum_gz, slots[1]) / static_cast<S>(a.cols);
        T* dx = static_cast<T*>(a.y) + row * a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kLong) {
            const S z = (to_compute<S>(x[c]) - mean) * rstd;
            S g = to_compute<S>(dy[c]);
            if (a.weight) g *= to_compute<S>(static_cast<const P*>(a.weight)[c]);
            dx[c] = from_compute<T, S>((g - mean_g - z * mean_gz) * rstd);
        }
    }
}

// The parameters' gradients of such rows: blockIdx.y takes every gridDim.y-th row, a thread one column.
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_long(const NormArgs a) {
    using S = typename stat_of<T>::type;
    S* mine = static_cast<S*>(a.partial) + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
    const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (c >= a.cols) return;
    S dw = 0, db = 0;
#pragma unroll 4
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const S mean = static_cast<const S*>(a.mean)[row], rstd = static_cast<const S*>(a.rstd)[row];
        const S d = to_compute<S>(static_cast<const T*>(a.dy)[row * a.dy_pitch + c]);
        dw += d * ((to_compute<S>(static_cast<const T*>(a.x)[row * a.x_pitch + c]) - mean) * rstd);
        db += d;
    }
    mine[c] = dw;
    mine[a.cols + c] = db;
}

// Adds the partial rows, in an order that depends on their number only. COLS columns per block and 1024 / COLS threads a column: 8 (a
// sector of 32 bytes, two or three loads a thread for a few hundred rows), 32 where that is blocks enough.
template <typename S, typename P, int COLS>
__global__ void __launch_bounds__(1024) norm_parameters(const S* partial, int blocks, int cols, P* __restrict__ dweight, P* __restrict__ dbias) {
    __shared__ S part[32][COLS + 1];
    chain_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // columns [0, cols) are the weight's, [cols, 2 cols) the bias's
    const int64_t all = static_cast<int64_t>(cols) * 2, c = static_cast<int64_t>(blockIdx.x) * COLS + lane % COLS;
    S sum = 0;
    if (c < all) {
#pragma unroll 4
        for (int b = threadIdx.x / COLS; b < blocks; b += 1024 / COLS) sum += partial[static_cast<int64_t>(b) * all + c];
    }
#pragma unroll
    for (int o = COLS; o < 32; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane < COLS) part[warp][lane] = sum;
    __syncthreads();
    if (warp >= COLS) return;
    sum = warp_sum(part[lane][warp]);  // column `warp`
    const int64_t out = static_cast<int64_t>(blockIdx.x) * COLS + warp;
    if (lane == 0 && out < all) {
        if (out < cols) {
            if (dweight) dweight[out] = from_compute<P, S>(sum);
        } else if (dbias) {
            dbias[out - cols] = from_compute<P, S>(sum);
        }
    }
}

// ------------------------------------------------------------------ host ---------------
int64_t rows_grid(int64_t rows, int groups) { return std::min<int64_t>(ceil_div(rows, groups), int64_t(1) << 30); }

struct Launch {
    NormArgs args;
    cudaStream_t stream;
    bool backward;
    void* dweight = nullptr;  // backward: parameter gradients, either may be null
    void* dbias = nullptr;
};

// Allocates the partial rows of a backward pass with `blocks` thread blocks.
template <typename S>
tn_status alloc_partial(Launch& l, int64_t blocks) {
    l.args.partial = nullptr;
    if (!l.dweight && !l.dbias) return TN_SUCCESS;
    return scratch_alloc(&l.args.partial, sizeof(S) * 2 * static_cast<size_t>(blocks) * static_cast<size_t>(l.args.cols), l.stream);
}

template <typename S, typename P>
tn_status finish_partial(Launch& l, int64_t blocks) {
    if (!l.args.partial) return TN_SUCCESS;
    const int64_t all = 2 * (int64_t)l.args.cols;
    const bool many = all >= 32 * (int64_t)sm_count();
    TN_CUDA(launch_chained(true, many ? norm_parameters<S, P, 32> : norm_parameters<S, P, 8>, (unsigned)ceil_div(all, many ? 32 : 8), 1024, 0, l.stream, 1,
                           static_cast<const S*>(l.args.partial), (int)blocks, l.args.cols, static_cast<P*>(l.dweight), static_cast<P*>(l.dbias)));
    return after_launch("norm_parameters");
}

// Thread blocks of a kernel that are on the GPU at once. The answer to the last question (device, threads, shared memory) is kept
// in `last`, one per kernel and thread.
struct Resident {
    int device = -1, allowed = -1, threads = 0;
    size_t smem = 0;
    int64_t blocks = 0;
};
template <typename K>
tn_status resident_blocks(K kernel, int threads, size_t smem, Resident& last) {
    int device = 0, per_sm = 0;
    TN_CUDA(cudaGetDevice(&device));
    if (last.device == device && last.threads == threads && last.smem == smem) return TN_SUCCESS;
    TN_TRY(allow_shared_memory(kernel, device, last.allowed));
    TN_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
    last.device = device;
    last.threads = threads;
    last.smem = smem;
    last.blocks = (int64_t)sm_count() * std::max(per_sm, 1);
    return TN_SUCCESS;
}

template <typename T, int VEC, int ITEMS, bool BLOCK>
int block_threads(int cols) {
    return BLOCK ? (int)(ceil_div(ceil_div(cols / VEC, ITEMS), 32) * 32) : 32 * kRowWarps;
}

template <typename T, typename P, int VEC, int ITEMS, bool BLOCK>
tn_status launch_forward(Launch& l) {
    constexpr int DEPTH = 3;
    const NormArgs& a = l.args;
    const int threads = block_threads<T, VEC, ITEMS, BLOCK>(a.cols);
    const size_t smem = Ring<T, VEC, ITEMS, 1, DEPTH, BLOCK>::bytes(a.cols, threads);
    static thread_local Resident resident;
    TN_TRY(resident_blocks(norm_forward<T, P, VEC, ITEMS, DEPTH, BLOCK>, threads, smem, resident));
    const int64_t blocks = std::min(resident.blocks, ceil_div(a.rows, BLOCK ? 1 : kRowWarps));
    norm_forward<T, P, VEC, ITEMS, DEPTH, BLOCK><<<(unsigned)blocks, threads, smem, l.stream>>>(a);
    return after_launch("norm_forward");
}

template <typename T, typename P, int VEC, int ITEMS, bool BLOCK, bool KEEP>
tn_status launch_backward(Launch& l) {
    using S = typename stat_of<T>::type;
    // what shared memory holds beside the blocks that the registers allow; one row of 16384 float32 twice is 128 KiB
    constexpr int DEPTH = VEC * ITEMS > 24 ? (sizeof(T) == 4 ? 1 : 3) : KEEP && sizeof(T) * VEC * ITEMS * 2 <= 96 ? 5 : 3;
    NormArgs& a = l.args;
    const int threads = block_threads<T, VEC, ITEMS, BLOCK>(a.cols);
    size_t smem = Ring<T, VEC, ITEMS, 2, DEPTH, BLOCK>::bytes(a.cols, threads);
    if (!BLOCK) smem = std::max(smem, sizeof(S) * 2 * (size_t)a.cols);
    // one resident wave: every block walks rows until the pass ends, then writes its partial row
    static thread_local Resident resident;
    TN_TRY(resident_blocks(norm_backward<T, P, VEC, ITEMS, DEPTH, BLOCK, KEEP>, threads, smem, resident));
    const int64_t blocks = std::min(resident.blocks, ceil_div(a.rows, BLOCK ? 1 : kRowWarps));
    TN_TRY(alloc_partial<S>(l, blocks));
    norm_backward<T, P, VEC, ITEMS, DEPTH, BLOCK, KEEP><<<(unsigned)blocks, threads, smem, l.stream>>>(a);
    tn_status st = after_launch("norm_backward");
    if (st == TN_SUCCESS) st = finish_partial<S, P>(l, blocks);
    if (a.partial) {
        const tn_status freed = scratch_free(a.partial, l.stream);
        if (st == TN_SUCCESS) st = freed;
    }
    return st;
}

template <typename T, typename P>
tn_status launch_long(Launch& l) {
    using S = typename stat_of<T>::type;
    if (!l.backward) {
        norm_forward_long<T, P><<<(unsigned)rows_grid(l.args.rows, 1), kLong, 0, l.stream>>>(l.args);
        return after_launch("norm_forward_long");
    }
    // the columns first: dx may take the place of dy or x
    const int64_t across = ceil_div(l.args.cols, 256);
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(l.args.rows, 1024), ceil_div((int64_t)sm_count() * 8, across)));
    TN_TRY(alloc_partial<S>(l, blocks));
    tn_status st = TN_SUCCESS;
    if (l.args.partial) {
        norm_columns_long<T><<<dim3((unsigned)across, (unsigned)blocks), 256, 0, l.stream>>>(l.args);
        st = after_launch("norm_columns_long");
        if (st == TN_SUCCESS) st = finish_partial<S, P>(l, blocks);
        const tn_status freed = scratch_free(l.args.partial, l.stream);
        if (st == TN_SUCCESS) st = freed;
    }
    if (st != TN_SUCCESS) return st;
    norm_backward_long<T, P><<<(unsigned)rows_grid(l.args.rows, 1), kLong, 0, l.stream>>>(l.args);
    return after_launch("norm_backward_long");
}

// ITEMS: vectors a thread holds. A warp takes a row of up to 32 (float64: 16) elements a lane. Element by element the steps are finer: every
// element beyond the row's end costs as much as one within (271 columns of float16 in 16 elements a lane: 33 us for 62447 rows, in 12: 29).
template <typename T, typename P, int VEC>
tn_status launch_sized(Launch& l) {
    const int c = l.args.cols;
    constexpr bool F64 = std::is_same<T, double>::value;
    constexpr int Q = F64 ? 16 / VEC : 32 / VEC;  // vectors of a full thread
    if constexpr (VEC == 1 && !F64) {
        const int each = (c + 31) / 32;
        if (!l.backward) {
            if (each <= 4) return launch_forward<T, P, 1, 4, false>(l);
            if (each <= 12 && each > 8) return launch_forward<T, P, 1, 12, false>(l);
            if (each <= 20 && each > 16) return launch_forward<T, P, 1, 20, false>(l);
        } else {
            if (each <= 4) return launch_backward<T, P, 1, 4, false, true>(l);
            if (each <= 12 && each > 8) return launch_backward<T, P, 1, 12, false, true>(l);
            if (each <= 20 && each > 16) return launch_backward<T, P, 1, 20, false, true>(l);
        }
    }
    if (!l.backward) {
        if (c <= 8 * Q * VEC) return launch_forward<T, P, VEC, Q / 4, false>(l);
        if (c <= 16 * Q * VEC) return launch_forward<T, P, VEC, Q / 2, false>(l);
        if constexpr (Q % 4 == 0)
            if (c <= 24 * Q * VEC) return launch_forward<T, P, VEC, Q / 4 * 3, false>(l);
        if (c <= 32 * Q * VEC) return launch_forward<T, P, VEC, Q, false>(l);
        if (c <= kMost * Q * VEC) return launch_forward<T, P, VEC, Q, true>(l);
    } else {
        if (c <= 8 * Q * VEC) return launch_backward<T, P, VEC, Q / 4, false, true>(l);
        if (c <= 16 * Q * VEC) return launch_backward<T, P, VEC, Q / 2, false, true>(l);
        if constexpr (!F64) {
            if (c <= 24 * Q * VEC) return launch_backward<T, P, VEC, Q / 4 * 3, false, VEC == 1 || sizeof(T) == 4>(l);
            if (c <= kMost * Q / 2 * VEC) return launch_backward<T, P, VEC, Q / 2, true, true>(l);
            if constexpr (VEC > 1)  // element by element the looping kernels are faster: 13531 columns of bfloat16, 5000 rows: 280 us against 640
                if (c <= kMost * Q * VEC) return launch_backward<T, P, VEC, Q, true, false>(l);
        } else {
            if (c <= kMost * Q / 4 * VEC) return launch_backward<T, P, VEC, Q / 4, true, true>(l);
        }
    }
    return launch_long<T, P>(l);
}

template <typename T, typename P>
tn_status launch_typed(Launch& l) {
    constexpr int VEC = 16 / sizeof(T);
    const NormArgs& a = l.args;
    // 16-byte accesses need every row of every operand to start on a 16-byte boundary
    auto fits = [](const void* p, int64_t pitch_bytes) { return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(pitch_bytes)) & 15) == 0; };
    bool wide = a.cols % VEC == 0 && fits(a.x, a.x_pitch * (int64_t)sizeof(T)) && fits(a.y, a.cols * (int64_t)sizeof(T)) && fits(a.weight, 0) && fits(a.bias, 0);
    if (l.backward) wide = wide && fits(a.dy, a.dy_pitch * (int64_t)sizeof(T));
    return wide ? launch_sized<T, P, VEC>(l) : launch_sized<T, P, 1>(l);
}

tn_status launch_any(Launch& l, int dtype, int param_dtype) {
    const bool wide_params = param_dtype == TN_FLOAT32;
    switch (dtype) {
        case TN_FLOAT16: return wide_params ? launch_typed<__half, float>(l) : launch_typed<__half, __half>(l);
        case TN_BFLOAT16: return wide_params ? launch_typed<__nv_bfloat16, float>(l) : launch_typed<__nv_bfloat16, __nv_bfloat16>(l);
        case TN_FLOAT32: return launch_typed<float, float>(l);
        default: return launch_typed<double, double>(l);
    }
}

bool dense(const tn_tensor_t* t) {
    int64_t expect = 1;
    for (int d = t->rank - 1; d >= 0; --d) {
        if (t->shape.sizes[d] != 1 && t->strides.sizes[d] != expect) return false;
        expect *= (int64_t)t->shape.sizes[d];
    }
    return true;
}

// An operand whose rows can be read in place: the last axis contiguous and all rows one pitch apart
// (any pitch, 0 for a broadcast row). Otherwise the view is copied dense into scratch memory first.
struct Rows {
    const void* base = nullptr;
    int64_t pitch = 0;
    void* scratch = nullptr;
};
tn_status rows_of(const tn_tensor_t* t, Rows* out, tn_stream_t stream) {
    const int last = t->rank - 1;
    out->base = t->address;
    out->pitch = (int64_t)t->shape.sizes[last];
    bool one = t->shape.sizes[last] == 1 || t->strides.sizes[last] == 1;
    int64_t expect = 0;
    bool any = false;
    for (int d = last - 1; one && d >= 0; --d) {
        if (t->shape.sizes[d] == 1) continue;
        if (!any) out->pitch = t->strides.sizes[d];
        else one = t->strides.sizes[d] == expect;
        any = true;
        expect = t->strides.sizes[d] * (int64_t)t->shape.sizes[d];
    }
    if (one) return TN_SUCCESS;
    tn_tensor_t copy = *t;
    int64_t run = 1;
    for (int d = last; d >= 0; --d) {
        copy.strides.sizes[d] = run;
        run *= (int64_t)t->shape.sizes[d];
    }
    copy.layout = TN_CONTIGUOUS;
    TN_TRY(scratch_alloc(&out->scratch, t->size * (size_t)dtype_bytes(t->dtype), as_cuda(stream)));
    copy.address = out->scratch;
    out->base = out->scratch;
    out->pitch = (int64_t)t->shape.sizes[last];
    return tn_cpy(t, &copy, stream);
}
tn_status release(Rows* r, cudaStream_t s, tn_status st) {
    if (!r->scratch) return st;
    const tn_status freed = scratch_free(r->scratch, s);
    r->scratch = nullptr;
    return st == TN_SUCCESS ? freed : st;
}

tn_status check_rows(const tn_tensor_t* x, const char* op) {
    if (!x) return fail(TN_ERROR, "%s: null tensor", op);
    if (x->rank < 1) return fail(TN_ERROR, "%s: the input needs an axis to normalise over", op);
    if (!is_float(x->dtype)) return fail(TN_UNSUPPORTED_DTYPE, "%s: dtype %d unsupported", op, (int)x->dtype);
    if (x->environment.kind != TN_DEVICE) return fail(TN_INCOMPATIBLE_DEVICES, "%s: device entry point called with a host tensor (no CPU fallback)", op);
    const size_t cols = x->shape.sizes[x->rank - 1];
    if (cols == 0) return fail(TN_ERROR, "%s: the last axis is empty", op);
    if (cols > (size_t(1) << 30)) return fail(TN_ERROR, "%s: %zu columns, at most 2^30", op, cols);
    return TN_SUCCESS;
}
tn_status same_device(const tn_tensor_t* x, const tn_tensor_t* t, const char* op) {
    if (t->environment.kind != TN_DEVICE || t->environment.resource.device.id != x->environment.resource.device.id)
        return fail(TN_INCOMPATIBLE_DEVICES, "%s: operands must live on one device", op);
    return TN_SUCCESS;
}
tn_status check_like(const tn_tensor_t* x, const tn_tensor_t* t, bool result, const char* op, const char* what) {
    if (!t) return fail(TN_ERROR, "%s: null %s", op, what);
    if (t->dtype != x->dtype) return fail(TN_UNSUPPORTED_DTYPE, "%s: %s has dtype %d, the input %d", op, what, (int)t->dtype, (int)x->dtype);
    bool same = t->rank == x->rank;
    for (int d = 0; same && d < x->rank; ++d) same = t->shape.sizes[d] == x->shape.sizes[d];
    if (!same) return fail(TN_ERROR, "%s: %s must have the input's shape", op, what);
    if (result && !dense(t)) return fail(TN_ERROR, "%s: %s must be dense", op, what);
    return same_device(x, t, op);
}
tn_status check_stat(const tn_tensor_t* x, const tn_tensor_t* t, const char* op, const char* what) {
    const tn_dtype want = x->dtype == TN_FLOAT64 ? TN_FLOAT64 : TN_FLOAT32;
    if (t->dtype != want) return fail(TN_UNSUPPORTED_DTYPE, "%s: %s has dtype %d, expected %d", op, what, (int)t->dtype, (int)want);
    const size_t rows = x->size / x->shape.sizes[x->rank - 1];
    if (t->size != rows) return fail(TN_ERROR, "%s: %s has %zu elements, the input has %zu rows", op, what, t->size, rows);
    if (!dense(t)) return fail(TN_ERROR, "%s: %s must be dense", op, what);
    return same_device(x, t, op);
}
// A parameter row (or its gradient): [columns], contiguous, of the input's dtype or float32 beside 16-bit rows.
tn_status check_param(const tn_tensor_t* x, const tn_tensor_t* t, const char* op, const char* what) {
    if (t->dtype != x->dtype && !(is_half(x->dtype) && t->dtype == TN_FLOAT32))
        return fail(TN_UNSUPPORTED_DTYPE, "%s: %s has dtype %d beside an input of dtype %d", op, what, (int)t->dtype, (int)x->dtype);
    if (t->rank != 1 || t->shape.sizes[0] != x->shape.sizes[x->rank - 1]) return fail(TN_ERROR, "%s: %s must be a vector as long as the last axis", op, what);
    if (!dense(t)) return fail(TN_ERROR, "%s: %s must be contiguous", op, what);
    return same_device(x, t, op);
}

}  // namespace
}  // namespace tnb

using namespace tnb;

extern "C" {

tn_status tn_layer_norm(const tn_tensor_t* x, const tn_tensor_t* weight, const tn_tensor_t* bias, tn_tensor_t* y, tn_tensor_t* mean, tn_tensor_t* rstd,
                        tn_stream_t stream, double eps) {
    const char* op = "layer_norm";
    TN_TRY(check_rows(x, op));
    TN_TRY(check_like(x, y, true, op, "the result"));
    if (weight) TN_TRY(check_param(x, weight, op, "weight"));
    if (bias) TN_TRY(check_param(x, bias, op, "bias"));
    if (weight && bias && weight->dtype != bias->dtype) return fail(TN_UNSUPPORTED_DTYPE, "layer_norm: weight and bias must share a dtype");
    if (mean) TN_TRY(check_stat(x, mean, op, "mean"));
    if (rstd) TN_TRY(check_stat(x, rstd, op, "rstd"));
    if (!(eps >= 0.0)) return fail(TN_ERROR, "layer_norm: eps must not be negative");
    TN_TRY(use_device_of(x));
    if (x->size == 0) return TN_SUCCESS;
    Rows rows;
    tn_status st = rows_of(x, &rows, stream);
    if (st == TN_SUCCESS) {
        Launch l = {};
        l.stream = as_cuda(stream);
        l.backward = false;
        NormArgs& a = l.args;
        a.x = rows.base;
        a.x_pitch = rows.pitch;
        a.weight = weight ? weight->address : nullptr;
        a.bias = bias ? bias->address : nullptr;
        a.y = y->address;
        a.mean = mean ? mean->address : nullptr;
        a.rstd = rstd ? rstd->address : nullptr;
        a.cols = (int)x->shape.sizes[x->rank - 1];
        a.rows = (int64_t)x->size / a.cols;
        a.eps = eps;
        st = launch_any(l, x->dtype, weight ? weight->dtype : bias ? bias->dtype : x->dtype);
    }
    return release(&rows, as_cuda(stream), st);
}

tn_status tn_layer_norm_grad(const tn_tensor_t* dy, const tn_tensor_t* x, const tn_tensor_t* mean, const tn_tensor_t* rstd, const tn_tensor_t* weight,
                             tn_tensor_t* dx, tn_tensor_t* dweight, tn_tensor_t* dbias, tn_stream_t stream) {
    const char* op = "layer_norm_grad";
    TN_TRY(check_rows(x, op));
    TN_TRY(check_like(x, dy, false, op, "the result's gradient"));
    TN_TRY(check_like(x, dx, true, op, "the input's gradient"));
    if (!mean || !rstd) return fail(TN_ERROR, "layer_norm_grad: null statistics");
    TN_TRY(check_stat(x, mean, op, "mean"));
    TN_TRY(check_stat(x, rstd, op, "rstd"));
    if (weight) TN_TRY(check_param(x, weight, op, "weight"));
    if (dweight) TN_TRY(check_param(x, dweight, op, "the weight's gradient"));
    if (dbias) TN_TRY(check_param(x, dbias, op, "the bias's gradient"));
    const int param = weight ? weight->dtype : dweight ? dweight->dtype : dbias ? dbias->dtype : x->dtype;
    if ((dweight && (int)dweight->dtype != param) || (dbias && (int)dbias->dtype != param))
        return fail(TN_UNSUPPORTED_DTYPE, "layer_norm_grad: the parameters and their gradients must share a dtype");
    TN_TRY(use_device_of(x));
    cudaStream_t s = as_cuda(stream);
    if (x->size == 0) {  // no rows: the sums over them are zero
        for (tn_tensor_t* t : {dweight, dbias})
            if (t) TN_CUDA(cudaMemsetAsync(t->address, 0, t->size * (size_t)dtype_bytes(t->dtype), s));
        return TN_SUCCESS;
    }
    Rows rx, rd;
    tn_status st = rows_of(x, &rx, stream);
    if (st == TN_SUCCESS) st = rows_of(dy, &rd, stream);
    if (st == TN_SUCCESS) {
        Launch l = {};
        l.stream = s;
        l.backward = true;
        l.dweight = dweight ? dweight->address : nullptr;
        l.dbias = dbias ? dbias->address : nullptr;
        NormArgs& a = l.args;
        a.x = rx.base;
        a.x_pitch = rx.pitch;
        a.dy = rd.base;
        a.dy_pitch = rd.pitch;
        a.weight = weight ? weight->address : nullptr;
        a.y = dx->address;
        a.mean = mean->address;
        a.rstd = rstd->address;
        a.cols = (int)x->shape.sizes[x->rank - 1];
        a.rows = (int64_t)x->size / a.cols;
        st = launch_any(l, x->dtype, param);
    }
    st = release(&rd, s, st);
    return release(&rx, s, st);
}

}  // extern "C"
