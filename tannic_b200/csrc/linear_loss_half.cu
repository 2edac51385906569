// The gradient of a linear layer's cross entropy for up to sixteen tokens of 16 bits.
//
// With lse known one pass over W does everything: for eight vocabulary rows at a time the logits, d = (exp(logit - lse) - [target]) grad
// from them, then dW = d^T h and dh += d W before the next rows take their place. The bound is memory: W is read once and dW written once.
// The products run as mma.sync with a tile of eight tokens, or two, on one side: tcgen05's smallest tile has 64 rows, reads both operands from shared
// memory, where d would have to be written first, and returns through TMEM, where dW would wait; here d stays in registers from one
// product's result to the next one's operand. Four tokens over 32000 x 4096 bfloat16: 107 us with dh's second kernel, 81 at copy speed (on the
// FP32 pipe the same pass took 136, the products for many tokens take 230); 8 over 131072 x 4096: 366 us, 90 % of copy speed. What is left is
// shared memory's: its pipe is busy 80 % of the time, with W and the tokens read twice a batch (16 tokens, in two tiles,
// over 50257 x 768: 70 us, the products for many tokens 124); a batch of 16 rows would read the tokens
// half as often, but two such batches of 4096 columns do not fit.
//
// A warp owns groups of 32 columns of all rows, fetches them with cp.async, reads each eight rows twice from shared memory (as they lie for
// the logits, transposed for dh) and fetches the next ones in their place, so the only barrier is the one over the warps' parts of the logits.
//   logits [tokens, 8 rows of W]    k = columns. A lane takes 16 bytes of a row of W, columns 8 t .. 8 t + 7 (t = lane % 4); h lies in
//                                   shared memory in the order that makes this the fragment of two steps.
//   dh [columns, 8 tokens]          k = the eight rows, once with d's upper part and once with its lower one.
//   dW [8 rows, columns]            k = the tokens; rows 0 to 7 of the product take d's upper part, rows 8 to 15 its lower one, and the two
//                                   are added. h's order puts eight neighbouring columns into a lane: one store of 16 bytes.
// d is the sum of two values of the operands' type (good to 2^-17 of it for bfloat16, 2^-22 for float16); float16's is relative to the largest
// gradient, like the larger products', and does not lose small ones.
#include <algorithm>

#include "linear_loss.cuh"

namespace tnb {
namespace {

constexpr int kTile = 8, kBatch = 8;    // tokens of a tile, and vocabulary rows at a time
constexpr int kGroup = 32;              // columns
constexpr int kMostGroups = 8;          // of a warp: 64 registers of dh's sums
template <int TILES, int EACH> constexpr int kSlots = TILES * EACH == kMostGroups && TILES == 1 ? 2 : 3;  // what fits beside the tokens

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 v = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&v); }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
};
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __nv_bfloat162 v = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&v); }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }
};

template <typename T>
__device__ __forceinline__ void mma_k16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Rows 0 to 7 and rows 8 to 15 of the product, added.
template <typename T>
__device__ __forceinline__ float2 mma_k8_rows(uint32_t a0, uint32_t a1, uint32_t b) {
    float c[4];
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(b), "f"(0.0f));
    else
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(b), "f"(0.0f));
    return make_float2(c[0] + c[2], c[1] + c[3]);
}
template <typename T>
__device__ __forceinline__ float2 mma_k16_rows(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    float c[4];
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                     : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    return make_float2(c[0] + c[2], c[1] + c[3]);
}
__device__ __forceinline__ void load4(uint32_t (&m)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load4_transposed(uint32_t (&m)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(m[0]), "=r"(m[1]), "=r"(m[2]), "=r"(m[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Bytes between the tokens in shared memory (16 more than a multiple of 64: eight rows fall on different banks) and between W's rows.
constexpr uint32_t h_bytes(int groups) { return groups * 64 + 16; }
constexpr uint32_t w_bytes(int groups) { return groups * 64; }

// EACH groups per warp; a row is taken to have WARPS * EACH of them, zeros behind its end, so that no branch keeps one group's loads from
// running under another's products. DW: with the weights' gradient. SLOTS batches of W lie in shared memory or are on their way there.
template <typename T, int TILES, int WARPS, int EACH, bool DW>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS) half_grad_kernel(const FewTokens p) {
    constexpr bool SCALED = std::is_same<T, __half>::value;
    extern __shared__ __align__(128) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    constexpr int GROUPS = WARPS * EACH, SLOTS = kSlots<TILES, EACH>;
    constexpr uint32_t h_row = h_bytes(GROUPS), w_row = w_bytes(GROUPS), slot_bytes = kBatch * w_row;
    const int group0 = warp * EACH;
    const int left = static_cast<int>(p.hidden) - group0 * kGroup - t * 8;  // columns from this lane's first on; may be negative
    uint8_t* tokens = smem + SLOTS * slot_bytes;
    float2* parts = reinterpret_cast<float2*>(tokens + TILES * kTile * h_row);  // [2][WARPS][TILES][32]
    const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)), hs = ring + SLOTS * slot_bytes;
    if (p.sums) chain_go();

    // Where the 16 bytes `chunk` (0 to 3) of this warp's group i of row r lie. The exchange of chunks by the row's bits, in reverse order, puts
    // both the eight rows of one chunk and two rows of four chunks on different banks.
    auto w_at = [&](int r, int chunk) {
        const int turn = (r & 1) << 2 | (r & 2) | (r >> 2 & 1);
        return ring + static_cast<uint32_t>(r) * w_row + group0 * 64 + (chunk ^ turn) * 16;
    };
    const uint32_t mine = w_at(g, t), matrix = w_at(lane & 7, lane >> 3);
    auto of_group = [](uint32_t at, int i) { return (i & 1 ? at ^ 64 : at) + (i >> 1) * 128; };
    // A copy takes 128 bytes, two groups, of four rows: 64 bytes of eight rows are twice as many transactions (113 us against 106 at 32000 x 4096).
    const int copy_row = lane >> 3, copy_left = static_cast<int>(p.hidden) - group0 * kGroup - (lane & 7) * 8;
    uint32_t copied[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) copied[k] = w_at(copy_row + 4 * k, lane & 7);
    const T* const w_first = static_cast<const T*>(p.w) + group0 * kGroup + (lane & 7) * 8;
    struct Rows { const T* from[2]; int bytes[2]; };
    // rows copy_row and copy_row + 4 of the batch at v; rows behind the last one are zeros
    auto rows_at = [&](int64_t v) {
        Rows r;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const bool row = v + copy_row + 4 * k < p.vocab;
            r.from[k] = w_first + (row ? v + copy_row + 4 * k : 0) * p.w_pitch;
            r.bytes[k] = row ? 16 : 0;
        }
        return r;
    };
    auto fetch = [&](const Rows& r, uint32_t slot, int i) {  // groups 2 i and 2 i + 1
        if (i * 2 * kGroup < copy_left)
#pragma unroll
            for (int k = 0; k < 2; ++k)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(copied[k] + slot + i * 128), "l"(r.from[k] + i * 2 * kGroup), "r"(r.bytes[k]) : "memory");
    };
    auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
    const int64_t step = static_cast<int64_t>(gridDim.x) * kBatch;
    int64_t v0 = static_cast<int64_t>(blockIdx.x) * kBatch;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const Rows rows = rows_at(v0 + s * step);
        // columns behind the row's end are zeros and stay so
#pragma unroll
        for (int i = 0; i < EACH / 2; ++i) {
            fetch(rows, s * slot_bytes, i);
            if (i * 2 * kGroup >= copy_left)
#pragma unroll
                for (int k = 0; k < 2; ++k) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(copied[k] + s * slot_bytes + i * 128), "r"(0) : "memory");
        }
        commit();
    }

    auto target_of = [&](int64_t n) { return p.wide ? static_cast<const int64_t*>(p.targets)[n] : static_cast<int64_t>(static_cast<const int32_t*>(p.targets)[n]); };
    // float16: the largest finite gradient lands at kTop (what is lost where top / kTop is no normal number, float16 cannot hold)
    const bool live = lane < p.tokens && target_of(lane) != p.ignore;
    const unsigned lives = __ballot_sync(0xFFFFFFFFu, live);
    float top = live ? fabsf(p.grad[lane]) : 0.0f;
    if (!isfinite(top)) top = 0.0f;
#pragma unroll
    for (int o = TILES * kTile / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    top = __shfl_sync(0xFFFFFFFFu, top, 0);
    if (top == 0.0f) top = 1.0f;
    const float back = top / kTop;
    // this lane's token of every tile
    bool counts[TILES];
    int64_t target[TILES];
    float lse[TILES], grad[TILES];
#pragma unroll
    for (int j = 0; j < TILES; ++j) {
        const int n = kTile * j + g;
        counts[j] = lives >> n & 1;
        target[j] = counts[j] ? target_of(n) : 0;
        lse[j] = counts[j] ? p.lse[n] : 0.0f;
        grad[j] = !counts[j] ? 0.0f : target[j] < 0 || target[j] >= p.vocab ? NAN : SCALED ? p.grad[n] / top * kTop : p.grad[n];
    }

    // The tokens, zeros where there is none or it does not count: column 8 a + 2 b + c of a group (a, b in 0..3, c in 0..1) at 8 b + 2 a + c.
    {
        struct alignas(16) Eight { uint16_t v[8]; };
        const uint16_t* from = static_cast<const uint16_t*>(p.h);
        const bool vectors = ((reinterpret_cast<uintptr_t>(from) | static_cast<uintptr_t>(p.h_pitch * 2)) & 15) == 0;
        constexpr int chunks = GROUPS * 4;
#pragma unroll 4
        for (int i = threadIdx.x; i < TILES * kTile * chunks; i += WARPS * 32) {
            const int n = i / chunks, k = i - n * chunks;
            Eight e = {};
            if ((lives >> n & 1) && k * 8 < p.hidden) {
                const uint16_t* at = from + n * p.h_pitch + k * 8;
                if (vectors) {
                    e = *reinterpret_cast<const Eight*>(at);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) e.v[j] = at[j];
                }
            }
            uint8_t* to = tokens + n * h_row + (k >> 2) * 64 + (k & 3) * 4;
#pragma unroll
            for (int b = 0; b < 4; ++b) *reinterpret_cast<uint32_t*>(to + b * 16) = e.v[2 * b] | static_cast<uint32_t>(e.v[2 * b + 1]) << 16;
        }
    }
    __syncthreads();

    float dh[EACH][TILES][8];
#pragma unroll
    for (int i = 0; i < EACH; ++i)
#pragma unroll
        for (int j = 0; j < TILES * 8; ++j) dh[i][j / 8][j % 8] = 0.0f;
    const uint32_t h_at = hs + (lane & 7) * h_row + (lane >> 3) * 16 + group0 * 64;  // this lane's row of the four matrices of a group
    uint32_t slot = 0;
    int parity = 0;
    for (; v0 < p.vocab; v0 += step, parity ^= 1) {
        asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 1) : "memory");
        __syncwarp();  // the other lanes' copies
        float sums[2][4] = {};
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            uint32_t a[4], x, y, z, u;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x), "=r"(y), "=r"(z), "=r"(u) : "r"(of_group(mine, i) + slot) : "memory");
            load4(a, h_at + i * 64);
            uint32_t more[4] = {};
            if constexpr (TILES == 2) load4(more, h_at + kTile * h_row + i * 64);
            mma_k16<T>(sums[0], a[0], more[0], a[1], more[1], x, y);
            mma_k16<T>(sums[1], a[2], more[2], a[3], more[3], z, u);
        }
        // token g of a tile, rows 2 t and 2 t + 1; the other parity's were read before the last barrier
#pragma unroll
        for (int j = 0; j < TILES; ++j)
            parts[((parity * WARPS + warp) * TILES + j) * 32 + lane] = make_float2(sums[0][2 * j] + sums[1][2 * j], sums[0][2 * j + 1] + sums[1][2 * j + 1]);
        __syncthreads();
        uint32_t hi[TILES], lo[TILES], hi_rows[TILES], lo_rows[TILES];
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
            float2 x = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < WARPS; ++k) {
                const float2 one = parts[((parity * WARPS + k) * TILES + j) * 32 + lane];
                x.x += one.x;
                x.y += one.y;
            }
            auto d_of = [&](float logit, int64_t v) {
                if (!counts[j] || v >= p.vocab) return 0.0f;
                return (v == target[j] ? expm1f(logit - lse[j]) : __expf(logit - lse[j])) * grad[j];
            };
            const float d0 = d_of(x.x, v0 + 2 * t), d1 = d_of(x.y, v0 + 2 * t + 1);
            hi[j] = Pair<T>::pack(d0, d1);
            const float2 upper = Pair<T>::unpack(hi[j]);
            // an infinity has no rest
            lo[j] = Pair<T>::pack(isinf(upper.x) ? 0.0f : d0 - upper.x, isinf(upper.y) ? 0.0f : d1 - upper.y);
            hi_rows[j] = transposed(hi[j]);  // row g, tokens 2 t and 2 t + 1 of the tile
            lo_rows[j] = transposed(lo[j]);
        }
        T* out = static_cast<T*>(p.dweight) + (v0 + g) * p.hidden + group0 * kGroup + t * 8;
        const int stores = v0 + g < p.vocab ? left : 0;
        const Rows next = rows_at(v0 + SLOTS * step);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            uint32_t m[4];
            load4_transposed(m, of_group(matrix, i) + slot);
            if (i & 1) {
                __syncwarp();  // all lanes have read the two groups: the next rows may take their place
                fetch(next, slot, i / 2);
            }
#pragma unroll
            for (int j = 0; j < TILES; ++j) {
                mma_k16<T>(dh[i][j], m[0], m[1], m[0], m[1], hi[j], lo[j]);
                mma_k16<T>(dh[i][j] + 4, m[2], m[3], m[2], m[3], hi[j], lo[j]);
            }
            if constexpr (DW) {
                uint32_t b[4], more[4], r[4];
                load4_transposed(b, h_at + i * 64);
                if constexpr (TILES == 2) load4_transposed(more, h_at + kTile * h_row + i * 64);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float2 c;
                    if constexpr (TILES == 2) c = mma_k16_rows<T>(hi_rows[0], lo_rows[0], hi_rows[TILES - 1], lo_rows[TILES - 1], b[k], more[k]);
                    else c = mma_k8_rows<T>(hi_rows[0], lo_rows[0], b[k]);
                    r[k] = SCALED ? Pair<T>::pack(c.x * back, c.y * back) : Pair<T>::pack(c.x, c.y);
                }
                if (i * kGroup < stores) *reinterpret_cast<uint4*>(out + i * kGroup) = make_uint4(r[0], r[1], r[2], r[3]);
            }
        }
        commit();
        slot = slot == (SLOTS - 1) * slot_bytes ? 0 : slot + slot_bytes;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (p.sums) {
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
#pragma unroll
            for (int j = 0; j < TILES * 8; ++j) {
                const int64_t c = (group0 + i) * kGroup + (j >> 2 & 1) * 16 + (j >> 1 & 1) * 8 + g;
                const int n = (j >> 3) * kTile + 2 * t + (j & 1);
                const float sum = dh[i][j / 8][j % 8];
                if (n < p.tokens && c < p.hidden) p.sums[(static_cast<int64_t>(blockIdx.x) * p.tokens + n) * p.hidden + c] = SCALED ? sum * back : sum;
            }
        }
    }
}

// ------------------------------------------------------------------ host ---------------
int groups_of(int64_t hidden) { return (int)((hidden + kGroup - 1) / kGroup); }
int tiles_for(int64_t tokens) { return tokens <= kTile ? 1 : 2; }
// Sums of dh of up to 2048 columns (two tiles: 1024) leave room for two blocks of eight warps on an SM, whose barriers cover for one another.
int warps_for(int64_t tokens, int64_t hidden) { return groups_of(hidden) * tiles_for(tokens) <= 8 * kMostGroups ? 8 : 16; }

template <typename T, int TILES, int WARPS, int EACH, bool DW>
tn_status launch(const FewTokens& p, cudaStream_t stream) {
    static thread_local int device = -1;  // the opt-in shared-memory size belongs to kernel and device
    constexpr int GROUPS = WARPS * EACH;
    constexpr size_t smem = kSlots<TILES, EACH> * kBatch * w_bytes(GROUPS) + TILES * kTile * h_bytes(GROUPS) + 2 * WARPS * TILES * 32 * sizeof(float2);
    static_assert(smem <= 227 * 1024 / (16 / WARPS) - (WARPS == 8 ? 1024 : 0), "does not fit");
    auto kernel = half_grad_kernel<T, TILES, WARPS, EACH, DW>;
    int dev = 0;
    TN_CUDA(cudaGetDevice(&dev));
    if (device != dev) {
        TN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        device = dev;
    }
    kernel<<<(unsigned)half_grad_blocks(p), WARPS * 32, smem, stream>>>(p);
    return after_launch("half_grad_kernel");
}
template <typename T, bool DW>
tn_status launch_sized(const FewTokens& p, cudaStream_t stream) {
    const int groups = groups_of(p.hidden);
    if (tiles_for(p.tokens) == 2) {
        if (groups <= 8 * 2) return launch<T, 2, 8, 2, DW>(p, stream);
        return groups <= 8 * 4 ? launch<T, 2, 8, 4, DW>(p, stream) : launch<T, 2, 16, 4, DW>(p, stream);
    }
    if (groups <= 8 * 2) return launch<T, 1, 8, 2, DW>(p, stream);
    if (groups <= 8 * 4) return launch<T, 1, 8, 4, DW>(p, stream);
    if (groups <= 8 * 6) return launch<T, 1, 8, 6, DW>(p, stream);
    if (groups <= 8 * 8) return launch<T, 1, 8, 8, DW>(p, stream);
    return groups <= 16 * 6 ? launch<T, 1, 16, 6, DW>(p, stream) : launch<T, 1, 16, 8, DW>(p, stream);
}
template <typename T>
tn_status launch_typed(const FewTokens& p, cudaStream_t stream) {
    return p.dweight ? launch_sized<T, true>(p, stream) : launch_sized<T, false>(p, stream);
}

}  // namespace

// Sixteen warps hold dh's sums of 4096 columns of eight tokens, or 2048 of sixteen. Rows that are not aligned to 16 bytes take the larger
// products, which copy the weights.
bool half_grad_fits(const FewTokens& p) {
    const bool wide = p.hidden % 8 == 0 && p.w_pitch % 8 == 0 && ((reinterpret_cast<uintptr_t>(p.w) | reinterpret_cast<uintptr_t>(p.dweight)) & 15) == 0;
    return (p.dtype == TN_FLOAT16 || p.dtype == TN_BFLOAT16) && p.tokens <= 2 * kTile && p.hidden * tiles_for(p.tokens) <= 16 * kMostGroups * kGroup && wide;
}
int64_t half_grad_blocks(const FewTokens& p) {
    return std::min<int64_t>((int64_t)p.sms * (16 / warps_for(p.tokens, p.hidden)), ceil_div(p.vocab, kBatch));
}

tn_status half_grad(const FewTokens& p, cudaStream_t stream) {
    TN_TRY(p.dtype == TN_FLOAT16 ? launch_typed<__half>(p, stream) : launch_typed<__nv_bfloat16>(p, stream));
    return p.dhidden ? few_dhidden(p, half_grad_blocks(p), stream) : TN_SUCCESS;
}

}  // namespace tnb
