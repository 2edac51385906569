// Softmax cross entropy of a linear layer over a large vocabulary, and its gradient, without the logits.
//
//   l = h W^T    lse = log sum_v exp(l_v)    loss = lse - l_target
//   d = (exp(l - lse) - onehot(target)) grad      dh = d W      dW = d^T h
//
// The products carry all the work (2 N H V for the loss, 6 N H V for the gradient, N tokens, H hidden, V
// vocabulary) and run on the tensor cores (tcgen05, fp32 accumulation in tensor memory); the [N, V] logits
// exist only as 128 x 256 tiles of tensor memory:
//
//   loss       The epilogue of the product keeps, per row and per half of a tile, the running maximum m and
//              s = sum exp(l - m), and picks the target's logit out of its registers. A small kernel joins the halves
//              of a row: lse = M + log sum s exp(m - M).
//   gradient   The vocabulary is cut into pieces. For each piece the product is formed again (by the same
//              kernel in the same order, so the same logits) and its epilogue writes d, rounded to the operands' type, into a
//              workspace (half a GiB, or 4096 entries of every token where that is more); two more products read it, dW's piece = d^T h and
//              dh += d W's piece, the latter in float32 in memory. Forming the logits again costs
//              2 N H V operations and saves writing, keeping and reading 4 N V bytes.
//
// Tokens without a target (ignore_index) take no part in the gradient: the rows of the others are
// gathered in front, and the products stop at the last one. Their number stays on the device.
//
// float32 operands are written as three bfloat16 parts (24 significand bits), and a product as the six
// products of parts that matter; a 64-wide block of K is six passes over those parts. bfloat16 and float16 are one part. A few tokens
// take kernels of their own (linear_loss.cuh).
//
// d is rounded to the operands' 16-bit type because the tensor cores take operands of one type. It is
// divided by the largest upstream gradient and multiplied by 2^14 first: float16 would lose the small
// probabilities otherwise (grad = 1/N and p = 1/V are below its smallest number), and where all tokens weigh the same, the usual
// mean, their weight is not rounded at all (1/N rounded to bfloat16 would be off by up to 2^-9 in every term
// alike). The results are multiplied back in float32.
//
// Kernel layout: warp 0 TMA producer, warp 1 MMA issuer, warp 2 tensor memory, warps 4..11 epilogue, persistent
// thread blocks, 64-wide K blocks, two accumulators so that the epilogue of a tile runs under the products of the
// next. Bounded waits throughout.
//
// A thread block on its own computes 128 x 256 and takes 48 KiB from L2 for every 64 of K. Two neighbouring SMs work as one
// (cta_group::2): 256 x 256, each SM holding its 128 rows of A and of the accumulator and half of B, 32 KiB for the
// same products, and five stages fit where three did. The even block of the pair issues the products for both; the loads of both report to
// its barriers, and its commits report to both. At full clocks it is the same time (8192 x 4096 by 32768: 1.50 ms against 1.51),
// with a third less traffic under the power cap that long runs meet. Up to 128 rows leave nothing to the second SM and take the single form.
//
// Measured (bfloat16, 8192 tokens, 4096 wide, 131072 entries): the gradient at 1190 TFLOP/s over 22 ms under the power cap, where cuBLAS
// alone, on the same three products, makes 1340; 16-bit loss of 4095 x 768 by 50257: 247 us for 316 GFLOP. The main loop without its
// epilogue reaches 1500 TFLOP/s at burst clocks; the epilogue's exponentials share the SM's power and issue slots with it.
//
// The tensor cores cut off, rather than round, what falls below an accumulator's last place: the more steps of 16 an accumulator takes, the
// further it is off, always towards zero. So one takes only `group` blocks, and the epilogue warps
// add it, in float32, to sums in their registers (128 a thread); its double hides that under the next blocks' products.
// Logits of 4096 products of either sign, rms in units of 2^-24 of theirs: float32 2.8, where the six passes of two blocks go smallest products
// first, so that only the last eight steps find anything to lose (20 with the largest first and 16 passes to an accumulator; the
// same loop on the FP32 pipe, one sum to a thread, 4.8). A group of one: 2.7, but 365 us for the gradient of 512 x 1024 by 14336 against 343
// (groups of three 337 us and 3.2). 16 bits, sixteen blocks: 17 (bfloat16) and 21 (float16), for products of one sign 33 and 93; eight blocks
// halve that and cost 3 to 12 % (8192 x 4096 by 16384: 822 us, 918), four 27 %.
// With the whole tile in registers an accumulator is free as soon as it is read, and the epilogue has 128 independent
// elements a thread to fill the gaps that two warps to a scheduler leave.
// The register split that takes is 40 a thread for warps 0..3 and 232 for the others, of 384 x 168 at launch.
#include <algorithm>

#include "linear_loss.cuh"
#include "tc_common.cuh"

namespace tnb {

tn_status tc_abort_counter(unsigned int** counter);  // of the current device

namespace {

constexpr int kChunks = BN / 64;                           // 32-column chunks of a warp
// A pair of thread blocks on neighbouring SMs (PAIR) shares a tile of 256 x 256: each loads its 128 rows of A and HALF of B.
template <bool PAIR> constexpr int kStages = PAIR ? 5 : 3;
template <bool PAIR> constexpr uint32_t kStageBytes = A_BYTES + (PAIR ? B_BYTES / 2 : B_BYTES);
constexpr int kEpilogueWarps = 8;                          // warps 4..11
constexpr int kThreads = 128 + 32 * kEpilogueWarps;
constexpr uint32_t kBoxBytes = 2048;                       // 32 rows x 64 bytes
constexpr uint32_t kWarpBytes = kChunks * kBoxBytes;       // a box per chunk, or 32 rows x 68 bytes
template <bool PAIR> constexpr uint32_t kSmemBytes = 1024 + kStages<PAIR> * kStageBytes<PAIR> + kEpilogueWarps * kWarpBytes + 256;
static_assert(kSmemBytes<true> <= 232448 && kSmemBytes<false> <= 232448, "exceeds the shared memory of an SM");
constexpr float kLog2e = 1.4426950408889634f;

// A row of the gradient's products: a token with a target, or (target kNoRow) nothing.
struct alignas(16) RowInfo {
    float lse;
    float grad;   // upstream gradient over the largest, times 2^14
    int target;
    int unused;
};
constexpr int kNoRow = -1;
// 64-wide blocks an accumulator takes before it is added up in registers; as many where the operands are float32 in parts; and for the logits
// of up to 128 tokens of 16 bits, where reading W is the time and the additions run under it.
constexpr int kGroup = 16, kGroupParts = 2, kGroupFew = 1;

// Passes over the parts of a float32 operand pair, smallest product first: an accumulator that holds little loses little.
__constant__ int kPartA[6] = {2, 1, 0, 1, 0, 0};
__constant__ int kPartB[6] = {0, 1, 2, 0, 1, 0};

enum { EPI_STATS = 0, EPI_D = 1, EPI_SUM = 2, EPI_RESULT = 3 };
// How the number of tokens that count bounds a product: not at all, its rows, or its K extent.
enum { COUNT_NONE = 0, COUNT_ROWS = 1, COUNT_K = 2 };

struct LossArgs {
    int64_t M, N;            // rows and columns of the result
    int n_tiles;
    int m_tiles;
    int k_blocks;            // 64-wide blocks of K, all splits together
    int most_splits;         // 1: K in one go
    int first_k_blocks;      // of the first piece, whose splits the others must not exceed
    int units;               // thread blocks, or pairs of them, that share the tiles
    int terms;               // 1, or 6 for float32 operands
    int group;               // 64-wide blocks of K that one accumulator takes
    int is_bf16;
    const int* count;        // tokens with a target
    int count_is;
    int64_t vocab0;          // first vocabulary entry of this piece
    // EPI_STATS
    const void* targets;
    int wide_targets;        // int64, else int32
    float2* halves;          // [2 * column tiles of all pieces][M]: maximum, sum of exponentials
    int64_t first_half;
    float* target_logit;     // [M]
    // EPI_D
    const RowInfo* rows;
    // EPI_SUM: add to what is there
    int add;
    // EPI_RESULT
    void* d;
    int64_t ldd;
    const float* scale;
    int tma_store;
    unsigned int* aborts;    // thread blocks that gave up on a bounded wait
};

// ---- a pair of thread blocks -----------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Address of the even block's copy of a shared-memory location.
__device__ __forceinline__ uint32_t in_even_block(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(0));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// A wait that also sees what the other block of the pair did before it arrived.
__device__ __forceinline__ bool mbar_wait_pair(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    for (uint32_t it = 0; it < kSpinLimit; ++it) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if (it >= kSpinFast) {
            if (*abort_flag) return false;
            __nanosleep(64);
        }
    }
    *abort_flag = 1;
    return false;
}
// A load into this block's memory that reports to a barrier of either block.
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t cluster_bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(cluster_bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrives at the barrier of both blocks once the products issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"(static_cast<uint16_t>(3))
        : "memory");
}

// Splits of the vocabulary when dh has `tiles` tiles for `units` blocks or pairs: as many as fill the GPU, each with at least four
// blocks of K. Decided on the device, where the number of tokens that count is known.
struct SplitPlan { int splits, blocks; };
__device__ __forceinline__ SplitPlan plan_splits(int tiles, int units, int k_blocks, int most) {
    int splits = tiles > 0 ? units / tiles : 1;
    splits = max(1, min(min(splits, most), k_blocks / 4));
    const int blocks = (k_blocks + splits - 1) / splits;
    return {(k_blocks + blocks - 1) / blocks, blocks};
}

__device__ __forceinline__ void tma_add_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
        ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

// Boxes of 32 rows x 64 bytes (a lane's row in `w`) on their way to TMA, which clips them at the tensor's edges: one per chunk, filled
// together and sent together, so that the warp waits for the previous tile's boxes only.
struct BoxStore {
    uint8_t* stage;
    const CUtensorMap* map;
    int lane;
    __device__ __forceinline__ void begin() const {
        if (lane == 0) bulk_wait_read_0();  // the boxes sent last have been read
        __syncwarp();
    }
    __device__ __forceinline__ void fill(int i, const uint32_t (&w)[16]) const {
        uint8_t* buf = stage + i * kBoxBytes;
        const int x = (lane >> 1) & 3;  // 64-byte swizzle
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(buf + lane * 64 + ((q ^ x) << 4)) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    }
    template <typename Send>
    __device__ __forceinline__ void send(int n, Send&& one) const {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
            for (int i = 0; i < n; ++i) one(i, smem_u32(stage + i * kBoxBytes));
            bulk_commit();
        }
    }
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// exp(x - base) = power(x) * rest with one multiply-add and one special-function instruction an x: 2^(x log2 e - base log2 e). What
// rounding base log2 e loses, up to 2^-24 of it and the same for every x, is in `rest`.
struct Exponent {
    float shift, rest;
    __device__ __forceinline__ explicit Exponent(float base) {
        shift = -base * kLog2e;
        const float lost = fmaf(base, kLog2e, shift);
        rest = isfinite(lost) ? exp2_approx(-lost) : 1.0f;
    }
    __device__ __forceinline__ float power(float x) const { return exp2_approx(fmaf(x, kLog2e, shift)); }
};

// exp(x - base) of two x, with the rounding of the difference like any float32 form and three more: t log2 e as the sum of two float32, log2 e
// itself as two, exp(t) = 2^hi 2^lo = 2^hi (1 + lo ln 2). In pairs this costs about half of what expf does: the
// gradient of 2000 x 512 by 30000, 1.32 ms, is 6 % longer than with Exponent, with expf 11 %; from 1024 columns on neither shows.
// Below -200 everything is zero; NaN stays.
__device__ __forceinline__ float2 exp_of_difference(float2 x, float base) {
    constexpr float kLog2eRest = static_cast<float>(1.4426950408889634 - static_cast<double>(kLog2e)), kLn2 = 0.6931471805599453f;
    float2 t = add2(x, make_float2(-base, -base));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(t.x) : "f"(-200.0f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(t.y) : "f"(-200.0f));
    const float2 hi = mul2(t, make_float2(kLog2e, kLog2e));
    float2 lo = fma2(t, make_float2(kLog2e, kLog2e), make_float2(-hi.x, -hi.y));
    lo = fma2(t, make_float2(kLog2eRest, kLog2eRest), lo);
    const float2 p = make_float2(exp2_approx(hi.x), exp2_approx(hi.y));
    return fma2(mul2(p, make_float2(kLn2, kLn2)), lo, p);
}

// x as bfloat16 (whose exponent range is float32's), the largest number where rounding would leave the range.
__device__ __forceinline__ float first_part(float x) {
    const float p = __bfloat162float(__float2bfloat16_rn(x));
    return isinf(p) && !isinf(x) ? copysignf(__uint_as_float(0x7F7F0000u), x) : p;
}
// x = p0 + p1 + p2, each part a bfloat16. An infinity or NaN stays in p0.
__device__ __forceinline__ void three_parts(float x, float& p0, float& p1, float& p2) {
    p0 = first_part(x);
    const float r = isfinite(x) ? x - p0 : 0.0f;
    p1 = __bfloat162float(__float2bfloat16_rn(r));
    p2 = r - p1;  // at most 8 significand bits are left; rounded when it is packed
}

// A_M: A is stored [K, M] (M contiguous), else [M, K]. B_N: B is stored [K, N], else [N, K]. T: operand type (bfloat16 parts
// for float32). OUT: result type of EPI_RESULT. PARTS: parts of d that EPI_D writes.
template <bool A_M, bool B_N, int EPI, typename T, typename OUT, int PARTS, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1)
loss_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_d, const LossArgs g) {
    constexpr int STAGES = kStages<PAIR>, ROWS = PAIR ? 2 * BM : BM;  // rows of a tile
    constexpr int B_COLS = PAIR ? BN / 2 : BN;                        // columns of B that this block loads
    constexpr uint32_t STAGE = kStageBytes<PAIR>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;  // swizzled tiles need 1024-byte alignment
    uint8_t* base_ptr = smem_raw + (base - raw);
    uint8_t* staging_ptr = base_ptr + STAGES * STAGE;
    const uint32_t bars = base + STAGES * STAGE + kEpilogueWarps * kWarpBytes;
    // barriers of 8 bytes: full[STAGES], empty[STAGES], accumulator full[2], accumulator empty[2]
    const uint32_t full0 = bars, empty0 = bars + 8 * STAGES, accf0 = bars + 16 * STAGES, acce0 = accf0 + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(staging_ptr + kEpilogueWarps * kWarpBytes + 16 * STAGES + 32);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = PAIR ? static_cast<int>(cluster_rank()) : 0;
    const uint32_t unit = PAIR ? blockIdx.x >> 1 : blockIdx.x, units = PAIR ? gridDim.x >> 1 : gridDim.x;
    auto wait = [&](uint32_t bar, uint32_t parity) { return PAIR ? mbar_wait_pair(bar, parity, abort_flag) : mbar_wait(bar, parity, abort_flag); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(accf0 + 8 * b, 1);
            mbar_init(acce0 + 8 * b, PAIR ? 2 * kEpilogueWarps : kEpilogueWarps);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();  // the other block's barriers exist before anything reports to them
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    // everything above ran under the kernel before this one; from here on its results are there
    chain_wait();
    if constexpr (EPI != EPI_RESULT) chain_go();  // that one may be the last of its call
    // the tokens that count bound the rows or the K extent
    int m_tiles = g.m_tiles, k_blocks = g.k_blocks;
    if (g.count_is != COUNT_NONE) {
        const int count = *g.count;
        if (g.count_is == COUNT_ROWS) m_tiles = (count + ROWS - 1) / ROWS;
        else k_blocks = (count + BK - 1) / BK;
    }
    SplitPlan plan = {1, k_blocks};
    if (g.most_splits > 1) {
        const int tiles = m_tiles * g.n_tiles;
        plan = plan_splits(tiles, g.units, k_blocks, plan_splits(tiles, g.units, g.first_k_blocks, g.most_splits).splits);
    }
    const uint32_t per_split = static_cast<uint32_t>(m_tiles) * static_cast<uint32_t>(g.n_tiles);
    const uint32_t total = per_split * static_cast<uint32_t>(plan.splits);
    // K blocks [first, first + n) of split z
    auto split_range = [&](int z, int& first, int& n) {
        first = z * plan.blocks;
        n = min(k_blocks - first, plan.blocks);
    };

    // all four warps of a group take part, so this comes before the roles
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 0) {
            // ------------------------------------------------------------ TMA producer ----
            if (lane == 0) {
                uint32_t it = 0;
                bool ok = true;
                for (uint32_t t = unit; ok && t < total; t += units) {
                    int z, mt, nt, first, blocks;
                    tile_coords(t, m_tiles, g.n_tiles, z, mt, nt);
                    split_range(z, first, blocks);
                    const int row = mt * ROWS + rank * BM, col = nt * BN + rank * B_COLS;  // what this block loads
                    // the blocks of one accumulator, once for every term
                    const int last = first + blocks;
                    for (int kb0 = first; ok && kb0 < last; kb0 += g.group) {
                        const int kb1 = min(kb0 + g.group, last);
                        for (int term = 0; ok && term < g.terms; ++term) {
                            const int pa = g.terms > 1 ? kPartA[term] : 0, pb = g.terms > 1 ? kPartB[term] : 0;
                            for (int kb = kb0; kb < kb1; ++kb, ++it) {
                                const int s = it % STAGES;
                                if (!wait(empty0 + 8 * s, ((it / STAGES) & 1) ^ 1)) { ok = false; break; }
                                const uint32_t sa = base + s * STAGE, sb = sa + A_BYTES;
                                uint32_t bar = full0 + 8 * s;
                                if (rank == 0) mbar_expect_tx(bar, PAIR ? 2 * STAGE : STAGE);
                                if constexpr (PAIR) bar = in_even_block(bar);
                                auto load = [&](uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2) {
                                    if constexpr (PAIR) tma_load_3d_pair(dst, map, bar, c0, c1, c2);
                                    else tma_load_3d(dst, map, bar, c0, c1, c2);
                                };
                                if constexpr (A_M) {
#pragma unroll
                                    for (int c = 0; c < BM / 64; ++c) load(sa + c * (64 * BK * 2), &map_a, row + c * 64, kb * BK, pa);
                                } else {
                                    load(sa, &map_a, kb * BK, row, pa);
                                }
                                if constexpr (B_N) {
#pragma unroll
                                    for (int c = 0; c < B_COLS / 64; ++c) load(sb + c * (64 * BK * 2), &map_b, col + c * 64, kb * BK, pb);
                                } else {
                                    load(sb, &map_b, kb * BK, col, pb);
                                }
                            }
                        }
                    }
                }
                if constexpr (PAIR) {
                    // the commits that free the last stages have arrived here before this block may go
                    for (uint32_t i = it > STAGES ? it - STAGES : 0; ok && i < it; ++i) ok = wait(empty0 + 8 * (i % STAGES), (i / STAGES) & 1);
                }
                if (!ok) {
                    // transactions that were already issued land before the shared memory goes away
                    for (int spin = 0; spin < 4096; ++spin) __nanosleep(64);
                }
            }
        } else if (warp == 1) {
            // ------------------------------------------------------------ MMA issuer ------
            if (lane == 0 && rank == 0) {
                // D = F32 (bits 4-5), A and B format (7-9, 10-12: 0 = F16, 1 = BF16), A and B stored with M / N contiguous (15, 16),
                // N >> 3 (17-22), M >> 4 (24-28)
                const uint32_t fmt = g.is_bf16 ? 1u : 0u;
                const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((A_M ? 1u : 0u) << 15) | ((B_N ? 1u : 0u) << 16) |
                                       (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>(ROWS >> 4) << 24);
                uint32_t it = 0, local = 0;
                bool ok = true;
                for (uint32_t t = unit; ok && t < total; t += units) {
                    int z, mt, nt, first, blocks;
                    tile_coords(t, m_tiles, g.n_tiles, z, mt, nt);
                    split_range(z, first, blocks);
                    const int steps = blocks * g.terms, period = g.group * g.terms;
                    for (int i0 = 0; ok && i0 < steps; i0 += period, ++local) {
                        const int buf = local & 1;
                        if (!wait(acce0 + 8 * buf, ((local >> 1) & 1) ^ 1)) { ok = false; break; }
                        tc_fence_after();
                        const uint32_t acc = tmem_base + buf * BN;
                        const int i1 = min(steps, i0 + period);
                        for (int i = i0; i < i1; ++i, ++it) {
                            const int s = it % STAGES;
                            if (!wait(full0 + 8 * s, (it / STAGES) & 1)) { ok = false; break; }
                            tc_fence_after();
                            const uint32_t sa = base + s * STAGE, sb = sa + A_BYTES;
#pragma unroll
                            for (int k = 0; k < BK / UMMA_K; ++k) {
                                // K contiguous: 32 bytes further along the swizzled row; else 16 rows of 128 bytes further, 64-wide boxes 8 KiB apart
                                const uint64_t da = A_M ? smem_desc(sa + k * UMMA_K * 128, 64 * BK * 2, 1024) : smem_desc(sa + k * UMMA_K * 2, 16, 1024);
                                const uint64_t db = B_N ? smem_desc(sb + k * UMMA_K * 128, 64 * BK * 2, 1024) : smem_desc(sb + k * UMMA_K * 2, 16, 1024);
                                if constexpr (PAIR) umma_f16_pair(acc, da, db, idesc, (i > i0 || k > 0) ? 1u : 0u);
                                else umma_f16(acc, da, db, idesc, (i > i0 || k > 0) ? 1u : 0u);
                            }
                            // frees the stage once these MMAs have read it
                            if constexpr (PAIR) umma_commit_pair(empty0 + 8 * s);
                            else umma_commit(empty0 + 8 * s);
                        }
                        if (ok) {
                            if constexpr (PAIR) umma_commit_pair(accf0 + 8 * buf);
                            else umma_commit(accf0 + 8 * buf);
                        }
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue --------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int ew = warp - 4;
        const int quarter = warp & 3;  // tensor-memory lanes [32 * quarter, 32 * quarter + 32)
        const int half = ew >> 2;      // this warp takes the 32-column chunks half, half + 2, ...
        BoxStore box = {staging_ptr + ew * kWarpBytes, &map_d, lane};
        const float scale = EPI == EPI_RESULT ? *g.scale : 1.0f;
        uint32_t local = 0;
        bool ok = true;
        for (uint32_t t = unit; ok && t < total; t += units) {
            int z, mt, nt, first, blocks;
            tile_coords(t, m_tiles, g.n_tiles, z, mt, nt);
            split_range(z, first, blocks);
            const int64_t row0 = static_cast<int64_t>(mt) * ROWS + rank * BM + quarter * 32, row = row0 + lane;
            const int64_t col0 = static_cast<int64_t>(nt) * BN;
            const int rows = static_cast<int>(max(int64_t(0), min(int64_t(32), g.M - row0)));
            const int cols = static_cast<int>(min(int64_t(BN), g.N - col0));
            // this warp's chunks that hold anything: chunk i starts at column 64 i + 32 half of the tile
            const int chunks = rows > 0 ? (cols - 32 * half + 63) >> 6 : 0;  // warp-uniform
            const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * 32;
            // The accumulators, added up: v[i][j] is column 64 i + 32 half + j of this lane's row. No steps at all (no token counts) leave zero.
            float v[kChunks][32];
#pragma unroll
            for (int i = 0; i < kChunks; ++i)
#pragma unroll
                for (int j = 0; j < 32; ++j) v[i][j] = 0.0f;
            for (int i0 = 0; i0 < blocks; i0 += g.group, ++local) {
                const int buf = local & 1;
                if (!wait(accf0 + 8 * buf, (local >> 1) & 1)) { ok = false; break; }
                tc_fence_after();
                // two chunks at a time, so that one load runs under the other
#pragma unroll
                for (int i = 0; i < kChunks; i += 2) {
                    if (i < chunks) {
                        uint32_t x[32], y[32];
                        tmem_load_issue(lanes + buf * BN + i * 64, x);
                        tmem_load_issue(lanes + buf * BN + (i + 1) * 64, y);
                        tmem_load_wait(x);
                        tmem_load_wait(y);
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            v[i][j] += __uint_as_float(x[j]);
                            v[i + 1][j] += __uint_as_float(y[j]);
                        }
                    }
                }
                // this warp has finished reading the accumulator: tell the block that issues the products
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) mbar_arrive_remote(in_even_block(acce0 + 8 * buf));
                    else mbar_arrive(acce0 + 8 * buf);
                }
            }
            if (!ok) break;
            if constexpr (EPI == EPI_STATS) {
                // where this row's target lies within the tile (anywhere outside when it has none here)
                int64_t target = -1;
                if (lane < rows) {
                    target = g.wide_targets ? static_cast<const int64_t*>(g.targets)[row] : static_cast<const int32_t*>(g.targets)[row];
                    target -= g.vocab0 + col0 + 32 * half;
                }
                const int at = target >= 0 && target < cols - 32 * half && ((target >> 5) & 1) == 0 ? static_cast<int>(target) : -1;
                if (chunks > 0) {
                    if (cols < BN) {  // warp-uniform: what lies behind the vocabulary's end has no weight
#pragma unroll
                        for (int i = 0; i < kChunks; ++i)
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (64 * i + 32 * half + j >= cols) v[i][j] = -INFINITY;
                    }
                    // independent maxima and sums for every chunk: with two warps to a scheduler, chains are what costs
                    float top[kChunks], s[kChunks];
#pragma unroll
                    for (int i = 0; i < kChunks; ++i) {
                        top[i] = v[i][0];
#pragma unroll
                        for (int j = 1; j < 32; ++j) top[i] = fmaxf(top[i], v[i][j]);
                        s[i] = 0.0f;
                    }
                    const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                    const Exponent e(m == -INFINITY ? 0.0f : m);  // nothing but -inf: the sum stays 0
#pragma unroll
                    for (int j = 0; j < 32; ++j)
#pragma unroll
                        for (int i = 0; i < kChunks; ++i) s[i] += e.power(v[i][j]);
                    if (lane < rows) {
                        g.halves[(g.first_half + 2 * nt + half) * g.M + row] = make_float2(m, ((s[0] + s[1]) + (s[2] + s[3])) * e.rest);
                        if (at >= 0) {
                            float hit = 0.0f;
#pragma unroll
                            for (int i = 0; i < kChunks; ++i)
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (at == 64 * i + j) hit = v[i][j];
                            g.target_logit[row] = hit;
                        }
                    }
                } else if (lane < rows) {
                    g.halves[(g.first_half + 2 * nt + half) * g.M + row] = make_float2(-INFINITY, 0.0f);
                }
            } else if constexpr (EPI == EPI_D) {
                RowInfo info = {0.0f, 0.0f, kNoRow, 0};
                if (lane < rows) info = g.rows[row];
                const int64_t target = info.target >= 0 ? info.target - g.vocab0 - col0 - 32 * half : -1;
                const int at = target >= 0 && target < cols - 32 * half && ((target >> 5) & 1) == 0 ? static_cast<int>(target) : -1;
                if (chunks > 0) {
                    float hit = 0.0f;
                    if (at >= 0) {
#pragma unroll
                        for (int i = 0; i < kChunks; ++i)
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (at == 64 * i + j) hit = v[i][j];
                        // p - 1 without cancellation: the gradient of a token that is almost certain
                        hit = expm1f(hit - info.lse) * info.grad;
                    }
                    const Exponent e(info.lse);
                    const float by = info.grad * e.rest;
#pragma unroll
                    for (int i = 0; i < kChunks; ++i)
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            // 16 bits hide what the short form leaves, a unit of 2^-24 for every one of |l - lse|; float32 does not
                            if constexpr (PARTS == 1) {
                                v[i][j] = e.power(v[i][j]) * by;
                                v[i][j + 1] = e.power(v[i][j + 1]) * by;
                            } else {
                                const float2 p = mul2(exp_of_difference(make_float2(v[i][j], v[i][j + 1]), info.lse), make_float2(info.grad, info.grad));
                                v[i][j] = p.x;
                                v[i][j + 1] = p.y;
                            }
                        }
                    if (info.target == kNoRow) {
#pragma unroll
                        for (int i = 0; i < kChunks; ++i)
#pragma unroll
                            for (int j = 0; j < 32; ++j) v[i][j] = 0.0f;  // whatever the logits are
                    }
                    if (at >= 0) {
#pragma unroll
                        for (int i = 0; i < kChunks; ++i)
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (at == 64 * i + j) v[i][j] = hit;
                    }
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        box.begin();
#pragma unroll
                        for (int i = 0; i < kChunks; ++i) {
                            uint32_t w[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                float &lo = v[i][2 * j], &hi = v[i][2 * j + 1];
                                if constexpr (PARTS == 1) {
                                    w[j] = pack2<T>(lo, hi);
                                } else {
                                    // one part goes out, what it leaves stays for the next
                                    const float a = first_part(lo), b = first_part(hi);
                                    w[j] = pack2<T>(a, b);
                                    lo = isfinite(lo) ? lo - a : 0.0f;
                                    hi = isfinite(hi) ? hi - b : 0.0f;
                                }
                            }
                            box.fill(i, w);
                        }
                        box.send(chunks, [&](int i, uint32_t from) { tma_store_3d(&map_d, from, static_cast<int>(col0) + 64 * i + 32 * half, static_cast<int>(row0), p); });
                    }
                }
            } else if constexpr (EPI == EPI_SUM) {
                if (chunks > 0) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {  // 16 columns of each chunk are 64 bytes
                        box.begin();
#pragma unroll
                        for (int i = 0; i < kChunks; ++i) {
                            uint32_t w[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(v[i][16 * q + j]);
                            box.fill(i, w);
                        }
                        box.send(chunks, [&](int i, uint32_t from) {
                            const int x = static_cast<int>(col0) + 64 * i + 32 * half + 16 * q;
                            if (x >= g.N) return;
                            if (g.add) tma_add_3d(&map_d, from, x, static_cast<int>(row0), z);
                            else tma_store_3d(&map_d, from, x, static_cast<int>(row0), z);
                        });
                    }
                }
            } else if (chunks > 0) {
                constexpr bool F32 = std::is_same<OUT, float>::value;
#pragma unroll
                for (int i = 0; i < kChunks; ++i)
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[i][j] = unscale(v[i][j], scale);
                if (g.tma_store) {
#pragma unroll
                    for (int q = 0; q < (F32 ? 2 : 1); ++q) {
                        box.begin();
#pragma unroll
                        for (int i = 0; i < kChunks; ++i) {
                            uint32_t w[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                if constexpr (F32) w[j] = __float_as_uint(v[i][16 * q + j]);
                                else w[j] = pack2<OUT>(v[i][2 * j], v[i][2 * j + 1]);
                            }
                            box.fill(i, w);
                        }
                        box.send(chunks, [&](int i, uint32_t from) {
                            const int x = static_cast<int>(col0) + 64 * i + 32 * half + 16 * q;
                            if (x < g.N) tma_store_3d(&map_d, from, x, static_cast<int>(row0), 0);
                        });
                    }
                } else {
                    // any alignment: through shared memory so that a store instruction runs along a row
                    float* mine = reinterpret_cast<float*>(box.stage);
#pragma unroll
                    for (int i = 0; i < kChunks; ++i)
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            __syncwarp();
#pragma unroll
                            for (int j = 0; j < 16; ++j) mine[lane * 17 + j] = v[i][16 * q + j];
                            __syncwarp();
                            const int64_t col = col0 + 64 * i + 32 * half + 16 * q + (lane & 15);
                            if (i < chunks && col < g.N)
                                for (int r = lane >> 4; r < rows; r += 2)
                                    static_cast<OUT*>(g.d)[(row0 + r) * g.ldd + col] = from_compute<OUT, float>(mine[r * 17 + (lane & 15)]);
                        }
                }
            }
        }
        if (lane == 0) bulk_wait_all();  // shared memory stays valid until the last box has left
    }

    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();  // neither block goes while the other may still report to it
    if (warp == 2) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
    if (threadIdx.x == 0 && *abort_flag) atomicAdd(g.aborts, 1u);
}

// Joins the halves of a row: R rows per block (32, or 1 when there are few), the halves of a row spread over 1024 / R threads. A
// thread takes eight at a time, so that eight loads are in flight and one maximum serves eight exponentials.
template <int R>
__global__ void __launch_bounds__(1024) loss_join(const float2* halves, int64_t n_halves, int64_t rows, const float* target_logit,
                                                  const void* targets, int wide, int64_t ignore, int64_t vocab, float* __restrict__ loss, float* __restrict__ lse) {
    __shared__ float2 part[32][33];
    chain_wait();
    constexpr int STEP = 1024 / R;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * R + threadIdx.x % R;
    float m = -INFINITY, s = 0.0f;
    if (row < rows) {
        for (int64_t i0 = threadIdx.x / R; i0 < n_halves; i0 += 8 * STEP) {
            float2 p[8];
            float top = m;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                p[q] = i0 + q * STEP < n_halves ? halves[(i0 + q * STEP) * rows + row] : make_float2(-INFINITY, 0.0f);
                top = fmaxf(top, p[q].x);
            }
            const float base = top == -INFINITY ? 0.0f : top;
            s *= __expf(m - base);
#pragma unroll
            for (int q = 0; q < 8; ++q) s += p[q].y * __expf(p[q].x - base);
            m = top;
        }
    }
    auto across = [&](float& top, float& sum) {  // over the lanes of a warp
        float all = top;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
        sum *= __expf(top - (all == -INFINITY ? 0.0f : all));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        top = all;
    };
    int64_t out;
    if constexpr (R == 32) {
        part[warp][lane] = make_float2(m, s);
        __syncthreads();
        m = part[lane][warp].x;  // lane: which share of the halves, warp: which row
        s = part[lane][warp].y;
        across(m, s);
        out = static_cast<int64_t>(blockIdx.x) * 32 + warp;
    } else {
        across(m, s);
        if (lane == 0) part[0][warp] = make_float2(m, s);
        __syncthreads();
        if (warp > 0) return;
        m = part[0][lane].x;
        s = part[0][lane].y;
        across(m, s);
        out = blockIdx.x;
    }
    if (lane == 0 && out < rows) {
        const float z = m + logf(s);
        const int64_t target = wide ? static_cast<const int64_t*>(targets)[out] : static_cast<const int32_t*>(targets)[out];
        if (lse) lse[out] = z;
        if (loss) loss[out] = target == ignore ? 0.0f : target < 0 || target >= vocab ? NAN : z - target_logit[out];
    }
}

// The rows of the gradient's products. Token i goes to row slot[i] where it has a target; the others fill the
// rows behind (slot[i] = -1 - row), as rows of nothing. Every block counts all targets for itself (they lie
// in L2), so there is no order between blocks to wait for.
__global__ void __launch_bounds__(256) loss_rows(const void* targets, int wide, int64_t n, const float* __restrict__ grad, const float* __restrict__ lse, int64_t ignore,
                                                 int64_t vocab, int per_block, RowInfo* __restrict__ info, int* __restrict__ slot, int* __restrict__ count,
                                                 float* __restrict__ scale) {
    __shared__ int ints[3][8];
    __shared__ float tops[8];
    chain_wait();
    chain_go();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * per_block;
    auto target_of = [&](int64_t i) { return wide ? static_cast<const int64_t*>(targets)[i] : static_cast<int64_t>(static_cast<const int32_t*>(targets)[i]); };
    int before = 0, all = 0;
    float top = 0.0f;
#pragma unroll 4
    for (int64_t i = tid; i < n; i += 256) {
        const bool one = target_of(i) != ignore;
        const float a = fabsf(grad[i]);
        all += one;
        before += one && i < n0;
        if (one && isfinite(a)) top = fmaxf(top, a);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        before += __shfl_xor_sync(0xFFFFFFFFu, before, o);
        all += __shfl_xor_sync(0xFFFFFFFFu, all, o);
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    }
    const int64_t mine = n0 + tid;
    const bool here = tid < per_block && mine < n;
    const int64_t target = here ? target_of(mine) : 0;
    const bool counts = here && target != ignore;
    const unsigned votes = __ballot_sync(0xFFFFFFFFu, counts);
    if (lane == 0) {
        ints[0][warp] = before;
        ints[1][warp] = all;
        ints[2][warp] = __popc(votes);
        tops[warp] = top;
    }
    __syncthreads();
    before = all = 0;
    top = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        before += ints[0][w] + (w < warp ? ints[2][w] : 0);
        all += ints[1][w];
        top = fmaxf(top, tops[w]);
    }
    before += __popc(votes & ((1u << lane) - 1u));
    if (top == 0.0f) top = 1.0f;
    if (here) {
        const int row = counts ? before : all + static_cast<int>(mine - before);
        slot[mine] = counts ? row : -1 - row;
        RowInfo r = {0.0f, 0.0f, kNoRow, 0};
        if (counts) {
            r.lse = lse[mine];
            const bool inside = target >= 0 && target < vocab;
            r.grad = inside ? grad[mine] / top * kTop : NAN;  // a target outside the vocabulary has no gradient
            r.target = inside ? static_cast<int>(target) : -2;
        }
        info[row] = r;
    }
    if (blockIdx.x == 0 && tid == 0) {
        *count = all;
        *scale = top;
    }
}

// Rows of an operand as the products read them: a multiple of 8 elements long (zeros behind the last), 16-byte aligned, in
// order, or row r at slot[r] (zeros where that is negative: row -1 - slot[r]); float32 as three parts of bfloat16.
template <typename T>
__global__ void __launch_bounds__(256) pack_rows(const T* __restrict__ src, int64_t pitch, int64_t rows, int64_t cols, int64_t padded, uint16_t* __restrict__ dst,
                                                 int64_t part_stride, const int* slot, int vectors) {
    chain_wait();
    chain_go();
    const int64_t groups = padded / 8, n = rows * groups;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = i / groups, c = (i - r * groups) * 8;
        int64_t to = r;
        bool zero = false;
        if (slot) {
            const int at = slot[r];
            zero = at < 0;
            to = zero ? -1 - at : at;
        }
        alignas(16) T x[8];
        if (!zero && vectors && c + 8 <= cols) {
#pragma unroll
            for (int q = 0; q < static_cast<int>(sizeof(T)) / 2; ++q) reinterpret_cast<uint4*>(x)[q] = reinterpret_cast<const uint4*>(src + r * pitch + c)[q];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = !zero && c + j < cols ? src[r * pitch + c + j] : T(0);
        }
        uint16_t* out = dst + to * padded + c;
        if constexpr (std::is_same<T, float>::value) {
            uint32_t w[3][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float lo[3], hi[3];
                three_parts(x[2 * j], lo[0], lo[1], lo[2]);
                three_parts(x[2 * j + 1], hi[0], hi[1], hi[2]);
#pragma unroll
                for (int p = 0; p < 3; ++p) w[p][j] = pack2<__nv_bfloat16>(lo[p], hi[p]);
            }
#pragma unroll
            for (int p = 0; p < 3; ++p) *reinterpret_cast<uint4*>(out + p * part_stride) = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
        } else {
            *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(x);
        }
    }
}

// dh: the float32 sums of the splits, added in order, scaled back, and put where the tokens stand. VEC: 4 where the rows of the
// result start on boundaries of four elements, else 1.
template <typename T, int VEC>
__global__ void __launch_bounds__(256) loss_dhidden(const float* sums, const int* count, int tile_rows, int n_tiles, int units, int k_blocks,
                                                    int most_splits, int64_t rows, int64_t cols, int64_t padded, const int* slot, const float* scale, T* out) {
    struct alignas(sizeof(T) * VEC) Result { T v[VEC]; };
    struct alignas(sizeof(float) * VEC) Sums { float v[VEC]; };
    constexpr int ROWS = 4;  // a thread's rows, their loads in flight together
    chain_wait();
    const float by = *scale;
    const int splits = plan_splits((*count + tile_rows - 1) / tile_rows * n_tiles, units, k_blocks, most_splits).splits;  // of the first piece
    const int64_t c = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * VEC;
    if (c >= cols) return;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.y) * ROWS; r0 < rows; r0 += static_cast<int64_t>(gridDim.y) * ROWS) {
        int at[ROWS];
        Sums total[ROWS];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            at[k] = r0 + k < rows ? slot[r0 + k] : -1;
#pragma unroll
            for (int j = 0; j < VEC; ++j) total[k].v[j] = 0.0f;
        }
        for (int z = 0; z < splits; ++z) {
            Sums one[ROWS];
#pragma unroll
            for (int k = 0; k < ROWS; ++k)
                if (at[k] >= 0) one[k] = *reinterpret_cast<const Sums*>(sums + (z * rows + at[k]) * padded + c);
#pragma unroll
            for (int k = 0; k < ROWS; ++k)
                if (at[k] >= 0) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) total[k].v[j] += one[k].v[j];
                }
        }
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            if (r0 + k < rows) {
                Result res;
#pragma unroll
                for (int j = 0; j < VEC; ++j) res.v[j] = from_compute<T, float>(at[k] >= 0 ? unscale(total[k].v[j], by) : 0.0f);
                *reinterpret_cast<Result*>(out + (r0 + k) * cols + c) = res;
            }
        }
    }
}

// ------------------------------------------------------------------ host ---------------
// Memory of one call, all of it released together.
struct Scratch {
    cudaStream_t stream;
    void* held[16];
    int n = 0;
    explicit Scratch(cudaStream_t s) : stream(s) {}
    template <typename P>
    tn_status take(P** out, size_t bytes) {
        if (n == 16) return fail(TN_ERROR, "linear_cross_entropy: too many workspaces");
        void* p = nullptr;
        TN_TRY(scratch_alloc(&p, bytes, stream));
        held[n++] = p;
        *out = static_cast<P*>(p);
        return TN_SUCCESS;
    }
    tn_status release(tn_status st) {
        while (n > 0) {
            const tn_status freed = scratch_free(held[--n], stream);
            if (st == TN_SUCCESS) st = freed;
        }
        return st;
    }
};

bool is_dense(const tn_tensor_t* t) {
    int64_t expect = 1;
    for (int d = t->rank - 1; d >= 0; --d) {
        if (t->shape.sizes[d] != 1 && t->strides.sizes[d] != expect) return false;
        expect *= (int64_t)t->shape.sizes[d];
    }
    return true;
}

// Address of a dense tensor with t's elements: t itself or a copy.
tn_status densely(const tn_tensor_t* t, const void** out, Scratch& mem, tn_stream_t stream) {
    *out = t->address;
    if (is_dense(t)) return TN_SUCCESS;
    tn_tensor_t copy = *t;
    int64_t run = 1;
    for (int d = t->rank - 1; d >= 0; --d) {
        copy.strides.sizes[d] = run;
        run *= (int64_t)t->shape.sizes[d];
    }
    copy.layout = TN_CONTIGUOUS;
    TN_TRY(mem.take(&copy.address, t->size * (size_t)dtype_bytes(t->dtype)));
    *out = copy.address;
    return tn_cpy(t, &copy, stream);
}

// A matrix of rows, read in place where its last axis is contiguous and its rows are one pitch apart.
struct RowsIn {
    const void* base;
    int64_t pitch;
};
tn_status rows_in(const tn_tensor_t* t, RowsIn* out, Scratch& mem, tn_stream_t stream) {
    const int last = t->rank - 1;
    const int64_t cols = (int64_t)t->shape.sizes[last];
    out->pitch = cols;
    bool one = cols == 1 || t->strides.sizes[last] == 1, any = false;
    int64_t expect = 0;
    for (int d = last - 1; one && d >= 0; --d) {
        if (t->shape.sizes[d] == 1) continue;
        if (!any) out->pitch = t->strides.sizes[d];
        else one = t->strides.sizes[d] == expect;
        any = true;
        expect = t->strides.sizes[d] * (int64_t)t->shape.sizes[d];
    }
    out->base = t->address;
    if (one) return TN_SUCCESS;
    out->pitch = cols;
    return densely(t, &out->base, mem, stream);
}

// An operand in the form the tensor maps address.
struct Operand {
    const void* ptr = nullptr;
    int64_t pitch = 0, part_stride = 0;
    int parts = 1;
};

struct Problem {
    int dtype;
    bool bf16;
    int parts, terms;
    int64_t tokens, hidden, vocab, padded;
    int sms;  // that the call may use. The margin is read once: what one kernel plans by it another one adds up by
    cudaStream_t stream;
    // Asked at each launch: whether a kernel of this call came before it.
    bool behind() const {
        const bool had = begun;
        begun = true;
        return had;
    }
    mutable bool begun = false;
};

bool in_place(const Problem& p, const RowsIn& r, int64_t rows) {
    return p.parts == 1 && mult8(r.pitch) && r.pitch >= p.hidden && aligned16(r.base) && rows > 0;
}

// Writes `rows` rows into `to` (room for parts * rows * padded elements).
tn_status pack(const Problem& p, const RowsIn& r, int64_t first, int64_t rows, uint16_t* to, const int* slot) {
    const int64_t size = p.parts == 1 ? 2 : 4;
    const uint8_t* src = static_cast<const uint8_t*>(r.base) + first * r.pitch * size;
    const int vectors = aligned16(src) && (r.pitch * size) % 16 == 0;
    const int64_t work = rows * (p.padded / 8);
    const int grid = (int)std::min<int64_t>(ceil_div(work, 256), (int64_t)sm_count() * 16);
    if (p.parts == 1)
        TN_CUDA(launch_chained(p.behind(), pack_rows<uint16_t>, grid, 256, 0, p.stream, 1, reinterpret_cast<const uint16_t*>(src), r.pitch, rows, p.hidden, p.padded, to, 0, slot, vectors));
    else
        TN_CUDA(launch_chained(p.behind(), pack_rows<float>, grid, 256, 0, p.stream, 1, reinterpret_cast<const float*>(src), r.pitch, rows, p.hidden, p.padded, to, rows * p.padded, slot, vectors));
    return after_launch("pack_rows");
}

// The weights' rows [first, first + rows): in place, or packed into `room`.
tn_status weight_piece(const Problem& p, const RowsIn& w, int64_t first, int64_t rows, uint16_t* room, Operand* out) {
    out->parts = p.parts;
    if (!room) {
        out->ptr = static_cast<const uint16_t*>(w.base) + first * w.pitch;
        out->pitch = w.pitch;
        return TN_SUCCESS;
    }
    out->ptr = room;
    out->pitch = p.padded;
    out->part_stride = rows * p.padded;
    return pack(p, w, first, rows, room, nullptr);
}

// Tensor map over an operand: (inner, rows, part).
tn_status operand_map(CUtensorMap* map, const Operand& o, bool bf16, int64_t inner, int64_t rows, int box_inner, int box_rows) {
    return make_map(map, o.ptr, bf16, inner, rows, o.parts, o.pitch, o.part_stride, box_inner, box_rows);
}

// Thread blocks, or pairs of them, that run at once.
int unit_count(const Problem& p, bool pair) { return std::max(1, pair ? p.sms / 2 : p.sms); }
// Whether a product with m result rows takes pairs: up to 128 rows the second block would have none.
bool takes_pairs(int64_t m) { return m > BM; }

template <bool A_M, bool B_N, int EPI, typename T, typename OUT, int PARTS, bool PAIR>
tn_status launch_as(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& d, LossArgs g, const Problem& p) {
    static thread_local int attr_device = -1;  // the opt-in shared-memory size belongs to kernel and device, the counter to the device
    static thread_local unsigned int* aborts = nullptr;
    auto kernel = loss_gemm<A_M, B_N, EPI, T, OUT, PARTS, PAIR>;
    int dev = 0;
    TN_CUDA(cudaGetDevice(&dev));
    if (attr_device != dev) {
        TN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes<PAIR>));
        TN_TRY(tc_abort_counter(&aborts));
        attr_device = dev;
    }
    g.aborts = aborts;
    const int64_t total = (int64_t)g.m_tiles * g.n_tiles * g.most_splits;
    if (total >= (int64_t(1) << 31)) return fail(TN_ERROR, "linear_cross_entropy: %lld tiles are too many", (long long)total);
    const unsigned grid = (unsigned)std::min<int64_t>(total, g.units) * (PAIR ? 2 : 1);
    TN_CUDA(launch_chained(p.behind(), kernel, grid, kThreads, kSmemBytes<PAIR>, p.stream, PAIR ? 2 : 1, a, b, d, g));
    return after_launch("loss_gemm");
}
template <bool A_M, bool B_N, int EPI, typename T, typename OUT, int PARTS>
tn_status launch_one(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& d, const LossArgs& g, const Problem& p) {
    return takes_pairs(g.M) ? launch_as<A_M, B_N, EPI, T, OUT, PARTS, true>(a, b, d, g, p)
                            : launch_as<A_M, B_N, EPI, T, OUT, PARTS, false>(a, b, d, g, p);
}

LossArgs gemm_args(const Problem& p, int64_t m, int64_t n, int64_t k) {
    LossArgs g = {};
    const bool pair = takes_pairs(m);
    g.M = m;
    g.N = n;
    g.m_tiles = (int)ceil_div(m, pair ? 2 * BM : BM);
    g.n_tiles = (int)ceil_div(n, BN);
    g.k_blocks = (int)ceil_div(k, BK);
    g.most_splits = 1;
    g.units = unit_count(p, pair);
    g.terms = p.terms;
    g.group = p.parts == 3 ? kGroupParts : kGroup;
    g.is_bf16 = p.bf16;
    return g;
}
// Loss and gradient form the logits of 16-bit operands alike: d = exp(l - lse) - 1 of a nearly certain token is the difference of two
// large numbers, and lse has to belong to the same l. Up to sixteen tokens half_grad_kernel forms the gradient's, in short sums of its own; what the
// loss cuts off has to be small then: logits of 20 over 4096 columns are low by 4e-5 to 1.1e-4 with sixteen blocks to an accumulator, by less
// than 4e-6 with one. Four tokens over 32768 x 4096: 95 us from memory against 93.
int logit_group(const Problem& p) { return takes_pairs(p.tokens) ? kGroup : kGroupFew; }
// Map of an operand B stored [N, K] for a product with m result rows: a block of a pair loads half the columns.
tn_status b_map(CUtensorMap* map, const Operand& o, bool bf16, int64_t k, int64_t n, int64_t m) {
    return operand_map(map, o, bf16, k, n, BK, takes_pairs(m) ? BN / 2 : BN);
}

// Vocabulary entries per piece: `bytes_each` is the workspace that one of them takes.
// 8192 tokens of 16 bits make pieces of 32768 entries. Every further piece reads and writes dh's float32 sums once more: at 4096 columns
// 40 us beside the 5.7 ms of such a piece's products; below 4096 entries it would show.
int64_t piece_entries(int64_t vocab, int64_t bytes_each) {
    if (bytes_each <= 0) return vocab;
    const int64_t fits = ((int64_t(512) << 20) / bytes_each) & ~int64_t(255);
    return std::min(vocab, std::max<int64_t>(fits, 4096));
}

tn_status check_problem(const char* op, const tn_tensor_t* hidden, const tn_tensor_t* weight, const tn_tensor_t* targets) {
    if (!hidden || !weight || !targets) return fail(TN_ERROR, "%s: null tensor", op);
    if (hidden->rank < 1) return fail(TN_ERROR, "%s: the hidden states need a last axis", op);
    if (!is_half(hidden->dtype) && hidden->dtype != TN_FLOAT32) return fail(TN_UNSUPPORTED_DTYPE, "%s: dtype %d unsupported (float16, bfloat16, float32)", op, (int)hidden->dtype);
    if (weight->dtype != hidden->dtype) return fail(TN_UNSUPPORTED_DTYPE, "%s: hidden states of dtype %d and weights of dtype %d", op, (int)hidden->dtype, (int)weight->dtype);
    if (targets->dtype != TN_INT32 && targets->dtype != TN_INT64) return fail(TN_UNSUPPORTED_DTYPE, "%s: targets of dtype %d, expected int32 or int64", op, (int)targets->dtype);
    for (const tn_tensor_t* t : {hidden, weight, targets})
        if (t->environment.kind != TN_DEVICE || hidden->environment.kind != TN_DEVICE || t->environment.resource.device.id != hidden->environment.resource.device.id)
            return fail(TN_INCOMPATIBLE_DEVICES, "%s: operands must live on one device (no CPU fallback)", op);
    if (weight->rank != 2) return fail(TN_ERROR, "%s: the weights must be a matrix [vocabulary, hidden]", op);
    const size_t h = hidden->shape.sizes[hidden->rank - 1];
    if (weight->shape.sizes[1] != h) return fail(TN_ERROR, "%s: hidden states of %zu and weights of %zu columns", op, h, (size_t)weight->shape.sizes[1]);
    if (h == 0 || weight->shape.sizes[0] == 0) return fail(TN_ERROR, "%s: an empty hidden axis or vocabulary", op);
    const size_t limit = (size_t(1) << 31) - 512;
    if (h > limit || weight->shape.sizes[0] > limit || hidden->size / h > limit) return fail(TN_ERROR, "%s: an extent of 2^31 or more", op);
    bool same = targets->rank == hidden->rank - 1;
    for (int d = 0; same && d < targets->rank; ++d) same = targets->shape.sizes[d] == hidden->shape.sizes[d];
    if (!same) return fail(TN_ERROR, "%s: the targets must have the hidden states' leading shape", op);
    return TN_SUCCESS;
}
tn_status check_tokens(const char* op, const tn_tensor_t* targets, const tn_tensor_t* t, bool result, const char* what) {
    if (t->dtype != TN_FLOAT32) return fail(TN_UNSUPPORTED_DTYPE, "%s: %s has dtype %d, expected float32", op, what, (int)t->dtype);
    bool same = t->rank == targets->rank;
    for (int d = 0; same && d < t->rank; ++d) same = t->shape.sizes[d] == targets->shape.sizes[d];
    if (!same) return fail(TN_ERROR, "%s: %s must have the targets' shape", op, what);
    if (result && !is_dense(t)) return fail(TN_ERROR, "%s: %s must be dense", op, what);
    if (t->environment.kind != TN_DEVICE || t->environment.resource.device.id != targets->environment.resource.device.id)
        return fail(TN_INCOMPATIBLE_DEVICES, "%s: operands must live on one device", op);
    return TN_SUCCESS;
}
tn_status check_result(const char* op, const tn_tensor_t* like, const tn_tensor_t* t, const char* what) {
    if (t->dtype != like->dtype) return fail(TN_UNSUPPORTED_DTYPE, "%s: %s has dtype %d, expected %d", op, what, (int)t->dtype, (int)like->dtype);
    bool same = t->rank == like->rank;
    for (int d = 0; same && d < t->rank; ++d) same = t->shape.sizes[d] == like->shape.sizes[d];
    if (!same) return fail(TN_ERROR, "%s: %s has the wrong shape", op, what);
    if (!is_dense(t)) return fail(TN_ERROR, "%s: %s must be dense", op, what);
    if (t->environment.kind != TN_DEVICE || t->environment.resource.device.id != like->environment.resource.device.id)
        return fail(TN_INCOMPATIBLE_DEVICES, "%s: operands must live on one device", op);
    return TN_SUCCESS;
}

Problem make_problem(const tn_tensor_t* hidden, const tn_tensor_t* weight, tn_stream_t stream) {
    Problem p;
    p.dtype = hidden->dtype;
    p.bf16 = hidden->dtype != TN_FLOAT16;
    p.parts = hidden->dtype == TN_FLOAT32 ? 3 : 1;
    p.terms = p.parts == 3 ? 6 : 1;
    p.hidden = (int64_t)hidden->shape.sizes[hidden->rank - 1];
    p.tokens = (int64_t)hidden->size / p.hidden;
    p.vocab = (int64_t)weight->shape.sizes[0];
    p.padded = (p.hidden + 7) & ~int64_t(7);
    p.sms = std::max(1, sm_count() - sm_margin());
    p.stream = as_cuda(stream);
    return p;
}

// Joins `n` groups of logits per row into lse and loss.
tn_status join(const Problem& p, const float2* halves, int64_t n, const float* target_logit, const void* targets, int wide, int64_t ignore, tn_tensor_t* loss, tn_tensor_t* lse) {
    const bool few = p.tokens <= 2 * sm_count();  // a block per row fills the GPU at most once
    TN_CUDA(launch_chained(true, few ? loss_join<1> : loss_join<32>, (unsigned)ceil_div(p.tokens, few ? 1 : 32), 1024, 0, p.stream, 1, halves, n, p.tokens, target_logit, targets, wide,
                           ignore, p.vocab, loss ? static_cast<float*>(loss->address) : nullptr, lse ? static_cast<float*>(lse->address) : nullptr));
    return after_launch("loss_join");
}

FewTokens few_tokens(const Problem& p, const RowsIn& h, const RowsIn& w, const void* targets, int wide, int64_t ignore) {
    FewTokens f;
    f.dtype = p.dtype;
    f.tokens = p.tokens;
    f.hidden = p.hidden;
    f.vocab = p.vocab;
    f.sms = p.sms;
    f.h = h.base;
    f.h_pitch = h.pitch;
    f.w = w.base;
    f.w_pitch = w.pitch;
    f.targets = targets;
    f.wide = wide;
    f.ignore = ignore;
    return f;
}

tn_status run_loss(const tn_tensor_t* hidden, const tn_tensor_t* weight, const tn_tensor_t* targets, tn_tensor_t* loss, tn_tensor_t* lse, tn_stream_t stream,
                   int64_t ignore, Scratch& mem) {
    const Problem p = make_problem(hidden, weight, stream);
    RowsIn h, w;
    const void* t = nullptr;
    TN_TRY(rows_in(hidden, &h, mem, stream));
    TN_TRY(rows_in(weight, &w, mem, stream));
    TN_TRY(densely(targets, &t, mem, stream));
    const int wide = targets->dtype == TN_INT64;
    float2* halves = nullptr;
    float* target_logit = nullptr;
    TN_TRY(mem.take(&target_logit, sizeof(float) * p.tokens));
    const bool few = few_loss_fits(p.dtype, p.tokens, p.hidden);
    if (few || f32_fits(p.dtype, p.tokens, p.hidden, false)) {
        FewTokens f = few_tokens(p, h, w, t, wide, ignore);
        const int64_t parts = few ? few_loss_parts(f) : f32_loss_parts(p.tokens, p.vocab);
        TN_TRY(mem.take(&halves, sizeof(float2) * (size_t)parts * p.tokens));
        f.parts = halves;
        f.target_logit = target_logit;
        if (few) {
            TN_TRY(few_loss(f, p.stream));
        } else {
            float* rows = nullptr;
            TN_TRY(mem.take(&rows, sizeof(float) * f32_row_floats(p.tokens, p.hidden)));
            TN_TRY(f32_loss(f, rows, p.stream));
        }
        return join(p, halves, parts, target_logit, t, wide, ignore, loss, lse);
    }
    Operand a;
    a.parts = p.parts;
    uint16_t* tokens = nullptr;
    if (in_place(p, h, p.tokens)) {
        a.ptr = h.base;
        a.pitch = h.pitch;
    } else {
        TN_TRY(mem.take(&tokens, (size_t)p.parts * p.tokens * p.padded * 2));
        a.ptr = tokens;
        a.pitch = p.padded;
        a.part_stride = p.tokens * p.padded;
    }
    const bool packed = !in_place(p, w, p.vocab);
    const int64_t piece = piece_entries(p.vocab, packed ? p.padded * 2 * p.parts : 0);
    uint16_t* room = nullptr;
    if (packed) TN_TRY(mem.take(&room, (size_t)p.parts * piece * p.padded * 2));
    int64_t tiles = 0;
    for (int64_t v0 = 0; v0 < p.vocab; v0 += piece) tiles += ceil_div(std::min(piece, p.vocab - v0), BN);
    TN_TRY(mem.take(&halves, sizeof(float2) * 2 * (size_t)tiles * p.tokens));
    if (tokens) TN_TRY(pack(p, h, 0, p.tokens, tokens, nullptr));
    CUtensorMap map_a, map_b;
    TN_TRY(operand_map(&map_a, a, p.bf16, p.hidden, p.tokens, BK, BM));
    int64_t first_half = 0;
    for (int64_t v0 = 0; v0 < p.vocab; v0 += piece) {
        const int64_t n = std::min(piece, p.vocab - v0);
        Operand b;
        TN_TRY(weight_piece(p, w, v0, n, room, &b));
        TN_TRY(b_map(&map_b, b, p.bf16, p.hidden, n, p.tokens));
        LossArgs g = gemm_args(p, p.tokens, n, p.hidden);
        if (p.parts == 1) g.group = logit_group(p);
        g.vocab0 = v0;
        g.targets = t;
        g.wide_targets = wide;
        g.halves = halves;
        g.first_half = first_half;
        g.target_logit = target_logit;
        TN_TRY((launch_one<false, false, EPI_STATS, __half, float, 1>(map_a, map_b, map_a, g, p)));
        first_half += 2 * (int64_t)g.n_tiles;
    }
    return join(p, halves, first_half, target_logit, t, wide, ignore, loss, lse);
}

template <typename T, typename OUT, int PARTS>
tn_status run_grad(const tn_tensor_t* grad, const tn_tensor_t* hidden, const tn_tensor_t* weight, const tn_tensor_t* targets, const tn_tensor_t* lse, tn_tensor_t* dhidden,
                   tn_tensor_t* dweight, tn_stream_t stream, int64_t ignore, Scratch& mem) {
    const Problem p = make_problem(hidden, weight, stream);
    RowsIn h, w;
    const void *t = nullptr, *up = nullptr, *z = nullptr;
    TN_TRY(rows_in(hidden, &h, mem, stream));
    TN_TRY(rows_in(weight, &w, mem, stream));
    TN_TRY(densely(targets, &t, mem, stream));
    TN_TRY(densely(grad, &up, mem, stream));
    TN_TRY(densely(lse, &z, mem, stream));
    const int wide = targets->dtype == TN_INT64;
    FewTokens f = few_tokens(p, h, w, t, wide, ignore);
    f.grad = static_cast<const float*>(up);
    f.lse = static_cast<const float*>(z);
    f.dhidden = dhidden ? dhidden->address : nullptr;
    f.dweight = dweight ? dweight->address : nullptr;
    const bool half = half_grad_fits(f), few = few_grad_fits(f);
    if (half || few || f32_fits(p.dtype, p.tokens, p.hidden, true)) {
        const int64_t blocks = half ? half_grad_blocks(f) : few ? few_grad_blocks(f) : f32_grad_shares(p.hidden, p.vocab);
        if (dhidden) TN_TRY(mem.take(&f.sums, sizeof(float) * (size_t)blocks * p.tokens * p.hidden));
        if (half) return half_grad(f, p.stream);
        if (few) return few_grad(f, p.stream);
        float *rows = nullptr, *d = nullptr;
        TN_TRY(mem.take(&rows, sizeof(float) * f32_row_floats(p.tokens, p.hidden)));
        TN_TRY(mem.take(&d, sizeof(float) * f32_d_floats(p.tokens, p.vocab)));
        return f32_grad(f, rows, d, p.stream);
    }
    RowInfo* info = nullptr;
    int *slot = nullptr, *count = nullptr;
    TN_TRY(mem.take(&info, sizeof(RowInfo) * p.tokens));
    TN_TRY(mem.take(&slot, sizeof(int) * p.tokens));
    TN_TRY(mem.take(&count, 2 * sizeof(int)));
    float* scale = reinterpret_cast<float*>(count + 1);
    uint16_t* gathered = nullptr;
    TN_TRY(mem.take(&gathered, (size_t)p.parts * p.tokens * p.padded * 2));
    Operand a;
    a.ptr = gathered;
    a.pitch = p.padded;
    a.part_stride = p.tokens * p.padded;
    a.parts = p.parts;

    const bool packed = !in_place(p, w, p.vocab);
    const int64_t piece = piece_entries(p.vocab, (p.tokens + (packed ? p.padded : 0)) * 2 * p.parts);
    uint16_t *room = nullptr, *d = nullptr;
    if (packed) TN_TRY(mem.take(&room, (size_t)p.parts * piece * p.padded * 2));
    const int64_t d_pitch = (piece + 7) & ~int64_t(7);
    TN_TRY(mem.take(&d, (size_t)p.parts * p.tokens * d_pitch * 2));
    Operand dd;
    dd.ptr = d;
    dd.pitch = d_pitch;
    dd.part_stride = p.tokens * d_pitch;
    dd.parts = p.parts;

    // dh has few tiles when there are few tokens: K (the vocabulary) is split until every SM has a tile, and the splits' sums are added
    // in order afterwards. Room for what the host can know; half of the tokens may turn out not to count.
    float* sums = nullptr;
    int splits = 1;
    const bool pair = takes_pairs(p.tokens);
    if (dhidden) {
        const int64_t tiles = ceil_div(p.tokens, pair ? 2 * BM : BM) * ceil_div(p.padded, BN);
        splits = (int)std::max<int64_t>(1, std::min<int64_t>(2 * (unit_count(p, pair) / tiles), ceil_div(piece, BK) / 4));
        TN_TRY(mem.take(&sums, sizeof(float) * (size_t)splits * p.tokens * p.padded));
    }

    // the scratch memory is all taken: what follows are kernels, one behind the other
    // every block reads all targets, so there are not too many of them
    const int per_block = (int)std::min<int64_t>(256, std::max<int64_t>(32, ceil_div(p.tokens, 256)));
    TN_CUDA(launch_chained(p.behind(), loss_rows, (unsigned)ceil_div(p.tokens, per_block), 256, 0, p.stream, 1, t, wide, p.tokens, f.grad, f.lse, ignore, p.vocab, per_block,
                           info, slot, count, scale));
    TN_TRY(after_launch("loss_rows"));
    TN_TRY(pack(p, h, 0, p.tokens, gathered, slot));

    CUtensorMap rows_a, rows_b, map;
    TN_TRY(operand_map(&rows_a, a, p.bf16, p.hidden, p.tokens, BK, BM));   // h as [tokens, hidden], K = hidden
    TN_TRY(operand_map(&rows_b, a, p.bf16, p.hidden, p.tokens, 64, BK));   // h as B of dW, K = tokens
    for (int64_t v0 = 0; v0 < p.vocab; v0 += piece) {
        const int64_t n = std::min(piece, p.vocab - v0);
        Operand b;
        TN_TRY(weight_piece(p, w, v0, n, room, &b));
        {   // d of this piece
            CUtensorMap map_d;
            TN_TRY(b_map(&map, b, p.bf16, p.hidden, n, p.tokens));
            const cuuint64_t dims[3] = {(cuuint64_t)n, (cuuint64_t)p.tokens, (cuuint64_t)p.parts};
            const cuuint64_t strides[2] = {(cuuint64_t)d_pitch * 2, (cuuint64_t)dd.part_stride * 2};
            const cuuint32_t box[3] = {32, 32, 1};
            TN_TRY(encode_as(&map_d, d, p.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_64B, 3, dims, strides, box));
            LossArgs g = gemm_args(p, p.tokens, n, p.hidden);
            if (p.parts == 1) g.group = logit_group(p);
            g.vocab0 = v0;
            g.count = count;
            g.count_is = COUNT_ROWS;
            g.rows = info;
            TN_TRY((launch_one<false, false, EPI_D, T, float, PARTS>(rows_a, map, map_d, g, p)));
        }
        if (dhidden) {
            CUtensorMap map_d, map_w;
            TN_TRY(operand_map(&map, dd, p.bf16, n, p.tokens, BK, BM));
            TN_TRY(operand_map(&map_w, b, p.bf16, p.hidden, n, 64, BK));
            TN_TRY(make_result_map(&map_d, sums, true, false, p.padded, p.tokens, splits, p.padded, p.tokens * p.padded));
            LossArgs g = gemm_args(p, p.tokens, p.padded, n);
            g.count = count;
            g.count_is = COUNT_ROWS;
            g.most_splits = splits;
            g.first_k_blocks = (int)ceil_div(piece, BK);
            g.add = v0 > 0;
            TN_TRY((launch_one<false, true, EPI_SUM, T, float, 1>(map, map_w, map_d, g, p)));
        }
        if (dweight) {
            CUtensorMap map_d;
            TN_TRY(operand_map(&map, dd, p.bf16, n, p.tokens, 64, BK));
            OUT* to = static_cast<OUT*>(dweight->address) + v0 * p.hidden;
            LossArgs g = gemm_args(p, n, p.hidden, p.tokens);
            g.count = count;
            g.count_is = COUNT_K;
            g.scale = scale;
            g.d = to;
            g.ldd = p.hidden;
            constexpr bool F32 = std::is_same<OUT, float>::value;
            g.tma_store = can_tma_store(to, p.hidden, p.hidden * 8, BN, F32);
            map_d = map;  // placeholder when the result does not leave through TMA
            if (g.tma_store) TN_TRY(make_result_map(&map_d, to, F32, p.bf16, p.hidden, n, 1, p.hidden, 0));
            TN_TRY((launch_one<true, true, EPI_RESULT, T, OUT, 1>(map, rows_b, map_d, g, p)));
        }
    }
    if (dhidden) {
        OUT* to = static_cast<OUT*>(dhidden->address);
        const bool wide = p.hidden % 4 == 0 && (reinterpret_cast<uintptr_t>(to) & (4 * sizeof(OUT) - 1)) == 0;
        const dim3 grid((unsigned)ceil_div(p.hidden, wide ? 1024 : 256), (unsigned)std::min<int64_t>(ceil_div(p.tokens, 4), 65535));
        TN_CUDA(launch_chained(true, wide ? loss_dhidden<OUT, 4> : loss_dhidden<OUT, 1>, grid, 256, 0, p.stream, 1, sums, count, pair ? 2 * BM : BM, (int)ceil_div(p.padded, BN),
                               unit_count(p, pair), (int)ceil_div(piece, BK), splits, p.tokens, p.hidden, p.padded, slot, scale, to));
        TN_TRY(after_launch("loss_dhidden"));
    }
    return TN_SUCCESS;
}

}  // namespace
}  // namespace tnb

using namespace tnb;

extern "C" {

tn_status tn_linear_cross_entropy(const tn_tensor_t* hidden, const tn_tensor_t* weight, const tn_tensor_t* targets, tn_tensor_t* loss, tn_tensor_t* lse,
                                  tn_stream_t stream, int64_t ignore_index) {
    const char* op = "linear_cross_entropy";
    TN_TRY(check_problem(op, hidden, weight, targets));
    if (!loss && !lse) return fail(TN_ERROR, "linear_cross_entropy: no output requested");
    if (loss) TN_TRY(check_tokens(op, targets, loss, true, "the loss"));
    if (lse) TN_TRY(check_tokens(op, targets, lse, true, "lse"));
    TN_TRY(use_device_of(hidden));
    if (hidden->size == 0) return TN_SUCCESS;
    Scratch mem(as_cuda(stream));
    return mem.release(run_loss(hidden, weight, targets, loss, lse, stream, ignore_index, mem));
}

tn_status tn_linear_cross_entropy_grad(const tn_tensor_t* grad, const tn_tensor_t* hidden, const tn_tensor_t* weight, const tn_tensor_t* targets, const tn_tensor_t* lse,
                                       tn_tensor_t* dhidden, tn_tensor_t* dweight, tn_stream_t stream, int64_t ignore_index) {
    const char* op = "linear_cross_entropy_grad";
    TN_TRY(check_problem(op, hidden, weight, targets));
    if (!grad || !lse) return fail(TN_ERROR, "%s: null tensor", op);
    TN_TRY(check_tokens(op, targets, grad, false, "the loss's gradient"));
    TN_TRY(check_tokens(op, targets, lse, false, "lse"));
    if (!dhidden && !dweight) return fail(TN_ERROR, "%s: no output requested", op);
    if (dhidden) TN_TRY(check_result(op, hidden, dhidden, "the hidden states' gradient"));
    if (dweight) TN_TRY(check_result(op, weight, dweight, "the weights' gradient"));
    TN_TRY(use_device_of(hidden));
    if (hidden->size == 0) {  // no tokens: the sum over them is zero
        if (dweight) TN_CUDA(cudaMemsetAsync(dweight->address, 0, dweight->size * (size_t)dtype_bytes(dweight->dtype), as_cuda(stream)));
        return TN_SUCCESS;
    }
    Scratch mem(as_cuda(stream));
    tn_status st;
    switch (hidden->dtype) {
        case TN_FLOAT16: st = run_grad<__half, __half, 1>(grad, hidden, weight, targets, lse, dhidden, dweight, stream, ignore_index, mem); break;
        case TN_BFLOAT16: st = run_grad<__nv_bfloat16, __nv_bfloat16, 1>(grad, hidden, weight, targets, lse, dhidden, dweight, stream, ignore_index, mem); break;
        default: st = run_grad<__nv_bfloat16, float, 3>(grad, hidden, weight, targets, lse, dhidden, dweight, stream, ignore_index, mem); break;
    }
    return mem.release(st);
}

}  // extern "C"
