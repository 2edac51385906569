// What the tensor-core kernels share: tile geometry, PTX wrappers (mbarrier, TMA, tcgen05), bounded waits, the walk over
// tiles, and the host side of TMA (tensor maps).
#pragma once

#include <cuda.h>

#include <cstdlib>
#include <mutex>

#include "common.cuh"

namespace tnb {

constexpr int BM = 128;
constexpr int BN = 256;
constexpr int BK = 64;            // 64 x 2 bytes = one 128-byte swizzle row
constexpr int UMMA_K = 16;
constexpr uint32_t A_BYTES = BM * BK * 2;        // 16 KiB
constexpr uint32_t B_BYTES = BN * BK * 2;        // 32 KiB
constexpr uint32_t STAGE_BYTES = A_BYTES + B_BYTES;
constexpr uint32_t TMEM_COLS = 512;              // two accumulators of BN fp32 columns

// Waits on an mbarrier are bounded: after this many polls a thread block gives up.
constexpr uint32_t kSpinFast = 2048;      // polls without sleeping
constexpr uint32_t kSpinLimit = 1u << 20; // then ~64 ns sleeps: gives up after roughly 0.1 s

// ------------------------------------------------------------------ PTX wrappers ------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// Bounded wait. Returns false when the CTA is aborting (this wait or another one ran out).
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t limit = kSpinLimit) {
    for (uint32_t it = 0; it < limit; ++it) {
        if (mbar_test(bar, parity)) return true;
        if (it >= kSpinFast) {
            if (*abort_flag) return false;
            __nanosleep(64);
        }
    }
    *abort_flag = 1;
    return false;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

// Result tiles leave through TMA as well: a warp writes a 32-row x 64-byte box into shared memory
// (64-byte swizzle) and one lane hands it to the copy engine, which clips it at the tensor's edges.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
        ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// Untiled copy of a 16-byte-aligned shared-memory range to a 16-byte-aligned global range.
__device__ __forceinline__ void bulk_store_linear(void* dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
        ::"l"(reinterpret_cast<uint64_t>(dst)), "r"(src), "r"(bytes)
        : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// until at most one of this thread's store groups still reads its shared-memory source
__device__ __forceinline__ void bulk_wait_read_1() { asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read_0() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void umma_f16(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// tcgen05.ld is asynchronous: the registers are valid only after tcgen05.wait::ld. The wait
// below names the registers as read-write operands so that no use of them can be scheduled
// ahead of it.
__device__ __forceinline__ void tmem_load_issue(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32"
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
        " %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_load_wait(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
        : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
          "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
          "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]),
          "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
        :
        : "memory");
}

// Shared-memory matrix descriptor of a 128-byte-swizzled tile (sm_100 format: start address,
// leading / stride byte offsets in 16-byte units, version 1 at bit 46, layout type 2 =
// SWIZZLE_128B at bits 61-63).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((addr & 0x3FFFF) >> 4);
    d |= static_cast<uint64_t>((lbo_bytes >> 4) & 0x3FFF) << 16;
    d |= static_cast<uint64_t>((sbo_bytes >> 4) & 0x3FFF) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// Tiles are walked in groups of 16 row-tiles so that the CTAs running at the same time share
// rows of A and columns of B in L2.
constexpr int kGroupM = 16;
__device__ __forceinline__ void tile_coords(uint32_t t, int m_tiles, int n_tiles, int& batch, int& mt, int& nt) {
    // tile counts are below 2^31 (checked on the host): 32-bit divisions only
    const uint32_t per_batch = static_cast<uint32_t>(m_tiles) * static_cast<uint32_t>(n_tiles);
    batch = static_cast<int>(t / per_batch);
    int r = static_cast<int>(t - static_cast<uint32_t>(batch) * per_batch);
    const int group_span = kGroupM * n_tiles;
    const int g = r / group_span;
    r -= g * group_span;
    const int rows_in_group = min(kGroupM, m_tiles - g * kGroupM);
    nt = r / rows_in_group;
    mt = g * kGroupM + (r - nt * rows_in_group);
}

// ------------------------------------------------------------------ host --------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

inline bool mult8(int64_t v) { return (v & 7) == 0; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Tiled map of rank `rank`, zero fill outside the tensor.
inline tn_status encode_as(CUtensorMap* map, const void* ptr, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, int rank,
                    const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box, const cuuint32_t* traversal = nullptr) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(TN_ERROR, "cuTensorMapEncodeTiled is not available from the driver");
    cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    if (traversal)
        for (int i = 0; i < rank; ++i) estr[i] = traversal[i];
    CUresult r = fn(map, type, (cuuint32_t)rank, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(TN_ERROR, "cuTensorMapEncodeTiled failed with code %d", (int)r);
    return TN_SUCCESS;
}

// Operand maps: 16-bit elements, 128-byte swizzle.
inline tn_status encode(CUtensorMap* map, const void* ptr, bool bf16, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                 const cuuint32_t* box, const cuuint32_t* traversal = nullptr) {
    return encode_as(map, ptr, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B,
                     rank, dims, strides, box, traversal);
}

// Result map (columns, rows, batch) for the epilogue's stores: boxes of 32 rows x 64 bytes, 64-byte
// swizzle. Usable when the base and both pitches are multiples of 16 bytes and every tile starts
// on a 16-byte column boundary.
inline bool can_tma_store(const void* d, int64_t ldd, int64_t d_batch, int64_t tile_n, bool f32) {
    const int64_t per16 = f32 ? 4 : 8;
    static const bool disabled = getenv("TN_TC_NO_TMA_STORE") != nullptr;
    if (disabled) return false;
    return aligned16(d) && ldd % per16 == 0 && d_batch % per16 == 0 && tile_n % per16 == 0;
}
inline tn_status make_result_map(CUtensorMap* map, void* d, bool f32, bool bf16, int64_t n, int64_t m, int64_t batches, int64_t ldd, int64_t d_batch) {
    const cuuint64_t es = f32 ? 4 : 2;
    cuuint64_t dims[3] = {(cuuint64_t)n, (cuuint64_t)m, (cuuint64_t)(batches > 0 ? batches : 1)};
    cuuint64_t pitch_batch = (cuuint64_t)(d_batch > 0 ? d_batch : ldd * m) * es;
    cuuint64_t strides[2] = {(cuuint64_t)ldd * es, pitch_batch};
    cuuint32_t box[3] = {(cuuint32_t)(64 / es), 32, 1};
    const CUtensorMapDataType type = f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return encode_as(map, d, type, CU_TENSOR_MAP_SWIZZLE_64B, 3, dims, strides, box);
}

// 3-D map (inner, rows, batch) over a 16-bit matrix; box = box_inner x box_rows x 1.
inline tn_status make_map(CUtensorMap* map, const void* ptr, bool bf16, int64_t inner, int64_t rows, int64_t batches,
                   int64_t row_pitch, int64_t batch_pitch, int box_inner, int box_rows) {
    cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)(batches > 0 ? batches : 1)};
    // a pitch is irrelevant for an extent of 1 but must still be a non-zero multiple of 16 bytes
    cuuint64_t pitch_rows = (cuuint64_t)row_pitch * 2;
    cuuint64_t pitch_batch = (cuuint64_t)(batch_pitch > 0 ? batch_pitch : row_pitch * rows) * 2;
    if (pitch_rows == 0) pitch_rows = (cuuint64_t)inner * 2;
    if (pitch_batch == 0) pitch_batch = pitch_rows;
    cuuint64_t strides[2] = {pitch_rows, pitch_batch};
    cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_rows, 1};
    return encode(map, ptr, bf16, 3, dims, strides, box);
}

}  // namespace tnb
