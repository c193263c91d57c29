// ============================================================================
//  tcgen05.cuh -- tensor-core products of 16-bit operands (sm_100a): shared
//  memory descriptors, TMA loads, tcgen05.mma and TMEM access, as the typed
//  products use them.
//
//  Operand tiles in shared memory are 128-byte rows with the 128-byte swizzle,
//  as TMA writes them:
//   inner    (the product's inner index is contiguous): one row per outer
//            index, 64 inner indexes; 8-row groups 1024 bytes apart.
//   outer    (the outer index is contiguous): one row per inner index, 64
//            outer indexes; 8 rows (8 inner indexes) are 1024 bytes, and the
//            next 64 outer indexes follow a whole chunk of 64 rows later.
// ============================================================================
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "launch.cuh"
#include "mbarrier.cuh"

namespace tg {
namespace tc {

constexpr int kInner = 64;            // inner indexes per stage: 64 16-bit values, one 128-byte row
constexpr uint32_t kChunkBytes = 64 * 128;  // 64 rows

// Descriptor bits common to both forms: address, SBO, version 1, 128-byte swizzle.
__device__ __forceinline__ uint64_t desc_base(uint32_t smem, uint32_t lbo, uint32_t sbo) {
    return static_cast<uint64_t>((smem >> 4) & 0x3FFF) | static_cast<uint64_t>(lbo >> 4) << 16 |
           static_cast<uint64_t>(sbo >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
// The 16 inner indexes [16 s, 16 s + 16) of a tile.
__device__ __forceinline__ uint64_t desc_inner(uint32_t tile, int s) { return desc_base(tile + s * 32, 16, 1024); }
__device__ __forceinline__ uint64_t desc_outer(uint32_t tile, int s) {
    return desc_base(tile + s * 2048, kChunkBytes, 1024);
}

// Instruction descriptor: 16-bit operands (bf16 or fp16), fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc(bool bf16, bool a_outer, bool b_outer, int m, int n) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_outer ? 1u << 15 : 0u) | (b_outer ? 1u << 16 : 0u) |
           (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(static_cast<uint32_t>(acc)));
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];"
                 ::"r"(mb::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;"); }

// One warp: `cols` columns of TMEM (a power of two >= 32), address to *out.
__device__ __forceinline__ void alloc(uint32_t* out, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(mb::smem_u32(out)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void dealloc(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}

// 32 columns of the warp's 32 TMEM lanes: lane l gets its lane's columns.
__device__ __forceinline__ void load32(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    __syncwarp();  // the load is a warp's: lanes may come from different branches
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}
__device__ __forceinline__ void tma3(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(mb::smem_u32(bar))
        : "memory");
}
// ── CTA pairs ────────────────────────────────────────────────────────────
// Two CTAs of a cluster multiply one tile of 256 rows (cta_group::2): each
// holds its 128 rows of A and half of B's columns in its own shared memory
// and its 128 rows of the accumulator in its own TMEM.  The CTA of rank 0
// issues the MMAs; its full barriers count both CTAs' copies.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of `bar` in the CTA of rank `rank`.
__device__ __forceinline__ uint32_t in_rank(const void* bar, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(mb::smem_u32(bar)), "r"(rank));
    return a;
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Bounded wait (as mb::wait) that sees what the other CTA did before it arrived.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, int* err, int code) {
    const uint32_t a = mb::smem_u32(bar);
    uint64_t t0 = 0;
    for (uint32_t i = 0;; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(a), "r"(parity)
            : "memory");
        if (ok) return true;
        if (i == 0) t0 = mb::global_ns();
        if ((i & 15) == 15 && mb::global_ns() - t0 > mb::kWaitNs) break;
        if (i > 32) __nanosleep(64);
    }
    atomicCAS(err, 0, code);
    return false;
}
// A copy into this CTA's shared memory that completes on a barrier of either CTA.
__device__ __forceinline__ void tma3_pair(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, "
        "%4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(static_cast<uint32_t>(acc)));
}
// Arrives on `bar` (the same offset) of both CTAs once the MMAs so far have retired.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(mb::smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
}
__device__ __forceinline__ void alloc_pair(uint32_t* out, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(mb::smem_u32(out)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void dealloc_pair(uint32_t tmem, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols));
}

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        cudaDriverEntryPointQueryResult q;
        void* p = nullptr;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) ==
                cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        else
            cudaGetLastError();
    });
    if (!fn) fail(TG_ERR_CUDA, "typed_linear: cuTensorMapEncodeTiled is unavailable");
    return fn;
}

// A tensor map of 16-bit elements, 128-byte swizzle, zeros out of range.
// dims / strides (elements; strides[0] is dimension 1's) / box: innermost first.
template <int R>
CUtensorMap map16(const void* base, bool bf16, const int64_t (&dims)[R], const int64_t (&strides)[R - 1],
                  const int (&box)[R]) {
    CUtensorMap m;
    cuuint64_t d[R], s[R - 1];
    cuuint32_t b[R], one[R];
    for (int i = 0; i < R; ++i) {
        d[i] = static_cast<cuuint64_t>(dims[i]);
        b[i] = static_cast<cuuint32_t>(box[i]);
        one[i] = 1;
        if (i) s[i - 1] = static_cast<cuuint64_t>(strides[i - 1]) * 2;
    }
    const CUresult r = encode_fn()(&m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, R,
                                   const_cast<void*>(base), d, s, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        fail(TG_ERR_CUDA, "typed_linear: tensor map encoding failed (" + std::to_string(r) + ")");
    return m;
}

}  // namespace tc
}  // namespace tg
