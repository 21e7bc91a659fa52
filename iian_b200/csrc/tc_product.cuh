// What the matrix products on tcgen05 share: barriers, TMA copies, matrix instructions, descriptors, on one SM and on pairs of them.
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace iian {

constexpr int TC_BM = 128;
constexpr int TC_BK = 64;                 // 64 bf16 = 128 bytes = one swizzle atom
constexpr int TC_THREADS = 192;           // warp 0: TMA, warp 1: MMA + TMEM, warps 2..5: epilogue
constexpr unsigned kSpinLimit = 2u * 1000u * 1000u;

struct TcStatus { int code; int where; };

__device__ __forceinline__ unsigned smem_addr(const void * p) { return (unsigned) __cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(unsigned bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(unsigned bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// bounded wait for the phase with this parity; false: gave up
__device__ __forceinline__ bool mbar_wait(unsigned bar, unsigned parity) {
    for (unsigned spin = 0; spin < kSpinLimit; spin++) {
        unsigned done;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ void tma_load_2d(unsigned dst, const CUtensorMap * map, int x, int y, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_mma(unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc,
                                       unsigned accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 lanes x 32 columns of 32-bit accumulators: thread i of the warp gets lane i's 32 columns
__device__ __forceinline__ void tc_ld32(unsigned taddr, unsigned * r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor: K-major tile with 128-byte rows, 128-byte swizzle, groups of 8 rows
// 1024 bytes apart.  Start address and offsets are in units of 16 bytes.
__device__ __forceinline__ unsigned long long smem_desc_sw128(unsigned addr) {
    unsigned long long d = 0;
    d |= (unsigned long long) ((addr & 0x3FFFF) >> 4);           // bits  0-13: start address
    d |= (unsigned long long) 1 << 16;                            // bits 16-29: leading byte offset (unused with swizzle)
    d |= (unsigned long long) (1024 >> 4) << 32;                  // bits 32-45: stride byte offset (8 rows)
    d |= (unsigned long long) 1 << 46;                            // bits 46-47: descriptor version of this architecture
    d |= (unsigned long long) 2 << 61;                            // bits 61-63: 128-byte swizzle
    return d;
}
// Instruction descriptor: bf16 x bf16 -> f32, both operands K-major, M x N tile.
__host__ __device__ constexpr unsigned instr_desc_bf16(int m, int n) {
    return (1u << 4)                      // accumulator format f32
         | (1u << 7) | (1u << 10)         // A and B are bf16
         | ((unsigned) (n >> 3) << 17)    // N / 8
         | ((unsigned) (m >> 4) << 24);   // M / 16
}

__device__ __forceinline__ void mbar_arrive(unsigned bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ---- pairs of SMs ----------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned cluster_cta_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned map_to_cta(unsigned addr, unsigned rank) {
    unsigned r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same in two halves, for work between them: every thread of the CTA takes both.  It says that all have arrived, and nothing of what they
// had written.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive_cluster(unsigned cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// no multicast: the tile lands in this CTA's shared memory; only the completion goes to the barrier of CTA 0
__device__ __forceinline__ void tma_load_2d_pair(unsigned dst, const CUtensorMap * map, int x, int y, unsigned bar_cluster) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar_cluster) : "memory");
}
__device__ __forceinline__ void tc_commit_pair(unsigned bar) {      // arrives on the barrier at this offset in both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"((unsigned short) 3) : "memory");
}
__device__ __forceinline__ void tc_mma_pair(unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc,
                                            unsigned accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// ---- the same issued by a whole warp, of which one lane is elected ------------------------------------------------
// Inside a branch that one lane takes, the compiler has to bring every operand of a matrix instruction or copy into a uniform register by
// itself (600 cycles for the four instructions and the commit of a K block); a warp that runs the loop as one keeps them there.
__device__ __forceinline__ void tc_mma4(unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n .reg .pred p, q, t;\n .reg .b64 a, b;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n"
                 " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
                 " add.s64 a, %1, 2;\n add.s64 b, %2, 2;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
                 " add.s64 a, %1, 4;\n add.s64 b, %2, 4;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n"
                 " add.s64 a, %1, 6;\n add.s64 b, %2, 6;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_mma4_pair(unsigned d_tmem, unsigned long long a_desc, unsigned long long b_desc, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n .reg .pred p, q, t;\n .reg .b64 a, b;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n"
                 " @q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
                 " add.s64 a, %1, 2;\n add.s64 b, %2, 2;\n @q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n"
                 " add.s64 a, %1, 4;\n add.s64 b, %2, 4;\n @q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n"
                 " add.s64 a, %1, 6;\n add.s64 b, %2, 6;\n @q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, t;\n}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_commit_warp(unsigned bar) {
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}"
                 ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_commit_pair_warp(unsigned bar, unsigned leader) {      // to the pair of CTAs leader, leader + 1 of the cluster
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
                 " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}"
                 ::"r"(bar), "h"((unsigned short) (3u << leader)) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx_warp(unsigned bar, unsigned bytes) {
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_load_2d_warp(unsigned dst, const CUtensorMap * map, int x, int y, unsigned bar) {
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
                 " @q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_2d_pair_warp(unsigned dst, const CUtensorMap * map, int x, int y, unsigned bar_cluster) {
    asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
                 " @q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n}"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar_cluster) : "memory");
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    if (fn == nullptr) {
        void * p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn) p;
    }
    return fn;
}

// a [rows, K] bf16 row-major matrix, rows `ld` entries apart (0: K), boxes of [box_rows, 64], 128-byte swizzle, zero fill outside
static int make_map(CUtensorMap * map, const void * base, int rows, int K, int box_rows, long long ld = 0) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) return IIAN_ERR_LIMIT;
    cuuint64_t dims[2] = {(cuuint64_t) K, (cuuint64_t) rows};
    cuuint64_t strides[1] = {(cuuint64_t) (ld > 0 ? ld : K) * 2};
    cuuint32_t box[2] = {(cuuint32_t) TC_BK, (cuuint32_t) box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? IIAN_OK : 2000 + (int) r;
}

}  // namespace iian
