// Device primitives of the tensor-core products: mbarriers, bulk tensor copies
// and tcgen05 (matrix instructions, tensor memory), sm_100a only.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <stdint.h>

namespace abft {

// cuTensorMapEncodeTiled (null when the driver does not provide it) and the
// polls of a wait (abft_set_wait_limit).
PFN_cuTensorMapEncodeTiled_v12000 encode_tiled();
int wait_limit();

namespace tensor {

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// Programmatic launch: every kernel of the products but the column checksum (which is
// launched plainly) first waits until the work before it in the stream is complete and
// visible, then lets the next one start up beside it. What a kernel does before the
// wait touches no global memory.
__device__ __forceinline__ void wait_for_stream() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// One lane of the warp (all lanes call). Copies and matrix instructions take
// their operands from the warp's uniform registers; in a branch on an elected
// lane they are cheaper to fill than in a branch on a lane number (0.30 us a
// chunk of copies and matrix instructions against 0.44).
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

// Address of the same shared variable in the cluster's CTA 0.
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The two halves of a cluster barrier whose first only says that a CTA runs.
__device__ __forceinline__ void cluster_arrive_relaxed() {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// Address of the same shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}

__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}

// --------------------------------------------------------------- mbarriers ---

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void bar_init_fence() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Arrive on a barrier of any CTA of the cluster (address from in_leader). What it
// announces is that tensor memory was read, so it needs no release of cluster
// scope, which would first wait for the warp's stores to global memory (bf16
// gradient of 4096 x 4096 weights from 64 tokens: 36 us with it, 26 us without).
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// -------------------------------------------------------- bulk tensor copy ---

// 2-d box at (x, y) into this CTA's shared memory; completes on `bar`, which
// for CG = 2 may lie in the pair's leader.
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
            "[%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
            "{%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ------------------------------------------------------------------ tcgen05 ---

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns) {
    if constexpr (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
}

template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
    else
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Arrive on `bar` when the matrix instructions issued so far have finished
// (CG = 2: on the same barrier of both CTAs of the pair).
template <int CG>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                     : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                bar),
            "h"((uint16_t)3)
            : "memory");
}

// D (+)= A B^T for one step of 32 bytes along K. INT8: 8-bit integers into
// 32-bit ones, else 16-bit floats into 32-bit ones.
template <int CG, bool INT8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    const uint32_t on = add ? 1u : 0u;
#define ABFT_MMA(group, kind)                                                                             \
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::" group ".kind::" kind \
                 " [%0], %1, %2, %3, p;\n}\n" ::"r"(d),                                                    \
                 "l"(a), "l"(b), "r"(idesc), "r"(on)                                                       \
                 : "memory")
    if constexpr (CG == 1 && INT8) ABFT_MMA("1", "i8");
    if constexpr (CG == 1 && !INT8) ABFT_MMA("1", "f16");
    if constexpr (CG == 2 && INT8) ABFT_MMA("2", "i8");
    if constexpr (CG == 2 && !INT8) ABFT_MMA("2", "f16");
#undef ABFT_MMA
}

// Shared-memory operand of a matrix instruction, 128-byte swizzle (the layout
// a bulk tensor copy with that swizzle writes; base aligned to 1024 bytes).
//   K-major: rows of 128 bytes along K, groups of 8 rows 1024 bytes apart.
//   MN-major: boxes of 64 elements along M/N (128 bytes) x 64 rows of K; groups
//   of 8 rows of K are 1024 bytes apart, the next 64 along M/N one box (8192
//   bytes) further.
__device__ __forceinline__ uint64_t operand(uint32_t addr, bool mn_major) {
    const uint64_t leading = mn_major ? 8192 >> 4 : 1;
    return (uint64_t)((addr & 0x3ffff) >> 4) | leading << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// Instruction descriptor: shape M x N, types (int8: S8 x S8 -> S32; else F16
// or BF16 -> F32), operands MN-major where set.
constexpr uint32_t instruction(int m, int n, bool int8, bool bf16, bool a_mn, bool b_mn) {
    const uint32_t type = int8 || bf16 ? 1u : 0u;
    return (int8 ? 2u : 1u) << 4 | type << 7 | type << 10 | (a_mn ? 1u : 0u) << 15 | (b_mn ? 1u : 0u) << 16 |
           (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

// 32 columns of this warp's 32 lanes of tensor memory.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}

#define ABFT_R8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), \
                      "+r"(r[i + 6]), "+r"(r[i + 7])
// Waits for the loads before it. The values pass through it, so that no use of
// them can be moved ahead of the wait; further arrays pass through after_wait.
__device__ __forceinline__ void tmem_wait_load(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : ABFT_R8(r, 0), ABFT_R8(r, 8), ABFT_R8(r, 16), ABFT_R8(r, 24)::"memory");
}
__device__ __forceinline__ void after_wait(uint32_t (&r)[32]) {
    asm volatile("" : ABFT_R8(r, 0), ABFT_R8(r, 8), ABFT_R8(r, 16), ABFT_R8(r, 24)::"memory");
}
#undef ABFT_R8

}  // namespace tensor
}  // namespace abft
