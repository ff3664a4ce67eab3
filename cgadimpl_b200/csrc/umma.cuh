// umma.cuh -- what the sm_100a matrix kernels are built from: tiled TMA loads, tensor memory, tcgen05.mma on bf16
// operands with fp32 accumulators, shared-memory and instruction descriptors, and waits that give up.
#pragma once
#include <cuda.h>

#include "agb_device.cuh"

namespace agb {

// ---------------------------------------------------------------- waits
// A wait that gives up after kTcPollLimit polls, or as soon as another role of the CTA has given up.  The polls carry no time
// hint: with the 10 us hint of mbar_try_wait the 4096 x 4096 x 18944 loss took 423 us, without it 413 us.  A poll takes 20 ns at
// least, so the limit is 80 ms or more, against the few milliseconds of the longest tile.
constexpr int kTcPollLimit = 1 << 22;
__device__ __forceinline__ bool mbar_poll(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status) {
    for (int i = 0; i < kTcPollLimit; ++i) {
        if (mbar_poll(bar, parity)) return true;
        if (*abort_flag) return false;
    }
    *abort_flag = 1;
    atomicExch(status, 6 /* AGB_ERR_TIMEOUT */);
    return false;
}
// One lane of the warp.  The branches that issue TMA and tcgen05 instructions are taken by elect.sync, not by comparing the lane
// number: those instructions want warp-uniform operands, and where the compiler sees that one lane alone runs the branch it needs no
// loop over lanes around each of them (4096 x 4096 x 18944 loss: 511 us with `lane == 0`, 423 us with this).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Arrives on the barrier of the CTA pair's leader (shared::cluster address).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t leader_address(const void* p) {
    uint32_t out;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(out) : "r"(smem_u32(p)));
    return out;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// Both CTAs of a pair; every thread of both takes part.
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// ---------------------------------------------------------------- tiled TMA load (no multicast)
// Coordinates in elements: x (innermost) is a multiple of 64 in every call, so each copy starts on a 128-byte boundary
// of the row.  Coordinates beyond the tensor read zeros.  `bar`: a shared::cluster address; in a pair (CG 2) it is the leader's,
// the data always goes to the issuing CTA.
template <int CG>
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    if (CG == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                         smem_u32(dst)),
                     "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                     : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                smem_u32(dst)),
            "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}

// ---------------------------------------------------------------- tensor memory
// CG 2: one warp of each CTA of the pair.
template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* smem_out, uint32_t columns) {
    if (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_out)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_out)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
    if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this thread's lane (the warp's quarter of the 128 lanes), fp32.  The values may be read after tmem_wait().
__device__ __forceinline__ void tmem_load32_async(uint32_t addr, uint32_t (&r)[32]) {
    __syncwarp();                                      // .aligned: the whole warp, together
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    tmem_load32_async(addr, r);
    tmem_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// ---------------------------------------------------------------- tiled TMA store
// A box of 128-byte rows from shared memory (128-byte swizzle) to coordinates (x, y, z); what lies beyond the tensor is not written.
// One thread issues it after every writer's fence_async() and a barrier between them.
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(smem_u32(src)), "r"(x),
                 "r"(y), "r"(z)
                 : "memory");
}
// The same, added to fp32 values in place.
__device__ __forceinline__ void tma_add_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                 "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// All but the last N groups of this thread have been read from shared memory.
template <int N>
__device__ __forceinline__ void tma_store_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void tma_store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// ---------------------------------------------------------------- descriptors
// Shared-memory matrix descriptor, 128-byte swizzle (layout 2), descriptor version 1.
//   K-major tile: rows of 64 elements (128 bytes), groups of 8 rows 1024 bytes apart (the stride field); the leading field is
//   not used.  The next 16 of K are 32 bytes further.
//   MN-major tile: for every block of 64 of M (or N) a run of K rows of 128 bytes; blocks `block_bytes` apart (the leading
//   field), groups of 8 K rows 1024 bytes apart (the stride field).  The next 16 of K are 2048 bytes further.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t block_bytes) {
    return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (static_cast<uint64_t>(block_bytes >> 4) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor of kind::f16: D fp32, A and B bf16, M x N, operands K-major unless the mn flags say otherwise.
__device__ __forceinline__ uint32_t mma_idesc(int M, int N, int a_mn, int b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a_mn) << 15) | (static_cast<uint32_t>(b_mn) << 16) |
           (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
template <int CG>
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    if (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
            : "memory");
}
// Arrives on `bar` (in a pair: on the barrier at this offset in both CTAs) once all MMAs issued so far by this thread have completed.
template <int CG>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    if (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                     "h"(static_cast<uint16_t>(3))
                     : "memory");
}

}  // namespace agb
