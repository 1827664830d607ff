// tcgen05 / TMA building blocks for kernels that run on one CTA or on a CTA pair (CG = 1 or 2), in
// addition to umsx_tc.cuh.
//
// In a pair (a cluster of two CTAs) one MMA of M = 256 takes 128 rows of A and half the rows of B from
// each CTA's shared memory, at the same offsets, and leaves 128 rows of D in each CTA's tensor memory.
// The even CTA (the leader) issues it; the barriers that its operands complete live with the leader.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "umsx_device.cuh"
#include "umsx_tc.cuh"

namespace umsx {
namespace tc {

template <int CG>
__device__ __forceinline__ void pair_tmem_alloc(uint32_t *dst_smem, uint32_t ncols) {
    if constexpr (CG == 1) {
        tmem_alloc(dst_smem, ncols);
        tmem_relinquish();
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst_smem)), "r"(ncols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG>
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    if constexpr (CG == 1) tmem_dealloc(taddr, ncols);
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// D (+)= A * B^T for one slice of 32 bytes of K; issued by one thread: 16-bit operands of a pair (by the leader) ...
__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}
// ... and 8-bit operands of one CTA.
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc),
                 "r"(idesc), "r"(accumulate)
                 : "memory");
}

// Arrive on `bar` (of both CTAs of a pair, at the same offset) once every MMA issued so far has completed.
template <int CG>
__device__ __forceinline__ void pair_commit(uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3)
            : "memory");
}

// The same to the leader's barrier alone.
template <int CG>
__device__ __forceinline__ void leader_commit(uint32_t bar) {
    if constexpr (CG == 1) pair_commit<1>(bar);
    else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrival at a barrier of the pair.  It orders tensor-memory reads (tcgen05 fences around it) but publishes no
// writes to the other CTA, so it needs no cluster scope, whose fence would wait for every store in flight.
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// The same, publishing this thread's writes to the other CTA.
__device__ __forceinline__ void publish_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Tiled TMA loads into this CTA that complete on the barrier at shared::cluster address `bar` (this CTA's, or its leader's).
template <int CG>
__device__ __forceinline__ void pair_tma_2d(uint32_t dst, const void *tmap, int x, int y, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
                     "[%4];" ::"r"(dst),
                     "l"(tmap), "r"(x), "r"(y), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
                     "{%2, %3}], [%4];" ::"r"(dst),
                     "l"(tmap), "r"(x), "r"(y), "r"(bar)
                     : "memory");
}
template <int CG>
__device__ __forceinline__ void pair_tma_3d(uint32_t dst, const void *tmap, int x, int y, int z, uint32_t bar) {
    if constexpr (CG == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
                     "%4}], [%5];" ::"r"(dst),
                     "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
                     "{%2, %3, %4}], [%5];" ::"r"(dst),
                     "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
                     : "memory");
}

// The leader's copy of a shared-memory object of this CTA, as a shared::cluster address.
__device__ __forceinline__ uint32_t leader_addr(uint32_t p) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(p));
    return a;
}

// Shared-memory matrix descriptor, 128-byte swizzle, 1024-byte atoms of eight 128-byte lines.
//   K-major:  a line is 128 bytes of K of one row; atoms of eight rows follow one another
//   MN-major: a line is 64 16-bit values of M (or N) at one k; atoms of eight k follow one another,
//             the next 64 values of M (or N) start `block` bytes on
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn_major, uint32_t block) {
    return ((addr & 0x3FFFFull) >> 4) | ((uint64_t)(mn_major ? block >> 4 : 1u) << 16) | (64ull << 32) | (1ull << 46) |
           (2ull << 61);
}

// Instruction descriptor: fp32 accumulators; a_fmt, b_fmt: kind::f16 0 f16, 1 bf16; kind::f8f6f4 0 e4m3.
__host__ __device__ constexpr uint32_t operand_idesc(int fmt, bool a_mn, bool b_mn, int M, int N) {
    return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// 16 consecutive fp32 columns of this warp's 32 TMEM lanes, in the fragment order of 8 x 8 matrices: r[8h + 4i + 2u + j]
// is lane 16h + 8u + (thread / 4), column 8i + 2 (thread % 4) + j.  Complete after tmem_wait_ld(r).
__device__ __forceinline__ void tmem_ld_frag_async(uint32_t taddr, uint32_t (&r)[16]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
        asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[8 * h]), "=r"(r[8 * h + 1]), "=r"(r[8 * h + 2]), "=r"(r[8 * h + 3]), "=r"(r[8 * h + 4]),
                       "=r"(r[8 * h + 5]), "=r"(r[8 * h + 6]), "=r"(r[8 * h + 7])
                     : "r"(taddr + ((uint32_t)(16 * h) << 16)));
}
// All loads so far are complete.  The values are operands of the wait, so that no use of them moves above it.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[16]) {
    tmem_ld_frag_async(taddr, r);
    tmem_wait_ld(r);
}

// Four 8 x 8 matrices of 16-bit values in fragment order, transposed, to the 16-byte rows that the lanes name
// (lanes 8m .. 8m + 7: the rows of matrix m).
__device__ __forceinline__ void stmatrix_trans4(void *row, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(row)), "r"(a), "r"(b),
                 "r"(c), "r"(d)
                 : "memory");
}

__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// True in one lane of a converged warp.  The copies and MMAs are issued under it and not under a test of the
// lane: their operands then stay in uniform registers (four MMAs took 490 cycles to issue under `lane == 0`).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}

// ---- bounded waits -----------------------------------------------------------------------------
//
// A wait that has not ended after the CTA's limit marks the CTA as given up; every other wait of the CTA whose phase is not
// complete then ends too, and the loops look at the mark once per tile.  One asm block each (a function with a loop in it took
// 250 cycles where a phase was complete, a block 50); mark and limit lie in shared memory, where only a wait that is not over
// at once looks at them.
constexpr long long kDrainCycles = 1ll << 25;  // 17 ms, for copies and MMAs in flight at the end, which take microseconds

struct GiveUp {
    int given_up;
    long long limit;  // SM cycles
};

#define UMSX_WAIT(sem, scale, ...)                                                                                \
    asm volatile(                                                                                                 \
        "{\n\t.reg .pred p, q;\n\t.reg .b32 g;\n\t.reg .b64 t0, t, m;\n\tmov.u32 %0, 0;\n\t"                      \
        "mbarrier.try_wait.parity" sem ".shared::cta.b64 p, [%1], %2;\n\t"                                        \
        "@p bra DONE;\n\tmov.u64 t0, %%clock64;\n"                                                               \
        "AGAIN:\n\tmbarrier.try_wait.parity" sem ".shared::cta.b64 p, [%1], %2;\n\t"                             \
        "@p bra DONE;\n\tld.volatile.shared.b32 g, [%3];\n\tsetp.ne.b32 q, g, 0;\n\t@q bra LOST;\n\t"            \
        "ld.shared.b64 m, [%3+8];\n\t" scale "mov.u64 t, %%clock64;\n\tsub.s64 t, t, t0;\n\t"                  \
        "setp.lt.s64 q, t, m;\n\t@q bra AGAIN;\n\tst.volatile.shared.b32 [%3], 1;\n"                            \
        "LOST:\n\tmov.u32 %0, 1;\nDONE:\n\t}"                                                                  \
        : "=&r"(lost)                                                                                             \
        : "r"(bar), "r"(parity), "r"(give_up) __VA_ARGS__                                                         \
        : "memory")

// Whether all lanes of the (converged) warp saw the phase complete.  Where they did not, the warp leaves its loops before it
// arrives with expected bytes, copies or multiplies any more: a barrier that it has not seen free would get a second
// arrival in a phase that awaits one.  bar, give_up: shared-memory addresses.  ACROSS: the barrier hands over what the
// other CTA's threads wrote (publish_at); an acquire of cluster scope costs about 200 cycles more, so the other waits
// stay at this CTA's scope.
template <bool ACROSS = false>
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, uint32_t give_up) {
    uint32_t lost;
    if constexpr (ACROSS) UMSX_WAIT(".acquire.cluster", "");
    else UMSX_WAIT("", "");
    return !__any_sync(kFull, lost);
}
// The same for `times` limits.
__device__ __forceinline__ bool wait_long(uint32_t bar, uint32_t parity, uint32_t give_up, uint32_t times) {
    uint32_t lost;
    UMSX_WAIT("", ".reg .b64 n;\n\tcvt.u64.u32 n, %4;\n\tmul.lo.s64 m, m, n;\n\t", , "r"(times));
    return !__any_sync(kFull, lost);
}
#undef UMSX_WAIT

// The same without a verdict, whose vote costs the e4m3 kernel 8 %, for warps that may run on to the end of their tile: their
// reads give garbage, which the mark says, and their plain arrivals only end phases early.  In a CTA that has given up it ends
// at once, as the first look at the barrier does not block.
__device__ __forceinline__ void wait_or_run_on(uint32_t bar, uint32_t parity, uint32_t give_up) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b32 g;\n\t.reg .b64 t0, t, m;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%0], %1;\n\t@p bra DONE;\n\tmov.u64 t0, %%clock64;\n"
        "AGAIN:\n\tld.volatile.shared.b32 g, [%2];\n\tsetp.ne.b32 q, g, 0;\n\t@q bra DONE;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1;\n\t@p bra DONE;\n\t"
        "ld.shared.b64 m, [%2+8];\n\tmov.u64 t, %%clock64;\n\tsub.s64 t, t, t0;\n\t"
        "setp.lt.s64 q, t, m;\n\t@q bra AGAIN;\n\tst.volatile.shared.b32 [%2], 1;\nDONE:\n\t}" ::"r"(bar),
        "r"(parity), "r"(give_up)
        : "memory");
}

// A ring position: stage and the parity of its next use.
template <int STAGES>
struct Ring {
    uint32_t s = 0, phase = 0;
    __device__ __forceinline__ void next() {
        if (++s == STAGES) s = 0, phase ^= 1u;
    }
};

}  // namespace tc
}  // namespace umsx
