// umsx_group_rows: a router's picks sorted into one run of rows per expert.
//
// A stable counting sort of T*k jobs by expert in ONE launch without global scratch: a cluster of
// up to sixteen CTAs splits the jobs into one contiguous piece per warp; each warp counts its piece
// per expert (lanes of equal expert find one another with a ballot per bit, so no atomics and one fixed
// order; a ballot takes an SM 5 cycles and match_any 50), the counts are scanned over the warps of a CTA, over the CTAs
// through distributed shared memory and over the experts, and a second walk over the piece gives every job its row.
// The second walk sorts a CTA's jobs in shared memory, so that row_token is written in runs: 32 lanes that
// store to 32 rows take the SM 32 cycles, which was most of the kernel's time.
// Bound: latency (the scans over warps, CTAs and experts, the barriers between them, two dependent walks): 4.5 us for 128
// jobs, 14.3 for 16384, a launch in a graph.  Where there are many, the ballots too, eight or eleven per 32 jobs at 5
// cycles each (131072 jobs on 16 SMs: 10 K cycles of 20 us), which is why they are spread over the largest cluster there is.
// The ids are read once and 8 bytes per job written once, some MB that memory would take a microsecond for.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "umsx_device.cuh"
#include "umsx_internal.h"
#include "umsx_products.h"

namespace cg = cooperative_groups;

namespace umsx {
namespace {

constexpr int kBatch = 16;  // kBatch: steps of 32 ids a warp has in flight
constexpr int kGroupSmemMax = 200 * 1024;

constexpr int kWarpsMax = 16;

// Shared memory: hist[warps][E], total[E], all[E], base[E], local[E], 32 partial sums, then `sorted` 16-bit job numbers.
size_t group_smem(int warps, int experts, int64_t sorted) {
    return ((size_t)(warps + 4) * experts + 32) * sizeof(int) + (size_t)sorted * sizeof(uint16_t);
}

// Lanes of the warp that hold the same expert (a number below 2^BITS).
template <int BITS>
__device__ __forceinline__ unsigned same_expert(int e) {
    unsigned same = kFull;
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
        const bool set = e >> b & 1;
        const unsigned v = __ballot_sync(kFull, set);
        same &= set ? v : ~v;
    }
    return same;
}

template <int BITS>
__global__ void __launch_bounds__(32 * kWarpsMax) k_group_rows(const int32_t *ids, int64_t jobs, int top_k, int E, int sort_local,
                                                     int32_t *offsets, int32_t *row_token, int32_t *row_of_job) {
    extern __shared__ int smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    int *hist = smem, *total = smem + warps * E, *all = total + E, *base = all + E, *local = base + E, *part = local + E;
    uint16_t *sorted = reinterpret_cast<uint16_t *>(part + 32);  // sort_local: this CTA's jobs by expert
    for (int i = tid; i < warps * E; i += blockDim.x) hist[i] = 0;
    __syncthreads();

    // this warp's piece: whole steps of 32 jobs
    const int64_t steps = (jobs + 31) / 32, per = (steps + ctas * warps - 1) / (ctas * warps);
    const int64_t first = (int64_t)(rank * warps + warp) * per * 32;
    const int64_t last = min(first + per * 32, jobs), cta_first = (int64_t)rank * warps * per * 32;
    int *mine = hist + warp * E;
    int id[kBatch];
    unsigned same[kBatch];
    auto fetch = [&](int64_t i) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            id[j] = i + 32 * j < last ? __ldg(ids + i + 32 * j) : E;
            if (id[j] < 0 || id[j] >= E) id[j] = E;  // of no group
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) same[j] = same_expert<BITS>(id[j]);  // under a condition a ballot costs 20 cycles
    };
    for (int64_t i = first + lane; i - lane < last; i += 32 * kBatch) {
        fetch(i);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (i - lane + 32 * j >= last) break;
            if (id[j] < E && lane == __ffs(same[j]) - 1) mine[id[j]] += __popc(same[j]);
            __syncwarp();
        }
    }
    __syncthreads();
    // per expert: counts -> starts within the CTA
    for (int e = tid; e < E; e += blockDim.x) {
        int run = 0;
        for (int w = 0; w < warps; ++w) {
            const int c = hist[w * E + e];
            hist[w * E + e] = run;
            run += c;
        }
        total[e] = run;
    }
    cluster.sync();
    for (int e = tid; e < E; e += blockDim.x) {
        int before = 0, sum = 0;
        for (int c = 0; c < ctas; ++c) {
            const int v = cluster.map_shared_rank(total, c)[e];
            if (c < rank) before += v;
            sum += v;
        }
        all[e] = sum;
        base[e] = before;
    }
    __syncthreads();
    // exclusive scans over the experts (smaller CTAs loop): of all jobs, and of this CTA's
    int carry = 0, carry_local = 0;
    for (int e0 = 0; e0 < E; e0 += blockDim.x) {
        const int e = e0 + tid;
        for (int which = 0; which < 2; ++which) {
            const int v = e < E ? (which ? total[e] : all[e]) : 0;
            int incl = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(kFull, incl, o);
                if (lane >= o) incl += u;
            }
            if (lane == 31) part[warp] = incl;
            __syncthreads();
            int sums = lane < warps ? part[lane] : 0;  // inclusive over the warps
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(kFull, sums, o);
                if (lane >= o) sums += u;
            }
            const int sum = __shfl_sync(kFull, sums, 31), lead = warp ? __shfl_sync(kFull, sums, warp - 1) : 0;
            const int start = (which ? carry_local : carry) + lead + incl - v;
            if (e < E) {
                if (which) {
                    local[e] = start;
                } else {
                    base[e] += start;
                    if (rank == 0) offsets[e] = start;
                }
            }
            (which ? carry_local : carry) += sum;
            __syncthreads();
        }
    }
    const int rows = carry;
    if (rank == 0 && tid == 0) offsets[E] = rows;
    const bool once = per <= kBatch;  // ids and lanes are still in registers
    for (int64_t i0 = first + lane; i0 - lane < last; i0 += 32 * kBatch) {
        if (!once) fetch(i0);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int64_t i = i0 + 32 * j;
            if (i - lane >= last) break;
            const int e = id[j], leader = __ffs(same[j]) - 1;
            int at = 0;  // place among this CTA's jobs of the expert
            if (e < E && lane == leader) {
                at = mine[e];
                mine[e] = at + __popc(same[j]);
            }
            at = __shfl_sync(kFull, at, leader) + __popc(same[j] & ((1u << lane) - 1u));
            if (i < last) row_of_job[i] = e < E ? base[e] + at : -1;
            if (e < E) {
                if (sort_local) sorted[local[e] + at] = (uint16_t)(i - cta_first);
                else row_token[base[e] + at] = (int32_t)((uint32_t)i / (uint32_t)top_k);
            }
            __syncwarp();
        }
    }
    if (sort_local) {
        __syncthreads();
        for (int e = warp; e < E; e += warps)
            for (int k = lane; k < total[e]; k += 32)
                row_token[base[e] + k] = (int32_t)((uint32_t)(cta_first + sorted[local[e] + k]) / (uint32_t)top_k);
    }
    // rows behind the last group name token 0, so that a gather by them stays inside x
    for (int64_t r = rows + (int64_t)rank * blockDim.x + tid; r < jobs; r += (int64_t)ctas * blockDim.x) row_token[r] = 0;
    cluster.sync();  // a CTA whose counts another one still reads must not exit
}

umsx_status fail(umsx_status s, const std::string &msg) {
    record_error(msg.c_str());
    return s;
}

}  // namespace
}  // namespace umsx

using namespace umsx;

extern "C" umsx_status umsx_group_rows(const int32_t *ids, int tokens, int top_k, int experts, int32_t *offsets,
                                       int32_t *row_token, int32_t *row_of_job, umsx_stream stream) {
    if (tokens < 0 || top_k < 1 || experts < 1 || experts > kMaxGroups || (int64_t)tokens * top_k > 0x7ffffff0)
        return fail(UMSX_EINVAL, "group_rows takes tokens >= 0, top_k >= 1, experts 1..1024 and fewer than 2^31 - 16 jobs");
    if (!offsets || (tokens && (!ids || !row_token || !row_of_job))) return fail(UMSX_EINVAL, "null buffer");
    const int64_t jobs = (int64_t)tokens * top_k;
    const Region r[4] = {region(ids, 4, jobs, 1, 0), region(offsets, 4, experts + 1, 1, 0), region(row_token, 4, jobs, 1, 0),
                         region(row_of_job, 4, jobs, 1, 0)};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j)
            if (overlap(r[i], r[j])) return fail(UMSX_EINVAL, "an output overlaps the ids or another output");
    for (const void *q : {static_cast<const void *>(ids), static_cast<const void *>(offsets), static_cast<const void *>(row_token),
                          static_cast<const void *>(row_of_job)})
        if (reinterpret_cast<uintptr_t>(q) % 4) return fail(UMSX_EINVAL, "a buffer is not aligned to its elements");
    const auto kernel = experts < 256 ? k_group_rows<8> : k_group_rows<11>;  // bits of 0..experts
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGroupSmemMax);
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    // One CTA for few jobs, where a cluster's barriers cost more than its SMs save (us in one CTA, in eight; 128 experts: 512
    // jobs 5.9, 9.3; 1024: 7.1, 9.8; 1536: 8.3, 9.8; 2048: 9.5, 8.9).  The border is that of 128 experts: the counters' scan grows
    // with the experts and eight CTAs repeat it, so 2048 jobs of 64 experts take 9.5, 7.6, of 256 10.9, 12.0 and of 1024 12.9, 23.4.
    // Sixteen CTAs, beyond the portable cluster size and
    // only if the device can hold them, for many (in eight, in sixteen, with the warps of then; 2048: 9.0, 10.2; 4096
    // jobs of 256 experts: 13.1, 12.5; 8192: 18.7, 13.4; 131072: 27.3, 23.1).
    int ctas = jobs <= 1536 ? 1 : 8;
    if (jobs >= 4096 && e == cudaSuccess) {
        int fit = 0;
        cfg.gridDim = dim3(16);
        cfg.blockDim = dim3(32 * kWarpsMax);
        cfg.dynamicSmemBytes = kGroupSmemMax;
        at[0].val.clusterDim.x = 16;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
            cudaOccupancyMaxActiveClusters(&fit, kernel, &cfg) == cudaSuccess && fit > 0)
            ctas = 16;
        else
            cudaGetLastError();  // not an error of this call
    }
    // Warps: each costs a row of the counters' scan, so sixteen at most (16384 jobs: 14.3 us, with 32 warps 19.3; 131072: 20.2,
    // 23.1), a step of 32 jobs each in a cluster (4096: 12.5, with two steps a warp 17.8), four in a single CTA (512: 5.9, with
    // one 7.8).
    const int64_t share = 32 * ctas * (ctas == 1 ? 4 : 1);
    const int warps = (int)std::min<int64_t>(kWarpsMax, std::max<int64_t>(4, (jobs + share - 1) / share));
    // one CTA's jobs, if their 16-bit numbers fit into shared memory (at 1024 experts up to 27 K of them)
    const int64_t piece = ((jobs + 31) / 32 + ctas * warps - 1) / (ctas * warps) * warps * 32;
    // (a single CTA's few jobs are written at once: its walk over the experts would take longer)
    const bool sort_local = ctas > 1 && piece <= 65536 && group_smem(warps, experts, piece) <= (size_t)kGroupSmemMax;
    const size_t smem = group_smem(warps, experts, sort_local ? piece : 0);
    if (e == cudaSuccess) {
        cfg.gridDim = dim3(ctas);
        cfg.blockDim = dim3(warps * 32);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = static_cast<cudaStream_t>(stream);
        at[0].val.clusterDim.x = ctas;
        e = cudaLaunchKernelEx(&cfg, kernel, ids, jobs, top_k, experts, (int)sort_local, offsets, row_token, row_of_job);
    }
    if (e != cudaSuccess) {
        (void)cudaGetLastError();  // reported here, not by the next launch's check
        return fail(UMSX_EDEVICE, std::string("group_rows launch: ") + cudaGetErrorString(e));
    }
    record_launches(1);
    return UMSX_OK;
}
