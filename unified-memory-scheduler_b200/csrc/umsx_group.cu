// umsx_group_rows: a router's picks sorted into one run of rows per expert.
//
// A stable counting sort of T*k jobs by expert in ONE launch without global scratch: a cluster of
// up to eight CTAs splits the jobs into one contiguous piece per warp; each warp counts its piece
// per expert (lanes of equal expert find one another with a ballot per bit, so no atomics and one fixed
// order; match_any takes an SM about 50 cycles a warp and bounded the kernel), the counts are scanned over the warps of a CTA, over the CTAs through distributed shared
// memory and over the experts, and a second walk over the piece gives every job its row.
// Bound: two dependent walks and three barriers, so latency; the ids are read twice (the second
// time from cache) and 8 bytes per job are written once.
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

constexpr int kGroupCluster = 8, kBatch = 8;  // kBatch: steps of ids a warp has in flight
constexpr int kGroupSmemMax = 200 * 1024;

// Shared memory: hist[warps][E], total[E], all[E], base[E], 32 partial sums.
size_t group_smem(int warps, int experts) { return ((size_t)(warps + 3) * experts + 32) * sizeof(int); }

// Lanes of the warp that hold the same expert.
__device__ __forceinline__ unsigned same_expert(int e, int bits) {
    unsigned same = kFull;
    for (int b = 0; b < bits; ++b) {
        const bool set = e >> b & 1;
        const unsigned v = __ballot_sync(kFull, set);
        same &= set ? v : ~v;
    }
    return same;
}

__global__ void __launch_bounds__(1024) k_group_rows(const int32_t *ids, int64_t jobs, int top_k, int E, int32_t *offsets,
                                                     int32_t *row_token, int32_t *row_of_job) {
    extern __shared__ int smem[];
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    int *hist = smem, *total = smem + warps * E, *all = total + E, *base = all + E, *part = base + E;
    for (int i = tid; i < warps * E; i += blockDim.x) hist[i] = 0;
    __syncthreads();

    // this warp's piece: whole steps of 32 jobs
    const int64_t steps = (jobs + 31) / 32, per = (steps + ctas * warps - 1) / (ctas * warps);
    const int64_t first = (int64_t)(rank * warps + warp) * per * 32;
    const int64_t last = min(first + per * 32, jobs);
    int *mine = hist + warp * E;
    const int bits = 32 - __clz(E);
    int id[kBatch];
    auto fetch = [&](int64_t i) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            id[j] = i + 32 * j < last ? __ldg(ids + i + 32 * j) : E;
            if (id[j] < 0 || id[j] >= E) id[j] = E;  // of no group
        }
    };
    for (int64_t i = first + lane; i - lane < last; i += 32 * kBatch) {
        fetch(i);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            if (i - lane + 32 * j >= last) break;
            const unsigned same = same_expert(id[j], bits);
            if (id[j] < E && lane == __ffs(same) - 1) mine[id[j]] += __popc(same);
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
    // exclusive scan over the experts (at most 1024: one value per thread; smaller CTAs loop)
    int carry = 0;
    for (int e0 = 0; e0 < E; e0 += blockDim.x) {
        const int e = e0 + tid, v = e < E ? all[e] : 0;
        int incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(kFull, incl, o);
            if (lane >= o) incl += u;
        }
        if (lane == 31) part[warp] = incl;
        __syncthreads();
        int lead = 0, sum = 0;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) lead += part[w];
            sum += part[w];
        }
        const int start = carry + lead + incl - v;
        if (e < E) {
            base[e] += start;
            if (rank == 0) offsets[e] = start;
        }
        carry += sum;
        __syncthreads();
    }
    const int rows = carry;
    if (rank == 0 && tid == 0) offsets[E] = rows;
    const bool once = per <= kBatch;  // the ids are still in registers
    for (int64_t i0 = first + lane; i0 - lane < last; i0 += 32 * kBatch) {
        if (!once) fetch(i0);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int64_t i = i0 + 32 * j;
            if (i - lane >= last) break;
            const int e = id[j];
            const unsigned same = same_expert(e, bits);
            int row = -1;
            if (e < E) row = base[e] + mine[e] + __popc(same & ((1u << lane) - 1u));
            __syncwarp();
            if (e < E && lane == __ffs(same) - 1) mine[e] += __popc(same);
            __syncwarp();
            if (i < last) row_of_job[i] = row;
            if (row >= 0) row_token[row] = (int32_t)((uint32_t)i / (uint32_t)top_k);
        }
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
    // One CTA up to 1024 jobs (one step per warp): a cluster's two extra barriers cost more than they save there.
    const int ctas = jobs <= 1024 ? 1 : kGroupCluster;
    // warps: no more than there are steps, no more than shared memory has counters for (E = 1024: 32 still fit)
    int warps = (int)std::min<int64_t>(32, std::max<int64_t>(4, (jobs + 32 * ctas - 1) / (32 * ctas)));
    const size_t smem = group_smem(warps, experts);
    cudaError_t e = cudaFuncSetAttribute(k_group_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, kGroupSmemMax);
    if (e == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(ctas);
        cfg.blockDim = dim3(warps * 32);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = static_cast<cudaStream_t>(stream);
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = ctas;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, k_group_rows, ids, jobs, top_k, experts, offsets, row_token, row_of_job);
    }
    if (e != cudaSuccess) return fail(UMSX_EDEVICE, std::string("group_rows launch: ") + cudaGetErrorString(e));
    record_launches(1);
    return UMSX_OK;
}
