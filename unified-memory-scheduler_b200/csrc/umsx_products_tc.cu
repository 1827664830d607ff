// Ragged products of 16-bit operands on the tensor cores (tcgen05), forward and both gradients.
//
// out[r][f] = sum_c R[r][c] F[f][c] with the FEATURES as the MMA's M (128 per CTA, TMEM lanes) and the
// group's ROWS as its N.  N goes in steps of 32, so a group of 140 rows costs 160 and not 256:
// with the rows as M, ragged groups would be padded to 128.  The rows of a group are split into equal
// tiles of at most 256.
//
//   forward  F = w (K-major), R = x (K-major)           contraction k
//   dx       F = w (MN-major: k is contiguous), R = dy  contraction n
//   dw       F = x, R = dy, both MN-major               contraction: the group's rows
//
// One persistent CTA pair per two SMs; pair i takes tiles i, i + pairs, ... of the list (group, feature
// tile, row tile), which every CTA derives from the offsets, so there is no scheduler state and the order of
// sums is fixed.  A pair's CTA reads half the rows' operand; single CTAs with tiles of 128 x 256 took 406, 401 and 500 us
// for forward, dx and dw where pairs took 356, 388 and 426 (bf16, 32 experts of 512 rows, 5760 x 2880; now, on another card,
// 363, 397 and 437), and were no faster for 128 features or fewer either (16 x 1024 rows, 128 x 2048: both 27 to 31 us).
// Roles: warp 0 TMA, warp 1 MMA, warps 2-9 epilogue, warp 10 (dw) the group's ragged end.
// Two accumulators of 256 columns: the epilogue drains one while the MMA fills the other.
//
// An accumulator of the tensor cores is less exact than rounded fp32 additions, the more so the longer it is added to (error
// 2.5e-6 of the result at a contraction of 2048, against 0.8e-6).  Outputs in fp32 therefore get a fresh accumulator
// every 512 of the contraction (kAccumulate32), which the epilogue adds up in registers.  In 16-bit outputs the last
// rounding hides 4096 of it (kAccumulate16), not any length: in one accumulator an f16 dw of 2^20 rows was 6.4e-3 of the value off.
//
// dw's contraction ends inside a block of 64 rows; the rows behind it belong to the next group.  Warp
// 10 zeroes them in both operands (a zero in one would leave 0 * NaN) up to the next multiple of 16, where
// the MMAs stop.  Only that last stage of a tile goes through it: handing every stage on cost 1.8 K cycles a stage.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>

#include "umsx_device.cuh"
#include "umsx_internal.h"
#include "umsx_pair.cuh"
#include "umsx_products.h"

namespace umsx {

__device__ uint32_t g_product_err;  // a bounded wait gave up (umsx_products_status)

namespace {

constexpr int kBF = 128, kBC = 64;  // features per CTA, contraction per stage
constexpr int kPair = 2;            // CTAs that share a tile of the 16-bit kernel
constexpr int kRowsMax = 256;       // rows of a tile (of a pair: 128 in each CTA)
constexpr int kRowBox = 32;         // rows of one K-major TMA box
constexpr int kThreads = 352, kEpilogueWarps = 8;
constexpr uint32_t kTmemCols = 512;
constexpr int kStageRow = 80;  // bytes of a staged output row: 64 of data; 80 spreads eight rows over all banks

struct TcParams {
    int groups, features, contraction, out_rows, out_dtype, fmt, vec, segment;
    int64_t rows;
    const int32_t *offsets;
    void *out;
    int64_t ldo, out_group;
    int fault_cta;
    long long wait_limit;
};

template <int MODE>
struct Shape {
    static constexpr bool kFMn = MODE != kForward, kRMn = MODE == kGradWeight;
    static constexpr int kBytesF = kBF * kBC * 2, kBytesR = kRowsMax / kPair * kBC * 2;
    static constexpr int kStages = 6;
    static constexpr size_t kSmem = 1024 + (size_t)kStages * (kBytesF + kBytesR) + kEpilogueWarps * 16 * kStageRow;
};

// One tile of the list: rows [row0, row0 + rows) x features [f0, f0 + 128 * CG) of group g; CG: CTAs that share it.
struct Tile {
    int g, f0, row0, rows, c0, c_len;  // c0: first contraction index (dw: a row of x and dy)
    int n;                             // rows rounded up to the MMA's N
};

template <int CG, int MODE>
struct Tiles {
    const int *start, *prefix;  // shared memory: first row of group g (and behind the last), tiles before group g
    int groups, f_tiles, features, contraction, out_rows;

    __device__ static int row_tiles(int rows) { return (rows + kRowsMax - 1) / kRowsMax; }

    // Tile t, by a converged warp that asks for ascending ones; `lo` is its group so far.
    __device__ __forceinline__ Tile get(int t, int &lo, int lane) const {
        while (true) {  // 32 groups a step: a binary search's dependent reads took 500 cycles of every tile
            const unsigned below = __ballot_sync(kFull, prefix[min(lo + 1 + lane, groups)] <= t);
            lo += __popc(below);
            if (below != kFull) break;
        }
        // A value that comes out of lane 0's register is the same in all lanes for the compiler too: the loops' counters and the
        // descriptors made of them then live in uniform registers, where the MMAs and copies want them.
        const auto uniform = [](int v) { return __shfl_sync(kFull, v, 0); };
        lo = uniform(lo);
        const int a = uniform(start[lo]), m = max(0, uniform(start[lo + 1]) - a);
        const int all = MODE == kGradWeight ? out_rows : m, rt = row_tiles(all);
        const int local = t - uniform(prefix[lo]);
        int i = 0, j = local, each = all;
        if (rt > 1) i = local % rt, j = local / rt, each = (all + rt - 1) / rt;
        // equal tiles, in steps of the MMA's N
        constexpr int kStep = 16 * CG;
        const int size = min(kRowsMax, (each + kStep - 1) / kStep * kStep);
        Tile x;
        x.g = lo;
        x.f0 = j * kBF * CG;
        x.row0 = i * size;
        x.rows = max(0, min(size, all - x.row0));
        x.n = (x.rows + kStep - 1) / kStep * kStep;
        if (MODE == kGradWeight) {
            x.c0 = a;
            x.c_len = m;
        } else {
            x.row0 += a;
            x.c0 = 0;
            x.c_len = contraction;
        }
        return x;
    }
};

// Tiles before every group, by one warp.
template <int CG, int MODE>
__device__ __forceinline__ void tile_prefix(const int *start, int *prefix, int groups, int f_tiles, int out_rows, int lane) {
    int carry = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {
        const int g = g0 + lane;
        int tiles = 0;
        if (g < groups)
            tiles = f_tiles * Tiles<CG, MODE>::row_tiles(MODE == kGradWeight ? out_rows : max(0, start[g + 1] - start[g]));
        int incl = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(kFull, incl, o);
            if (lane >= o) incl += v;
        }
        if (g < groups) prefix[g] = carry + incl - tiles;
        carry += __shfl_sync(kFull, incl, 31);
    }
    if (lane == 0) prefix[groups] = carry;
}

// ---- epilogue ---------------------------------------------------------------------------------
//
// A warp holds 32 features (its TMEM lanes) x 16 rows in fragment order.  16-bit outputs are transposed through
// shared memory (stmatrix), so that a lane stores 16 bytes of one row: one store instruction instead of eight.
struct OutTile {
    void *out;
    int64_t at, ldo;  // element of the warp's first feature in the tile's first row
    int dtype, features, rows;  // valid features of the warp's 32, valid rows of the tile
    bool vec;         // 16-byte stores: base and rows are aligned, features is a multiple of 8 from an aligned start
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack16(uint32_t lo, uint32_t hi) {
    const float a = __uint_as_float(lo), b = __uint_as_float(hi);
    if constexpr (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 16 rows of 32 16-bit features from v (fragment order) to shared memory, row by row.
template <bool BF16>
__device__ __forceinline__ void stage16(uint8_t *to, int lane, const uint32_t (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t m[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int e = 8 * (q >> 1) + 4 * i + 2 * (q & 1);
            m[q] = pack16<BF16>(v[e], v[e + 1]);
        }
        tc::stmatrix_trans4(to + (8 * i + (lane & 7)) * kStageRow + (lane >> 3) * 16, m[0], m[1], m[2], m[3]);
    }
}

// Rows c0 .. c0 + 15 of the tile from v (fragment order), through the warp's staging of 16 rows.  RUNS: where 16-byte
// stores cannot be used, a store of 32 neighbours for each row, not eight elements of a row by each lane (bf16 5759 x 2880, 32
// experts of 512 rows: 365 us, now 377, and 600; e4m3 346, 668).  Not for dw, whose width is odd only where an operand is too, unless that
// is padded: the code's registers cost its fp32 outputs 5 %.
template <bool RUNS>
__device__ __forceinline__ void store_chunk(const OutTile &o, uint8_t *stage, int lane, int c0, const uint32_t (&v)[16]) {
    if (o.dtype == UMSX_DTYPE_F32) {
        float *p = static_cast<float *>(o.out) + o.at + (int64_t)(c0 + 2 * (lane & 3)) * o.ldo + (lane >> 2);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const bool on = c0 + 8 * i + 2 * (lane & 3) + j < o.rows;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (on && 8 * q + (lane >> 2) < o.features)
                        p[(8 * i + j) * o.ldo + 8 * q] = __uint_as_float(v[8 * (q >> 1) + 4 * i + 2 * (q & 1) + j]);
            }
        return;
    }
    __syncwarp();  // the previous rows have been read out of the staging
    if (o.dtype == UMSX_DTYPE_BF16) stage16<true>(stage, lane, v);
    else stage16<false>(stage, lane, v);
    __syncwarp();
    uint16_t *p = static_cast<uint16_t *>(o.out) + o.at;
    if (RUNS && !o.vec) {
        const int rows = min(16, o.rows - c0);
        if (lane < o.features) {
            p += (int64_t)c0 * o.ldo + lane;
#pragma unroll
            for (int r = 0; r < 16; ++r, p += o.ldo)
                if (r < rows) *p = *reinterpret_cast<const uint16_t *>(stage + r * kStageRow + lane * 2);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = 8 * i + (lane >> 2), f = 8 * (lane & 3);
        if (c0 + row >= o.rows || f >= o.features) continue;
        const uint4 w = *reinterpret_cast<const uint4 *>(stage + row * kStageRow + f * 2);
        uint16_t *d = p + (int64_t)(c0 + row) * o.ldo + f;
        if ((RUNS || o.vec) && f + 8 <= o.features) {
            *reinterpret_cast<uint4 *>(d) = w;
        } else {
            const uint16_t *h = reinterpret_cast<const uint16_t *>(&w);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (f + j < o.features) d[j] = h[j];
        }
    }
}

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1) k_product_tc(const __grid_constant__ CUtensorMap map_f,
                                                            const __grid_constant__ CUtensorMap map_r, const TcParams p) {
    using S = Shape<MODE>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    uint8_t *sF = smem, *sR = smem + S::kStages * S::kBytesF;
    __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages], d_full[2], d_empty[2];
    // dw, a tile's ragged last stage: its copies to this CTA, and both CTAs' zeroing
    __shared__ __align__(8) uint64_t tail[S::kStages], fixed[S::kStages], last;
    __shared__ uint32_t tmem_s;
    __shared__ tc::GiveUp give_up;
    __shared__ int start[kMaxGroups + 1], prefix[kMaxGroups + 1];

    const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
    const uint32_t rank = tc::cluster_rank();
    const int cluster = blockIdx.x / kPair, clusters = gridDim.x / kPair;

    for (int g = tid; g <= p.groups; g += kThreads) start[g] = group_start(p.offsets, g, p.rows);
    if (tid == 0) {
        give_up.given_up = 0;
        give_up.limit = p.wait_limit;
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&tail[s], 1);
            mbar_init(&fixed[s], kPair);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&last, 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&d_full[b], 1);
            mbar_init(&d_empty[b], kPair * kEpilogueWarps);
        }
    }
    if (warp == 1) tc::pair_tmem_alloc<kPair>(&tmem_s, kTmemCols);
    __syncthreads();
    const int f_tiles = (p.features + kBF * kPair - 1) / (kBF * kPair);
    if (warp == 0) tile_prefix<kPair, MODE>(start, prefix, p.groups, f_tiles, p.out_rows, lane);
    tc::fence_before_sync();
    tc::cluster_sync_all();  // barriers are initialised before the peer's copies and arrivals reach them
    tc::fence_after_sync();
    const uint32_t tmem = __shfl_sync(kFull, tmem_s, 0);
    const int total = __shfl_sync(kFull, prefix[p.groups], 0);
    const Tiles<kPair, MODE> tiles{start, prefix, p.groups, f_tiles, p.features, p.contraction, p.out_rows};

    const uint32_t up = smem_u32(&give_up), aF = smem_u32(sF), aR = smem_u32(sR);
    const uint32_t b_full = smem_u32(full), b_empty = smem_u32(empty), b_dfull = smem_u32(d_full), b_dempty = smem_u32(d_empty),
                   b_tail = smem_u32(tail), b_fixed = smem_u32(fixed);
    const auto stop = [&] { return __shfl_sync(kFull, *const_cast<volatile int *>(&give_up.given_up), 0) != 0; };

    if (warp == 0) {
        tc::Ring<S::kStages> r;
        uint32_t tails = 0, tail_phase = 0, used = 0;  // bit s: stage s holds a ragged end; uses of tail[s], mod 2; stages in use
        int group = 0;
        bool withhold = (int)blockIdx.x == p.fault_cta, on = true;
        for (int t = cluster; on && t < total && !stop(); t += clusters) {
            const Tile x = tiles.get(t, group, lane);
            const int kb = (x.c_len + kBC - 1) / kBC;
            if (!x.rows) continue;
            const int half = x.n / kPair;  // rows of this CTA's part of R
            const int boxes = S::kRMn ? (half + 63) / 64 : (half + kRowBox - 1) / kRowBox;
            const uint32_t bytes = S::kBytesF + boxes * (S::kRMn ? 64 : kRowBox) * kBC * 2;
            const int f0 = x.f0 + (int)rank * kBF, r0 = x.row0 + (int)rank * half;
            for (int kk = 0; kk < kb; ++kk, r.next()) {
                if (!(on = tc::wait(b_empty + 8 * r.s, r.phase ^ 1u, up))) break;
                if (withhold) {
                    withhold = false;
                    continue;
                }
                const bool ragged = MODE == kGradWeight && kk == kb - 1 && (x.c_len & 15);
                used |= 1u << r.s;
                if (ragged) tails |= 1u << r.s, tail_phase ^= 1u << r.s;
                else tails &= ~(1u << r.s);
                if (tc::elect_one()) {
                    uint32_t bar = (ragged ? b_tail : b_full) + 8 * r.s;
                    if (ragged) {
                        tc::expect_tx(bar, bytes);  // each CTA's own, for its warp 10
                        if (rank == 0) tc::arrive(b_full + 8 * r.s);
                    } else {
                        if (rank == 0) tc::expect_tx(bar, kPair * bytes);
                        bar = tc::leader_addr(bar);
                    }
                    const int c = x.c0 + kk * kBC;
                    const uint32_t dF = aF + r.s * S::kBytesF, dR = aR + r.s * S::kBytesR;
                    if constexpr (MODE == kForward) {
                        tc::pair_tma_3d<kPair>(dF, &map_f, c, f0, x.g, bar);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if constexpr (MODE == kGradInput) tc::pair_tma_3d<kPair>(dF + h * 8192, &map_f, f0 + 64 * h, c, x.g, bar);
                            else tc::pair_tma_2d<kPair>(dF + h * 8192, &map_f, f0 + 64 * h, c, bar);
                        }
                    }
                    for (int b = 0; b < boxes; ++b) {
                        if constexpr (S::kRMn) tc::pair_tma_2d<kPair>(dR + b * 8192, &map_r, r0 + 64 * b, c, bar);
                        else tc::pair_tma_2d<kPair>(dR + b * kRowBox * 128, &map_r, c, r0 + kRowBox * b, bar);
                    }
                }
                __syncwarp();
            }
        }
        // A CTA must not exit before the last arrivals at its barriers, nor, where a wait gave up and the MMAs did not
        // read them, under copies in flight: those of the odd CTA complete on the leader's barrier, and land long before
        // its own wait here has run out.
        for (uint32_t s = 0; s < (uint32_t)S::kStages; ++s) {
            if (!(used >> s & 1u)) continue;
            const uint32_t last_phase = r.phase ^ (s >= r.s ? 1u : 0u);
            if (mbar_wait_bounded(&empty[s], last_phase, tc::kDrainCycles)) continue;
            if (tails >> s & 1u) mbar_wait_bounded(&tail[s], (tail_phase >> s & 1u) ^ 1u, tc::kDrainCycles);
            else if (rank == 0) mbar_wait_bounded(&full[s], last_phase, tc::kDrainCycles);
        }
    } else if (warp == 1) {
        if (rank == 0) {
            tc::Ring<S::kStages> r;
            uint32_t n_item = 0, fixed_phase = 0;
            int group = 0;
            bool on = true;
            for (int t = cluster; on && t < total && !stop(); t += clusters) {
                const Tile x = tiles.get(t, group, lane);
                const int kb = (x.c_len + kBC - 1) / kBC;
                if (!x.rows || !kb) continue;
                const uint32_t idesc = tc::operand_idesc(p.fmt, S::kFMn, S::kRMn, kBF * kPair, x.n);
                uint32_t buf = 0, d_tm = 0;
                for (int kk = 0, in_seg = 0; kk < kb; ++kk, r.next()) {
                    if (in_seg == 0) {
                        buf = n_item & 1u, d_tm = tmem + buf * kRowsMax;
                        if (!(on = tc::wait(b_dempty + 8 * buf, ((n_item >> 1) & 1u) ^ 1u, up))) break;
                        ++n_item;
                    }
                    if (!(on = tc::wait(b_full + 8 * r.s, r.phase, up))) break;
                    if (MODE == kGradWeight && kk == kb - 1 && (x.c_len & 15)) {
                        if (!(on = tc::wait<true>(b_fixed + 8 * r.s, fixed_phase >> r.s & 1u, up))) break;
                        fixed_phase ^= 1u << r.s;
                    }
                    tc::fence_after_sync();
                    if (tc::elect_one()) {
                        const uint64_t df = tc::operand_desc(aF + r.s * S::kBytesF, S::kFMn, 8192);
                        const uint64_t dr = tc::operand_desc(aR + r.s * S::kBytesR, S::kRMn, 8192);
                        // 16 of the contraction per MMA: 32 bytes along K, or two atoms of eight lines
                        const int left = x.c_len - kk * kBC;
#pragma unroll
                        for (int j = 0; j < kBC / 16; ++j)
                            if (16 * j < left)
                                tc::mma_f16_pair(d_tm, df + j * (S::kFMn ? 128 : 2), dr + j * (S::kRMn ? 128 : 2), idesc,
                                                               (in_seg | j) != 0);
                        tc::pair_commit<kPair>(b_empty + 8 * r.s);
                        if (kk == kb - 1 || in_seg == p.segment - 1) tc::pair_commit<kPair>(b_dfull + 8 * buf);
                    }
                    __syncwarp();
                    if (++in_seg == p.segment) in_seg = 0;
                }
            }
            // nor under MMAs in flight
            if (tc::elect_one()) tc::leader_commit<kPair>(smem_u32(&last));
            mbar_wait_bounded(&last, 0, tc::kDrainCycles);
        }
    } else if (warp < 2 + kEpilogueWarps) {
        const int quad = warp & 3, part = (warp - 2) >> 2;  // TMEM lanes 32 * quad.., columns in turns of 16
        uint8_t *stage = smem + S::kStages * (S::kBytesF + S::kBytesR) + (warp - 2) * 16 * kStageRow;
        uint32_t n_item = 0;
        int group = 0;
        bool on = true;
        for (int t = cluster; on && t < total && !stop(); t += clusters) {
            const Tile x = tiles.get(t, group, lane);
            if (!x.rows) continue;
            const int f = x.f0 + (int)rank * kBF + quad * 32;
            const OutTile o{p.out, (MODE == kGradWeight ? x.g * p.out_group : 0) + (int64_t)x.row0 * p.ldo + f, p.ldo, p.out_dtype,
                            p.features - f, x.rows, p.vec != 0};
            const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
            const int kb = (x.c_len + kBC - 1) / kBC, segments = kb > p.segment ? (kb + p.segment - 1) / p.segment : kb > 0;
            // The next accumulator, and its return.
            auto take = [&] {
                const uint32_t buf = n_item & 1u;
                on = tc::wait(b_dfull + 8 * buf, (n_item >> 1) & 1u, up);
                tc::fence_after_sync();
                ++n_item;
                return buf;
            };
            auto give = [&](uint32_t buf) {
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::arrive_at(tc::leader_addr(b_dempty + 8 * buf));
            };
            if (segments <= 1) {
                const uint32_t buf = segments ? take() : 0;
                if (!on) break;
                for (int c0 = part * 16; c0 < x.rows; c0 += 32) {
                    uint32_t v[16] = {};  // an expert without rows: dw is zero
                    if (segments) tc::tmem_ld_frag(lanes + buf * kRowsMax + c0, v);
                    store_chunk<MODE != kGradWeight>(o, stage, lane, c0, v);
                }
                if (segments) give(buf);
                continue;
            }
            float acc[kRowsMax / 32][16];
#pragma unroll
            for (int c = 0; c < kRowsMax / 32; ++c)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[c][j] = 0.0f;
            for (int g = 0; g < segments; ++g) {
                const uint32_t buf = take();
                if (!on) break;
#pragma unroll
                for (int c = 0; c < kRowsMax / 32; ++c)
                    if (32 * c + part * 16 < x.rows) {
                        uint32_t v[16];
                        tc::tmem_ld_frag(lanes + buf * kRowsMax + 32 * c + part * 16, v);
#pragma unroll
                        for (int j = 0; j < 16; ++j) acc[c][j] += __uint_as_float(v[j]);
                    }
                give(buf);
            }
            if (!on) break;
#pragma unroll
            for (int c = 0; c < kRowsMax / 32; ++c)
                if (32 * c + part * 16 < x.rows) {
                    uint32_t v[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(acc[c][j]);
                    store_chunk<MODE != kGradWeight>(o, stage, lane, 32 * c + part * 16, v);
                }
        }
    } else if (MODE == kGradWeight) {
        // This warp passes over tiles without a ragged end and waits for the next one that has one, however far ahead; the
        // epilogue waits for every accumulator up to there, so it may wait for as many limits.
        uint32_t s_next = 0, tail_phase = 0, limits = 1;
        int group = 0;
        for (int t = cluster; t < total && !stop(); t += clusters) {
            const Tile x = tiles.get(t, group, lane);
            const int kb = (x.c_len + kBC - 1) / kBC;
            if (!x.rows) continue;
            s_next = (s_next + kb) % S::kStages;
            limits += (kb - 1) / p.segment + 1;
            if (!(x.c_len & 15)) continue;
            const int boxes = (x.n / kPair + 63) / 64, s = (s_next + S::kStages - 1) % S::kStages;
            if (!tc::wait_long(b_tail + 8 * s, tail_phase >> s & 1u, up, limits)) break;
            tail_phase ^= 1u << s;
            limits = 1;
            // lines (one contraction row each) from `valid` up to the last multiple of 16 that the MMAs read
            const int valid = x.c_len - (kb - 1) * kBC, lines = 16 - (valid & 15);
            for (int i = lane; i < (2 + boxes) * lines * 8; i += 32) {
                const int box = i / (lines * 8), rest = i - box * lines * 8;
                uint8_t *b = box < 2 ? sF + s * S::kBytesF + box * 8192 : sR + s * S::kBytesR + (box - 2) * 8192;
                *reinterpret_cast<uint4 *>(b + (valid + (rest >> 3)) * 128 + (rest & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) tc::publish_at(tc::leader_addr(b_fixed + 8 * s));
        }
    }
    if (stop() && lane == 0) atomicOr(&g_product_err, 1u);
    __syncwarp();
    tc::fence_before_sync();
    tc::cluster_sync_all();  // the peer's shared and tensor memory are no longer in use
    tc::fence_after_sync();
    if (warp == 1) tc::pair_tmem_dealloc<kPair>(tmem, kTmemCols);
}

// ---- e4m3 operands with a scale per block of 128 -------------------------------------------------
//
// out[r][f] = sum_b xs[r][b] ws[f / 128][b] D_b[r][f] with D_b the product over block b of the contraction.  A stage
// is one block: its MMAs start a fresh accumulator, and the epilogue warps add it, times the scales, to fp32
// sums in registers.  The scale is one per column of the accumulator (a row of x) and CTA (128 features: one
// block of w), so warp 2 puts xs * ws of a stage's rows into shared memory and a thread multiplies
// pairs of columns with one packed FMA.
//
// A tile's rows are two halves, each with accumulators (two of 128 columns), an issuing warp (1 and 3) and four promotion
// warps of its own, so that one half's waits and tile changes run under the other's arithmetic; with both halves in
// one accumulator the eight warps waited together.  2048 x 10944 x 2048 takes 68 us, 1.47 K cycles for each of a CTA's 80
// blocks (start and tile changes included) where the MMAs take 512 (tensor pipe 38 %).  No single part bounds it: copies that
// left one out took 61 (MMAs), 59 (TMEM loads), 66 (scale loads), 72 (stores) and 82 us (FMAs).  At 256 rows shared
// memory carries 112 KB a block, 875 cycles at 128 bytes a cycle, the floor of this tiling.  The promotion
// needs the number of column chunks as a compile-time constant and, at 128 columns, 16 columns a load (with 32
// the sums spill).
//
// Single CTAs, not pairs: the promotion, not the operands' traffic, bounds the tiles, and a pair's CTAs wait for one
// another's eight warps at every block (4096 x 4 rows, 128 experts of 5760 x 2880: 553 us in pairs, 485 alone).  The warps
// store their sums themselves; a staging for TMA stores takes a stage and two barriers a tile and was slower (560 us).

constexpr int kThreadsF8 = 384, kHalfCols = 128, kSlots = 4, kHalfWarps = 4;

// Half h of a tile: columns [at, at + n) of its n, and its accumulators: slot h + 2 * (block & 1).
struct Half {
    int at, n;
};
__device__ __forceinline__ Half tile_half(int n, int h) {
    const int first = (n / 2 + 15) / 16 * 16;
    return h ? Half{first, n - first} : Half{0, first};
}

struct F8Params {
    TcParams t;
    const float *xs, *ws;
    int64_t xs_row, xs_blk, ws_row, ws_blk, ws_group;
};

struct ShapeF8 {
    static constexpr int kBC8 = 128;  // contraction per stage, in bytes too
    static constexpr int kBytesF = kBF * kBC8, kBytesR = kRowsMax * kBC8, kBytesHalf = kBytesR / 2;
    static constexpr int kStages = 4;
    static constexpr size_t kOperands = (size_t)kStages * (kBytesF + kBytesR);
    static constexpr size_t kSmem = 1024 + kOperands + kSlots * kHalfCols * sizeof(float) + kEpilogueWarps * 16 * kStageRow;
};

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) { return (uint64_t)lo | ((uint64_t)hi << 32); }
__device__ __forceinline__ void fma2(uint64_t &acc, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}

// What a promotion warp needs of its CTA.
struct F8Sync {
    uint32_t d_full, d_empty, sc_empty, give_up;  // shared-memory addresses
    uint32_t lanes;                               // TMEM address of the warp's lanes
    const float *scales;
    uint8_t *stage;  // the warp's
};

// Half `part` of a tile by one promotion warp: NCH chunks of 32 columns.  `it`: blocks of this half so far.
template <int NCH>
__device__ __forceinline__ void promote_half(const F8Sync &y, uint32_t &it, const TcParams &p, const Tile &x, const Half &half,
                                             int f, int kb, int part, int lane) {
    uint64_t acc[2 * NCH][8];  // 16 columns, pairs of columns in fragment order: 0.0f
#pragma unroll
    for (int h = 0; h < 2 * NCH; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[h][i] = 0;
    constexpr int kTogether = NCH <= 2 ? 2 * NCH : 1;  // loads of 16 columns under one wait
    for (int kk = 0; kk < kb; ++kk, ++it) {
        const int slot = part + 2 * (int)(it & 1u);
        tc::wait_or_run_on(y.d_full + 8 * slot, (it >> 1) & 1u, y.give_up);
        tc::fence_after_sync();
        const float *sc = y.scales + slot * kHalfCols + 2 * (lane & 3);
        const uint32_t src = y.lanes + slot * kHalfCols;
#pragma unroll
        for (int h0 = 0; h0 < 2 * NCH; h0 += kTogether) {
            uint32_t v[kTogether][16];
#pragma unroll
            for (int j = 0; j < kTogether; ++j) tc::tmem_ld_frag_async(src + 16 * (h0 + j), v[j]);
#pragma unroll
            for (int j = 0; j < kTogether; ++j) tc::tmem_wait_ld(v[j]);
#pragma unroll
            for (int j = 0; j < kTogether; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint64_t s2 = *reinterpret_cast<const uint64_t *>(sc + 16 * (h0 + j) + 8 * i);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int e = 8 * (q >> 1) + 4 * i + 2 * (q & 1);
                        fma2(acc[h0 + j][e >> 1], pack2(v[j][e], v[j][e + 1]), s2);
                    }
                }
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane < 2)  // one lane per barrier
            tc::arrive((lane ? y.sc_empty : y.d_empty) + 8 * slot);
    }
    // a half ends at a multiple of 16, its last chunk may not
    const OutTile o{p.out, (int64_t)x.row0 * p.ldo + f, p.ldo, p.out_dtype, p.features - f, min(x.rows, half.at + half.n), p.vec != 0};
#pragma unroll
    for (int h = 0; h < 2 * NCH; ++h) {
        uint32_t v[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[2 * i] = (uint32_t)acc[h][i];
            v[2 * i + 1] = (uint32_t)(acc[h][i] >> 32);
        }
        store_chunk<true>(o, y.stage, lane, half.at + 16 * h, v);
    }
}

__global__ void __launch_bounds__(kThreadsF8, 1) k_product_f8(const __grid_constant__ CUtensorMap map_f,
                                                              const __grid_constant__ CUtensorMap map_r, const F8Params fp) {
    using S = ShapeF8;
    const TcParams &p = fp.t;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    uint8_t *sF = smem, *sR = smem + S::kStages * S::kBytesF;  // a stage of R: the rows of half 0, from its middle those of half 1
    float *scales = reinterpret_cast<float *>(smem + S::kOperands);  // [slot][column]: xs * ws
    uint8_t *staging = smem + S::kOperands + kSlots * kHalfCols * sizeof(float);
    // d_full: a slot's MMAs and its scales; d_empty, sc_empty: both read by the four warps of its half
    __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages], d_full[kSlots], d_empty[kSlots], sc_empty[kSlots], last;
    __shared__ uint32_t tmem_s;
    __shared__ tc::GiveUp give_up;
    __shared__ int start[kMaxGroups + 1], prefix[kMaxGroups + 1];

    const int tid = threadIdx.x, warp = __shfl_sync(kFull, tid >> 5, 0), lane = tid & 31;
    for (int g = tid; g <= p.groups; g += kThreadsF8) start[g] = group_start(p.offsets, g, p.rows);
    if (tid == 0) {
        give_up.given_up = 0;
        give_up.limit = p.wait_limit;
        mbar_init(&last, 2);
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 2);
        }
        for (int s = 0; s < kSlots; ++s) {
            mbar_init(&d_full[s], 2);
            mbar_init(&d_empty[s], kHalfWarps);
            mbar_init(&sc_empty[s], kHalfWarps);
        }
    }
    if (warp == 1) tc::pair_tmem_alloc<1>(&tmem_s, kTmemCols);
    __syncthreads();
    const int f_tiles = (p.features + kBF - 1) / kBF;
    if (warp == 0) tile_prefix<1, kForward>(start, prefix, p.groups, f_tiles, p.out_rows, lane);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = __shfl_sync(kFull, tmem_s, 0);
    const int total = __shfl_sync(kFull, prefix[p.groups], 0), kb = (p.contraction + S::kBC8 - 1) / S::kBC8;
    const Tiles<1, kForward> tiles{start, prefix, p.groups, f_tiles, p.features, p.contraction, p.out_rows};

    const uint32_t up = smem_u32(&give_up), aF = smem_u32(sF), aR = smem_u32(sR);
    const uint32_t b_full = smem_u32(full), b_empty = smem_u32(empty), b_dfull = smem_u32(d_full), b_dempty = smem_u32(d_empty),
                   b_sempty = smem_u32(sc_empty);
    const auto stop = [&] { return __shfl_sync(kFull, *const_cast<volatile int *>(&give_up.given_up), 0) != 0; };

    if (warp == 0) {
        tc::Ring<S::kStages> r;
        uint32_t used = 0;  // stages in use
        int group = 0;
        bool withhold = (int)blockIdx.x == p.fault_cta, on = true;
        for (int t = blockIdx.x; on && t < total && !stop(); t += gridDim.x) {
            const Tile x = tiles.get(t, group, lane);
            if (!x.rows) continue;
            const Half h0 = tile_half(x.n, 0), h1 = tile_half(x.n, 1);
            const int boxes0 = (h0.n + kRowBox - 1) / kRowBox, boxes1 = (h1.n + kRowBox - 1) / kRowBox;
            const uint32_t bytes = S::kBytesF + (boxes0 + boxes1) * kRowBox * S::kBC8;
            for (int kk = 0; kk < kb; ++kk, r.next()) {
                if (!(on = tc::wait(b_empty + 8 * r.s, r.phase ^ 1u, up))) break;
                if (withhold) {
                    withhold = false;
                    continue;
                }
                used |= 1u << r.s;
                if (tc::elect_one()) {
                    const uint32_t bar = b_full + 8 * r.s;
                    tc::expect_tx(bar, bytes);
                    const int c = kk * S::kBC8;
                    const uint32_t dR = aR + r.s * S::kBytesR;
                    tc::pair_tma_3d<1>(aF + r.s * S::kBytesF, &map_f, c, x.f0, x.g, bar);
                    for (int b = 0; b < boxes0; ++b)
                        tc::pair_tma_2d<1>(dR + b * kRowBox * S::kBC8, &map_r, c, x.row0 + kRowBox * b, bar);
                    for (int b = 0; b < boxes1; ++b)
                        tc::pair_tma_2d<1>(dR + S::kBytesHalf + b * kRowBox * S::kBC8, &map_r, c, x.row0 + h1.at + kRowBox * b, bar);
                }
                __syncwarp();
            }
        }
        for (uint32_t s = 0; s < (uint32_t)S::kStages; ++s) {  // as in k_product_tc: no exit before the last arrivals and copies
            if (!(used >> s & 1u)) continue;
            const uint32_t last_phase = r.phase ^ (s >= r.s ? 1u : 0u);
            if (!mbar_wait_bounded(&empty[s], last_phase, tc::kDrainCycles)) mbar_wait_bounded(&full[s], last_phase, tc::kDrainCycles);
        }
    } else if (warp == 1 || warp == 3) {
        const int h = warp >> 1;
        tc::Ring<S::kStages> r;
        uint32_t it = 0;  // blocks of this half so far
        int group = 0;
        bool on = true;
        for (int t = blockIdx.x; on && t < total && !stop(); t += gridDim.x) {
            const Tile x = tiles.get(t, group, lane);
            if (!x.rows) continue;
            const int n = tile_half(x.n, h).n;
            const uint32_t idesc = tc::operand_idesc(0, false, false, kBF, n);
            for (int kk = 0; kk < kb; ++kk, r.next()) {
                if (!(on = tc::wait(b_full + 8 * r.s, r.phase, up))) break;
                const int slot = h + 2 * (int)(it & 1u);
                if (n && !(on = tc::wait(b_dempty + 8 * slot, ((it >> 1) & 1u) ^ 1u, up))) break;
                tc::fence_after_sync();
                if (tc::elect_one()) {
                    if (n) {
                        const uint64_t df = tc::operand_desc(aF + r.s * S::kBytesF, false, 0);
                        const uint64_t dr = tc::operand_desc(aR + r.s * S::kBytesR + h * S::kBytesHalf, false, 0);
                        const int left = p.contraction - kk * S::kBC8;
#pragma unroll
                        for (int j = 0; j < S::kBC8 / 32; ++j)
                            if (32 * j < left)
                                tc::mma_e4m3(tmem + slot * kHalfCols, df + 2 * j, dr + 2 * j, idesc, j != 0);
                        tc::pair_commit<1>(b_dfull + 8 * slot);
                    }
                    tc::pair_commit<1>(b_empty + 8 * r.s);
                }
                __syncwarp();
                if (n) ++it;
            }
        }
        if (tc::elect_one()) tc::leader_commit<1>(smem_u32(&last));  // nor under MMAs in flight
        mbar_wait_bounded(&last, 0, tc::kDrainCycles);
    } else if (warp == 2) {
        // ---- scales, two blocks ahead: registers [block & 1][half][32 columns] ------------------------------
        uint32_t it[2] = {0, 0};
        int group = 0;
        for (int t = blockIdx.x; t < total && !stop(); t += gridDim.x) {
            const Tile x = tiles.get(t, group, lane);
            if (!x.rows) continue;
            const Half h1 = tile_half(x.n, 1);
            const float *ws = fp.ws + x.g * fp.ws_group + (int64_t)(x.f0 / kScaleBlock) * fp.ws_row;
            const float *xs[2] = {fp.xs + (int64_t)(x.row0 + lane) * fp.xs_row, fp.xs + (int64_t)(x.row0 + h1.at + lane) * fp.xs_row};
            const int first[2] = {lane, h1.at + lane};
            const int valid[2] = {min(x.rows, h1.at), x.rows};
            float v[2][2][4], w[2];
            auto fetch = [&](int kk, float (&v)[2][4], float &w) {
                w = kk < kb ? __ldg(ws + kk * fp.ws_blk) : 0.0f;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        v[h][i] = kk < kb && first[h] + 32 * i < valid[h]
                                      ? __ldg(xs[h] + (int64_t)(32 * i) * fp.xs_row + kk * fp.xs_blk)
                                      : 0.0f;
            };
            fetch(0, v[0], w[0]);
            fetch(1, v[1], w[1]);
            for (int k0 = 0; k0 < kb; k0 += 2)
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    if (k0 + d >= kb) break;
                    float s[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[h][i] = v[d][h][i] * w[d];
                    fetch(k0 + d + 2, v[d], w[d]);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (h && !h1.n) break;
                        const int slot = h + 2 * (int)(it[h] & 1u);
                        tc::wait_or_run_on(b_sempty + 8 * slot, ((it[h] >> 1) & 1u) ^ 1u, up);
#pragma unroll
                        for (int i = 0; i < 4; ++i) scales[slot * kHalfCols + lane + 32 * i] = s[h][i];
                        __syncwarp();
                        if (lane == 0) tc::arrive(b_dfull + 8 * slot);
                        ++it[h];
                    }
                }
        }
    } else {
        const int quad = warp & 3, part = (warp - 4) >> 2;  // TMEM lanes 32 * quad.., half
        const F8Sync y{b_dfull, b_dempty, b_sempty, up, tmem + ((uint32_t)(quad * 32) << 16), scales,
                       staging + (warp - 4) * 16 * kStageRow};
        uint32_t it = 0;
        int group = 0;
        for (int t = blockIdx.x; t < total && !stop(); t += gridDim.x) {
            const Tile x = tiles.get(t, group, lane);
            if (!x.rows) continue;
            const Half half = tile_half(x.n, part);
            const int f = x.f0 + quad * 32, chunks = (half.n + 31) / 32;
            if (chunks == 0) continue;
            if (chunks == 1) promote_half<1>(y, it, p, x, half, f, kb, part, lane);
            else if (chunks == 2) promote_half<2>(y, it, p, x, half, f, kb, part, lane);
            else if (chunks == 3) promote_half<3>(y, it, p, x, half, f, kb, part, lane);
            else promote_half<4>(y, it, p, x, half, f, kb, part, lane);
        }
    }
    if (stop() && lane == 0) atomicOr(&g_product_err, 1u);
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (warp == 1) tc::pair_tmem_dealloc<1>(tmem, kTmemCols);
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static EncodeTiled fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *q = nullptr;
        cudaDriverEntryPointQueryResult r{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &q, cudaEnableDefault, &r) == cudaSuccess &&
            r == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(q);
    });
    return fn;
}

// A tensor map over a matrix of 128-byte box lines: dims (inner, lines[, matrices]), strides in bytes.
bool encode(CUtensorMap *m, int dtype, const void *base, int rank, uint64_t inner, uint64_t lines, uint64_t matrices,
            uint64_t line_bytes, uint64_t matrix_bytes, uint32_t box_lines) {
    EncodeTiled enc = encoder();
    if (!enc) return false;
    const CUtensorMapDataType t = dtype == UMSX_DTYPE_BF16  ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                  : dtype == UMSX_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                            : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const cuuint64_t dims[3] = {inner, lines, matrices};
    const cuuint64_t strides[2] = {line_bytes, matrix_bytes};
    const cuuint32_t box[3] = {dtype == UMSX_DTYPE_E4M3 ? 128u : 64u, box_lines, 1};
    const cuuint32_t step[3] = {1, 1, 1};
    return enc(m, t, (cuuint32_t)rank, const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int MODE>
int launch(const CUtensorMap &mf, const CUtensorMap &mr, const TcParams &t, int64_t tiles_most, int sms, cudaStream_t s) {
    auto *kernel = k_product_tc<MODE>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<MODE>::kSmem) != cudaSuccess)
        return -1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(kPair * std::max<int64_t>(1, std::min<int64_t>(tiles_most, sms / kPair))));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Shape<MODE>::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kPair;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, mf, mr, t) == cudaSuccess ? 1 : -1;
}

int launch_mode(const Product &p, const CUtensorMap &mf, const CUtensorMap &mr, const TcParams &t, int sms, cudaStream_t s) {
    const int64_t ft = (p.features() + kBF * kPair - 1) / (kBF * kPair);
    const int64_t rt = p.mode == kGradWeight ? (int64_t)p.groups * ((p.n + kRowsMax - 1) / kRowsMax)
                                             : p.rows / kRowsMax + std::min<int64_t>(p.groups, p.rows);
    if (p.mode == kForward) return launch<kForward>(mf, mr, t, ft * rt, sms, s);
    if (p.mode == kGradInput) return launch<kGradInput>(mf, mr, t, ft * rt, sms, s);
    return launch<kGradWeight>(mf, mr, t, ft * rt, sms, s);
}

int launch_f8(const CUtensorMap &mf, const CUtensorMap &mr, const F8Params &fp, int sms, cudaStream_t s) {
    if (cudaFuncSetAttribute(k_product_f8, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ShapeF8::kSmem) != cudaSuccess) return -1;
    const int64_t tiles = (int64_t)((fp.t.features + kBF - 1) / kBF) * (fp.t.rows / kRowsMax + std::min<int64_t>(fp.t.groups, fp.t.rows));
    k_product_f8<<<(unsigned)std::min<int64_t>(tiles, sms), kThreadsF8, ShapeF8::kSmem, s>>>(mf, mr, fp);
    return 1;
}

bool aligned(const void *p, int64_t stride, int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}

}  // namespace

bool product_tc_takes(const Product &p) {
    const int size = p.dtype == UMSX_DTYPE_E4M3 ? 1 : 2;
    if (p.x && !aligned(p.x, p.ldx, size)) return false;
    if (p.dy && !aligned(p.dy, p.lddy, size)) return false;
    if (p.w && (!aligned(p.w, p.ldw, size) || (p.groups > 1 && p.w_stride * size % 16))) return false;
    return p.rows > 0;
}

int launch_product_tc(const Product &p, int sms, cudaStream_t s) {
    CUtensorMap mf, mr;
    bool ok;
    if (p.mode == kGradWeight) {
        ok = encode(&mf, p.dtype, p.x, 2, p.k, p.rows, 1, p.ldx * 2, 0, kBC) &&
             encode(&mr, p.dtype, p.dy, 2, p.n, p.rows, 1, p.lddy * 2, 0, kBC);
    } else {
        const int size = p.dtype == UMSX_DTYPE_E4M3 ? 1 : 2;
        const uint64_t ws = (p.groups > 1 ? p.w_stride : p.ldw) * size;
        ok = encode(&mf, p.dtype, p.w, 3, p.k, p.n, p.groups, p.ldw * size, ws, p.mode == kForward ? kBF : kBC) &&
             encode(&mr, p.dtype, p.mode == kForward ? p.x : p.dy, 2, p.mode == kForward ? p.k : p.n, p.rows, 1,
                    (p.mode == kForward ? p.ldx : p.lddy) * size, 0, kRowBox);
    }
    if (!ok) return -1;
    TcParams t{};
    t.groups = p.groups;
    t.features = p.features();
    t.contraction = p.mode == kForward ? p.k : p.n;
    t.out_rows = p.n;
    t.out_dtype = p.out_dtype;
    t.fmt = p.dtype == UMSX_DTYPE_BF16 ? 1 : 0;
    t.rows = p.rows;
    t.offsets = p.offsets;
    t.out = p.out;
    t.ldo = p.ldo;
    t.out_group = p.out_stride;
    t.vec = aligned(p.out, p.ldo, 2) && p.out_stride % 8 == 0;
    t.fault_cta = p.fault_cta;
    t.wait_limit = p.wait_limit ? p.wait_limit : kWaitCycles;
    t.segment = (p.out_dtype == UMSX_DTYPE_F32 ? kAccumulate32 : kAccumulate16) / kBC;
    if (p.dtype == UMSX_DTYPE_E4M3) {
        const F8Params fp{t, p.xs, p.ws, p.xs_row, p.xs_blk, p.ws_row, p.ws_blk, p.ws_group};
        return launch_f8(mf, mr, fp, sms, s);
    }
    return launch_mode(p, mf, mr, t, sms, s);
}

uint32_t *product_err_word() {
    void *a = nullptr;
    return cudaGetSymbolAddress(&a, g_product_err) == cudaSuccess ? static_cast<uint32_t *>(a) : nullptr;
}

}  // namespace umsx
