// Entry points of the ragged products (umsx_grouped_mm and its gradients, umsx_fp8_grouped_mm), and the kernel that takes
// every shape, stride and alignment.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "umsx_device.cuh"
#include "umsx_internal.h"
#include "umsx_products.h"

namespace umsx {
namespace {

umsx_status fail(umsx_status s, const std::string &msg) {
    record_error(msg.c_str());
    return s;
}

// ---- any shape ---------------------------------------------------------------------------
//
// out[r][f] = sum_c R[r][c] F[f][c] for every stride and alignment: what the tcgen05 kernel cannot address, since TMA wants
// bases and row strides that are multiples of 16 bytes (odd widths, slices that start anywhere).  Tiles of 64 rows x 128
// features; a step takes 128 bytes of every line, as it lies in memory (along c, or along the rows or features for the
// gradients), one step ahead in registers.  A lane loads the aligned word that holds its first byte and shifts its four out of
// that and the next lane's; a line's alignment is the same in every step.  From shared memory into mma.sync, by ldmatrix
// with or without a transposition.  e4m3 codes become f16 (exact); a step is a block of 128, scaled once and added in fp32.
// 16-bit operands get a fresh accumulator every 512 of the contraction (kAccumulate16 of it for 16-bit outputs), added up in fp32
// in shared memory: the tensor cores add less exactly than fp32 additions round, the more so the longer they add.  From there a
// warp stores 32 neighbours.
// Bound by the latency of a step where there are few tiles (e4m3 511 x 308 x 1323: 24 tiles, 37 us; with steps of 32 values
// 80), by issue where there are many: bf16 4096 x 4096 x 2049 takes 483 us forward (142 TFLOP/s), 522 for dx, 508 for dw
// (500, 523 for fp32 outputs, forward and dw), e4m3 446; with single-element loads 573, 784, 891 and 1116, and with a test in front of every load and shift 778 forward.

constexpr int kAnyRows = 64, kAnyF = 128, kLineBytes = 128, kAnyWarps = 8;
constexpr int kSumLine = kAnyF + 8;  // a half warp's pairs of sums lie in different banks

template <int DTYPE>
struct AnyShape {
    static constexpr int kSize = DTYPE == UMSX_DTYPE_E4M3 ? 1 : 2;
    static constexpr int kC = kLineBytes / kSize;  // contraction a step
    static_assert(kSize == 2 || kC == kScaleBlock, "a step of e4m3 codes is a block");
    static constexpr int kLine = kC + 8;           // 16-bit values from line to line: eight lines spread over all banks
    static constexpr int kOperands = (kAnyRows + kAnyF) * kLine * 2, kSums = kAnyRows * kSumLine * 4;
    static constexpr int kSmem = kOperands + kSums;
};

struct AnyParams {
    int out_dtype, groups, segment;  // segment: contraction that shares an accumulator
    int64_t rows;
    int features, contraction;  // contraction: forward k, dx n (dw: the group's rows)
    int out_rows;               // dw: n
    const int32_t *offsets;
    const uint8_t *R, *F, *R_end, *F_end;  // first byte, and behind the last
    int64_t r_pitch, f_pitch, f_group;     // bytes: between lines in memory, F's from group to group
    const float *rs, *fs;
    int64_t rs_row, rs_blk, fs_row, fs_blk, fs_group;
    void *out;
    int64_t ldo, out_group;
};

// The bytes of an aligned word that lie in [begin, end).
__device__ __noinline__ uint32_t edge_word(const uint8_t *at, const uint8_t *begin, const uint8_t *end) {
    uint32_t v = 0;
    for (int i = 0; i < 4; ++i)
        if (at + i >= begin && at + i < end) v |= (uint32_t)__ldg(at + i) << 8 * i;
    return v;
}

// One step of an operand of LINES rows or features, held by 256 threads between its load and its store.  ALONG: lines in memory
// run along the contraction, LINES of them; otherwise along the rows or features, 64 of them in LINES / 64 parts of 128 bytes.
// Warp w takes lines w, w + 8, ..., lane j their word j; lane i also the word behind the i-th.
template <bool ALONG, int LINES>
struct Words {
    static constexpr int kPer = LINES / kAnyWarps, kParts = ALONG ? 1 : LINES / 64;
    uint32_t w[kPer], behind;
    int bytes;  // of a line that are inside

    __device__ __forceinline__ void load(const uint8_t *p, int64_t pitch, int lines, int line_bytes, const uint8_t *begin,
                                         const uint8_t *end) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        bytes = line_bytes;
        if (lines <= 0 || line_bytes <= 0) lines = 0;
        const uint8_t *line = p + warp * pitch;
        const int skew = (int)(reinterpret_cast<uintptr_t>(line) & 3);
        const uint8_t *at = line - skew + 4 * lane;
        const int i_b = lane / kParts, part_b = lane % kParts;
        const uint8_t *at_b = line - skew + kLineBytes + (int64_t)i_b * kAnyWarps * pitch + part_b * kLineBytes;
        const bool in_b = skew && lane < kPer && warp + kAnyWarps * i_b < lines &&
                          kLineBytes - skew < min(kLineBytes, bytes - part_b * kLineBytes);
        // words may reach over the operand's first or last byte in the tiles there
        const uint8_t *low = p - (reinterpret_cast<uintptr_t>(p) & 3);
        const uint8_t *high = p + (lines - 1) * pitch + bytes;
        high += -reinterpret_cast<uintptr_t>(high) & 3;
        const bool inside = low >= begin && high <= end;
        if (inside && lines >= (ALONG ? LINES : 64) && bytes >= kParts * kLineBytes) {  // no test in front of any load
            const uint8_t *q = at;
            const int64_t down = kAnyWarps * pitch;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                w[i] = __ldg(reinterpret_cast<const uint32_t *>(q + i % kParts * kLineBytes));
                if ((i + 1) % kParts == 0) q += down;
            }
            behind = in_b ? __ldg(reinterpret_cast<const uint32_t *>(at_b)) : 0;
            return;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int part = i % kParts, l = warp + kAnyWarps * (i / kParts);
            const bool in = l < lines && 4 * lane - skew < min(kLineBytes, bytes - part * kLineBytes);
            const uint8_t *q = at + (int64_t)(i / kParts) * kAnyWarps * pitch + part * kLineBytes;
            w[i] = in && inside ? __ldg(reinterpret_cast<const uint32_t *>(q)) : 0;
        }
        behind = in_b && inside ? __ldg(reinterpret_cast<const uint32_t *>(at_b)) : 0;
        if (inside) return;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int part = i % kParts, l = warp + kAnyWarps * (i / kParts);
            const bool in = l < lines && 4 * lane - skew < min(kLineBytes, bytes - part * kLineBytes);
            if (in) w[i] = edge_word(at + (int64_t)(i / kParts) * kAnyWarps * pitch + part * kLineBytes, begin, end);
        }
        if (in_b) behind = edge_word(at_b, begin, end);
    }

    // To lines of `kLine` 16-bit values (not ALONG: part after part); zero behind the end, where a NaN may lie.
    template <int DTYPE>
    __device__ __forceinline__ void store(uint16_t *to, const uint8_t *p, int64_t pitch) const {
        constexpr int kLine = AnyShape<DTYPE>::kLine;
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const int skew = (int)(reinterpret_cast<uintptr_t>(p + warp * pitch) & 3);
        uint32_t mask[kParts];
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            const int left = bytes - part * kLineBytes - 4 * lane;
            mask[part] = left >= 4 ? ~0u : left > 0 ? (1u << 8 * left) - 1u : 0u;
        }
        uint16_t *d = to + warp * kLine + (DTYPE == UMSX_DTYPE_E4M3 ? 4 : 2) * lane;
        const auto put = [&](int i, uint32_t v) {
            uint16_t *at = d + (i % kParts * 64 + kAnyWarps * (i / kParts)) * kLine;
            v &= mask[i % kParts];
            if constexpr (DTYPE == UMSX_DTYPE_E4M3) {
                const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v & 0xffffu), __NV_E4M3),
                                  hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v >> 16), __NV_E4M3);
                *reinterpret_cast<uint2 *>(at) = make_uint2(lo.x | (uint32_t)lo.y << 16, hi.x | (uint32_t)hi.y << 16);
            } else {
                *reinterpret_cast<uint32_t *>(at) = v;
            }
        };
        if (skew) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const uint32_t next = __shfl_down_sync(kFull, w[i], 1), last = __shfl_sync(kFull, behind, i);
                put(i, __funnelshift_r(w[i], lane == 31 ? last : next, 8 * skew));
            }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) put(i, w[i]);
        }
    }
};

template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const uint16_t *p) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(smem_u32(p)));
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(smem_u32(p)));
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void store_el(void *p, int64_t i, int dtype, float v) {
    if (dtype == UMSX_DTYPE_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == UMSX_DTYPE_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half *>(p)[i] = __float2half_rn(v);
}

template <int DTYPE, int MODE>
__global__ void __launch_bounds__(32 * kAnyWarps, 2) k_product_any(const AnyParams p) {
    using S = AnyShape<DTYPE>;
    constexpr bool kF8 = DTYPE == UMSX_DTYPE_E4M3, dw = MODE == kGradWeight;
    constexpr bool kRAlong = !dw, kFAlong = MODE == kForward;
    constexpr int kSize = S::kSize, kC = S::kC, kLine = S::kLine;
    extern __shared__ __align__(16) uint8_t any_smem[];
    uint16_t *sR = reinterpret_cast<uint16_t *>(any_smem), *sF = sR + kAnyRows * kLine;
    float *sums = reinterpret_cast<float *>(any_smem + S::kOperands);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, f0 = blockIdx.x * kAnyF;
    const int wr = (warp & 1) * 32, wf = (warp >> 1) * 32;  // the warp's 32 x 32 of the tile
    // row tiles of all groups in order; this CTA takes every gridDim.y-th
    for (int t = blockIdx.y;; t += gridDim.y) {
        __syncthreads();
        int g = 0, tile = 0;
        if (dw) {
            const int each = (p.out_rows + kAnyRows - 1) / kAnyRows;
            g = t / each;
            tile = t % each;
            if (g >= p.groups) return;
        } else if (!find_tile(p.offsets, p.groups, p.rows, kAnyRows, t, g, tile)) {
            return;
        }
        int a, b;
        group_bounds(p.offsets, g, p.rows, a, b);
        const int r0 = tile * kAnyRows, nr = min(kAnyRows, (dw ? p.out_rows : b - a) - r0), nf = min(kAnyF, p.features - f0);
        const int nc = dw ? b - a : p.contraction;
        // the tile's first line, and from step to step
        const uint8_t *R = p.R + (dw ? a * p.r_pitch + (int64_t)r0 * kSize : (int64_t)(a + r0) * p.r_pitch);
        const uint8_t *F = p.F + g * p.f_group + (kFAlong ? f0 * p.f_pitch : (int64_t)f0 * kSize + (dw ? a * p.f_pitch : 0));
        const int64_t r_step = kRAlong ? kLineBytes : kC * p.r_pitch, f_step = kFAlong ? kLineBytes : kC * p.f_pitch;
        Words<kRAlong, kAnyRows> er;
        Words<kFAlong, kAnyF> ef;
        const auto load = [&](int c0) {
            const int left = min(kC, nc - c0);
            const uint8_t *r = R + c0 / kC * r_step, *f = F + c0 / kC * f_step;
            er.load(r, p.r_pitch, kRAlong ? nr : left, (kRAlong ? left : nr) * kSize, p.R, p.R_end);
            ef.load(f, p.f_pitch, kFAlong ? nf : left, (kFAlong ? left : nf) * kSize, p.F, p.F_end);
        };
        if (nc > 0) load(0);
        int c0 = 0;
        do {  // at least once: the sums of nothing are zero
            const int end = c0 + (kF8 ? nc : min(nc - c0, p.segment));
            const bool first = c0 == 0;
            float acc[2][4][4] = {};  // [16 rows][8 features]
            for (; c0 < end; c0 += kC) {
                __syncthreads();  // the previous step has been read
                er.template store<DTYPE>(sR, R, p.r_pitch);
                ef.template store<DTYPE>(sF, F, p.f_pitch);
                __syncthreads();
                const int left = nc - c0;
                if (c0 + kC < nc) load(c0 + kC);
                float blk[2][4][4] = {};  // e4m3: of this block
#pragma unroll
                for (int k = 0; k < kC; k += 16) {
                    if (k >= left) break;
                    uint32_t x[2][4], y[2][4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // rows x contraction: 8 x 8 matrices (0, 0), (8, 0), (0, 8), (8, 8); features: (0, 0), (0, 8), (8, 0), (8, 8)
                        const int r = wr + 16 * i, f = wf + 16 * i;
                        if constexpr (kRAlong) ldmatrix4<false>(x[i], sR + (r + (lane & 15)) * kLine + k + 8 * (lane >> 4));
                        else ldmatrix4<true>(x[i], sR + (k + (lane & 7) + 8 * (lane >> 4)) * kLine + r + 8 * ((lane >> 3) & 1));
                        if constexpr (kFAlong)
                            ldmatrix4<false>(y[i], sF + (f + (lane & 7) + 8 * (lane >> 4)) * kLine + k + 8 * ((lane >> 3) & 1));
                        else
                            ldmatrix4<true>(y[i], sF + ((f & 64) + k + (lane & 7) + 8 * ((lane >> 3) & 1)) * kLine + (f & 63) + 8 * (lane >> 4));
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            mma16816<DTYPE == UMSX_DTYPE_BF16>(kF8 ? blk[i][j] : acc[i][j], x[i], y[j >> 1][2 * (j & 1)],
                                                               y[j >> 1][2 * (j & 1) + 1]);
                }
                if constexpr (kF8) {
                    const int cb = c0 / kScaleBlock;
                    const float w = __ldg(p.fs + g * p.fs_group + (int64_t)(f0 / kScaleBlock) * p.fs_row + cb * p.fs_blk);
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int r = wr + 16 * i + 8 * h + (lane >> 2);
                            const float sc = r < nr ? w * __ldg(p.rs + (int64_t)(a + r0 + r) * p.rs_row + cb * p.rs_blk) : 0.0f;
#pragma unroll
                            for (int j = 0; j < 4; ++j)
#pragma unroll
                                for (int q = 0; q < 2; ++q)
                                    acc[i][j][2 * h + q] = fmaf(sc, blk[i][j][2 * h + q], acc[i][j][2 * h + q]);
                        }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float2 *to = reinterpret_cast<float2 *>(sums + (wr + 16 * i + 8 * h + (lane >> 2)) * kSumLine + wf + 8 * j + 2 * (lane & 3));
                        const float2 had = first ? make_float2(0.0f, 0.0f) : *to;
                        *to = make_float2(had.x + acc[i][j][2 * h], had.y + acc[i][j][2 * h + 1]);
                    }
        } while (c0 < nc);
        __syncthreads();
        for (int r = warp; r < nr; r += kAnyWarps) {
            const int64_t at = (dw ? g * p.out_group + (int64_t)(r0 + r) * p.ldo : (int64_t)(a + r0 + r) * p.ldo) + f0;
#pragma unroll
            for (int f = lane; f < kAnyF; f += 32)
                if (f < nf) store_el(p.out, at + f, p.out_dtype, sums[r * kSumLine + f]);
        }
    }
}

template <int DTYPE, int MODE>
int launch_any(const AnyParams &a, dim3 grid, cudaStream_t s) {
    auto *kernel = k_product_any<DTYPE, MODE>;
    constexpr int kSmem = AnyShape<DTYPE>::kSmem;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) return -1;
    kernel<<<grid, 32 * kAnyWarps, kSmem, s>>>(a);
    return 1;
}
template <int DTYPE>
int launch_any(const AnyParams &a, ProductMode mode, dim3 grid, cudaStream_t s) {
    if (mode == kForward) return launch_any<DTYPE, kForward>(a, grid, s);
    return mode == kGradInput ? launch_any<DTYPE, kGradInput>(a, grid, s) : launch_any<DTYPE, kGradWeight>(a, grid, s);
}

}  // namespace

int launch_product_any(const Product &p, int sms, cudaStream_t s) {
    const int size = p.dtype == UMSX_DTYPE_E4M3 ? 1 : 2;
    const auto bytes = [](const void *q) { return static_cast<const uint8_t *>(q); };
    AnyParams a{};
    a.out_dtype = p.out_dtype;
    a.groups = p.groups;
    a.segment = (p.out_dtype == UMSX_DTYPE_F32 ? kAccumulate32 : kAccumulate16);
    a.rows = p.rows;
    a.offsets = p.offsets;
    a.features = p.features();
    a.contraction = p.mode == kForward ? p.k : p.n;
    a.out_rows = p.n;
    a.out = p.out;
    a.ldo = p.ldo;
    a.out_group = p.out_stride;
    a.rs = p.xs;
    a.rs_row = p.xs_row;
    a.rs_blk = p.xs_blk;
    a.fs = p.ws;
    a.fs_row = p.ws_row;
    a.fs_blk = p.ws_blk;
    a.fs_group = p.ws_group;
    const bool fwd = p.mode == kForward, dw = p.mode == kGradWeight;
    a.R = bytes(fwd ? p.x : p.dy);
    a.r_pitch = (fwd ? p.ldx : p.lddy) * size;
    a.R_end = a.R + (p.rows - 1) * a.r_pitch + (int64_t)(fwd ? p.k : p.n) * size;
    a.F = bytes(dw ? p.x : p.w);
    a.f_pitch = (dw ? p.ldx : p.ldw) * size;
    a.f_group = dw ? 0 : p.groups > 1 ? p.w_stride * size : 0;
    a.F_end = a.F + (p.groups - 1) * a.f_group + ((dw ? p.rows : p.n) - 1) * a.f_pitch + (int64_t)p.k * size;
    const int64_t tiles = dw ? (int64_t)p.groups * ((p.n + kAnyRows - 1) / kAnyRows)
                             : p.rows / kAnyRows + std::min<int64_t>(p.groups, p.rows);
    const dim3 grid((unsigned)((a.features + kAnyF - 1) / kAnyF), (unsigned)std::max<int64_t>(1, std::min<int64_t>(tiles, 32 * sms)));
    if (p.dtype == UMSX_DTYPE_BF16) return launch_any<UMSX_DTYPE_BF16>(a, p.mode, grid, s);
    if (p.dtype == UMSX_DTYPE_F16) return launch_any<UMSX_DTYPE_F16>(a, p.mode, grid, s);
    return launch_any<UMSX_DTYPE_E4M3, kForward>(a, grid, s);
}

namespace {

bool out_ok(int t) { return t == UMSX_DTYPE_F32 || t == UMSX_DTYPE_BF16 || t == UMSX_DTYPE_F16; }

// Shape checks shared by the entry points; the sizes are those that the kernels' 32-bit row and column indexes hold.
umsx_status check_product(const Product &p) {
    if (p.groups < 1 || p.groups > kMaxGroups) return fail(UMSX_EINVAL, "experts must be 1..1024");
    if (p.n < 1 || p.k < 1 || p.n > (1 << 24) || p.k > (1 << 24)) return fail(UMSX_EINVAL, "n and k must be 1..2^24");
    if (p.rows < 0 || p.rows > kMaxRows) return fail(UMSX_EINVAL, "rows must be 0..2^31 - 512");
    if (!out_ok(p.out_dtype)) return fail(UMSX_EINVAL, "the output's type must be F32, BF16 or F16");
    return UMSX_OK;
}

// The kernels write while other CTAs still read: an output inside an operand would race.
bool out_overlaps(const Product &p) {
    const int size = p.dtype == UMSX_DTYPE_E4M3 ? 1 : 2, out_size = p.out_dtype == UMSX_DTYPE_F32 ? 4 : 2;
    const bool dw = p.mode == kGradWeight;
    const Region out = dw ? region(p.out, out_size, p.k, p.n, p.ldo, p.groups, p.out_stride)
                          : region(p.out, out_size, p.features(), p.rows, p.ldo);
    const int64_t kb = (p.k + kScaleBlock - 1) / kScaleBlock, nb = (p.n + kScaleBlock - 1) / kScaleBlock;
    return (p.rows && (overlap(out, region(p.x, size, p.k, p.rows, p.ldx)) || overlap(out, region(p.dy, size, p.n, p.rows, p.lddy)) ||
                       overlap(out, region(p.xs, 4, (p.rows - 1) * p.xs_row + (kb - 1) * p.xs_blk + 1, 1, 0)))) ||
           overlap(out, region(p.w, size, p.k, p.n, p.ldw, p.groups, p.w_stride)) ||
           overlap(out, region(p.ws, 4, (p.groups - 1) * p.ws_group + (nb - 1) * p.ws_row + (kb - 1) * p.ws_blk + 1, 1, 0)) ||
           overlap(out, region(p.offsets, 4, p.groups + 1, 1, 0));
}

bool misaligned(const void *p, int size) { return reinterpret_cast<uintptr_t>(p) % size; }

// What umsx_products_inject_fault left for the calling thread's next product on the tcgen05 kernels.
struct Fault {
    int cta = -1;
    long long wait_limit = 0;
};
thread_local Fault g_fault;

umsx_status run_product(Product &p, umsx_stream stream) {
    if (out_overlaps(p)) return fail(UMSX_EINVAL, "the output overlaps an input");
    const int size = p.dtype == UMSX_DTYPE_E4M3 ? 1 : 2, out_size = p.out_dtype == UMSX_DTYPE_F32 ? 4 : 2;
    if (misaligned(p.x, size) || misaligned(p.dy, size) || misaligned(p.w, size) || misaligned(p.out, out_size) ||
        misaligned(p.xs, 4) || misaligned(p.ws, 4) || misaligned(p.offsets, 4))
        return fail(UMSX_EINVAL, "a buffer is not aligned to its elements");
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail(UMSX_EDEVICE, std::string("device query: ") + cudaGetErrorString(e));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    (void)cudaGetLastError();  // an earlier call's error is not this launch's
    const bool few = product_few_takes(p), tc = !few && product_tc_takes(p);
    if (tc) p.fault_cta = g_fault.cta, p.wait_limit = g_fault.wait_limit, g_fault = Fault{};
    const int n = few ? launch_product_few(p, sms, s)
                  : tc ? launch_product_tc(p, sms, s)
                       : launch_product_any(p, sms, s);
    e = cudaGetLastError();
    if (n < 0) return fail(UMSX_EDEVICE, std::string("the product's kernel could not be set up: ") + cudaGetErrorString(e));
    record_launches((uint64_t)n);
    if (e != cudaSuccess) return fail(UMSX_EDEVICE, std::string("product launch: ") + cudaGetErrorString(e));
    return UMSX_OK;
}

bool dtype16(int t) { return t == UMSX_DTYPE_BF16 || t == UMSX_DTYPE_F16; }

}  // namespace
}  // namespace umsx

using namespace umsx;

extern "C" {

umsx_status umsx_grouped_mm(const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t w_stride,
                            const int32_t *offsets, int experts, int64_t rows, int n, int k, int dtype, void *out,
                            int64_t ldo, int out_dtype, umsx_stream stream) {
    Product p{};
    p.mode = kForward;
    p.dtype = dtype, p.out_dtype = out_dtype;
    p.groups = experts, p.rows = rows, p.n = n, p.k = k, p.offsets = offsets;
    p.x = x, p.ldx = ldx, p.w = w, p.ldw = ldw, p.w_stride = w_stride;
    p.out = out, p.ldo = ldo;
    if (!dtype16(dtype)) return fail(UMSX_EINVAL, "the operands' type must be BF16 or F16");
    if (umsx_status st = check_product(p)) return st;
    if (ldx < k || ldw < k || w_stride < (int64_t)(n - 1) * ldw + k || ldo < n) return fail(UMSX_EINVAL, "a stride is shorter than a row");
    if (rows == 0) return UMSX_OK;
    if (!x || !w || !offsets || !out) return fail(UMSX_EINVAL, "null buffer");
    return run_product(p, stream);
}

umsx_status umsx_grouped_mm_dx(const void *dy, int64_t lddy, const void *w, int64_t ldw, int64_t w_stride,
                               const int32_t *offsets, int experts, int64_t rows, int n, int k, int dtype, void *dx,
                               int64_t lddx, int out_dtype, umsx_stream stream) {
    Product p{};
    p.mode = kGradInput;
    p.dtype = dtype, p.out_dtype = out_dtype;
    p.groups = experts, p.rows = rows, p.n = n, p.k = k, p.offsets = offsets;
    p.dy = dy, p.lddy = lddy, p.w = w, p.ldw = ldw, p.w_stride = w_stride;
    p.out = dx, p.ldo = lddx;
    if (!dtype16(dtype)) return fail(UMSX_EINVAL, "the operands' type must be BF16 or F16");
    if (umsx_status st = check_product(p)) return st;
    if (lddy < n || ldw < k || w_stride < (int64_t)(n - 1) * ldw + k || lddx < k) return fail(UMSX_EINVAL, "a stride is shorter than a row");
    if (rows == 0) return UMSX_OK;
    if (!dy || !w || !offsets || !dx) return fail(UMSX_EINVAL, "null buffer");
    return run_product(p, stream);
}

umsx_status umsx_grouped_mm_dw(const void *dy, int64_t lddy, const void *x, int64_t ldx, const int32_t *offsets,
                               int experts, int64_t rows, int n, int k, int dtype, void *dw, int64_t lddw,
                               int64_t dw_stride, int out_dtype, umsx_stream stream) {
    Product p{};
    p.mode = kGradWeight;
    p.dtype = dtype, p.out_dtype = out_dtype;
    p.groups = experts, p.rows = rows, p.n = n, p.k = k, p.offsets = offsets;
    p.dy = dy, p.lddy = lddy, p.x = x, p.ldx = ldx;
    p.out = dw, p.ldo = lddw, p.out_stride = dw_stride;
    if (!dtype16(dtype)) return fail(UMSX_EINVAL, "the operands' type must be BF16 or F16");
    if (umsx_status st = check_product(p)) return st;
    if (lddy < n || ldx < k || lddw < k || dw_stride < (int64_t)(n - 1) * lddw + k) return fail(UMSX_EINVAL, "a stride is shorter than a row");
    // without rows every group's gradient is zero, and is written
    if ((rows && (!dy || !x)) || !offsets || !dw) return fail(UMSX_EINVAL, "null buffer");
    return run_product(p, stream);
}

umsx_status umsx_fp8_grouped_mm(const void *x, int64_t ldx, const float *xs, int64_t xs_row, int64_t xs_blk, const void *w,
                                int64_t ldw, int64_t w_stride, const float *ws, int64_t ws_row, int64_t ws_blk,
                                int64_t ws_stride, const int32_t *offsets, int experts, int64_t rows, int n, int k,
                                void *out, int64_t ldo, int out_dtype, umsx_stream stream) {
    Product p{};
    p.mode = kForward;
    p.dtype = UMSX_DTYPE_E4M3, p.out_dtype = out_dtype;
    p.groups = experts, p.rows = rows, p.n = n, p.k = k, p.offsets = offsets;
    p.x = x, p.ldx = ldx, p.w = w, p.ldw = ldw, p.w_stride = w_stride;
    p.xs = xs, p.xs_row = xs_row, p.xs_blk = xs_blk;
    p.ws = ws, p.ws_row = ws_row, p.ws_blk = ws_blk, p.ws_group = ws_stride;
    p.out = out, p.ldo = ldo;
    if (umsx_status st = check_product(p)) return st;
    if (!offsets && experts != 1) return fail(UMSX_EINVAL, "offsets may be null for one expert only");
    if (ldx < k || ldw < k || (experts > 1 && w_stride < (int64_t)(n - 1) * ldw + k) || ldo < n)
        return fail(UMSX_EINVAL, "a stride is shorter than a row");
    if (xs_row < 0 || xs_blk < 0 || ws_row < 0 || ws_blk < 0 || ws_stride < 0) return fail(UMSX_EINVAL, "negative scale stride");
    if (rows == 0) return UMSX_OK;
    if (!x || !xs || !w || !ws || !out) return fail(UMSX_EINVAL, "null buffer");
    return run_product(p, stream);
}

umsx_status umsx_products_status(umsx_stream stream) {
    uint32_t *word = product_err_word(), v = 0;
    if (!word) return fail(UMSX_EDEVICE, "the device's status word has no address");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaMemcpyAsync(&v, word, sizeof v, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e == cudaSuccess && v) e = cudaMemsetAsync(word, 0, sizeof v, s);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();  // reported here, not by the next launch's check
        return fail(UMSX_EDEVICE, std::string("products status: ") + cudaGetErrorString(e));
    }
    return v ? fail(UMSX_ETIMEOUT, "a bounded wait of a product's kernel gave up: its output is not complete") : UMSX_OK;
}

umsx_status umsx_products_inject_fault(int cta, int64_t wait_limit_cycles) {
    if (cta < 0 || wait_limit_cycles < 1 || wait_limit_cycles > kWaitCycles)  // a wait may be for many limits: no overflow
        return fail(UMSX_EINVAL, "cta must not be negative, wait_limit_cycles must be 1..2000000000");
    g_fault = {cta, wait_limit_cycles};
    return UMSX_OK;
}

}  // extern "C"
