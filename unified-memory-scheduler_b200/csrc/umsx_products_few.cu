// Ragged products of few rows (decoding): a stream of weights past eight rows at a time.
//
// With a handful of rows per expert the product is the reading of the weights.  A warp takes 16 features x 8 * NT rows of one
// group; SPLIT of a CTA's eight warps share the same ones and take turns along the contraction: eight where a step reads
// little (one token through one matrix, which all SMs have to read together), one where there are more 16-feature blocks
// than warps on the device (then eight only repeated the search for the group: 16 sequences x 6 of 64 experts took 145 us).
// Each lane loads 16 bytes of a weight row straight into the registers of mma.sync, U steps ahead.  A fragment wants
// elements (2t, 2t+1, 2t+8, 2t+9) of 16; any other eight of the contraction do as well if both operands use the same ones, so
// lane t takes eight neighbours and feeds two MMAs with them.  e4m3 codes become f16 (exact) and the fp32 sums of a
// block of 128 are scaled once; 16-bit operands get a fresh accumulator every U steps (at most 256 of the contraction), added up
// in fp32, since the tensor cores add less exactly than fp32 additions round.  The eight warps' sums are added in a fixed order.
//
// Bound: memory (e4m3, 96 rows over 64 experts of 2816 x 2048: 61 us, 4.9 TB/s, 75 % of a copy's rate).  The tcgen05
// kernel's tiles of 128 or 256 features leave SMs without work here (8 experts of 1536 features: 48 tiles for 74 pairs) and
// go through a pipeline that costs more than the weights of one step.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "umsx_device.cuh"
#include "umsx_products.h"

namespace umsx {
namespace {

constexpr int kWarps = 8, kFewF = 16;  // kWarps: find_tile's CTA

struct FewParams {
    int groups, n, k, out_dtype;
    int64_t rows;
    const int32_t *offsets;
    const uint8_t *x, *w;
    int64_t ldx, ldw, w_stride;  // bytes
    const float *xs, *ws;
    int64_t xs_row, xs_blk, ws_row, ws_blk, ws_group;
    void *out;
    int64_t ldo;
    int split;  // warps of a CTA that share 16 features: 1, 2, 4 or 8
};

__device__ __forceinline__ uint4 load_stream(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <int DTYPE>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (DTYPE == UMSX_DTYPE_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four e4m3 codes as two f16 pairs, exact.
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t v, uint32_t &lo, uint32_t &hi) {
    asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }" : "=r"(lo), "=r"(hi) : "r"(v));
}

// d += the 16 bytes of contraction that the lanes hold of weight rows g, g + 8 (a, b) and row g of x (c).
template <int DTYPE>
__device__ __forceinline__ void multiply(float (&d)[4], const uint4 &a, const uint4 &b, const uint4 &c) {
    if constexpr (DTYPE == UMSX_DTYPE_E4M3) {
        const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w}, cv[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t a0, a2, a1, a3, b0, b1;
            e4m3x4_to_f16(av[i], a0, a2);
            e4m3x4_to_f16(bv[i], a1, a3);
            e4m3x4_to_f16(cv[i], b0, b1);
            mma16816<UMSX_DTYPE_F16>(d, a0, a1, a2, a3, b0, b1);
        }
    } else {
        mma16816<DTYPE>(d, a.x, b.x, a.y, b.y, c.x, c.y);
        mma16816<DTYPE>(d, a.z, b.z, a.w, b.w, c.z, c.w);
    }
}

// DTYPE: of the operands; NT: tiles of eight rows; U: steps in flight.  A step is 128 bytes of a row: 64 16-bit values, or one
// block of 128 codes.
template <int DTYPE, int NT, int U>
__global__ void __launch_bounds__(kWarps * 32, 2) k_product_few(const FewParams p) {
    constexpr int kRows = 8 * NT;
    constexpr bool kF8 = DTYPE == UMSX_DTYPE_E4M3;
    __shared__ float part[kWarps][kFewF * kRows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gl = lane >> 2, tl = lane & 3;

    // the blockIdx.y-th chunk of kRows rows, counted over the groups
    int group = 0, chunk = blockIdx.y, a = 0, b = (int)p.rows;
    if (p.offsets) {
        if (!find_tile(p.offsets, p.groups, p.rows, kRows, blockIdx.y, group, chunk)) return;
        group_bounds(p.offsets, group, p.rows, a, b);
    }
    const int row0 = a + chunk * kRows, rows = min(kRows, b - row0);
    const int f0 = (blockIdx.x * (kWarps / p.split) + warp / p.split) * kFewF, turn = warp % p.split, stride = p.split * 128;
    const int bytes = p.k * (kF8 ? 1 : 2);

    // rows behind the matrix or the chunk read its last one; their results are dropped
    const uint8_t *w0 = p.w + group * p.w_stride + (int64_t)min(f0 + gl, p.n - 1) * p.ldw + tl * 16;
    const uint8_t *w1 = p.w + group * p.w_stride + (int64_t)min(f0 + gl + 8, p.n - 1) * p.ldw + tl * 16;
    const uint8_t *xr[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) xr[t] = p.x + (int64_t)(row0 + min(8 * t + gl, rows - 1)) * p.ldx + tl * 16;
    const int left = bytes - tl * 16;  // of a row from this lane's first byte on
    float acc[NT][4] = {};
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int s0 = f0 < p.n ? turn * 128 : bytes; s0 < bytes; s0 += stride * U) {
        uint4 wa[U][2], wb[U][2], xv[U][NT][2];
        float ws[U] = {}, xs[U][NT][2] = {};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * stride;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = s + 64 * h;
                const bool on = at < left;
                wa[u][h] = on ? load_stream(w0 + at) : zero;
                wb[u][h] = on ? load_stream(w1 + at) : zero;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * stride;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < NT; ++t) xv[u][t][h] = s + 64 * h < left ? __ldg(reinterpret_cast<const uint4 *>(xr[t] + s + 64 * h)) : zero;
            if (kF8 && s < bytes) {
                const int blk = s / 128;
                ws[u] = __ldg(p.ws + group * p.ws_group + (int64_t)(f0 / kScaleBlock) * p.ws_row + blk * p.ws_blk);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 2; ++j)  // of the accumulator's columns: rows 2 * tl + j of the tile
                        xs[u][t][j] = __ldg(p.xs + (int64_t)(row0 + min(8 * t + 2 * tl + j, rows - 1)) * p.xs_row + blk * p.xs_blk);
            }
        }
        float seg[NT][4] = {};  // 16-bit: of these steps
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                if constexpr (kF8) {
                    float d[4] = {};
#pragma unroll
                    for (int h = 0; h < 2; ++h) multiply<DTYPE>(d, wa[u][h], wb[u][h], xv[u][t][h]);
                    // a step behind the last has zero sums and zero scales
                    const float c0 = ws[u] * xs[u][t][0], c1 = ws[u] * xs[u][t][1];
                    acc[t][0] = fmaf(d[0], c0, acc[t][0]);
                    acc[t][1] = fmaf(d[1], c1, acc[t][1]);
                    acc[t][2] = fmaf(d[2], c0, acc[t][2]);
                    acc[t][3] = fmaf(d[3], c1, acc[t][3]);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) multiply<DTYPE>(seg[t], wa[u][h], wb[u][h], xv[u][t][h]);
                }
            }
        if constexpr (!kF8)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[t][i] += seg[t][i];
    }
    // part[warp][row][feature]
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[warp][(8 * t + 2 * tl + (i & 1)) * kFewF + gl + 8 * (i >> 1)] = acc[t][i];
    __syncthreads();
    const int wide = kWarps / p.split * kFewF;  // features of the CTA
    for (int i = tid; i < wide * rows; i += kWarps * 32) {
        const int row = i / wide, j = i - row * wide;
        const float *v0 = &part[j / kFewF * p.split][row * kFewF + j % kFewF];
        float v = *v0;
        for (int w = 1; w < p.split; ++w) v += v0[w * kFewF * kRows];
        const int f = blockIdx.x * wide + j;
        if (f >= p.n) continue;
        const int64_t o = (int64_t)(row0 + row) * p.ldo + f;
        if (p.out_dtype == UMSX_DTYPE_F32) static_cast<float *>(p.out)[o] = v;
        else if (p.out_dtype == UMSX_DTYPE_BF16) static_cast<__nv_bfloat16 *>(p.out)[o] = __float2bfloat16_rn(v);
        else static_cast<__half *>(p.out)[o] = __float2half_rn(v);
    }
}

template <int DTYPE>
void launch(const FewParams &p, int nt, int64_t chunks, cudaStream_t s) {
    const int features = kWarps / p.split * kFewF;
    const dim3 grid((p.n + features - 1) / features, (unsigned)chunks);
    constexpr bool kF8 = DTYPE == UMSX_DTYPE_E4M3;  // steps in flight: what 128 registers hold
    if (nt == 1) k_product_few<DTYPE, 1, kF8 ? 3 : 4><<<grid, kWarps * 32, 0, s>>>(p);
    else k_product_few<DTYPE, 2, 2><<<grid, kWarps * 32, 0, s>>>(p);
}

}  // namespace

// Tiles of eight rows a CTA takes, or 0 where the tcgen05 kernel is to be used.  Decoding, up to four rows an expert on average:
// the weights are all there is to read (2816 x 2048 e4m3, 1536 x 2048 bf16, this kernel / the other: 3 rows an expert 82 / 78 us
// and 123 / 125, 6 rows 88 / 88, 8 rows in bf16 160 / 147).  Up to 2^17 outputs: the other has few tiles, each alone with its
// contraction, which this one splits over eight warps (us, bf16; 57 rows of 640 x 9728: 19.5 / 39.9, 256 of 136 x 5648: 13.3 /
// 35.8, 64 of 640 x 128: 8.2 / 10.2, 8 x 8 of 1536 x 2048: 18.5 / 22.6, 128 of 1024 x 4096: 21.5 / 23.6); with more of them it
// reads the weights too often (8 x 32 of 1536 x 2048: 30.8 / 22.5, 128 of 2048 x 4096: 37.9 / 25.6).  e4m3, with half the bytes,
// changes over a little later (the same seven: 18.5 / 43.0, 12.3 / 36.9, 8.2 / 10.3, 16.4 / 16.4, 19.5 / 28.7, then
// 26.6 / 18.4 and 30.7 / 26.6; between them 256 of 640 x 9728, 160 K outputs: 38.9 / 55.3, in bf16 47.1 / 55.3).  The rows of the longest group are not known on
// the host: where one of many experts gets them all, its weights are read once for every eight or sixteen.
static int few_tiles(const Product &p) {
    const double mean = (double)p.rows / p.groups;
    if (p.rows > 1024) return 0;  // one expert may have got them all, and is then read rows / 8 times
    if (mean <= 4) return 1;
    return p.rows * ((p.n + kFewF - 1) / kFewF * kFewF) <= 1 << 17 ? (mean <= 8 ? 1 : 2) : 0;
}

bool product_few_takes(const Product &p) {
    const int size = p.dtype == UMSX_DTYPE_E4M3 ? 1 : 2;
    const auto ok = [&](const void *b, int64_t ld) { return reinterpret_cast<uintptr_t>(b) % 16 == 0 && ld * size % 16 == 0; };
    return p.mode == kForward && p.rows > 0 && p.k * size % 16 == 0 && ok(p.x, p.ldx) && ok(p.w, p.ldw) &&
           (p.groups == 1 || p.w_stride * size % 16 == 0) && few_tiles(p) > 0;
}

int launch_product_few(const Product &p, int sms, cudaStream_t s) {
    const int size = p.dtype == UMSX_DTYPE_E4M3 ? 1 : 2, nt = few_tiles(p);
    FewParams f{};
    f.groups = p.groups, f.n = p.n, f.k = p.k, f.out_dtype = p.out_dtype;
    f.rows = p.rows, f.offsets = p.offsets;
    f.x = static_cast<const uint8_t *>(p.x), f.w = static_cast<const uint8_t *>(p.w);
    f.ldx = p.ldx * size, f.ldw = p.ldw * size, f.w_stride = p.w_stride * size;
    f.xs = p.xs, f.ws = p.ws;
    f.xs_row = p.xs_row, f.xs_blk = p.xs_blk, f.ws_row = p.ws_row, f.ws_blk = p.ws_blk, f.ws_group = p.ws_group;
    f.out = p.out, f.ldo = p.ldo;
    // chunks of 8 * nt rows: at most one that is not full for each group that has rows
    const int64_t chunks = p.offsets ? p.rows / (8 * nt) + std::min<int64_t>(p.groups, p.rows) : (p.rows + 8 * nt - 1) / (8 * nt);
    // As many warps as are resident (16 an SM) for the blocks of 16 features that have rows, and at most 2 KB of a row to a
    // warp: 8 bf16 experts of 1536 features 18.5 us with two warps a block (four: 20.5), 16 tokens' 92 us (one: 98).
    const int64_t blocks = std::min<int64_t>(p.groups, p.rows) * ((p.n + kFewF - 1) / kFewF);
    f.split = 1;
    while (f.split < 8 && (2 * f.split * blocks <= 16 * sms || f.split * 2048 < p.k * size)) f.split *= 2;
    if (p.dtype == UMSX_DTYPE_BF16) launch<UMSX_DTYPE_BF16>(f, nt, chunks, s);
    else if (p.dtype == UMSX_DTYPE_F16) launch<UMSX_DTYPE_F16>(f, nt, chunks, s);
    else launch<UMSX_DTYPE_E4M3>(f, nt, chunks, s);
    return 1;
}

}  // namespace umsx
