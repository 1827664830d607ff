// Ragged products over the caller's own expert weights: what the entry points
// (umsx_products.cu) hand to the kernels.
//
// Every direction is one form: out[r][f] = sum_c R[r][c] * F[f][c].
//   forward  r: rows of the group, f: n, c: k    R = x,        F = w[e]
//   dx       r: rows of the group, f: k, c: n    R = dy,       F = w[e] transposed
//   dw       r: n, f: k, c: rows of the group    R = dy transposed, F = x transposed
// so that f is contiguous in the output and w is read as it lies in memory.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/umsx.h"

namespace umsx {

enum ProductMode { kForward = 0, kGradInput = 1, kGradWeight = 2 };

constexpr int kMaxGroups = 1024;
constexpr int64_t kMaxRows = (1ll << 31) - 512;  // a row plus a tile of rows, or a step of the contraction, is an int
// Contraction of 16-bit operands that shares a tensor-core accumulator, for fp32 and for 16-bit outputs, whose last rounding hides
// an error of 2^-15 of the value (25 units of 2^-23 for each 512 at worst, half an f16's unit is 2^-11).
constexpr int kAccumulate32 = 512, kAccumulate16 = 4096;
constexpr long long kWaitCycles = 2000000000ll;  // limit of a bounded wait, about a second
constexpr int kScaleBlock = 128;  // values that share one scale of an e4m3 operand

struct Product {
    ProductMode mode;
    int dtype;      // operands: UMSX_DTYPE_BF16, _F16 or _E4M3
    int out_dtype;  // UMSX_DTYPE_F32, _BF16 or _F16
    int groups;
    int64_t rows;  // of x and dy
    int n, k;
    const int32_t *offsets;  // [groups + 1], or null: one group of all rows
    const void *x, *dy, *w;  // [rows][k], [rows][n], [groups][n][k]; strides in elements, the last is 1
    int64_t ldx, lddy, ldw, w_stride;
    const float *xs, *ws;  // e4m3: xs(row, block of k), ws(group, block of n, block of k)
    int64_t xs_row, xs_blk, ws_row, ws_blk, ws_group;
    void *out;  // forward [rows][n], dx [rows][k], dw [groups][n][k]
    int64_t ldo, out_stride;
    int fault_cta;         // CTA that withholds its first copies (umsx_products_inject_fault), -1: none
    long long wait_limit;  // SM cycles of a bounded wait, 0: the usual ones

    int features() const { return mode == kForward ? n : k; }
};

// Where a tensor lies: `blocks` blocks, `block` bytes apart, of `lines` lines of `width` bytes, `line` bytes apart.
struct Region {
    const void *base;
    int64_t width, lines, line, blocks, block;
    int64_t extent() const { return (blocks - 1) * block + (lines - 1) * line + width; }
};
// A matrix or a stack of them, strides in elements of `size` bytes.
inline Region region(const void *base, int size, int64_t width, int64_t lines, int64_t line, int64_t blocks = 1, int64_t block = 0) {
    return {base, width * size, lines, lines > 1 ? line * size : 0, blocks, blocks > 1 ? block * size : 0};
}
// Whether the two may share a byte.  Slices of one buffer that lie beside one another share none although their ranges
// do: columns of equal line stride, or lines of equal block stride.
inline bool overlap(const Region &a, const Region &b) {
    if (!a.base || !b.base || a.extent() <= 0 || b.extent() <= 0) return false;
    const int64_t at = (int64_t)((uintptr_t)b.base - (uintptr_t)a.base);
    if (at >= a.extent() || -at >= b.extent()) return false;
    const auto beside = [at](int64_t period, int64_t wa, int64_t wb) {
        if (period <= 0) return false;
        const int64_t r = (at % period + period) % period;
        return r >= wa && r + wb <= period;
    };
    const auto whole = [](const Region &x, int64_t period) { return x.blocks == 1 || x.block % period == 0; };
    if (a.line == b.line && a.line > 0 && whole(a, a.line) && whole(b, a.line) && beside(a.line, a.width, b.width)) return false;
    const int64_t ba = (a.lines - 1) * a.line + a.width, bb = (b.lines - 1) * b.line + b.width;
    return !(a.block == b.block && beside(a.block, ba, bb));
}

#ifdef __CUDACC__
// First row of group g, and for g = groups the row behind the last one.  Offsets are clamped to the matrix, so that wrong
// ones cannot lead outside it; a group whose end lies before its start is empty.
__device__ __forceinline__ int group_start(const int32_t *offsets, int g, int64_t rows) {
    if (!offsets) return g ? (int)rows : 0;
    return min(max(__ldg(offsets + g), 0), (int)rows);
}
// Rows [a, b) of group g.
__device__ __forceinline__ void group_bounds(const int32_t *offsets, int g, int64_t rows, int &a, int &b) {
    a = group_start(offsets, g, rows);
    b = max(a, group_start(offsets, g + 1, rows));
}
// The index-th tile of `per` rows, counted over the groups, by all threads of a CTA of 256 (a barrier in front of the next
// call); false behind the last.
__device__ __forceinline__ bool find_tile(const int32_t *offsets, int groups, int64_t rows, int per, int index, int &group,
                                          int &tile) {
    __shared__ int s_group, s_tile, s_sum[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int g0 = 0; g0 < groups; g0 += 256) {
        const int g = g0 + tid;
        int a = 0, b = 0;
        if (g < groups) group_bounds(offsets, g, rows, a, b);
        const int tiles = (b - a + per - 1) / per;
        int incl = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) s_sum[warp] = incl;
        if (tid == 0) s_group = -1;
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            if (w < warp) before += s_sum[w];
            all += s_sum[w];
        }
        const int first = before + incl - tiles;
        if (index >= first && index < first + tiles) s_group = g, s_tile = index - first;
        __syncthreads();
        group = s_group;
        tile = s_tile;
        if (group >= 0) return true;
        index -= all;
        __syncthreads();  // s_sum is written again
    }
    return false;
}
#endif

// Each returns the number of kernels launched, -1 when the driver refuses something.
int launch_product_any(const Product &p, int sms, cudaStream_t s);
int launch_product_tc(const Product &p, int sms, cudaStream_t s);  // where product_tc_takes(p)
bool product_tc_takes(const Product &p);
int launch_product_few(const Product &p, int sms, cudaStream_t s);  // where product_few_takes(p)
bool product_few_takes(const Product &p);
uint32_t *product_err_word();  // of the current device: nonzero after a bounded wait gave up

}  // namespace umsx
