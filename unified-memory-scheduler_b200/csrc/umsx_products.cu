// Entry points of the ragged products (umsx_grouped_mm and its gradients, umsx_fp8_mm,
// umsx_fp8_grouped_mm), and the kernel that takes every shape, stride and alignment.
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
// features, 32 of the contraction a step: single-element loads, neighbouring lanes along the axis that is contiguous in
// memory, one step ahead in registers; from shared memory into mma.sync.  e4m3 codes become f16 (exact); the sums of
// a block of 128 are scaled once and added in fp32.  Bound by the issue of those loads (bf16 4096 x 4096 x 2049: 573 us,
// 120 TFLOP/s; fp32 FMAs in place of mma.sync took 3441 us, 64-bit addresses per element instead of a step per thread 1295).

constexpr int kAnyRows = 64, kAnyF = 128, kStep = 32, kLine = kStep + 8;  // kLine: 80 bytes spread eight lines over all banks

struct AnyParams {
    int out_dtype, groups, mode;
    int64_t rows;
    int features, contraction;  // contraction: forward k, dx n (dw: the group's rows)
    int out_rows;               // dw: n
    const int32_t *offsets;
    const void *R, *F;
    int64_t r_row, r_c, f_feat, f_c, f_group;  // element strides
    const float *rs, *fs;
    int64_t rs_row, rs_blk, fs_row, fs_blk, fs_group;
    void *out;
    int64_t ldo, out_group;
};

// LINES x kStep elements of an operand, held by 256 threads between their load and their store: element i of a thread.
template <int DTYPE, int LINES>
struct Elements {
    static constexpr int kPer = LINES * kStep / 256;
    uint16_t v[kPer];

    // Neighbouring threads lie along c where that is contiguous, along the lines otherwise; a thread's next element is a fixed
    // step further in memory either way.
    __device__ __forceinline__ void load(const void *p, int64_t s_line, int64_t s_c, int lines, int steps) {
        constexpr int kSize = DTYPE == UMSX_DTYPE_E4M3 ? 1 : 2;
        const bool along_c = s_c == 1;
        const int l = along_c ? threadIdx.x / kStep : threadIdx.x % LINES, c = along_c ? threadIdx.x % kStep : threadIdx.x / LINES;
        const int64_t by = (along_c ? 256 / kStep * s_line : 256 / LINES * s_c) * kSize;
        const uint8_t *at = static_cast<const uint8_t *>(p) + (l * s_line + c * s_c) * kSize;
        // elements of this thread that lie inside: the other coordinate is fixed
        const int in = along_c ? (c < steps ? (lines - l + 256 / kStep - 1) / (256 / kStep) : 0)
                               : (l < lines ? (steps - c + 256 / LINES - 1) / (256 / LINES) : 0);
#pragma unroll
        for (int i = 0; i < kPer; ++i, at += by) {
            if constexpr (kSize == 1) v[i] = i < in ? __ldg(at) : 0;
            else v[i] = i < in ? __ldg(reinterpret_cast<const unsigned short *>(at)) : 0;
        }
    }
    __device__ __forceinline__ void store(uint16_t *to, bool along_c) const {
        const int l = along_c ? threadIdx.x / kStep : threadIdx.x % LINES, c = along_c ? threadIdx.x % kStep : threadIdx.x / LINES;
        uint16_t *at = to + l * kLine + c;
        const int by = along_c ? 256 / kStep * kLine : 256 / LINES;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            uint16_t h = v[i];
            if constexpr (DTYPE == UMSX_DTYPE_E4M3) h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)h, __NV_E4M3).x;
            at[i * by] = h;
        }
    }
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], const uint16_t *p) {
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

template <int DTYPE>
__global__ void __launch_bounds__(256, 2) k_product_any(const AnyParams p) {
    constexpr bool kF8 = DTYPE == UMSX_DTYPE_E4M3;
    constexpr int kSize = kF8 ? 1 : 2;
    __shared__ __align__(16) uint16_t sR[kAnyRows * kLine], sF[kAnyF * kLine];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, f0 = blockIdx.x * kAnyF;
    const int wr = (warp & 1) * 32, wf = (warp >> 1) * 32;  // the warp's 32 x 32 of the tile
    const bool r_along = p.r_c == 1, f_along = p.f_c == 1;
    // row tiles of all groups in order; this CTA takes every gridDim.y-th
    for (int t = blockIdx.y;; t += gridDim.y) {
        __syncthreads();
        int g = 0, tile = 0;
        if (p.mode == kGradWeight) {
            const int each = (p.out_rows + kAnyRows - 1) / kAnyRows;
            g = t / each;
            tile = t % each;
            if (g >= p.groups) return;
        } else if (!find_tile(p.offsets, p.groups, p.rows, kAnyRows, t, g, tile)) {
            return;
        }
        int a, b;
        group_bounds(p.offsets, g, p.rows, a, b);
        const bool dw = p.mode == kGradWeight;
        const int r0 = tile * kAnyRows, nr = min(kAnyRows, (dw ? p.out_rows : b - a) - r0), nf = min(kAnyF, p.features - f0);
        const int nc = dw ? b - a : p.contraction;
        const uint8_t *R = static_cast<const uint8_t *>(p.R) + (a * (dw ? p.r_c : p.r_row) + r0 * p.r_row) * kSize;
        const uint8_t *F = static_cast<const uint8_t *>(p.F) + (dw ? a * p.f_c : g * p.f_group) * kSize + f0 * p.f_feat * kSize;
        Elements<DTYPE, kAnyRows> er;
        Elements<DTYPE, kAnyF> ef;
        er.load(R, p.r_row, p.r_c, nr, nc);
        ef.load(F, p.f_feat, p.f_c, nf, nc);
        float acc[2][4][4] = {}, blk[2][4][4] = {};  // [16 rows][8 features]; blk: e4m3, of the present block of 128
        for (int c0 = 0; c0 < nc; c0 += kStep) {
            __syncthreads();  // the previous step has been read
            er.store(sR, r_along);
            ef.store(sF, f_along);
            __syncthreads();
            if (c0 + kStep < nc) {
                er.load(R + (c0 + kStep) * p.r_c * kSize, p.r_row, p.r_c, nr, nc - c0 - kStep);
                ef.load(F + (c0 + kStep) * p.f_c * kSize, p.f_feat, p.f_c, nf, nc - c0 - kStep);
            }
#pragma unroll
            for (int k = 0; k < kStep; k += 16) {
                uint32_t x[2][4], y[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    // rows x contraction: 8 x 8 matrices (0, 0), (8, 0), (0, 8), (8, 8); features: (0, 0), (0, 8), (8, 0), (8, 8)
                    ldmatrix4(x[i], sR + (wr + 16 * i + (lane & 15)) * kLine + k + 8 * (lane >> 4));
                    ldmatrix4(y[i], sF + (wf + 16 * i + (lane & 7) + 8 * (lane >> 4)) * kLine + k + 8 * ((lane >> 3) & 1));
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma16816<DTYPE == UMSX_DTYPE_BF16>(kF8 ? blk[i][j] : acc[i][j], x[i], y[j >> 1][2 * (j & 1)], y[j >> 1][2 * (j & 1) + 1]);
            }
            if (kF8 && (c0 % kScaleBlock == kScaleBlock - kStep || c0 + kStep >= nc)) {
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
                            for (int q = 0; q < 2; ++q) {
                                acc[i][j][2 * h + q] = fmaf(sc, blk[i][j][2 * h + q], acc[i][j][2 * h + q]);
                                blk[i][j][2 * h + q] = 0.0f;
                            }
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = wr + 16 * i + 8 * h + (lane >> 2);
                if (r >= nr) continue;
                const int64_t at = (dw ? g * p.out_group + (int64_t)(r0 + r) * p.ldo : (int64_t)(a + r0 + r) * p.ldo) + f0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int f = wf + 8 * j + 2 * (lane & 3) + q;
                        if (f < nf) store_el(p.out, at + f, p.out_dtype, acc[i][j][2 * h + q]);
                    }
            }
    }
}

}  // namespace

int launch_product_any(const Product &p, int sms, cudaStream_t s) {
    AnyParams a{};
    a.out_dtype = p.out_dtype;
    a.groups = p.groups;
    a.mode = p.mode;
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
    if (p.mode == kForward) {
        a.R = p.x, a.r_row = p.ldx, a.r_c = 1;
        a.F = p.w, a.f_feat = p.ldw, a.f_c = 1, a.f_group = p.w_stride;
    } else if (p.mode == kGradInput) {
        a.R = p.dy, a.r_row = p.lddy, a.r_c = 1;
        a.F = p.w, a.f_feat = 1, a.f_c = p.ldw, a.f_group = p.w_stride;
    } else {
        a.R = p.dy, a.r_row = 1, a.r_c = p.lddy;
        a.F = p.x, a.f_feat = 1, a.f_c = p.ldx;
    }
    const int64_t tiles = p.mode == kGradWeight ? (int64_t)p.groups * ((p.n + kAnyRows - 1) / kAnyRows)
                                                : p.rows / kAnyRows + std::min<int64_t>(p.groups, p.rows);
    const dim3 grid((unsigned)((a.features + kAnyF - 1) / kAnyF), (unsigned)std::max<int64_t>(1, std::min<int64_t>(tiles, 32 * sms)));
    if (p.dtype == UMSX_DTYPE_BF16) k_product_any<UMSX_DTYPE_BF16><<<grid, 256, 0, s>>>(a);
    else if (p.dtype == UMSX_DTYPE_F16) k_product_any<UMSX_DTYPE_F16><<<grid, 256, 0, s>>>(a);
    else k_product_any<UMSX_DTYPE_E4M3><<<grid, 256, 0, s>>>(a);
    return 1;
}

namespace {

bool out_ok(int t) { return t == UMSX_DTYPE_F32 || t == UMSX_DTYPE_BF16 || t == UMSX_DTYPE_F16; }

// Shape checks shared by the entry points; the sizes are those that the kernels' 32-bit row and column indexes hold.
umsx_status check_product(const Product &p) {
    if (p.groups < 1 || p.groups > kMaxGroups) return fail(UMSX_EINVAL, "experts must be 1..1024");
    if (p.n < 1 || p.k < 1 || p.n > (1 << 24) || p.k > (1 << 24)) return fail(UMSX_EINVAL, "n and k must be 1..2^24");
    if (p.rows < 0 || p.rows > 0x7ffffff0) return fail(UMSX_EINVAL, "rows must be 0..2^31 - 16");
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

umsx_status run_product(const Product &p, umsx_stream stream) {
    if (out_overlaps(p)) return fail(UMSX_EINVAL, "the output overlaps an input");
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail(UMSX_EDEVICE, std::string("device query: ") + cudaGetErrorString(e));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int n = product_few_takes(p, sms) ? launch_product_few(p, sms, s) : product_tc_takes(p) ? launch_product_tc(p, sms, s) : launch_product_any(p, sms, s);
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
    if (e != cudaSuccess) return fail(UMSX_EDEVICE, std::string("products status: ") + cudaGetErrorString(e));
    return v ? fail(UMSX_ETIMEOUT, "a bounded wait of a product's kernel gave up: its output is not complete") : UMSX_OK;
}

}  // extern "C"
