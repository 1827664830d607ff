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
// out[r][f] = sum_c R[r][c] F[f][c] in 64 x 64 tiles with fp32 FMAs, element loads and bounds
// checks everywhere.  It takes what the tensor-core kernels cannot address: TMA wants bases
// and row strides that are multiples of 16 bytes.  e4m3 operands are dequantised as they are
// staged (code * scale, one rounding).

constexpr int kTile = 64, kStep = 16;

struct AnyParams {
    int dtype, out_dtype, groups, mode;
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

__device__ __forceinline__ float load_el(const void *p, int64_t i, int dtype) {
    if (dtype == UMSX_DTYPE_E4M3) {
        const __nv_fp8_e4m3 v = static_cast<const __nv_fp8_e4m3 *>(p)[i];
        return (float)v;
    }
    const uint32_t h = __ldg(static_cast<const unsigned short *>(p) + i);
    return dtype == UMSX_DTYPE_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}

__device__ __forceinline__ void store_el(void *p, int64_t i, int dtype, float v) {
    if (dtype == UMSX_DTYPE_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == UMSX_DTYPE_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half *>(p)[i] = __float2half_rn(v);
}

__global__ void __launch_bounds__(256) k_product_any(const AnyParams p) {
    __shared__ float sR[kStep][kTile + 4], sF[kStep][kTile + 4];
    __shared__ int s_group, s_tile;
    const int tid = threadIdx.x, f0 = blockIdx.x * kTile;
    // row tiles of all groups in order; this CTA takes every gridDim.y-th
    for (int t = blockIdx.y;; t += gridDim.y) {
        __syncthreads();
        if (tid == 0) {
            int left = t, g = 0;
            for (; g < p.groups; ++g) {
                int a, b;
                group_bounds(p.offsets, g, p.rows, a, b);
                const int tiles = p.mode == kGradWeight ? (p.out_rows + kTile - 1) / kTile : (b - a + kTile - 1) / kTile;
                if (left < tiles) break;
                left -= tiles;
            }
            s_group = g;
            s_tile = left;
        }
        __syncthreads();
        if (s_group == p.groups) return;
        int a, b;
        group_bounds(p.offsets, s_group, p.rows, a, b);
        const bool dw = p.mode == kGradWeight;
        const int r0 = s_tile * kTile, nr = dw ? p.out_rows : b - a, nc = dw ? b - a : p.contraction;
        const int64_t r_base = dw ? (int64_t)a * p.r_c : (int64_t)a * p.r_row;
        const int64_t f_base = dw ? (int64_t)a * p.f_c : (int64_t)s_group * p.f_group;
        float acc[4][4] = {};
        for (int c0 = 0; c0 < nc; c0 += kStep) {
            for (int i = tid; i < kTile * kStep; i += 256) {
                // neighbouring threads along the axis that is contiguous in memory
                int rr = p.r_c == 1 ? i / kStep : i % kTile, cc = p.r_c == 1 ? i % kStep : i / kTile;
                float v = 0.0f;
                if (r0 + rr < nr && c0 + cc < nc) {
                    v = load_el(p.R, r_base + (int64_t)(r0 + rr) * p.r_row + (int64_t)(c0 + cc) * p.r_c, p.dtype);
                    if (p.rs) v *= __ldg(p.rs + (int64_t)(a + r0 + rr) * p.rs_row + (int64_t)((c0 + cc) / kScaleBlock) * p.rs_blk);
                }
                sR[cc][rr] = v;
                rr = p.f_c == 1 ? i / kStep : i % kTile, cc = p.f_c == 1 ? i % kStep : i / kTile;
                v = 0.0f;
                if (f0 + rr < p.features && c0 + cc < nc) {
                    v = load_el(p.F, f_base + (int64_t)(f0 + rr) * p.f_feat + (int64_t)(c0 + cc) * p.f_c, p.dtype);
                    if (p.fs)
                        v *= __ldg(p.fs + s_group * p.fs_group + (int64_t)((f0 + rr) / kScaleBlock) * p.fs_row +
                                   (int64_t)((c0 + cc) / kScaleBlock) * p.fs_blk);
                }
                sF[cc][rr] = v;
            }
            __syncthreads();
#pragma unroll
            for (int cc = 0; cc < kStep; ++cc) {
                float x[4], y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = sR[cc][(tid >> 4) * 4 + i];
                    y[i] = sF[cc][(tid & 15) * 4 + i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
            }
            __syncthreads();
        }
        for (int i = 0; i < 4; ++i) {
            const int r = r0 + (tid >> 4) * 4 + i;
            if (r >= nr) break;
            for (int j = 0; j < 4; ++j) {
                const int f = f0 + (tid & 15) * 4 + j;
                if (f >= p.features) break;
                const int64_t o = dw ? s_group * p.out_group + (int64_t)r * p.ldo + f : (int64_t)(a + r) * p.ldo + f;
                store_el(p.out, o, p.out_dtype, acc[i][j]);
            }
        }
    }
}

}  // namespace

int launch_product_any(const Product &p, int sms, cudaStream_t s) {
    AnyParams a{};
    a.dtype = p.dtype;
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
    const int64_t tiles = p.mode == kGradWeight ? (int64_t)p.groups * ((p.n + kTile - 1) / kTile)
                                                : (p.rows + kTile - 1) / kTile + p.groups;
    const dim3 grid((unsigned)((a.features + kTile - 1) / kTile), (unsigned)std::min<int64_t>(tiles, 32 * sms));
    k_product_any<<<grid, 256, 0, s>>>(a);
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

umsx_status run_product(const Product &p, umsx_stream stream) {
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
