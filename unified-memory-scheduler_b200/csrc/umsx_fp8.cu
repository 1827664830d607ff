// umsx_fp8_quantize: values to e4m3 codes with one fp32 scale per block of 1 x 128 (rows of
// activations) or 128 x 128 (weight matrices).
//
//   scale = max(amax / 448, 2^-126)     amax over the block's finite values
//   code  = e4m3 nearest to x / scale   ties to even; inf and NaN become the NaN code
//
// 448 is the largest e4m3 value, so a block's largest entry lands on it.  The floor 2^-126 (the
// smallest normal float) keeps the quotient finite for blocks of zeros and subnormals.  scale and
// quotient are IEEE divisions, one rounding each, so the codes are those of the same formula on a CPU.
// Bound: memory, (2 + 1) bytes per bf16 value plus 4 per block, read and written once.
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

struct QuantParams {
    const void *x;
    int64_t ldx, x_stride;
    int matrices, cols, vec;  // vec: rows start at multiples of 16 bytes (x) and 8 bytes (q)
    int64_t rows;
    uint8_t *q;
    int64_t ldq, q_stride;
    float *scales;
    int64_t s_row, s_blk, s_stride;
};

template <class T>
__device__ __forceinline__ float to_f32(T v) {
    return (float)v;
}

// Eight consecutive values of a row from column c on; zeros behind the last column.
template <class T>
__device__ __forceinline__ void load8(const T *row, int c, int cols, bool vec, float (&v)[8]) {
    if (vec && c + 8 <= cols) {
        constexpr int kVecs = 8 * sizeof(T) / 16;
        uint4 raw[kVecs];
#pragma unroll
        for (int i = 0; i < kVecs; ++i) raw[i] = __ldg(reinterpret_cast<const uint4 *>(row + c) + i);
        const T *e = reinterpret_cast<const T *>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(e[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? to_f32(row[c + i]) : 0.0f;
}

__device__ __forceinline__ float amax8(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float a = fabsf(v[i]);
        if (a < INFINITY) m = fmaxf(m, a);  // false for inf and NaN
    }
    return m;
}

__device__ __forceinline__ float block_scale(float amax) { return fmaxf(__fdiv_rn(amax, 448.0f), 0x1p-126f); }

__device__ __forceinline__ void store8(uint8_t *row, int c, int cols, bool vec, const float (&v)[8], float scale) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float2 t;
        // inf / scale would saturate to 448: make it the NaN that it stands for
        t.x = fabsf(v[i]) < INFINITY ? __fdiv_rn(v[i], scale) : __uint_as_float(0x7fc00000u);
        t.y = fabsf(v[i + 1]) < INFINITY ? __fdiv_rn(v[i + 1], scale) : __uint_as_float(0x7fc00000u);
        w[i >> 2] |= (uint32_t)__nv_cvt_float2_to_fp8x2(t, __NV_SATFINITE, __NV_E4M3) << (16 * ((i >> 1) & 1));
    }
    if (vec && c + 8 <= cols) {
        *reinterpret_cast<uint2 *>(row + c) = make_uint2(w[0], w[1]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < cols) row[c + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
}

// 1 x 128 blocks: sixteen lanes per block, eight values each.
template <class T>
__global__ void __launch_bounds__(256) k_quant_rows(const QuantParams p) {
    const int nb = (p.cols + kScaleBlock - 1) / kScaleBlock, l = threadIdx.x & 15;
    const int64_t blocks = (int64_t)p.matrices * p.rows * nb;
    // whole warps step together: the shuffles below need both halves
    for (int64_t i0 = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; 2 * i0 < blocks;
         i0 += ((int64_t)gridDim.x * blockDim.x) >> 5) {
        const int64_t i = 2 * i0 + ((threadIdx.x >> 4) & 1);
        const bool on = i < blocks;
        const int64_t mr = on ? i / nb : 0, mat = mr / p.rows, r = mr - mat * p.rows;
        const int b = on ? (int)(i - mr * nb) : 0, c = b * kScaleBlock + l * 8;
        float v[8] = {};
        if (on) load8(static_cast<const T *>(p.x) + mat * p.x_stride + r * p.ldx, c, p.cols, p.vec, v);
        float m = amax8(v);
#pragma unroll
        for (int s = 8; s >= 1; s >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, s));
        const float scale = block_scale(m);
        if (!on) continue;
        store8(p.q + mat * p.q_stride + r * p.ldq, c, p.cols, p.vec, v, scale);
        if (l == 0) p.scales[mat * p.s_stride + r * p.s_row + b * p.s_blk] = scale;
    }
}

// 128 x 128 blocks: one CTA per block; the block stays in registers between its maximum and its codes.
template <class T>
__global__ void __launch_bounds__(256) k_quant_blocks(const QuantParams p) {
    __shared__ float part[8];
    const int64_t nbr = (p.rows + kScaleBlock - 1) / kScaleBlock;
    const int nb = (p.cols + kScaleBlock - 1) / kScaleBlock;
    const int64_t blocks = (int64_t)p.matrices * nbr * nb;
    for (int64_t i = blockIdx.x; i < blocks; i += gridDim.x) {
        const int64_t mbr = i / nb, mat = mbr / nbr, br = mbr - mat * nbr;
        const int b = (int)(i - mbr * nb), c = b * kScaleBlock + (threadIdx.x & 15) * 8;
        const int64_t r0 = br * kScaleBlock + (threadIdx.x >> 4);
        float v[8][8], m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t r = r0 + 16 * j;
            if (r < p.rows) load8(static_cast<const T *>(p.x) + mat * p.x_stride + r * p.ldx, c, p.cols, p.vec, v[j]);
            else
#pragma unroll
                for (int q = 0; q < 8; ++q) v[j][q] = 0.0f;
            m = fmaxf(m, amax8(v[j]));
        }
        m = warp_max(m);
        __syncthreads();  // the previous block's readers are done with part
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) m = fmaxf(m, part[w]);
        const float scale = block_scale(m);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t r = r0 + 16 * j;
            if (r < p.rows) store8(p.q + mat * p.q_stride + r * p.ldq, c, p.cols, p.vec, v[j], scale);
        }
        if (threadIdx.x == 0) p.scales[mat * p.s_stride + br * p.s_row + b * p.s_blk] = scale;
    }
}

template <class T>
void launch_quant(const QuantParams &p, int block_rows, int sms, cudaStream_t s) {
    const int64_t nb = (p.cols + kScaleBlock - 1) / kScaleBlock;
    if (block_rows == 1) {
        const int64_t ctas = ((int64_t)p.matrices * p.rows * nb + 15) / 16;
        k_quant_rows<T><<<(unsigned)std::min<int64_t>(ctas, 8 * sms), 256, 0, s>>>(p);
    } else {
        const int64_t blocks = (int64_t)p.matrices * ((p.rows + kScaleBlock - 1) / kScaleBlock) * nb;
        k_quant_blocks<T><<<(unsigned)std::min<int64_t>(blocks, 64 * sms), 256, 0, s>>>(p);
    }
}

umsx_status fail(umsx_status s, const std::string &msg) {
    record_error(msg.c_str());
    return s;
}

}  // namespace
}  // namespace umsx

using namespace umsx;

extern "C" umsx_status umsx_fp8_quantize(const void *x, int64_t ldx, int64_t x_stride, int x_dtype, int matrices,
                                         int64_t rows, int cols, int block_rows, void *q, int64_t ldq, int64_t q_stride,
                                         float *scales, int64_t s_row, int64_t s_blk, int64_t s_stride,
                                         umsx_stream stream) {
    if (x_dtype != UMSX_DTYPE_F32 && x_dtype != UMSX_DTYPE_BF16 && x_dtype != UMSX_DTYPE_F16)
        return fail(UMSX_EINVAL, "x must be F32, BF16 or F16");
    if (block_rows != 1 && block_rows != kScaleBlock) return fail(UMSX_EINVAL, "block_rows must be 1 or 128");
    if (matrices < 0 || rows < 0 || rows > 0x7ffffff0 || cols < 1 || cols > (1 << 24))
        return fail(UMSX_EINVAL, "matrices and rows must not be negative, cols must be 1..2^24");
    if (ldx < cols || ldq < cols || x_stride < 0 || s_row < 0 || s_blk < 0 || s_stride < 0 ||
        (matrices > 1 && q_stride < (rows - 1) * ldq + cols))
        return fail(UMSX_EINVAL, "a stride is shorter than a row");
    if (matrices == 0 || rows == 0) return UMSX_OK;
    if (!x || !q || !scales) return fail(UMSX_EINVAL, "null buffer");
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail(UMSX_EDEVICE, std::string("device query: ") + cudaGetErrorString(e));
    const int64_t size = x_dtype == UMSX_DTYPE_F32 ? 4 : 2;
    QuantParams p{};
    p.x = x, p.ldx = ldx, p.x_stride = x_stride;
    p.matrices = matrices, p.rows = rows, p.cols = cols;
    p.q = static_cast<uint8_t *>(q), p.ldq = ldq, p.q_stride = q_stride;
    p.scales = scales, p.s_row = s_row, p.s_blk = s_blk, p.s_stride = s_stride;
    p.vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx * size % 16 == 0 && x_stride * size % 16 == 0 &&
            reinterpret_cast<uintptr_t>(q) % 8 == 0 && ldq % 8 == 0 && q_stride % 8 == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x_dtype == UMSX_DTYPE_F32) launch_quant<float>(p, block_rows, sms, s);
    else if (x_dtype == UMSX_DTYPE_BF16) launch_quant<__nv_bfloat16>(p, block_rows, sms, s);
    else launch_quant<__half>(p, block_rows, sms, s);
    record_launches(1);
    e = cudaGetLastError();
    if (e != cudaSuccess) return fail(UMSX_EDEVICE, std::string("quantize launch: ") + cudaGetErrorString(e));
    return UMSX_OK;
}
