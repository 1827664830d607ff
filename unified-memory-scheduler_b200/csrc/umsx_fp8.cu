// umsx_fp8_quantize: values to e4m3 codes with one fp32 scale per block of 1 x 128 (rows of
// activations) or 128 x 128 (weight matrices).
//
//   scale = max(amax / 448, 2^-126)     amax over the block's finite values
//   code  = e4m3 nearest to x / scale   ties to even; inf and NaN become the NaN code
//
// 448 is the largest e4m3 value, so a block's largest entry lands on it.  The floor 2^-126 (the
// smallest normal float) keeps the quotient finite for blocks of zeros and subnormals.  scale and
// quotient are rounded once each, as IEEE divisions are, so the codes are those of the same formula on a CPU.
// Bound: memory, (2 + 1) bytes per bf16 value plus 4 per block, read and written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <array>
#include <string>
#include <type_traits>
#include <utility>

#include "umsx_device.cuh"
#include "umsx_internal.h"
#include "umsx_products.h"

namespace umsx {
namespace {

struct QuantParams {
    const void *x;
    int64_t ldx, x_stride;
    int matrices, cols, steps;
    bool vec;  // rows start at multiples of 16 bytes (x) and 8 bytes (q)
    int64_t rows;
    uint8_t *q;
    int64_t ldq, q_stride;
    float *scales;
    int64_t s_row, s_blk, s_stride;
};

// A lane's 32 values of a 128-block, as pieces of 16 bytes: four lanes hold a block, piece j of lane l starts at column
// 128 / kPieces * j + kPer * l, so that the lanes of one load are neighbours in memory.  Values stay in their own type until
// they are scaled, which halves the registers of 16-bit inputs.  (With eight lanes to a block the work per block, a
// division, a reciprocal, shuffles and addresses, took as many instructions as the values.)
template <class T>
struct Values {
    static constexpr int kWords = 32 * sizeof(T) / 4, kPer = 16 / sizeof(T), kPieces = 32 / kPer;
    uint32_t w[kWords];

    static __device__ __forceinline__ int column(int b, int l, int j) { return b * kScaleBlock + kScaleBlock / kPieces * j + kPer * l; }

    // Block b's values of lane l of a row of `cols` values; zeros behind its end.
    __device__ __forceinline__ void load(const T *row, int b, int l, int cols, bool vec) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int c = column(b, l, j);
            if (vec && c + kPer <= cols) {
                *reinterpret_cast<uint4 *>(w + 4 * j) = __ldg(reinterpret_cast<const uint4 *>(row + c));
                continue;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (sizeof(T) == 4) {
                    w[4 * j + i] = c + i < cols ? __ldg(reinterpret_cast<const uint32_t *>(row) + c + i) : 0u;
                } else {
                    const unsigned short *h = reinterpret_cast<const unsigned short *>(row) + c + 2 * i;
                    w[4 * j + i] = (c + 2 * i < cols ? __ldg(h) : 0u) | (c + 2 * i + 1 < cols ? (uint32_t)__ldg(h + 1) << 16 : 0u);
                }
            }
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else {
            const uint32_t h = i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xffffu;
            if constexpr (std::is_same<T, __nv_bfloat16>::value) return i & 1 ? __uint_as_float(w[i >> 1] & 0xffff0000u) : bf16_bits_to_f32(h);
            else return f16_bits_to_f32(h);
        }
    }
    // Bits of |v| order like |v|; those of inf and NaN are at least kInf.  top: the largest of the 32 (16-bit types: of the
    // even and of the odd ones); finite: of the finite ones.
    static constexpr uint32_t kInf = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
    __device__ __forceinline__ uint32_t top() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) m = max(m, w[i] & 0x7fffffffu);
            else m = __vmaxu2(m, w[i] & 0x7fff7fffu);
        }
        return m;
    }
    __device__ __forceinline__ uint32_t finite() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint32_t a = sizeof(T) == 4 ? w[i] & 0x7fffffffu : (w[i >> 1] >> 16 * (i & 1)) & 0x7fffu;
            if (a < kInf) m = max(m, a);
        }
        return m;
    }
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return sizeof(T) == 4 ? max(a, b) : __vmaxu2(a, b); }
    static __device__ __forceinline__ uint32_t one(uint32_t m) { return sizeof(T) == 4 ? m : max(m >> 16, m & 0xffffu); }
    static __device__ __forceinline__ float as_float(uint32_t m) {
        if constexpr (sizeof(T) == 4) return __uint_as_float(m);
        else if constexpr (std::is_same<T, __nv_bfloat16>::value) return bf16_bits_to_f32(m);
        else return f16_bits_to_f32(m);
    }
};

// x / d as an IEEE division rounds it, Markstein's way (1990): with y = 1 / d correctly rounded, q = x y and r = x - q d
// (exact), q + r y rounds to x / d.  Three operations instead of ten, which would bound the kernel; not for quotients or
// residuals that may be subnormal.
__device__ __forceinline__ float quotient(float x, float d, float y) {
    const float q = __fmul_rn(x, y);
    return __fmaf_rn(__fmaf_rn(-q, d, x), y, q);
}
// Smallest block maximum for it.  The residual is exact down to |x| = 2^-102 (the last bit of q d is at least 2^-149 there);
// below, x / d is at most 2^-102 * 448 * 2^80 < 2^-13, which no error of an ulp lifts to the 2^-10 where codes begin.
constexpr float kPlain = 0x1p-80f;

// -x / d for two values at once (packed fp32 operations); yy, dd: -y and d in both halves.  The negative, because a sum of
// opposite zeros is +0: x = -0 meets one on the way, and its code is to keep the sign.
__device__ __forceinline__ uint64_t twice(float v) { return (uint64_t)__float_as_uint(v) << 32 | __float_as_uint(v); }
__device__ __forceinline__ float2 quotients(float a, float b, uint64_t dd, uint64_t yy) {
    uint64_t x, q, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a), "f"(b));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(x), "l"(yy));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(q), "l"(dd), "l"(x));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(q) : "l"(r), "l"(yy), "l"(q));
    float2 t;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(t.x), "=f"(t.y) : "l"(q));
    return t;
}

__device__ __forceinline__ float block_scale(float amax) {
    if (amax >= kPlain) return quotient(amax, 448.0f, 1.0f / 448.0f);
    return fmaxf(__fdiv_rn(amax, 448.0f), 0x1p-126f);
}

// Codes of a lane's values.  plain: every value is finite and the block's maximum at least kPlain.
template <class T>
__device__ __forceinline__ void store_codes(uint8_t *row, int b, int l, int cols, bool vec, const Values<T> &v, float scale, bool plain) {
    uint32_t w[8];
    if (plain) {
        const uint64_t yy = twice(-__frcp_rn(scale)), dd = twice(scale);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 a = quotients(v.value(4 * i), v.value(4 * i + 1), dd, yy);
            const float2 b = quotients(v.value(4 * i + 2), v.value(4 * i + 3), dd, yy);
            w[i] = ((uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
                    (uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16) ^ 0x80808080u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = 0;
            for (int j = 0; j < 4; ++j) {  // inf / scale would saturate to 448: make it the NaN that it stands for
                const float x = v.value(4 * i + j), t = fabsf(x) < INFINITY ? __fdiv_rn(x, scale) : __uint_as_float(0x7fc00000u);
                w[i] |= (uint32_t)__nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3) << (8 * j);
            }
        }
    }
    constexpr int kPer = Values<T>::kPer;
#pragma unroll
    for (int j = 0; j < Values<T>::kPieces; ++j) {
        const int c = Values<T>::column(b, l, j);
        if (vec && c + kPer <= cols) {
            if constexpr (kPer == 8) *reinterpret_cast<uint2 *>(row + c) = make_uint2(w[2 * j], w[2 * j + 1]);
            else *reinterpret_cast<uint32_t *>(row + c) = w[j];
            continue;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (c + i < cols) row[c + i] = (uint8_t)(w[(kPer * j + i) >> 2] >> (8 * (i & 3)));
    }
}

// 1 x 128 blocks: four lanes per block, a warp takes p.steps times eight blocks of a row, the next ones loaded before
// these are used.
template <class T>
__global__ void __launch_bounds__(256) k_quant_rows(const QuantParams p) {
    const int l = threadIdx.x & 3, sub = (threadIdx.x >> 2) & 7;
    const int nb = (p.cols + kScaleBlock - 1) / kScaleBlock;
    const uint32_t segs = (nb + 8 * p.steps - 1) / (8 * p.steps);
    const int64_t items = (int64_t)p.matrices * p.rows * segs, step = ((int64_t)gridDim.x * blockDim.x) >> 5;
    for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < items; i += step) {
        const int64_t mr = items < (1ll << 32) ? (uint32_t)i / segs : i / segs;
        const int b0 = (int)(i - mr * segs) * 8 * p.steps + sub, b1 = min(nb, b0 - sub + 8 * p.steps);
        int64_t r = mr, mat = 0;
        if (p.matrices > 1) mat = mr / p.rows, r = mr - mat * p.rows;
        const T *x = static_cast<const T *>(p.x) + mat * p.x_stride + r * p.ldx;
        uint8_t *q = p.q + mat * p.q_stride + r * p.ldq;
        float *s = p.scales + mat * p.s_stride + r * p.s_row;
        Values<T> v, next;
        next.load(x, b0, l, p.cols, p.vec);
        for (int b = b0; b - sub < b1; b += 8) {  // whole warps: lanes behind the last block hold zeros
            v = next;
            if (b - sub + 8 < b1) next.load(x, b + 8, l, p.cols, p.vec);
            uint32_t m = v.top();
            m = Values<T>::larger(m, __shfl_xor_sync(kFull, m, 2));
            m = Values<T>::one(Values<T>::larger(m, __shfl_xor_sync(kFull, m, 1)));
            const bool fine = m < Values<T>::kInf;
            if (__any_sync(kFull, !fine)) {
                m = v.finite();
                m = max(m, __shfl_xor_sync(kFull, m, 2));
                m = max(m, __shfl_xor_sync(kFull, m, 1));
            }
            if (b >= b1) continue;
            const float amax = Values<T>::as_float(m), scale = block_scale(amax);
            store_codes(q, b, l, p.cols, p.vec, v, scale, fine && amax >= kPlain);
            if (l == 0) s[b * p.s_blk] = scale;
        }
    }
}

// 128 x 128 blocks: one CTA per block; the block stays in registers between its maximum and its codes.  bf16 8 x 5760 x 2880:
// 92 us, 4.3 TB/s (66 % of a copy's rate); bound by issue (64 % active) and, at half the warps, by the two barriers a block.
template <class T>
__global__ void __launch_bounds__(256) k_quant_blocks(const QuantParams p) {
    __shared__ uint32_t part[2][8];
    const int64_t nbr = (p.rows + kScaleBlock - 1) / kScaleBlock;
    const int nb = (p.cols + kScaleBlock - 1) / kScaleBlock;
    const int64_t blocks = (int64_t)p.matrices * nbr * nb;
    for (int64_t i = blockIdx.x; i < blocks; i += gridDim.x) {
        const int64_t mbr = i / nb, mat = mbr / nbr, br = mbr - mat * nbr;
        const int b = (int)(i - mbr * nb), l = threadIdx.x & 3;
        const int64_t r0 = br * kScaleBlock + (threadIdx.x >> 2);
        Values<T> v[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t r = r0 + 64 * j;
            v[j].load(static_cast<const T *>(p.x) + mat * p.x_stride + r * p.ldx, b, l, r < p.rows ? p.cols : 0, p.vec);
        }
        uint32_t m = 0, f = 0;  // over all values, over the finite ones
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            m = max(m, Values<T>::one(v[j].top()));
            f = max(f, v[j].finite());
        }
        m = __reduce_max_sync(kFull, m);
        f = __reduce_max_sync(kFull, f);
        __syncthreads();  // the previous block's readers are done with part
        if ((threadIdx.x & 31) == 0) part[0][threadIdx.x >> 5] = m, part[1][threadIdx.x >> 5] = f;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) m = max(m, part[0][w]), f = max(f, part[1][w]);
        const float amax = Values<T>::as_float(f), scale = block_scale(amax);
        const bool plain = m < Values<T>::kInf && amax >= kPlain;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int64_t r = r0 + 64 * j;
            if (r < p.rows) store_codes(p.q + mat * p.q_stride + r * p.ldq, b, l, p.cols, p.vec, v[j], scale, plain);
        }
        if (threadIdx.x == 0) p.scales[mat * p.s_stride + br * p.s_row + b * p.s_blk] = scale;
    }
}

template <class T>
void launch_quant(QuantParams p, int block_rows, int sms, cudaStream_t s) {
    const int64_t nb = (p.cols + kScaleBlock - 1) / kScaleBlock, rows = (int64_t)p.matrices * p.rows;
    if (block_rows == 1) {
        // eight blocks a warp where that leaves warps idle, otherwise up to 32
        p.steps = 1;
        while (p.steps < 4 && rows * ((nb + 16 * p.steps - 1) / (16 * p.steps)) >= 64 * sms) p.steps *= 2;
        const int64_t items = rows * ((nb + 8 * p.steps - 1) / (8 * p.steps));
        k_quant_rows<T><<<(unsigned)std::min<int64_t>((items + 7) / 8, 64 * sms), 256, 0, s>>>(p);
    } else {
        const int64_t blocks = (int64_t)p.matrices * ((p.rows + kScaleBlock - 1) / kScaleBlock) * nb;
        k_quant_blocks<T><<<(unsigned)std::min<int64_t>(blocks, 64 * sms), 256, 0, s>>>(p);
    }
}

// Whether an array's strides give each element an address of its own: from the shortest on, each spans the shorter ones.
bool distinct(std::array<std::pair<int64_t, int64_t>, 3> dims) {  // (stride, length)
    std::sort(dims.begin(), dims.end());
    int64_t span = 0;  // from the first element to the last
    for (const auto &[stride, length] : dims) {
        if (length <= 1) continue;
        if (stride <= span) return false;
        span += (length - 1) * stride;
    }
    return true;
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
    const int64_t br = (rows + block_rows - 1) / block_rows, bc = (cols + kScaleBlock - 1) / kScaleBlock;
    if (!distinct({{{s_stride, matrices}, {s_row, br}, {s_blk, bc}}})) return fail(UMSX_EINVAL, "the strides of the scales give two blocks one address");
    const Region rx = region(x, x_dtype == UMSX_DTYPE_F32 ? 4 : 2, cols, rows, ldx, matrices, x_stride),
                 rq = region(q, 1, cols, rows, ldq, matrices, q_stride),
                 rs = region(scales, 4, (matrices - 1) * s_stride + (br - 1) * s_row + (bc - 1) * s_blk + 1, 1, 0);
    if (overlap(rq, rx) || overlap(rs, rx) || overlap(rs, rq)) return fail(UMSX_EINVAL, "an output overlaps the input or the other output");
    if (reinterpret_cast<uintptr_t>(x) % (x_dtype == UMSX_DTYPE_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(scales) % 4)
        return fail(UMSX_EINVAL, "a buffer is not aligned to its elements");
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
    (void)cudaGetLastError();  // an earlier call's error is not this launch's
    if (x_dtype == UMSX_DTYPE_F32) launch_quant<float>(p, block_rows, sms, s);
    else if (x_dtype == UMSX_DTYPE_BF16) launch_quant<__nv_bfloat16>(p, block_rows, sms, s);
    else launch_quant<__half>(p, block_rows, sms, s);
    record_launches(1);
    e = cudaGetLastError();
    if (e != cudaSuccess) return fail(UMSX_EDEVICE, std::string("quantize launch: ") + cudaGetErrorString(e));
    return UMSX_OK;
}
