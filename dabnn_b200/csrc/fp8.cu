// 8-bit float matrices with a scale for each block of 128: the quantiser and the product.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "scalar_types.cuh"

namespace dabnn {

constexpr int F8_BLOCK = 128;

// The scale of a block whose largest finite magnitude has the bits `top` (fp32): the least power of two 2^e, e >= -126, with
// top <= 448 * 2^e, 448 = 1.75 * 2^8 being the largest e4m3 value.  As bits; the reciprocal's bits are (254 << 23) - scale.
__device__ __forceinline__ uint32_t f8_scale_bits(uint32_t top) {
    const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)(max(e, -126) + 127) << 23;
}

// one CTA per block of block_rows x 128
template <typename T>
__global__ void __launch_bounds__(128) fp8_quantize_kernel(const T* __restrict__ in, const long long ld_in, uint8_t* __restrict__ out, const long long ld_out,
                                                           float* __restrict__ scales, const long long scale_row, const long long scale_block,
                                                           const int rows, const int k, const int block_rows) {
    __shared__ uint32_t top_s;
    const int kb = blockIdx.y, col = kb * F8_BLOCK + threadIdx.x;
    const long long r0 = (long long)blockIdx.x * block_rows;
    const int nr = (int)min((long long)block_rows, rows - r0);
    if (threadIdx.x == 0) top_s = 0;
    __syncthreads();
    uint32_t top = 0;
    for (int r = 0; r < nr && col < k; r++) {
        const uint32_t a = __float_as_uint(to_f32(in[(r0 + r) * ld_in + col])) & 0x7fffffffu;
        if (a < 0x7f800000u) top = max(top, a);
    }
    atomicMax(&top_s, top);
    __syncthreads();
    const uint32_t scale = f8_scale_bits(top_s);
    const float inv = __uint_as_float((254u << 23) - scale);
    if (threadIdx.x == 0) scales[blockIdx.x * scale_row + kb * scale_block] = __uint_as_float(scale);
    for (int r = 0; r < nr && col < k; r++) {
        const float x = to_f32(in[(r0 + r) * ld_in + col]);
        const bool finite = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
        out[(r0 + r) * ld_out + col] = finite ? __nv_cvt_float_to_fp8(x * inv, __NV_SATFINITE, __NV_E4M3) : 0x7f;
    }
}

__device__ __forceinline__ float f8_to_f32(uint8_t v) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3))); }

// 16 x 16 outputs per CTA, one block of K at a time
template <typename T>
__global__ void __launch_bounds__(256) fp8_gemm_kernel(const uint8_t* __restrict__ a, const long long lda, const float* __restrict__ as, const long long as_row,
                                                       const long long as_block, const uint8_t* __restrict__ b, const long long ldb,
                                                       const float* __restrict__ bs, const long long bs_row, const long long bs_block,
                                                       const float* __restrict__ bias, T* __restrict__ c, const long long ldc, const int M, const int N, const int K) {
    __shared__ float sa[16][F8_BLOCK + 1], sb[16][F8_BLOCK + 1];
    const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
    const long long m0 = (long long)blockIdx.y * 16, n0 = (long long)blockIdx.x * 16;
    float acc = 0.f;
    for (int kb = 0; kb * F8_BLOCK < K; kb++) {
        for (int i = threadIdx.x; i < 16 * F8_BLOCK; i += 256) {
            const int r = i >> 7, k = kb * F8_BLOCK + (i & 127);
            sa[r][i & 127] = k < K && m0 + r < M ? f8_to_f32(a[(m0 + r) * lda + k]) : 0.f;
            sb[r][i & 127] = k < K && n0 + r < N ? f8_to_f32(b[(n0 + r) * ldb + k]) : 0.f;
        }
        __syncthreads();
        float part = 0.f;
        for (int k = 0; k < F8_BLOCK; k++) part = fmaf(sa[ty][k], sb[tx][k], part);
        if (m0 + ty < M && n0 + tx < N) acc = fmaf(as[(m0 + ty) * as_row + kb * as_block] * bs[((n0 + tx) >> 7) * bs_row + kb * bs_block], part, acc);
        __syncthreads();
    }
    if (m0 + ty < M && n0 + tx < N) c[(m0 + ty) * ldc + n0 + tx] = from_f32<T>(acc + (bias ? bias[n0 + tx] : 0.f));
}

}  // namespace dabnn

using namespace dabnn;

static bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

extern "C" int dabnn_fp8_quantize(const void* in, int in_type, long long ld_in, uint8_t* out, long long ld_out, float* scales, long long scale_row,
                                  long long scale_block, int rows, int k, int block_rows, dabnn_stream_t s) {
    DABNN_REQUIRE(in_type >= DABNN_F32 && in_type <= DABNN_BF16, DABNN_ERR_ARG, "fp8_quantize: unknown input type");
    DABNN_REQUIRE(rows >= 0 && k >= 0, DABNN_ERR_ARG, "fp8_quantize: bad dims");
    DABNN_REQUIRE(block_rows == 1 || block_rows == F8_BLOCK, DABNN_ERR_ARG, "fp8_quantize: a scale's block has 1 or 128 rows");
    if (rows == 0 || k == 0) return DABNN_OK;
    DABNN_REQUIRE(in && out && scales, DABNN_ERR_ARG, "fp8_quantize: null pointer");
    DABNN_REQUIRE(ld_in >= k && ld_out >= k, DABNN_ERR_SHAPE, "fp8_quantize: a row pitch is below k");
    DABNN_REQUIRE(aligned_to(in, in_type == DABNN_F32 ? 4 : 2) && aligned_to(scales, 4), DABNN_ERR_ARG, "fp8_quantize: misaligned pointer");
    const cudaStream_t stream = static_cast<cudaStream_t>(s);
    const dim3 grid((rows + block_rows - 1) / block_rows, (k + F8_BLOCK - 1) / F8_BLOCK);
    auto launch = [&](auto tag) {
        using T = decltype(tag);
        fp8_quantize_kernel<T><<<grid, 128, 0, stream>>>(static_cast<const T*>(in), ld_in, out, ld_out, scales, scale_row, scale_block, rows, k, block_rows);
    };
    if (in_type == DABNN_F32) launch(float{});
    else if (in_type == DABNN_F16) launch(__half{});
    else launch(__nv_bfloat16{});
    return check_launch("fp8_quantize_kernel");
}

extern "C" int dabnn_fp8_gemm(const uint8_t* a, long long lda, const float* a_scales, long long as_row, long long as_block, const uint8_t* b,
                              long long ldb, const float* b_scales, long long bs_row, long long bs_block, const float* bias, void* c, int c_type,
                              long long ldc, int m, int n, int k, dabnn_stream_t s) {
    DABNN_REQUIRE(c_type >= DABNN_F32 && c_type <= DABNN_BF16, DABNN_ERR_ARG, "fp8_gemm: unknown output type");
    DABNN_REQUIRE(m >= 0 && n >= 0 && k >= 0, DABNN_ERR_ARG, "fp8_gemm: bad dims");
    if (m == 0 || n == 0) return DABNN_OK;
    DABNN_REQUIRE(c && (k == 0 || (a && b && a_scales && b_scales)), DABNN_ERR_ARG, "fp8_gemm: null pointer");
    DABNN_REQUIRE((lda >= k || m == 1) && (ldb >= k || n == 1) && (ldc >= n || m == 1), DABNN_ERR_SHAPE, "fp8_gemm: a row pitch is below the row");
    DABNN_REQUIRE(k == 0 || (aligned_to(a, 16) && aligned_to(b, 16) && (m == 1 || lda % 16 == 0) && (n == 1 || ldb % 16 == 0)), DABNN_ERR_SHAPE,
                  "fp8_gemm: rows of a and b must begin on 16-byte boundaries");
    DABNN_REQUIRE(aligned_to(c, c_type == DABNN_F32 ? 4 : 2) && aligned_to(a_scales, 4) && aligned_to(b_scales, 4) && aligned_to(bias, 4), DABNN_ERR_ARG,
                  "fp8_gemm: misaligned pointer");
    const cudaStream_t stream = static_cast<cudaStream_t>(s);
    const dim3 grid((n + 15) / 16, (m + 15) / 16);
    auto launch = [&](auto tag) {
        using T = decltype(tag);
        fp8_gemm_kernel<T><<<grid, 256, 0, stream>>>(a, lda, a_scales, as_row, as_block, b, ldb, b_scales, bs_row, bs_block, bias, static_cast<T*>(c), ldc, m, n, k);
    };
    if (c_type == DABNN_F32) launch(float{});
    else if (c_type == DABNN_F16) launch(__half{});
    else launch(__nv_bfloat16{});
    return check_launch("fp8_gemm_kernel");
}
