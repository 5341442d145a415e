// 8-bit float matrices with a scale for each block of 128: the quantiser and the product.
#include <cuda_fp8.h>

#include <algorithm>
#include <climits>

#include "fp8_gemm.cuh"
#include "kernels.h"

namespace dabnn {

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

static bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// -------------------------------------------------------------------------------------------------
// The product: which tile (its columns: 16, 32, 64 activation rows or 128, 256 weight rows), how many CTAs share one.
static int f8_columns(int m, int n) {
    if (m <= 16) return 16;
    if (m <= 32) return 32;
    if (m <= 64 || ((long long)m + 127) / 128 * ((n + 127) / 128) < sm_count()) return 64;
    return ((long long)m + 255) / 256 * ((n + 255) / 256) < sm_count() / 2 ? 128 : 256;
}
static int f8_splits(long long ntiles, int nkb) {
    int s = 1;
    while (s < F8_MAX_SPLIT && 2 * s * ntiles <= 2 * sm_count() && 4 * s <= nkb) s *= 2;
    return s;
}

template <int NT, bool SPLIT, typename T>
static int f8_launch(const Fp8Params& p, int splits, const CUtensorMap& lane_map, const CUtensorMap& col_map, cudaStream_t stream) {
    using Cfg = Fp8Cfg<NT>;
    auto kern = fp8_gemm_kernel<NT, SPLIT, T>;
    static thread_local int ready_device = -1, resident = 0;   // teams that run at once
    int dev = 0;
    DABNN_CUDA_OK(cudaGetDevice(&dev));
    if (dev != ready_device) {
        DABNN_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    }
    cudaLaunchConfig_t cfg{};
    const int team = SPLIT ? splits : Cfg::PAIR ? 2 : 1;
    cfg.blockDim = dim3(Cfg::THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    int n = 0;
    if (team > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = team;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    cfg.numAttrs = n;
    cfg.gridDim = dim3(team);
    if (dev != ready_device) {
        if (Cfg::PAIR) DABNN_CUDA_OK(cudaOccupancyMaxActiveClusters(&resident, kern, &cfg));
        else resident = sm_count() * Cfg::CTAS_PER_SM;
        DABNN_REQUIRE(resident > 0, DABNN_ERR_CUDA, "fp8_gemm: the device runs no pair of CTAs");
        ready_device = dev;
    }
    cfg.gridDim = dim3((SPLIT ? p.ntiles : std::min(p.ntiles, resident)) * team);
    if (g_overlap_launches) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    cfg.numAttrs = n;
    DABNN_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, p, splits, lane_map, col_map));
    return DABNN_OK;
}

template <typename T>
static int f8_gemm(Fp8Params p, const uint8_t* a, long long lda, const uint8_t* b, long long ldb, int k, cudaStream_t stream) {
    const int nt = f8_columns(p.M, p.N), rows_m = nt <= 64 ? nt : nt == 128 ? 128 : 256, rows_n = nt <= 64 ? 128 : nt;
    p.tiles_n = (p.N + rows_n - 1) / rows_n;
    const long long ntiles = (long long)p.tiles_n * ((p.M + rows_m - 1) / rows_m);
    DABNN_REQUIRE(ntiles < (1ll << 30), DABNN_ERR_SHAPE, "fp8_gemm: too many outputs");
    p.ntiles = (int)ntiles;
    p.nkb = (k + F8_BLOCK - 1) / F8_BLOCK;
    p.vec = aligned_to(p.c, 32) && (p.M == 1 || p.ldc * sizeof(T) % 32 == 0);
    CUtensorMap w_map{}, x_map{};
    if (k > 0) {   // a single row's pitch is of no account, but the descriptor wants one
        const unsigned long long whole = ((unsigned long long)k + 15) / 16 * 16;
        const unsigned long long wdims[2] = {(unsigned long long)k, (unsigned long long)p.N}, wpitch[1] = {p.N > 1 ? (unsigned long long)ldb : whole};
        const unsigned long long xdims[2] = {(unsigned long long)k, (unsigned long long)p.M}, xpitch[1] = {p.M > 1 ? (unsigned long long)lda : whole};
        const unsigned wbox[2] = {F8_BLOCK, (unsigned)std::min(rows_n, 128)}, xbox[2] = {F8_BLOCK, (unsigned)std::min(rows_m, 128)};   // (a pair loads halves)
        DABNN_REQUIRE(make_u8_tensor_map(&w_map, b, 2, wdims, wpitch, wbox) && make_u8_tensor_map(&x_map, a, 2, xdims, xpitch, xbox), DABNN_ERR_CUDA,
                      "fp8_gemm: cannot make a tensor map (no CUDA device, or a pitch beyond 2^40)");
    }
    const int splits = nt <= 64 ? f8_splits(ntiles, p.nkb) : 1;
    switch (nt) {
        case 16: return splits > 1 ? f8_launch<16, true, T>(p, splits, w_map, x_map, stream) : f8_launch<16, false, T>(p, 1, w_map, x_map, stream);
        case 32: return splits > 1 ? f8_launch<32, true, T>(p, splits, w_map, x_map, stream) : f8_launch<32, false, T>(p, 1, w_map, x_map, stream);
        case 64: return splits > 1 ? f8_launch<64, true, T>(p, splits, w_map, x_map, stream) : f8_launch<64, false, T>(p, 1, w_map, x_map, stream);
        case 128: return f8_launch<128, false, T>(p, 1, x_map, w_map, stream);
        default: return f8_launch<256, false, T>(p, 1, x_map, w_map, stream);
    }
}

int fp8_status_word(int** addr) {
    DABNN_CUDA_OK(cudaGetSymbolAddress(reinterpret_cast<void**>(addr), g_fp8_status));
    return DABNN_OK;
}

}  // namespace dabnn

using namespace dabnn;

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
    DABNN_REQUIRE(m < INT_MAX - 512 && n < INT_MAX - 512 && k < INT_MAX - 512, DABNN_ERR_SHAPE, "fp8_gemm: too large a matrix");
    const cudaStream_t stream = static_cast<cudaStream_t>(s);
    const Fp8Params p{a_scales, b_scales, bias, as_row, as_block, bs_row, bs_block, ldc, c, m, n};
    if (c_type == DABNN_F32) return f8_gemm<float>(p, a, lda, b, ldb, k, stream);
    if (c_type == DABNN_F16) return f8_gemm<__half>(p, a, lda, b, ldb, k, stream);
    return f8_gemm<__nv_bfloat16>(p, a, lda, b, ldb, k, stream);
}
