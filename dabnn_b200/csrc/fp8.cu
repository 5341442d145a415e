// 8-bit float matrices with a scale for each block of 128: the quantiser and the product.
#include <cuda_fp8.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "fp8_gemm.cuh"
#include "kernels.h"

namespace dabnn {

// -------------------------------------------------------------------------------------------------
// The quantiser: per block, A = the largest finite |x|, scale = 2^e with e = max(-126, least integer with A <= 448 * 2^e),
// q = e4m3(x * 2^-e).  A power of two, so that the product is exact, the rounding to e4m3 the only one, and a block's values
// the same whichever order or width they are computed in; 8-bit floats lose nothing by it but the lowest binade.
// One pass over the data: a thread keeps its values in registers between the maximum and the conversion.  Bound by HBM: 8192 x
// 4096 bf16 by rows 17.7 us (5.8 TB/s), fp32 by blocks of 128 x 128 27.4 us (6.1 TB/s).

// the scale's bits from those of A (fp32), 448 = 1.75 * 2^8; the reciprocal's bits are (254 << 23) - scale
__device__ __forceinline__ uint32_t f8_scale_bits(uint32_t top) {
    const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return (uint32_t)(max(e, -126) + 127) << 23;
}

// 16 neighbouring values of a row, as they lie in memory
template <typename T>
struct Sixteen {
    static constexpr int WORDS = 16 * sizeof(T) / 4;
    uint32_t w[WORDS];

    __device__ __forceinline__ void load(const T* at, int left, bool vec) {   // left: values before the row's end; the others read as zeros
        if (left >= 16 && vec) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(at) + i / 4);
                w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i++) w[i] = 0;
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (i < left) {
                    if constexpr (sizeof(T) == 4) w[i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
                    else w[i / 2] |= (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(at) + i) << (i % 2 * 16);
                }
        }
    }
    __device__ __forceinline__ float value(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        else return __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (i % 2 * 16))));
    }
    // fp32 bits of the largest magnitude; an infinity or a NaN counts (>= 0x7f800000), or with finite = true is passed over
    __device__ __forceinline__ uint32_t top(bool finite) const {
        uint32_t m = 0;
        if (finite) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const uint32_t a = __float_as_uint(value(i)) & 0x7fffffffu;
                if (a < 0x7f800000u) m = max(m, a);
            }
            return m;
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < WORDS; i++) m = max(m, w[i] & 0x7fffffffu);
            return m;
        } else {   // two at a time: the order of magnitudes is that of their bits
#pragma unroll
            for (int i = 0; i < WORDS; i++) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            const unsigned short s = (unsigned short)max(m & 0xffffu, m >> 16);
            if constexpr (std::is_same_v<T, __nv_bfloat16>) return (uint32_t)s << 16;
            else return __float_as_uint(__half2float(__ushort_as_half(s)));
        }
    }
    __device__ __forceinline__ uint4 bytes(float inv, bool special) const {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(value(4 * i) * inv, value(4 * i + 1) * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(value(4 * i + 2) * inv, value(4 * i + 3) * inv), __NV_SATFINITE, __NV_E4M3);
            o[i] = lo | hi << 16;
        }
        if (special) {   // the conversion makes infinities the largest value
#pragma unroll
            for (int i = 0; i < 16; i++)
                if ((__float_as_uint(value(i)) & 0x7f800000u) == 0x7f800000u) o[i / 4] |= 0x7fu << (i % 4 * 8);
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
};

__device__ __forceinline__ void f8_store16(uint8_t* at, uint4 v, int left, bool vec) {
    if (left >= 16 && vec) {
        *reinterpret_cast<uint4*>(at) = v;
    } else {
        const uint32_t o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (i < left) at[i] = (uint8_t)(o[i / 4] >> (i % 4 * 8));
    }
}

// Blocks of one row.  Eight lanes a block, 16 values each; a warp has 2^kshift neighbouring blocks of 4 >> kshift rows (four
// of one row unless rows have fewer), a CTA eight warps' rows, whose scales it writes side by side.
constexpr int FQ_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(FQ_WARPS * 32) fp8_quantize_rows_kernel(const T* __restrict__ in, const long long ld_in, uint8_t* __restrict__ out,
                                                                          const long long ld_out, float* __restrict__ scales, const long long scale_row,
                                                                          const long long scale_block, const int rows, const int k, const int kshift,
                                                                          const int kgroups, const int vec_in, const int vec_out) {
    __shared__ float scale_s[FQ_WARPS * 4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, unit = lane >> 3;
    const int rows_warp = 4 >> kshift;
    const int kb = ((int)(blockIdx.x % kgroups) << kshift) + (unit & ((1 << kshift) - 1));
    const long long row0 = (long long)(blockIdx.x / kgroups) * (FQ_WARPS * rows_warp);
    const int r = warp * rows_warp + (unit >> kshift);
    const long long row = row0 + r;
    const int col = kb * F8_BLOCK + (lane & 7) * 16, left = row < rows ? k - col : 0;
    grid_dependency_wait();

    Sixteen<T> v;
    v.load(in + row * ld_in + col, left, vec_in);
    auto eight = [](uint32_t m) {
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
        return m;
    };
    uint32_t top = eight(v.top(false));
    const bool special = top >= 0x7f800000u;
    if (__any_sync(0xffffffffu, special)) top = eight(v.top(true));
    const uint32_t scale = f8_scale_bits(top);
    if (left > 0) f8_store16(out + row * ld_out + col, v.bytes(__uint_as_float((254u << 23) - scale), special), left, vec_out);
    if ((lane & 7) == 0) scale_s[(unit & ((1 << kshift) - 1)) * (FQ_WARPS * rows_warp) + r] = __uint_as_float(scale);
    __syncthreads();
    if (threadIdx.x < FQ_WARPS * 4) {
        const int b = threadIdx.x / (FQ_WARPS * rows_warp), rr = threadIdx.x % (FQ_WARPS * rows_warp);
        const long long q = ((long long)(blockIdx.x % kgroups) << kshift) + b;
        if (row0 + rr < rows && q * F8_BLOCK < k) scales[(row0 + rr) * scale_row + q * scale_block] = scale_s[threadIdx.x];
    }
}

// Blocks of 128 x 128, one CTA each: 64 values of a thread, of four rows
template <typename T>
__global__ void __launch_bounds__(256) fp8_quantize_blocks_kernel(const T* __restrict__ in, const long long ld_in, uint8_t* __restrict__ out, const long long ld_out,
                                                                  float* __restrict__ scales, const long long scale_row, const long long scale_block,
                                                                  const int rows, const int k, const int kblocks, const int vec_in, const int vec_out) {
    __shared__ uint32_t top_s[2][8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int kb = blockIdx.x % kblocks, rb = blockIdx.x / kblocks;
    const int col = kb * F8_BLOCK + (threadIdx.x & 7) * 16;
    const long long row = (long long)rb * F8_BLOCK + (threadIdx.x >> 3);
    grid_dependency_wait();

    Sixteen<T> v[4];
    int left[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        left[j] = row + j * 32 < rows ? k - col : 0;
        v[j].load(in + (row + j * 32) * ld_in + col, left[j], vec_in);
    }
    auto all = [&](bool finite, uint32_t* shared) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) m = max(m, v[j].top(finite));
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) shared[warp] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; i++) m = max(m, shared[i]);
        return m;
    };
    uint32_t top = all(false, top_s[0]);
    const bool special = top >= 0x7f800000u;
    if (special) top = all(true, top_s[1]);
    const uint32_t scale = f8_scale_bits(top);
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (left[j] > 0) f8_store16(out + (row + j * 32) * ld_out + col, v[j].bytes(__uint_as_float((254u << 23) - scale), special), left[j], vec_out);
    if (threadIdx.x == 0) scales[rb * scale_row + kb * scale_block] = __uint_as_float(scale);
}

static bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// -------------------------------------------------------------------------------------------------
// The product: which tile (its columns: 16, 32, 64 activation rows or 128, 256 weight rows).  More than 64 rows have tiles of
// 128 x 128 (512 x 4096 x 4096: 13.8 us, 17.5 in columns of 64), unless those are too few for a quarter of the SMs and K is
// better divided (100 x 1000 x 4096: 7.1 us in columns of 64, 13 in eight tiles of 128), or more than one for an SM: then pairs
// of CTAs have 256 x 256 (2048 x 2048 x 2048: 12.7 us, 14.7 in tiles of 128; 1024 x 1024 x 4096, 64 tiles: 17.3 and 13.1).
static int f8_columns(int m, int n) {
    if (m <= 16) return 16;
    if (m <= 32) return 32;
    const long long tiles = ((long long)m + 127) / 128 * ((n + 127) / 128);
    if (m <= 64 || 4 * tiles < sm_count()) return 64;
    return tiles <= sm_count() ? 128 : 256;
}
// How many CTAs share a tile: as many as find room, two to an SM, with four blocks of K or more each.  Joining their parts takes
// 2 us, what a CTA needs for about eight blocks: 8 x 1024 x 4096 4.5 us (10.7 undivided), 1 x 8192 x 4096 9.2 (13.0), 256 x 2048
// x 1024, of eight blocks, 7.5 divided and 5.6 undivided.
static int f8_splits(long long ntiles, int nkb) {
    int s = 1;
    if (nkb >= 12)
        while (s < F8_MAX_SPLIT && 2 * s * ntiles <= 2 * sm_count() && 8 * s <= nkb) s *= 2;
    return s;
}

template <int NT, bool SPLIT, typename T>
static int f8_launch(const Fp8Params& p, int splits, const CUtensorMap& lane_map, const CUtensorMap& col_map, const CUtensorMap& out_map,
                     cudaStream_t stream) {
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
    DABNN_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, p, splits, lane_map, col_map, out_map));
    return DABNN_OK;
}

static int g_give_up_group = -1, g_give_up_rank = 0;   // dabnn_debug_fp8_give_up

template <typename T>
static int f8_gemm(Fp8Params p, const uint8_t* a, long long lda, const uint8_t* b, long long ldb, int k, cudaStream_t stream) {
    const int nt = f8_columns(p.M, p.N), rows_m = nt <= 64 ? nt : nt == 128 ? 128 : 256, rows_n = nt <= 64 ? 128 : nt;
    p.tiles_n = (p.N + rows_n - 1) / rows_n;
    const long long ntiles = (long long)p.tiles_n * ((p.M + rows_m - 1) / rows_m);
    DABNN_REQUIRE(ntiles < (1ll << 30), DABNN_ERR_SHAPE, "fp8_gemm: too many outputs");
    p.ntiles = (int)ntiles;
    p.nkb = (k + F8_BLOCK - 1) / F8_BLOCK;
    p.give_up_group = g_give_up_group;
    p.give_up_rank = g_give_up_rank;
    CUtensorMap w_map{}, x_map{};
    if (k > 0) {   // a single row's pitch is of no account, but the descriptor wants one
        const unsigned long long whole = ((unsigned long long)k + 15) / 16 * 16;
        const unsigned long long wdims[2] = {(unsigned long long)k, (unsigned long long)p.N}, wpitch[1] = {p.N > 1 ? (unsigned long long)ldb : whole};
        const unsigned long long xdims[2] = {(unsigned long long)k, (unsigned long long)p.M}, xpitch[1] = {p.M > 1 ? (unsigned long long)lda : whole};
        const unsigned wbox[2] = {F8_BLOCK, (unsigned)std::min(rows_n, 128)}, xbox[2] = {F8_BLOCK, (unsigned)std::min(rows_m, 128)};   // (a pair loads halves)
        DABNN_REQUIRE(make_u8_tensor_map(&w_map, b, 2, wdims, wpitch, wbox) && make_u8_tensor_map(&x_map, a, 2, xdims, xpitch, xbox), DABNN_ERR_CUDA,
                      "fp8_gemm: cannot make a tensor map (no CUDA device, or a pitch beyond 2^40)");
    }
    CUtensorMap out_map{};
    p.tma_out = 0;   // (a tensor store writes whole 16 bytes: rows that end inside them would have what lies behind them overwritten)
    if (nt > 64 && aligned_to(p.c, 16) && p.ldc * sizeof(T) % 16 == 0 && p.N * sizeof(T) % 16 == 0 && (unsigned long long)p.ldc * sizeof(T) < (1ull << 40) && p.N * sizeof(T) < INT_MAX) {
        const unsigned long long dims[2] = {p.N * sizeof(T), (unsigned long long)p.M}, pitch[1] = {p.ldc * sizeof(T)};
        const unsigned box[2] = {128, 32};
        p.tma_out = make_u8_tensor_map(&out_map, static_cast<const unsigned char*>(p.c), 2, dims, pitch, box);
    }
    const int splits = nt <= 64 ? f8_splits(ntiles, p.nkb) : 1;
    switch (nt) {
        case 16: return splits > 1 ? f8_launch<16, true, T>(p, splits, w_map, x_map, out_map, stream) : f8_launch<16, false, T>(p, 1, w_map, x_map, out_map, stream);
        case 32: return splits > 1 ? f8_launch<32, true, T>(p, splits, w_map, x_map, out_map, stream) : f8_launch<32, false, T>(p, 1, w_map, x_map, out_map, stream);
        case 64: return splits > 1 ? f8_launch<64, true, T>(p, splits, w_map, x_map, out_map, stream) : f8_launch<64, false, T>(p, 1, w_map, x_map, out_map, stream);
        case 128: return f8_launch<128, false, T>(p, 1, x_map, w_map, out_map, stream);
        default: return f8_launch<256, false, T>(p, 1, x_map, w_map, out_map, stream);
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
    DABNN_REQUIRE(k < INT_MAX - 512, DABNN_ERR_SHAPE, "fp8_quantize: too large a matrix");
    DABNN_REQUIRE(block_rows == 1 || block_rows == F8_BLOCK, DABNN_ERR_ARG, "fp8_quantize: a scale's block has 1 or 128 rows");
    if (rows == 0 || k == 0) return DABNN_OK;
    DABNN_REQUIRE(in && out && scales, DABNN_ERR_ARG, "fp8_quantize: null pointer");
    DABNN_REQUIRE(ld_in >= k && ld_out >= k, DABNN_ERR_SHAPE, "fp8_quantize: a row pitch is below k");
    DABNN_REQUIRE(aligned_to(in, in_type == DABNN_F32 ? 4 : 2) && aligned_to(scales, 4), DABNN_ERR_ARG, "fp8_quantize: misaligned pointer");
    const cudaStream_t stream = static_cast<cudaStream_t>(s);
    auto launch = [&](auto tag) -> int {
        using T = decltype(tag);
        const T* x = static_cast<const T*>(in);
        const int vec_in = aligned_to(in, 16) && (rows == 1 || ld_in * sizeof(T) % 16 == 0), vec_out = aligned_to(out, 16) && (rows == 1 || ld_out % 16 == 0);
        const long long kblocks = ((long long)k + F8_BLOCK - 1) / F8_BLOCK;
        if (block_rows == 1) {
            const int kshift = kblocks >= 4 ? 2 : kblocks >= 2 ? 1 : 0, rows_cta = FQ_WARPS * (4 >> kshift);
            const long long kgroups = (kblocks + (1 << kshift) - 1) >> kshift, ctas = kgroups * (((long long)rows + rows_cta - 1) / rows_cta);
            DABNN_REQUIRE(ctas < INT_MAX, DABNN_ERR_SHAPE, "fp8_quantize: too large a matrix");
            DABNN_CUDA_OK(launch_overlapped(fp8_quantize_rows_kernel<T>, dim3((unsigned)ctas), dim3(FQ_WARPS * 32), 0, stream, x, ld_in, out, ld_out, scales, scale_row,
                                            scale_block, rows, k, kshift, (int)kgroups, vec_in, vec_out));
        } else {
            const long long ctas = kblocks * (((long long)rows + F8_BLOCK - 1) / F8_BLOCK);
            DABNN_REQUIRE(ctas < INT_MAX, DABNN_ERR_SHAPE, "fp8_quantize: too large a matrix");
            DABNN_CUDA_OK(launch_overlapped(fp8_quantize_blocks_kernel<T>, dim3((unsigned)ctas), dim3(256), 0, stream, x, ld_in, out, ld_out, scales, scale_row,
                                            scale_block, rows, k, (int)kblocks, vec_in, vec_out));
        }
        return DABNN_OK;
    };
    if (in_type == DABNN_F32) return launch(float{});
    if (in_type == DABNN_F16) return launch(__half{});
    return launch(__nv_bfloat16{});
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

extern "C" int dabnn_debug_fp8_give_up(int group, int rank) {
    DABNN_REQUIRE(group >= -1 && rank >= 0 && rank < F8_MAX_SPLIT, DABNN_ERR_ARG, "fp8_give_up: group must be -1 or more, rank 0 - 7");
    g_give_up_group = group;
    g_give_up_rank = rank;
    return DABNN_OK;
}
