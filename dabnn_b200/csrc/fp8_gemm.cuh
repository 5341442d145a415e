// Product of 8-bit float matrices with a scale for each block of 128, on tcgen05.mma kind::f8f6f4:
//
//   c[i][j] = sum over blocks q of 128 along K of as(i, q) bs(j / 128, q) sum_{h in q} a[i][h] b[j][h]   (+ bias[j])
//
// The weights b are the M = 128 operand and the activations a the N operand (16 .. 256 columns), so an accumulator holds 128
// outputs (lanes) of each activation row (columns):
//   * a tile's 128 weight rows are one block of scales: bs is one number per tile and block of K, as one per column;
//   * few activation rows fill narrow instructions instead of an eighth of a wide one;
//   * a warp's 32 lanes hold 32 neighbouring outputs of a row, so results go to memory straight from registers, coalesced.
// A block of K is four instructions into one of two accumulators.  The epilogue warps read it while the other one fills,
// multiply by as * bs and add to fp32 sums in their registers (one fused multiply-add per value and block): the tensor core's
// own additions never run over more than 128 products.
//
// Warps: 0 TMA loads (128-byte-swizzled boxes of 128 bytes of K; rows and bytes beyond the matrices read as zeros), 1 MMA
// issue, then the epilogue.  Few rows leave few tiles: a cluster then shares a tile, each CTA with a run of K's blocks, and
// adds up the parts over distributed shared memory in a fixed order.
//
// Every wait on an mbarrier is bounded; one that gives up records a code (51 loader, 52 / 53 MMA warp waiting for an
// accumulator / a stage, 54 epilogue), raises the CTA's abort flag, and the CTA frees its tensor memory and returns.
#pragma once
#include "bcontract_tc5.cuh"
#include "scalar_types.cuh"

namespace dabnn {

constexpr int F8_BLOCK = 128;
constexpr int F8_W_BYTES = 128 * F8_BLOCK;            // the weights of a stage
constexpr int F8_MAX_SPLIT = 8;

__device__ int g_fp8_status;   // 0 = ok; 51 - 54 as above

struct Fp8Params {
    const float *as, *bs, *bias;
    long long as_row, as_block, bs_row, bs_block, ldc;
    void* c;
    int M, N, nkb;                                     // activation rows, weight rows, blocks of K
    int tiles_n, ntiles;                               // tiles of 128 weight rows; all tiles
};

template <int NT>
struct Fp8Cfg {                                        // NT: activation rows of a tile
    static constexpr int EPI_WARPS = NT <= 64 ? 4 : 8;
    static constexpr int THREADS = 64 + EPI_WARPS * 32;
    static constexpr int COLS = NT / (EPI_WARPS / 4);  // accumulator columns of an epilogue warp
    static constexpr int STAGE_BYTES = F8_W_BYTES + NT * F8_BLOCK;
    static constexpr int STAGES = NT <= 32 ? 5 : NT == 64 ? 4 : NT == 128 ? 6 : 4;
    static constexpr int CTAS_PER_SM = NT <= 64 ? 2 : 1;
    static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES;
};

__device__ __forceinline__ void f8_mma(uint32_t d_tmem, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accum) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}\n"
                 ::"r"(d_tmem), "l"(ad), "l"(bd), "r"(idesc), "r"(accum), "r"(0), "r"(0), "r"(0), "r"(0) : "memory");
}
// K-major SWIZZLE_128B: rows of 128 bytes, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t f8_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void f8_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void f8_tmem_ld16(uint32_t (&v)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(at));
}
__device__ __forceinline__ void f8_tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float f8_ld_cluster(uint32_t addr, int rank) {
    uint32_t remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
    return v;
}
__device__ __forceinline__ void f8_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// SPLIT: the CTAs of a cluster share one tile (the grid then has one cluster per tile); otherwise a CTA walks the tiles
template <int NT, bool SPLIT, typename T>
__global__ void __launch_bounds__(Fp8Cfg<NT>::THREADS, Fp8Cfg<NT>::CTAS_PER_SM)
    fp8_gemm_kernel(const Fp8Params p, const int splits, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map) {
    using Cfg = Fp8Cfg<NT>;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) uint64_t bar_full[Cfg::STAGES], bar_empty[Cfg::STAGES], bar_acc_full[2], bar_acc_empty[2];
    __shared__ __align__(16) float scale_s[Cfg::EPI_WARPS][Cfg::COLS];
    __shared__ uint32_t tmem_base_s;
    __shared__ int s_abort;

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const uint32_t stage0 = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    const volatile int* abort_flag = &s_abort;
    constexpr int TMEM_COLS = 2 * NT;
    const int rank = SPLIT ? (int)blockIdx.x % splits : 0, first = SPLIT ? (int)blockIdx.x / splits : (int)blockIdx.x, step = SPLIT ? p.ntiles : (int)gridDim.x;
    const int kb0 = SPLIT ? (int)((long long)p.nkb * rank / splits) : 0, kb1 = SPLIT ? (int)((long long)p.nkb * (rank + 1) / splits) : p.nkb;

    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < Cfg::STAGES; i++) { mbar_init(&bar_full[i], 1); mbar_init(&bar_empty[i], 1); }
        for (int i = 0; i < 2; i++) { mbar_init(&bar_acc_full[i], 1); mbar_init(&bar_acc_empty[i], Cfg::EPI_WARPS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::);
        s_abort = 0;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = tmem_base_s;
    grid_launch_dependents();
    grid_dependency_wait();

    if (warp == 0) {
        // =========================== TMA loads: one lane ===========================
        if (elect_lane()) {
            uint32_t s = 0, use = 0;
            bool ok = true;
            for (int tile = first; tile < p.ntiles && ok; tile += step) {
                const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
                for (int kb = kb0; kb < kb1; kb++) {
                    if (use >= 1 && !mbar_wait(&bar_empty[s], (use - 1) & 1, abort_flag)) {
                        atomicCAS(&g_fp8_status, 0, 51);
                        s_abort = 1;
                        ok = false;
                        break;
                    }
                    const uint32_t bar = smem_u32(&bar_full[s]), at = stage0 + s * Cfg::STAGE_BYTES;
                    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(Cfg::STAGE_BYTES) : "memory");
                    f8_load(at, &w_map, kb * F8_BLOCK, tn * 128, bar);
                    f8_load(at + F8_W_BYTES, &x_map, kb * F8_BLOCK, tm * NT, bar);
                    if (++s == Cfg::STAGES) { s = 0; use++; }
                }
            }
        }
    } else if (warp == 1) {
        // =========================== MMA issue: the whole warp walks, one lane issues ===========================
        const bool leader = elect_lane();
        constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);   // D f32, A = B = e4m3, K-major
        uint32_t s = 0, par = 0;
        bool ok = true;
        int i = 0;   // blocks so far
        for (int tile = first; tile < p.ntiles && ok; tile += step)
            for (int kb = kb0; kb < kb1; kb++, i++) {
                const int acc = i & 1;
                if (i >= 2 && !mbar_wait_warp(&bar_acc_empty[acc], ((i >> 1) - 1) & 1, abort_flag)) {
                    atomicCAS(&g_fp8_status, 0, 52);
                    s_abort = 1;
                    ok = false;
                    break;
                }
                if (!mbar_wait_warp(&bar_full[s], par, abort_flag)) {
                    atomicCAS(&g_fp8_status, 0, 53);
                    s_abort = 1;
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t w = f8_desc(stage0 + s * Cfg::STAGE_BYTES), x = w + (F8_W_BYTES >> 4);
                if (leader) {
#pragma unroll
                    for (int j = 0; j < F8_BLOCK / 32; j++) f8_mma(tmem_base + acc * NT, w + 2 * j, x + 2 * j, idesc, j > 0);
                    umma_commit(&bar_empty[s]);
                    umma_commit(&bar_acc_full[acc]);
                }
                __syncwarp();
                if (++s == Cfg::STAGES) { s = 0; par ^= 1u; }
            }
    } else {
        // =========================== epilogue ===========================
        const int ew = warp - 2, quarter = warp & 3, col0 = (ew >> 2) * Cfg::COLS;   // TMEM lane quarter of a warp = warp % 4
        const uint32_t t_mine = tmem_base + ((uint32_t)(quarter * 32) << 16) + col0;
        float* const my_scales = scale_s[ew];
        constexpr int SC = (Cfg::COLS + 31) / 32;      // scales that a lane fetches
        int i = 0;
        bool ok = true;
        for (int tile = first; tile < p.ntiles && ok; tile += step) {
            const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
            const int m0 = tm * NT + col0;
            float sum[Cfg::COLS];
#pragma unroll
            for (int e = 0; e < Cfg::COLS; e++) sum[e] = 0.f;
            // the scales of a block, fetched two blocks ahead
            float next[2][SC], wnext[2];
            auto fetch = [&](int kb, float (&v)[SC], float& w) {
                w = kb < kb1 ? __ldg(p.bs + tn * p.bs_row + kb * p.bs_block) : 0.f;
#pragma unroll
                for (int e = 0; e < SC; e++) {
                    const int m = m0 + e * 32 + lane;
                    v[e] = kb < kb1 && m < p.M && e * 32 + lane < Cfg::COLS ? __ldg(p.as + m * p.as_row + kb * p.as_block) : 0.f;
                }
            };
            fetch(kb0, next[0], wnext[0]);
            fetch(kb0 + 1, next[1], wnext[1]);
            for (int kb = kb0; kb < kb1; kb++, i++) {
                __syncwarp();                          // the scales of the block before have been read
#pragma unroll
                for (int e = 0; e < SC; e++)
                    if (e * 32 + lane < Cfg::COLS) my_scales[e * 32 + lane] = next[0][e] * wnext[0];
#pragma unroll
                for (int e = 0; e < SC; e++) next[0][e] = next[1][e];
                wnext[0] = wnext[1];
                fetch(kb + 2, next[1], wnext[1]);
                __syncwarp();
                const int acc = i & 1;
                if (!mbar_wait_warp(&bar_acc_full[acc], (i >> 1) & 1, abort_flag)) {
                    atomicCAS(&g_fp8_status, 0, 54);
                    s_abort = 1;
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t v[2][16];
                f8_tmem_ld16(v[0], t_mine + acc * NT);
#pragma unroll
                for (int h = 0; h < Cfg::COLS / 16; h++) {
                    f8_tmem_wait();
                    if (h + 1 < Cfg::COLS / 16) {
                        f8_tmem_ld16(v[(h + 1) & 1], t_mine + acc * NT + (h + 1) * 16);
                    } else {                           // all of it is in registers: the MMA warp may reuse the accumulator
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar_acc_empty[acc]);
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 sc = lds128f(smem_u32(my_scales + h * 16 + e));
                        sum[h * 16 + e] = fmaf(__uint_as_float(v[h & 1][e]), sc.x, sum[h * 16 + e]);
                        sum[h * 16 + e + 1] = fmaf(__uint_as_float(v[h & 1][e + 1]), sc.y, sum[h * 16 + e + 1]);
                        sum[h * 16 + e + 2] = fmaf(__uint_as_float(v[h & 1][e + 2]), sc.z, sum[h * 16 + e + 2]);
                        sum[h * 16 + e + 3] = fmaf(__uint_as_float(v[h & 1][e + 3]), sc.w, sum[h * 16 + e + 3]);
                    }
                }
            }
            if (SPLIT) {
                // this CTA's part -> its shared memory (the ring is idle: its last loads have been multiplied), [column][output]
                const uint32_t part = stage0 + (uint32_t)((col0 * 128 + quarter * 32 + lane) * 4);
                if (ok)
#pragma unroll
                    for (int e = 0; e < Cfg::COLS; e++) asm volatile("st.shared.f32 [%0], %1;" ::"r"(part + e * 512), "f"(sum[e]) : "memory");
            } else if (ok) {
                const int n = tn * 128 + quarter * 32 + lane;
                if (n < p.N) {
                    const float bias = p.bias ? __ldg(p.bias + n) : 0.f;
                    T* out = static_cast<T*>(p.c) + m0 * p.ldc + n;
                    const int left = p.M - m0;
#pragma unroll
                    for (int e = 0; e < Cfg::COLS; e++) {
                        if (e < left) *out = from_f32<T>(sum[e] + bias);
                        out += p.ldc;
                    }
                }
            }
        }
    }

    if (SPLIT) {
        // every CTA of the cluster adds up an equal share of the tile's outputs over all parts, in the order of K
        __syncwarp();
        f8_cluster_sync();
        const int tile = first, tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
        const int total = min(NT, p.M - tm * NT) * 128;
        const int lo = (int)((long long)total * rank / splits), hi = (int)((long long)total * (rank + 1) / splits);
        for (int idx = lo + (int)threadIdx.x; idx < hi; idx += Cfg::THREADS) {
            float part[F8_MAX_SPLIT];
#pragma unroll
            for (int r = 0; r < F8_MAX_SPLIT; r++) part[r] = r < splits ? f8_ld_cluster(stage0 + idx * 4, r) : 0.f;
            float v = part[0];
#pragma unroll
            for (int r = 1; r < F8_MAX_SPLIT; r++) v += part[r];
            const int m = tm * NT + (idx >> 7), n = tn * 128 + (idx & 127);
            if (n < p.N) static_cast<T*>(p.c)[m * p.ldc + n] = from_f32<T>(v + (p.bias ? __ldg(p.bias + n) : 0.f));
        }
        f8_cluster_sync();                             // no CTA leaves while its part is being read
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
    }
}

}  // namespace dabnn
