// Product of 8-bit float matrices with a scale for each block of 128, on tcgen05.mma kind::f8f6f4:
//
//   c[i][j] = sum over blocks q of 128 along K of as(i, q) bs(j / 128, q) sum_{h in q} a[i][h] b[j][h]   (+ bias[j])
//
// A block of K is four instructions into one of two accumulators.  The epilogue warps read it while the other one fills,
// multiply by as * bs and add to fp32 sums in their registers (one fused multiply-add per value and block): the tensor core's
// own additions never run over more than 128 products.  Which operand takes the accumulator's 128 lanes and which its columns:
//   * many rows (FEW = false): lanes are activation rows, columns weight rows.  A thread has one as, a warp one bs per block:
//     the factor is one register, and reading the accumulator is all that passes through the shared-memory pipe.
//   * few rows (FEW): lanes are weight rows, columns 16 .. 64 activation rows, so that they fill a narrow instruction instead of
//     an eighth of a wide one.  The factors differ by column and come from shared memory.  A tile's 128 weight rows are one
//     block of scales.  Few rows leave few tiles: a cluster then shares a tile (SPLIT), each CTA with a run of K's blocks, and
//     adds up the parts over distributed shared memory in a fixed order.
//
// Warps: 0 TMA loads (128-byte-swizzled boxes of 128 bytes of K; rows and bytes beyond the matrices read as zeros), 1 MMA
// issue, 2 factors (scales of any strides, fetched four blocks at a time, their products left in a ring in shared memory: an
// epilogue that fetched its own waited for them, 8192 x 8192 x 4096 in 294 us), then the epilogue.
//
// What bounds it: at many rows the epilogue, whose trips to tensor memory take 735 cycles a block where the four instructions take
// 512 (8192 x 8192 x 4096 233 us, 2.4 PFLOP/s; in long runs the power cap, 277 us), in tiles of 128 x 128 L2 (512 x 4096 x 4096
// 14 us); at few rows HBM and set-up (1 x 16384 x 16384 49 us, 5.5 TB/s; 1 x 8192 x 4096 9.5 us, 3.5 TB/s).
//
// Every wait on an mbarrier is bounded; one that gives up records a code (51 loader, 52 / 53 MMA warp waiting for an
// accumulator / a stage, 54 epilogue, 55 factors) and raises the abort flag, in both CTAs of a pair, at which every role stops.
// What was started goes on without them: before the tensor memory is freed and a CTA leaves, the instructions issued so far and
// the loads still on their way, the other CTA's among them, are waited for, again with a limit.
#pragma once
#include "bcontract_tc5.cuh"
#include "scalar_types.cuh"

namespace dabnn {

constexpr int F8_BLOCK = 128;
constexpr int F8_L_BYTES = 128 * F8_BLOCK;            // the lane operand of a stage
constexpr int F8_MAX_SPLIT = 8;
constexpr int F8_OUT_BYTES = 32 * 128;                // where a warp leaves 32 rows of 128 bytes of the result for a tensor store
constexpr int F8_GROUPS = 2, F8_GROUP = 4;            // the ring of factors: groups of blocks, fetched and handed over together

__device__ int g_fp8_status;   // 0 = ok; 51 - 55 as above

struct Fp8Params {
    const float *as, *bs, *bias;
    long long as_row, as_block, bs_row, bs_block, ldc;
    void* c;
    int M, N, nkb;                                     // activation rows, weight rows, blocks of K
    int tiles_n, ntiles;                               // tiles along the weight rows; all tiles
    int tma_out;                                       // rows of c begin and end on 16-byte boundaries: tensor stores
    int give_up_group, give_up_rank;                   // dabnn_debug_fp8_give_up: which group of factors of which CTA of a team is held to have run out of time; none: -1
};

template <int NT>
struct Fp8Cfg {                                        // NT: columns of a tile
    static constexpr bool FEW = NT <= 64, PAIR = NT == 256;
    static constexpr int EPI_WARPS = FEW ? 4 : NT / 16;
    static constexpr int EPI_WARP0 = PAIR ? 4 : 3, THREADS = (EPI_WARP0 + EPI_WARPS) * 32;
    static constexpr int COLS = NT / (EPI_WARPS / 4);  // accumulator columns of an epilogue warp
    static constexpr int FACTORS = NT;                 // of a block: one per column / per lane and 128 columns
    static constexpr int COL_ROWS = PAIR ? NT / 2 : NT;  // rows of the column operand that a CTA loads
    static constexpr int STAGE_BYTES = F8_L_BYTES + COL_ROWS * F8_BLOCK;
    static constexpr int STAGES = NT <= 32 ? 5 : NT == 64 ? 4 : NT == 128 ? 5 : 4;
    static constexpr int OUT_BYTES = FEW ? 0 : EPI_WARPS * F8_OUT_BYTES;
    static constexpr int CTAS_PER_SM = FEW ? 2 : 1;
    static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + OUT_BYTES;
};

// A bounded wait of a whole warp (that no abort flag ends where it is null)
__device__ __forceinline__ bool f8_wait(uint32_t bar, uint32_t parity, const volatile int* abort_flag) {
    for (uint32_t it = 0; it < TC5_SPIN_LIMIT; it++) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred P1;\n\tmbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2;\n\tselp.b32 %0, 1, 0, P1;\n\t}"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (__all_sync(0xffffffffu, done)) return true;
        if (abort_flag && (it & 255u) == 255u && __any_sync(0xffffffffu, *abort_flag)) return false;
    }
    return false;
}
__device__ __forceinline__ void f8_arrive(uint32_t bar) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0];\n\t}" ::"r"(bar) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void f8_mma(uint32_t d_tmem, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accum) {
    if (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
                     ::"r"(d_tmem), "l"(ad), "l"(bd), "r"(idesc), "r"(accum) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
                     ::"r"(d_tmem), "l"(ad), "l"(bd), "r"(idesc), "r"(accum) : "memory");
}
// the barrier of this CTA, or those at the same place in both CTAs of the pair
template <bool PAIR>
__device__ __forceinline__ void f8_commit(uint32_t bar) {
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((unsigned short)3) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t f8_in_cta(uint32_t addr, int rank) {   // the same place in another CTA of the cluster
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(addr), "r"(rank));
    return there;
}
// (relaxed: what it follows are loads from tensor memory that have been waited for; a release across the cluster takes hundreds of cycles)
__device__ __forceinline__ void f8_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// K-major SWIZZLE_128B: rows of 128 bytes, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t f8_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
template <bool PAIR>
__device__ __forceinline__ void f8_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if (PAIR)   // the barrier may be the other CTA's
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void f8_tmem_ld16(uint32_t (&v)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                   "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(at));
}
// two fused multiply-adds: (x, y) += (a, b) * (sx, sy)
__device__ __forceinline__ void f8_fma2(float2& sum, uint32_t a, uint32_t b, float sx, float sy) {
    asm("{\n\t.reg .b64 s, v, c;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 c, {%4, %5};\n\t"
        "fma.rn.f32x2 s, v, c, s;\n\tmov.b64 {%0, %1}, s;\n\t}" : "+f"(sum.x), "+f"(sum.y) : "r"(a), "r"(b), "f"(sx), "f"(sy));
}
__device__ __forceinline__ void f8_tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 f8_ld_cluster(uint32_t addr, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(f8_in_cta(addr, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void f8_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Waits for the loads that nothing else waits for after an abort; called by one thread, of a pair's first CTA.  Load n of a CTA
// belongs to phase n / STAGES of its stage's barrier - for a pair the first CTA's, which announces the bytes of both.  The
// loaders stop by themselves: of the loads that only one of the two has issued, the first CTA's are announced with bytes of the
// other that will not come, which are counted as having come, and the other's have not been announced at all, which is made up
// for.  (At most STAGES loads lie between the two: both wait for the same instructions to free a stage.)
template <bool PAIR, int STAGES, int BYTES>
__device__ __forceinline__ void f8_await_loads(uint64_t* bar_full, const int* loads) {
    const int mine = *loads;
    int other = mine;
    if (PAIR) asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(other) : "r"(f8_in_cta(smem_u32(loads), 1)) : "memory");
    const int all = max(mine, other), never = 0;
#pragma unroll 1
    for (int n = min(mine, other); n < all; n++) {
        const uint32_t bar = smem_u32(&bar_full[n % STAGES]);
        if (n < mine) asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(BYTES) : "memory");
        else asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(BYTES) : "memory");
    }
#pragma unroll 1
    for (int n = max(0, all - STAGES); n < all; n++) mbar_wait(&bar_full[n % STAGES], (n / STAGES) & 1, &never);
}

// SPLIT: the CTAs of a cluster share one tile (the grid then has one cluster per tile); otherwise a CTA walks the tiles
template <int NT, bool SPLIT, typename T>
__global__ void __launch_bounds__(Fp8Cfg<NT>::THREADS, Fp8Cfg<NT>::CTAS_PER_SM)
    fp8_gemm_kernel(const Fp8Params p, const int splits, const __grid_constant__ CUtensorMap lane_map, const __grid_constant__ CUtensorMap col_map,
                    const __grid_constant__ CUtensorMap out_map) {
    using Cfg = Fp8Cfg<NT>;
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) uint64_t bar_full[Cfg::STAGES], bar_empty[Cfg::STAGES], bar_acc_full[2], bar_acc_empty[2];
    __shared__ __align__(8) uint64_t bar_factor_full[F8_GROUPS], bar_factor_empty[F8_GROUPS], bar_issued;
    __shared__ __align__(16) float factors[F8_GROUPS][F8_GROUP][Cfg::FACTORS];
    __shared__ uint32_t tmem_base_s;
    __shared__ int s_abort, s_loads;

    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const uint32_t stage0 = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    const volatile int* abort_flag = &s_abort;
    constexpr int TMEM_COLS = 2 * NT;
    constexpr bool PAIR = Cfg::PAIR;
    const int team = SPLIT ? splits : PAIR ? 2 : 1;    // CTAs that share a tile: the cluster
    const int rank = (int)blockIdx.x % team, first = (int)blockIdx.x / team, step = (int)gridDim.x / team;
    const int kb0 = SPLIT ? (int)((long long)p.nkb * rank / splits) : 0, kb1 = SPLIT ? (int)((long long)p.nkb * (rank + 1) / splits) : p.nkb;

    if (warp == 1) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(TMEM_COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(TMEM_COLS));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        }
    }
    if (threadIdx.x == 0) {
        if (!Cfg::FEW && p.tma_out) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&out_map)));
        for (int i = 0; i < Cfg::STAGES; i++) { mbar_init(&bar_full[i], 1); mbar_init(&bar_empty[i], 1); }
        for (int i = 0; i < F8_GROUPS; i++) { mbar_init(&bar_factor_full[i], 1); mbar_init(&bar_factor_empty[i], Cfg::EPI_WARPS); }
        for (int i = 0; i < 2; i++) { mbar_init(&bar_acc_full[i], 1); mbar_init(&bar_acc_empty[i], (PAIR ? 2 : 1) * Cfg::EPI_WARPS); }
        mbar_init(&bar_issued, 1);                     // every instruction of the MMA warp is complete
        asm volatile("fence.mbarrier_init.release.cluster;" ::);
        s_abort = 0;
        s_loads = 0;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (PAIR) f8_cluster_sync();                       // the other CTA's barriers are set up
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = tmem_base_s;
    // In this order: a kernel that this lets start may read its constants at once, and they may come from a launch before this one.
    grid_dependency_wait();
    grid_launch_dependents();
    auto give_up = [&](int code) {                     // a wait ran out: nothing of the team's tile can be finished
        atomicCAS(&g_fp8_status, 0, code);
        s_abort = 1;
        if (PAIR) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(f8_in_cta(smem_u32(&s_abort), rank ^ 1)), "r"(1) : "memory");
    };
    if (warp < Cfg::EPI_WARP0) {
        // a pair's 20 warps have 96 registers each at launch: these four give 32 of theirs to the epilogue's sixteen, whose sums and two
        // chunks of an accumulator take 96 (with 16-bit results five values spill: 20 bytes stored, 40 loaded)
        if (PAIR) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 0) {
            // =========================== TMA loads: one lane ===========================
            if (elect_lane()) {
                uint32_t s = 0, use = 0;
                bool ok = true;
                for (int tile = first; tile < p.ntiles && ok; tile += step) {
                    const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
                    for (int kb = kb0; kb < kb1; kb++) {
                        if (use >= 1 && !mbar_wait(&bar_empty[s], (use - 1) & 1, abort_flag)) {
                            give_up(51);
                            ok = false;
                            break;
                        }
                        const uint32_t at = stage0 + s * Cfg::STAGE_BYTES;
                        uint32_t bar = smem_u32(&bar_full[s]);
                        if (!PAIR || rank == 0)
                            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"((PAIR ? 2 : 1) * Cfg::STAGE_BYTES) : "memory");
                        if (PAIR) bar = f8_in_cta(bar, 0);   // the CTA that issues for both waits for both
                        f8_load<PAIR>(at, &lane_map, kb * F8_BLOCK, (Cfg::FEW ? tn : PAIR ? tm * 2 + rank : tm) * 128, bar);
                        f8_load<PAIR>(at + F8_L_BYTES, &col_map, kb * F8_BLOCK, (Cfg::FEW ? tm : tn) * NT + (PAIR ? rank * Cfg::COL_ROWS : 0), bar);
                        if (++s == Cfg::STAGES) { s = 0; use++; }
                    }
                }
                s_loads = (int)(use * Cfg::STAGES + s);
            }
        } else if (warp == 1) {
            // =========================== MMA issue: the whole warp walks, one lane issues, for a pair the first CTA's ===========================
            const bool leader = elect_lane();
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)((PAIR ? 256 : 128) >> 4) << 24);   // D f32, A = B = e4m3, K-major
            uint32_t s = 0, par = 0;
            bool ok = !PAIR || rank == 0;
            int i = 0;   // blocks so far
            for (int tile = first; tile < p.ntiles && ok; tile += step)
                for (int kb = kb0; kb < kb1; kb++, i++) {
                    const int acc = i & 1;
                    if (i >= 2 && !f8_wait(smem_u32(&bar_acc_empty[acc]), ((i >> 1) - 1) & 1, abort_flag)) {
                        give_up(52);
                        ok = false;
                        break;
                    }
                    if (!f8_wait(smem_u32(&bar_full[s]), par, abort_flag)) {
                        give_up(53);
                        ok = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint64_t l = f8_desc(stage0 + s * Cfg::STAGE_BYTES), c = l + (F8_L_BYTES >> 4);
                    if (leader) {
#pragma unroll
                        for (int j = 0; j < F8_BLOCK / 32; j++) f8_mma<PAIR>(tmem_base + acc * NT, l + 2 * j, c + 2 * j, idesc, j > 0);
                        f8_commit<PAIR>(smem_u32(&bar_empty[s]));
                        f8_commit<PAIR>(smem_u32(&bar_acc_full[acc]));
                    }
                    __syncwarp();
                    if (++s == Cfg::STAGES) { s = 0; par ^= 1u; }
                }
            if (leader && (!PAIR || rank == 0)) f8_commit<PAIR>(smem_u32(&bar_issued));
        } else if (warp == 2) {
            // =========================== factors as * bs ===========================
            // FEW: a lane has the columns lane, lane + 32; else rows lane + 32 j of the tile, each with the bs of every 128 columns
            constexpr int MINE = Cfg::FEW ? (NT + 31) / 32 : 4, BLOCKS = Cfg::FEW ? 1 : NT / 128;
            int i = 0;
            bool ok = true;
            for (int tile = first; tile < p.ntiles && ok; tile += step) {
                const int tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
                const int m0 = (Cfg::FEW ? tm * NT : (PAIR ? tm * 2 + rank : tm) * 128) + lane;
                const float* a = p.as + m0 * p.as_row + kb0 * p.as_block;
                const float* b = p.bs + (long long)tn * BLOCKS * p.bs_row + kb0 * p.bs_block;
                for (int kb = kb0; kb < kb1; kb += F8_GROUP, i++) {   // (a tile begins with a new group)
                    float av[F8_GROUP][MINE], bv[F8_GROUP][BLOCKS];
#pragma unroll
                    for (int g = 0; g < F8_GROUP; g++) {
#pragma unroll
                        for (int e = 0; e < MINE; e++) av[g][e] = kb + g < kb1 && m0 + e * 32 < p.M ? __ldg(a + e * 32 * p.as_row) : 0.f;
#pragma unroll
                        for (int e = 0; e < BLOCKS; e++) bv[g][e] = kb + g < kb1 && (tn * BLOCKS + e) * 128 < p.N ? __ldg(b + e * p.bs_row) : 0.f;
                        a += p.as_block;
                        b += p.bs_block;
                    }
                    const int slot = i % F8_GROUPS;
                    if ((i >= F8_GROUPS && !f8_wait(smem_u32(&bar_factor_empty[slot]), (i / F8_GROUPS - 1) & 1, abort_flag)) ||
                        (i == p.give_up_group && rank == p.give_up_rank)) {
                        give_up(55);
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int g = 0; g < F8_GROUP; g++)
#pragma unroll
                        for (int e = 0; e < MINE; e++)
#pragma unroll
                            for (int h = 0; h < BLOCKS; h++)
                                if (!Cfg::FEW || e * 32 + lane < NT) factors[slot][g][h * 128 + e * 32 + lane] = av[g][e] * bv[g][h];
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar_factor_full[slot]);
                }
            }
        }
    } else {
        // =========================== epilogue ===========================
        if (PAIR) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const int ew = warp - Cfg::EPI_WARP0, quarter = warp & 3, col0 = (ew >> 2) * Cfg::COLS;   // TMEM lane quarter of a warp = warp % 4
        const uint32_t t_mine = tmem_base + ((uint32_t)(quarter * 32) << 16) + col0;
        // Walking state: one accumulator further with every block, one slot of factors with every group of them.
        uint32_t slot = 0, slot_par = 0, acc = 0, acc_par = 0;
        const uint32_t acc_full = smem_u32(bar_acc_full), acc_empty = PAIR ? f8_in_cta(smem_u32(bar_acc_empty), 0) : smem_u32(bar_acc_empty), factor_full = smem_u32(bar_factor_full),
                       factor_empty = smem_u32(bar_factor_empty);
        const uint32_t my_factors = smem_u32(factors) + (Cfg::FEW ? col0 : (col0 & ~127) + quarter * 32 + lane) * 4;
        bool ok = true;
        int tm = first / p.tiles_n, tn = first - tm * p.tiles_n;
        const int step_m = step / p.tiles_n, step_n = step - step_m * p.tiles_n;
        for (int tile = first; tile < p.ntiles && ok; tile += step) {
            float2 sum[Cfg::COLS / 2];
#pragma unroll
            for (int e = 0; e < Cfg::COLS / 2; e++) sum[e] = make_float2(0.f, 0.f);
            auto sum_of = [&](int e) { return e & 1 ? sum[e >> 1].y : sum[e >> 1].x; };
            uint32_t mine = 0;                         // this block's factors
            int in_group = F8_GROUP;
#pragma unroll 1
            for (int left = kb1 - kb0; left > 0; left--) {
                bool there = true;
                if (in_group == F8_GROUP) {
                    there = f8_wait(factor_full + slot * 8, slot_par, abort_flag);
                    mine = my_factors + slot * (F8_GROUP * Cfg::FACTORS * 4);
                    in_group = 0;
                }
                if (!there || !f8_wait(acc_full + acc * 8, acc_par, abort_flag)) {
                    give_up(54);
                    ok = false;
                    break;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                // 16 columns at a time, two loads to a wait
                constexpr int CHUNKS = Cfg::COLS / 16;
                const uint32_t t_acc = t_mine + acc * NT;
                uint32_t v[2][16];
                f8_tmem_ld16(v[0], t_acc);
                if (CHUNKS > 1) f8_tmem_ld16(v[1], t_acc + 16);
                const float factor = Cfg::FEW ? 0.f : lds_f32(mine);
#pragma unroll
                for (int h = 0; h < CHUNKS; h++) {
                    if (h % 2 == 0) f8_tmem_wait();
                    if (h == max(CHUNKS - 2, 0)) {     // all of it is in registers: the MMA warp may reuse the accumulator
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        if (elect_lane()) {
                            if (PAIR) f8_arrive_cluster(acc_empty + acc * 8);
                            else f8_arrive(acc_empty + acc * 8);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 sc = Cfg::FEW ? lds128f(mine + (h * 16 + e) * 4) : make_float4(factor, factor, factor, factor);
                        f8_fma2(sum[(h * 16 + e) / 2], v[h & 1][e], v[h & 1][e + 1], sc.x, sc.y);
                        f8_fma2(sum[(h * 16 + e) / 2 + 1], v[h & 1][e + 2], v[h & 1][e + 3], sc.z, sc.w);
                    }
                    if (h + 2 < CHUNKS) f8_tmem_ld16(v[h & 1], t_acc + (h + 2) * 16);
                }
                mine += Cfg::FACTORS * 4;
                if (++in_group == F8_GROUP || left == 1) {
                    in_group = F8_GROUP;
                    __syncwarp();
                    if (elect_lane()) f8_arrive(factor_empty + slot * 8);
                    if (++slot == F8_GROUPS) { slot = 0; slot_par ^= 1; }
                }
                acc ^= 1;
                if (!acc) acc_par ^= 1;
            }
            if (!ok) break;
            const int m0 = Cfg::FEW ? tm * NT + col0 : (PAIR ? tm * 2 + rank : tm) * 128 + quarter * 32;   // first activation row and output of the warp
            const int n0 = Cfg::FEW ? tn * 128 + quarter * 32 : tn * NT + col0;
            tm += step_m;                              // the next tile's place
            if ((tn += step_n) >= p.tiles_n) { tn -= p.tiles_n; tm++; }
            if (SPLIT) {
                // this CTA's part -> its shared memory (the ring is idle: its last loads have been multiplied), [column][output]
                const uint32_t part = stage0 + (uint32_t)((col0 * 128 + quarter * 32 + lane) * 4);
#pragma unroll
                for (int e = 0; e < Cfg::COLS; e++) asm volatile("st.shared.f32 [%0], %1;" ::"r"(part + e * 512), "f"(sum_of(e)) : "memory");
            } else if (Cfg::FEW) {
                // a warp's lanes are neighbouring outputs of a row
                const int n = n0 + lane;
                if (n < p.N) {
                    const float bias = p.bias ? __ldg(p.bias + n) : 0.f;
                    T* out = static_cast<T*>(p.c) + m0 * p.ldc + n;
                    const int left = p.M - m0;
#pragma unroll
                    for (int e = 0; e < Cfg::COLS; e++) {
                        if (e < left) *out = from_f32<T>(sum_of(e) + bias);
                        out += p.ldc;
                    }
                }
            } else {
                // A thread has neighbouring outputs of its row: 128 bytes of each of the warp's rows go to shared memory in the
                // swizzled layout of a tensor store, which writes whole lines while the warp goes on (stores from registers, 32
                // bytes of 32 rows each, held the next tile up for 5000 cycles: 8192 x 8192 x 4096 in 243 us).
                const uint32_t out = stage0 + Cfg::STAGES * Cfg::STAGE_BYTES + ew * F8_OUT_BYTES;
                auto stored = [] {                     // the last store has read its bytes
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    __syncwarp();
                };
                stored();
                if (p.bias) {                          // through shared memory: a warp's columns are the same in all its lanes
#pragma unroll
                    for (int e = 0; e < Cfg::COLS; e += 32)
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(out + (e + lane) * 4), "f"(__ldg(p.bias + min(n0 + e + lane, p.N - 1))) : "memory");
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < Cfg::COLS; e += 4) {
                        const float4 b = lds128f(out + e * 4);
                        sum[e / 2].x += b.x; sum[e / 2].y += b.y; sum[e / 2 + 1].x += b.z; sum[e / 2 + 1].y += b.w;
                    }
                    __syncwarp();
                }
                constexpr int W = 128 / (int)sizeof(T);
#pragma unroll
                for (int h = 0; h < Cfg::COLS; h += W) {
                    if (h) stored();
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        alignas(16) T o[W / 8];
#pragma unroll
                        for (int e = 0; e < W / 8; e++) o[e] = from_f32<T>(sum_of(h + q * (W / 8) + e));
                        const uint4 u = *reinterpret_cast<const uint4*>(o);
                        sts128(out + lane * 128 + ((q ^ (lane & 7)) << 4), u.x, u.y, u.z, u.w);
                    }
                    if (p.tma_out) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0 && n0 + h < p.N && m0 < p.M) {   // what lies outside c is not written
                            asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];"
                                         ::"l"(reinterpret_cast<uint64_t>(&out_map)), "r"((n0 + h) * (int)sizeof(T)), "r"(m0), "r"(out) : "memory");
                            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                        }
                    } else {                           // a row at a time, its outputs side by side
                        __syncwarp();
#pragma unroll 4
                        for (int r = 0; r < 32; r++) {
                            if (m0 + r >= p.M) break;
#pragma unroll
                            for (int e = lane; e < W; e += 32) {
                                const uint32_t at = out + r * 128 + (((e * (int)sizeof(T) >> 4) ^ (r & 7)) << 4) + (e * (int)sizeof(T) & 15);
                                T v;
                                if constexpr (sizeof(T) == 4) v = lds_f32(at);
                                else asm volatile("ld.shared.b16 %0, [%1];" : "=h"(reinterpret_cast<unsigned short&>(v)) : "r"(at));
                                if (n0 + h + e < p.N) static_cast<T*>(p.c)[(long long)(m0 + r) * p.ldc + n0 + h + e] = v;
                            }
                        }
                        __syncwarp();
                    }
                }
            }
        }
        if (!Cfg::FEW) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // the stores are complete before the CTA winds down
    }

    if (SPLIT) {
        // every CTA of the cluster adds up an equal share of the tile's outputs over all parts, in the order of K
        __syncwarp();
        f8_cluster_sync();
        const int tile = first, tm = tile / p.tiles_n, tn = tile - tm * p.tiles_n;
        const int total = min(NT, p.M - tm * NT) * 32;   // in fours, whose trip over the cluster is what this takes
        const int lo = (int)((long long)total * rank / splits), hi = (int)((long long)total * (rank + 1) / splits);
        for (int idx = lo + (int)threadIdx.x; idx < hi; idx += Cfg::THREADS) {
            float4 part[F8_MAX_SPLIT];
#pragma unroll
            for (int r = 0; r < F8_MAX_SPLIT; r++)
                if (r < splits) part[r] = f8_ld_cluster(stage0 + idx * 16, r);
            float4 v = part[0];
#pragma unroll
            for (int r = 1; r < F8_MAX_SPLIT; r++)
                if (r < splits) { v.x += part[r].x; v.y += part[r].y; v.z += part[r].z; v.w += part[r].w; }
            const int m = tm * NT + (idx >> 5), n = tn * 128 + (idx & 31) * 4;
            T* const out = static_cast<T*>(p.c) + m * p.ldc + n;
            const float o[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (n + e < p.N) out[e] = from_f32<T>(o[e] + (p.bias ? __ldg(p.bias + n + e) : 0.f));
        }
        __syncwarp();
        f8_cluster_sync();                             // no CTA leaves while its part is being read
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) f8_wait(smem_u32(&bar_issued), 0, nullptr);   // the instructions read and write both CTAs' memory, and arrive at their barriers
    __syncwarp();
    if (PAIR) f8_cluster_sync();                       // neither arrives at the other's barriers any more, nor raises its flag: the two are the same
    if (s_abort) {
        if (threadIdx.x == 0 && (!PAIR || rank == 0)) f8_await_loads<PAIR, Cfg::STAGES, Cfg::STAGE_BYTES>(bar_full, &s_loads);
        __syncwarp();
        if (PAIR) f8_cluster_sync();                   // neither leaves while loads for it are on their way
    }
    if (warp == 1) {
        __syncwarp();
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
    }
}

}  // namespace dabnn
