// Scoring of rows of logits: log probability and rank of a given class, entropy, the top alternatives.
//
//   m = max x_j, d_j = x_j - m, S = sum e^d_j, W = sum d_j e^d_j
//   log p_j = d_j - ln S,   entropy = -sum p ln p = ln S - W / S
//
// Classes are ordered by value, larger first, equal ones (the two zeros are) by index, a NaN before everything.
//
// One pass over a row: a lane keeps its own m, S, W (rescaled when its m grows) and its own count of classes before the label;
// a warp keeps its best classes in order, one to a lane.  A batch of a warp - 64 bytes of each lane - is looked at for
// alternatives only if some lane's maximum passes a threshold.  With r = ceil(k / 4), the fourth largest of the eight warps'
// r-th best classes is one (4 r >= k classes reach it), and so is the warp's own k-th best.  A row's first batches have no best
// classes yet: there the r-th largest of a warp's 64 half-lane maxima stands for its r-th best, and the warps meet once to
// compare them.  The lanes that pass leave their 64 bytes in shared memory, where the warp looks at the values of one lane (two
// of fp32) at a time, inserting what belongs among the best.
//
// A row is scored by one warp, or by a CTA of eight, or by a cluster of such CTAs where rows are few: the warps take the row's
// batches in turn and their parts are joined at the end, lists of best classes by counting, for each entry, the better ones.
//
// What bounds it: with many rows the latency of a warp's steps (its batch from L2 first), of the pipes issue, 11 instructions for 32
// logits, and ex2 most; then HBM.  4096 rows of 65536 bf16, top 8: 124 us
// (4.3 TB/s; 101 us without alternatives); 4096 of 32768 fp32 without them 88 us (6.1 TB/s); 1 row of 131072, top 20: 12 us.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "scalar_types.cuh"

namespace dabnn {

constexpr int LP_WARPS = 8, LP_MAX_CLUSTER = 8;        // warps of a CTA that share a row, CTAs of a cluster
constexpr int LP_ROWS = 4;                             // warps of a CTA that have a row each
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;
constexpr float LP_FLOOR = -1e30f;                     // a difference below it has e^d = 0; keeps d e^d a number
constexpr float LP_GONE = 1024.f;                      // a maximum this far below another (in units of ln 2) has e^d = 0; its product with a sum of as many terms as a row has is a number

// fp32 -> unsigned, order preserved; a NaN is the largest, the zeros are one value, nothing is 0
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    if (x != x) return 0xffffffffu;
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
    return key == 0xffffffffu ? __int_as_float(0x7fc00000) : __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
// t with: not (v <= t) exactly where v's key is at least `key` (for the key of -inf t is a NaN, which all pass)
__device__ __forceinline__ float pass_from(uint32_t key) {
    if (key == 0xffffffffu) return INFINITY;           // NaN alone
    const uint32_t below = key - (key == 0x80000000u ? 2 : 1);
    return __uint_as_float(below & 0x80000000u ? below ^ 0x80000000u : ~below);
}
// t with: not (v <= t) exactly where v's key is above `key`
__device__ __forceinline__ float pass_above(uint32_t key) { return key == 0xffffffffu ? INFINITY : pass_from(key + 1); }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float exp2_fast(float x) {   // ex2.approx: off by 2^-22
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// two fp32 operations in an instruction
__device__ __forceinline__ float2 two_add(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 two_mul(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 two_fma(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}

// Part of a row: its maximum, and S and W relative to it, W in units of ln 2 (the argument that ex2 wants anyway)
struct Part {
    float m, s, w;
    __device__ __forceinline__ void raise(float to) {   // to >= m
        const float delta = m == -INFINITY ? 0.f : fminf((to - m) * LP_LOG2E, LP_GONE), scale = exp2_fast(-delta);
        w = scale * (w - delta * s);
        s *= scale;
        m = to;
    }
    __device__ __forceinline__ void join(Part o) {
        const float to = fmaxf(m, o.m);
        raise(to);
        o.raise(to);
        s += o.s;
        w += o.w;
    }
};

template <typename T>
struct Vec {                                           // 16 bytes of a row
    static constexpr int N = 16 / (int)sizeof(T);
    uint4 raw;
    __device__ __forceinline__ float value(int i) const {
        const uint32_t w = sizeof(T) == 4 ? (i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w) : (i < 2 ? raw.x : i < 4 ? raw.y : i < 6 ? raw.z : raw.w);
        if constexpr (sizeof(T) == 4) return __uint_as_float(w);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
        else return __half2float(__ushort_as_half((unsigned short)(i % 2 ? w >> 16 : w)));
    }
    __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w; }
    // values at [first, first + N) of a row of n, -inf outside it; `row` + first is on a 16-byte boundary
    __device__ __forceinline__ void load(const T* row, int first, int n) {
        if (first >= 0 && first + N <= n) {
            raw = __ldg(reinterpret_cast<const uint4*>(row + first));
            return;
        }
        uint32_t w[4];
        constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : std::is_same_v<T, __nv_bfloat16> ? 0xff80ff80u : 0xfc00fc00u;
        w[0] = w[1] = w[2] = w[3] = NONE;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (first + i >= 0 && first + i < n) {
                if constexpr (sizeof(T) == 4) w[i] = __ldg(reinterpret_cast<const uint32_t*>(row) + first + i);
                else {
                    const uint32_t v = __ldg(reinterpret_cast<const unsigned short*>(row) + first + i);
                    w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | v << 16 : (w[i / 2] & 0xffff0000u) | v;
                }
            }
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// The best classes of a warp so far, in order: entry lane (and, with two, lane + 32) is key << 32 | ~index; 0: none yet
template <int ENTRIES>
struct Best {
    unsigned long long e[ENTRIES == 0 ? 1 : ENTRIES];
    __device__ __forceinline__ void insert(unsigned long long x) {   // x: the same in all lanes
        const int lane = threadIdx.x & 31;
        int pos = 0;
#pragma unroll
        for (int h = 0; h < ENTRIES; h++) pos += __popc(__ballot_sync(0xffffffffu, e[h] > x));
        unsigned long long carry = 0;
#pragma unroll
        for (int h = 0; h < ENTRIES; h++) {
            const unsigned long long up = __shfl_up_sync(0xffffffffu, e[h], 1), last = __shfl_sync(0xffffffffu, e[h], 31);
            const int at = h * 32 + lane;
            if (at > pos) e[h] = lane ? up : carry;
            else if (at == pos) e[h] = x;
            carry = last;
        }
    }
    __device__ __forceinline__ unsigned long long at(int i) const {   // i: the same in all lanes
        unsigned long long x = __shfl_sync(0xffffffffu, e[0], i & 31);
        if (ENTRIES > 1) {
            const unsigned long long y = __shfl_sync(0xffffffffu, e[ENTRIES - 1], i & 31);
            if (i >= 32) x = y;
        }
        return x;
    }
};

struct LogprobsParams {
    const void* logits;
    long long ld, ld_group;                            // between rows of a group, between groups
    const int64_t* labels;
    long long label_group;
    float *label_logprob, *entropy, *top_logprob;
    int64_t *label_rank, *top_index;
    int group_rows, rows, classes, top;
    // where the logits and the label of a warp's row lie (the address from one lane: known to be the same in all, it stays in
    // uniform registers; 4096 rows of 65536 bf16 132 us otherwise)
    template <typename T>
    __device__ __forceinline__ const T* place(int row, int64_t& label) const {
        const int g = row < group_rows ? 0 : row / group_rows, i = row - g * group_rows;
        label = labels ? labels[g * label_group + i] : -1;
        const unsigned long long at = reinterpret_cast<unsigned long long>(static_cast<const T*>(logits) + g * ld_group + i * ld);
        const uint32_t lo = __shfl_sync(0xffffffffu, (uint32_t)at, 0), hi = __shfl_sync(0xffffffffu, (uint32_t)(at >> 32), 0);
        return reinterpret_cast<const T*>((unsigned long long)hi << 32 | lo);
    }
};

__device__ __forceinline__ void lp_write(const LogprobsParams& p, long long row, int64_t label, float mine, const Part& all, unsigned long long before) {
    const bool have = label >= 0 && label < p.classes, nothing = all.m == -INFINITY && all.s == 0.f;   // a row of -inf alone has no distribution
    const float ls = logf(all.s);
    if (p.label_logprob) p.label_logprob[row] = have ? (nothing ? -INFINITY : (mine - all.m) - ls) : label < 0 ? 0.f : __int_as_float(0x7fc00000);
    if (p.label_rank) p.label_rank[row] = have ? (int64_t)before : -1;
    if (p.entropy) p.entropy[row] = nothing ? 0.f : ls - all.w / all.s * LP_LN2;
}
__device__ __forceinline__ void lp_write_top(const LogprobsParams& p, long long row, int i, unsigned long long entry, const Part& all) {
    const bool nothing = all.m == -INFINITY && all.s == 0.f;
    p.top_logprob[row * p.top + i] = nothing ? -INFINITY : (key_value((uint32_t)(entry >> 32)) - all.m) - logf(all.s);
    p.top_index[row * p.top + i] = (int64_t)(uint32_t)~(uint32_t)entry;
}

// Two 16-bit values at a time: the larger (a NaN wins), and how many pass a threshold, not (v <= t), as two small floats
template <typename T> struct Pair16;
template <> struct Pair16<__half> {
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
    static __device__ __forceinline__ uint32_t count(uint32_t v, uint32_t t, uint32_t sum) {
        uint32_t r;
        asm("{\n\t.reg .b32 c;\n\tset.gtu.f16x2.f16x2 c, %1, %2;\n\tadd.f16x2 %0, c, %3;\n\t}" : "=r"(r) : "r"(v), "r"(t), "r"(sum));
        return r;
    }
    static __device__ __forceinline__ uint32_t bits(float t) { return __half_as_ushort(__float2half_rd(t)); }
    static __device__ __forceinline__ float value(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }
};
template <> struct Pair16<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { uint32_t r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r; }
    static __device__ __forceinline__ uint32_t count(uint32_t v, uint32_t t, uint32_t sum) {
        uint32_t r;
        asm("{\n\t.reg .b32 c;\n\tset.gtu.bf16x2.bf16x2 c, %1, %2;\n\tadd.bf16x2 %0, c, %3;\n\t}" : "=r"(r) : "r"(v), "r"(t), "r"(sum));
        return r;
    }
    static __device__ __forceinline__ uint32_t bits(float t) { return __bfloat16_as_ushort(__float2bfloat16_rd(t)); }
    static __device__ __forceinline__ float value(uint32_t b) { return __uint_as_float(b << 16); }
};

// the largest of two vectors (a NaN wins)
template <typename T>
__device__ __forceinline__ float vec_max(const Vec<T>& a, const Vec<T>& b) {
    if constexpr (sizeof(T) == 4) {
        float m = max_nan(a.value(0), b.value(0));
#pragma unroll
        for (int i = 1; i < 4; i++) m = max_nan(m, max_nan(a.value(i), b.value(i)));
        return m;
    } else {
        uint32_t m = Pair16<T>::max(a.raw.x, b.raw.x);
#pragma unroll
        for (int i = 1; i < 4; i++) m = Pair16<T>::max(m, Pair16<T>::max(a.word(i), b.word(i)));
        return max_nan(Pair16<T>::value(m & 0xffffu), Pair16<T>::value(m >> 16));
    }
}
// How many values of a vector pass, not (v <= t), added to a running count: whole numbers in one float, or in two small ones
// (t rounded down to a 16-bit type passes the same values of it)
template <typename T>
struct Count {
    using Threshold = std::conditional_t<sizeof(T) == 4, float, uint32_t>;
    static __device__ __forceinline__ Threshold threshold(float t) {
        if constexpr (sizeof(T) == 4) return t;
        else return Pair16<T>::bits(t) * 0x10001u;
    }
    Threshold sum = 0;
    __device__ __forceinline__ void add(const Vec<T>& v, Threshold t) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if constexpr (sizeof(T) == 4) sum += v.value(i) <= t ? 0.f : 1.f;
            else sum = Pair16<T>::count(v.word(i), t, sum);
    }
    __device__ __forceinline__ int total() const {
        if constexpr (sizeof(T) == 4) return (int)sum;
        else return (int)(Pair16<T>::value(sum & 0xffffu) + Pair16<T>::value(sum >> 16));
    }
};

// how many entries of a list in order come before x (zeros, which stand for none, are at the end)
__device__ __forceinline__ int entries_before(const unsigned long long* list, int n, unsigned long long x) {
    int at = 0;
#pragma unroll
    for (int s = DABNN_LOGPROBS_MAX_TOP; s; s >>= 1)
        if (at + s <= n && list[at + s - 1] > x) at += s;
    return at;
}

// What the warps of a CTA share about their row's best classes
template <int ENTRIES>
struct Shared {
    unsigned long long lists[LP_WARPS][ENTRIES ? ENTRIES * 32 : 1];   // each warp's, in order, at the end
    uint32_t reach[LP_WARPS];                          // a key that ceil(top / 4) classes of a warp reach, 0: none yet
};
// the fourth largest of the eight
__device__ __forceinline__ uint32_t fourth_of(const uint32_t* reach) {
    const volatile uint32_t* const r = reach;
    const int lane = threadIdx.x & 31;
    const uint32_t mine = lane < LP_WARPS ? r[lane] : 0;
    int larger = 0;
#pragma unroll
    for (int i = 0; i < LP_WARPS; i++) {
        const uint32_t o = __shfl_sync(0xffffffffu, mine, i);
        larger += o > mine || (o == mine && i < lane);
    }
    return __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, larger == 3 && lane < LP_WARPS)) - 1);
}
__device__ __forceinline__ void team_sync() { asm volatile("bar.sync 1, %0;" ::"n"(LP_WARPS * 32) : "memory"); }
// Where the lanes of a warp leave a batch
struct Stash {
    uint4 bytes[32][4];
    int first[32];                                     // the index of a lane's first value
};

// A warp's share of a row: batches `part`, part + parts, ...
template <typename T, int ENTRIES, bool TEAM>
__device__ __forceinline__ void lp_scan(const LogprobsParams& p, const T* row, int64_t label64, float& mine, int part, int parts, Stash* stash,
                                        Shared<ENTRIES>* shared, Part& all, unsigned& before, Best<ENTRIES>& best) {
    constexpr int N = Vec<T>::N, VECS = 4, BATCH = 32 * VECS * N;
    const int warp = uniform_warp(), lane = threadIdx.x & 31, n = p.classes;
    // vectors are counted from the 16-byte boundary at or below the row's first element, which is element `shift` there
    const int shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int step = parts * BATCH;
    int first = part * BATCH - shift + lane * N;       // this lane's first element of the batch
    Vec<T> v[VECS];
    auto load = [&](int b) {
        if (b * BATCH >= shift && (b + 1) * BATCH - shift <= n) {   // (the same in all lanes)
            const uint4* const at = reinterpret_cast<const uint4*>(row + first);
#pragma unroll
            for (int i = 0; i < VECS; i++) v[i].raw = __ldg(at + i * 32);
        } else if constexpr (TEAM) {
#pragma unroll
            for (int i = 0; i < VECS; i++) v[i].load(row, first + i * 32 * N, n);
        } else {                                       // (less code: 4096 rows of 65536 bf16 124 us instead of 130, 1024 of 1000 fp32 6.2 instead of 5.6)
#pragma unroll 1
            for (int i = 0; i < VECS; i++) {
                Vec<T> u;
                u.load(row, first + i * 32 * N, n);
#pragma unroll
                for (int k = 0; k < VECS; k++)
                    if (i == k) v[k] = u;
            }
        }
    };
    load(part);

    const bool have = __shfl_sync(0xffffffffu, label64 >= 0 && label64 < n, 0);
    const int label = __shfl_sync(0xffffffffu, have ? (int)label64 : -1, 0);   // (known to be the same in all lanes)
    mine = have ? to_f32(row[label]) : 0.f;
    // classes before the label: those at least as large as it in front of it, those larger behind it
    const uint32_t mykey = order_key(mine);
    const auto many_front = Count<T>::threshold(pass_from(mykey)), many_behind = Count<T>::threshold(pass_above(mykey));
    const bool all_front = mine == -INFINITY, none_behind = mine != mine;   // (thresholds that would pass what is outside the row, or a NaN)

    all = Part{-INFINITY, 0.f, 0.f};
    before = 0;
    if (have && all_front && part == 0 && lane == 0) before = label;
#pragma unroll
    for (int h = 0; h < ENTRIES; h++) best.e[h] = 0;
    float thr = __int_as_float(0x7fc00000);            // an alternative is what passes: not (v <= thr)
    const int reach_at = (p.top + 3) / 4 - 1;
    const int batches = (int)(((long long)n + shift + BATCH - 1) / BATCH);
    if (TEAM && ENTRIES && part >= batches) team_sync();   // nothing to do but to let the others pass
    for (int b = part; b < batches; b += parts) {
        if (b != part) load(b);
        {   // the next batch on its way to L2 (one ahead: 2048 rows of 32768 fp32 67 us, 71 without, four ahead 71)
            const long long next = (long long)(b + parts) * BATCH - shift + lane * (128 / (int)sizeof(T));
            if (lane < VECS * 4 && next >= 0 && next < n) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + next));
        }
        const float half[2] = {vec_max(v[0], v[1]), vec_max(v[2], v[3])};
        const float top = max_nan(half[0], half[1]);
        const float to = fmaxf(all.m, top);        // (a NaN is passed over: it makes S one)
        if (to > all.m) all.raise(to);
        const float base = all.m == -INFINITY ? 0.f : all.m;
        float2 s = make_float2(0.f, 0.f), w = s;
#pragma unroll
        for (int i = 0; i < VECS; i++)
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                float2 t = two_mul(two_add(make_float2(v[i].value(e), v[i].value(e + 1)), make_float2(-base, -base)), make_float2(LP_LOG2E, LP_LOG2E));
                t = make_float2(max_nan(t.x, LP_FLOOR), max_nan(t.y, LP_FLOOR));
                const float2 x = make_float2(exp2_fast(t.x), exp2_fast(t.y));
                s = two_add(s, x);
                w = two_fma(t, x, w);
            }
        all.s += s.x + s.y;
        all.w += w.x + w.y;

        // nothing of most batches comes before a label that is among the likeliest (4096 rows of 65536 bf16, top 8: 113 us with the
        // likeliest classes as labels, 127 with any)
        if (have && __any_sync(0xffffffffu, !(top < mine))) {
            int count = 0;
            auto pick = [&](int i) {                   // v[i], i not known to the compiler
                Vec<T> u = v[0];
#pragma unroll
                for (int k = 1; k < VECS; k++)
                    if (i == k) u = v[k];
                return u;
            };
            if (!all_front && !none_behind) {
                Count<T> c;
#pragma unroll
                for (int i = 0; i < VECS; i++) c.add(v[i], first + i * 32 * N + N <= label ? many_front : many_behind);
                count = c.total();
                const unsigned off = (unsigned)(label - first), at = off % (32 * N);
                if (off < VECS * 32 * N && at < N) {   // the label's own vector: what equals it in front of it is still to be counted
                    const Vec<T> u = pick(off / (32 * N));
#pragma unroll
                    for (int e = 0; e < N - 1; e++) count += e < (int)at && u.value(e) == mine;
                }
            } else {                                   // no threshold serves: one by one
                const float thr_front = pass_from(order_key(mine)), thr_behind = pass_above(order_key(mine));
#pragma unroll 1
                for (int i = 0; i < VECS; i++) {
                    const Vec<T> u = pick(i);
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const int at = first + i * 32 * N + e;
                        if (at >= 0 && at < n && (at < label ? !all_front && !(u.value(e) <= thr_front) : at > label && !none_behind && !(u.value(e) <= thr_behind))) count++;
                    }
                }
            }
            before += count;
        }

        if (ENTRIES) {
            // the nth largest of the 64 half-lane maxima: as many classes are that large
            auto nth_maximum = [&](int nth) {
                uint32_t a = order_key(half[0]), c = order_key(half[1]), key = 0;
                for (int k = 0; k < nth; k++) {
                    const uint32_t mx = max(a, c);
                    key = __reduce_max_sync(0xffffffffu, mx);
                    const int who = __ffs(__ballot_sync(0xffffffffu, mx == key)) - 1;
                    if (lane == who) { if (a >= c) a = 0; else c = 0; }
                }
                return key;
            };
            auto raise_to = [&](uint32_t key) {        // (-inf may stand for what is outside the row)
                if (key > 0x007fffffu) {
                    const float t = pass_from(key);    // what equals it may still come before it
                    if (!(t <= thr)) thr = t;
                }
            };
            if (TEAM && b == part) {
                const uint32_t key = nth_maximum(reach_at + 1);
                if (lane == 0) shared->reach[warp] = key;
                team_sync();
            }
            uint32_t hot = __ballot_sync(0xffffffffu, !(top <= thr));
            if (TEAM && hot) {
                raise_to(fourth_of(shared->reach));
                hot = __ballot_sync(0xffffffffu, !(top <= thr));
            }
            if (__popc(hot) > 8) {
                raise_to(nth_maximum(p.top));
                hot = __ballot_sync(0xffffffffu, !(top <= thr));
            }
            if (hot) {
                if (hot >> lane & 1) {
                    const int slot = __popc(hot & ((1u << lane) - 1));
#pragma unroll
                    for (int i = 0; i < VECS; i++) stash->bytes[slot][i] = v[i].raw;
                    stash->first[slot] = first;
                }
                __syncwarp();
                unsigned long long last = best.at(p.top - 1);
                constexpr int AT_ONCE = 32 / (VECS * N);   // lanes' batches that a warp looks at together
                const int nhot = __popc(hot), j = lane % (VECS * N);
#pragma unroll 1
                for (int q = 0; q < nhot; q += AT_ONCE) {
                    const int slot = q + lane / (VECS * N);
                    unsigned long long x = 0;
                    if (slot < nhot) {
                        const float u = to_f32(reinterpret_cast<const T*>(stash->bytes[slot])[j]);
                        const int at = stash->first[slot] + j / N * 32 * N + j % N;
                        if (!(u <= thr) && (unsigned)at < (unsigned)n) x = (unsigned long long)order_key(u) << 32 | (uint32_t)~at;
                    }
                    for (uint32_t mask = __ballot_sync(0xffffffffu, x > last); mask; mask &= mask - 1) {
                        const unsigned long long y = __shfl_sync(0xffffffffu, x, __ffs(mask) - 1);
                        if (y > last) {
                            best.insert(y);
                            last = best.at(p.top - 1);
                        }
                    }
                }
                __syncwarp();
                if (last) {                        // in a warp's own order what equals it comes after it
                    const float t = pass_above((uint32_t)(last >> 32));
                    if (!(t <= thr)) thr = t;
                }
                if (TEAM) {
                    const uint32_t key = (uint32_t)(best.at(reach_at) >> 32);
                    volatile uint32_t* const mine_s = &shared->reach[warp];
                    if (lane == 0 && key > *mine_s) *mine_s = key;
                }
            }
        }
        first += step;
    }
    // the lanes' parts
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        Part o;
        o.m = __shfl_xor_sync(0xffffffffu, all.m, d);
        o.s = __shfl_xor_sync(0xffffffffu, all.s, d);
        o.w = __shfl_xor_sync(0xffffffffu, all.w, d);
        all.join(o);
    }
    before = __reduce_add_sync(0xffffffffu, before);
}

// a warp per row
template <typename T, int ENTRIES>
__global__ void __launch_bounds__(LP_ROWS * 32, 7) logprobs_warp_kernel(const LogprobsParams p) {
    __shared__ Stash stash[ENTRIES ? LP_ROWS : 1];
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * LP_ROWS + warp;
    grid_dependency_wait();
    if (row >= p.rows) return;
    int64_t label;
    const T* const logits = p.place<T>((int)row, label);
    float mine;
    Part all;
    unsigned before;
    Best<ENTRIES> best;
    lp_scan<T, ENTRIES, false>(p, logits, label, mine, 0, 1, &stash[ENTRIES ? warp : 0], nullptr, all, before, best);
    if (lane == 0) lp_write(p, row, label, mine, all, before);
    if (ENTRIES)
#pragma unroll
        for (int h = 0; h < ENTRIES; h++)
            if (h * 32 + lane < p.top) lp_write_top(p, row, h * 32 + lane, best.e[h], all);
}

// a cluster of CTAs (one, where rows are many) per row
template <typename T, int ENTRIES>
__global__ void __launch_bounds__(LP_WARPS * 32, 4) logprobs_team_kernel(const LogprobsParams p, const int ctas) {
    constexpr int LIST = ENTRIES ? ENTRIES * 32 : 1;
    __shared__ Stash stash[ENTRIES ? LP_WARPS : 1];
    __shared__ Shared<ENTRIES> shared;
    __shared__ unsigned long long merged[LIST], gathered[LP_MAX_CLUSTER * LIST];
    __shared__ Part parts[LP_WARPS], part_s;
    __shared__ unsigned before_s[LP_WARPS], before_cta;
    const int warp = uniform_warp(), lane = threadIdx.x & 31, rank = blockIdx.x % ctas;
    const long long row = blockIdx.x / ctas;
    if (threadIdx.x < LP_WARPS) shared.reach[threadIdx.x] = 0;
    __syncthreads();
    grid_dependency_wait();
    int64_t label;
    const T* const logits = p.place<T>((int)row, label);
    float mine;
    Part all;
    unsigned before;
    Best<ENTRIES> best;
    lp_scan<T, ENTRIES, true>(p, logits, label, mine, warp * ctas + rank, LP_WARPS * ctas, &stash[ENTRIES ? warp : 0], &shared, all, before, best);
    if (lane == 0) { parts[warp] = all; before_s[warp] = before; }
    if (ENTRIES)
#pragma unroll
        for (int h = 0; h < ENTRIES; h++) shared.lists[warp][h * 32 + lane] = best.e[h];
    __syncthreads();
    // an entry's place: how many of the others come before it (no two are alike; 0 stands for none)
    auto place = [&](const unsigned long long* entries, int count, unsigned long long x) {
        int better = 0;
        for (int i = 0; i < count; i++) better += entries_before(entries + i * LIST, p.top, x);
        return better;
    };
    if (warp == 0) {
        all = parts[lane % LP_WARPS];
        before = before_s[lane % LP_WARPS];
#pragma unroll
        for (int d = LP_WARPS / 2; d; d >>= 1) {
            Part o;
            o.m = __shfl_xor_sync(0xffffffffu, all.m, d);
            o.s = __shfl_xor_sync(0xffffffffu, all.s, d);
            o.w = __shfl_xor_sync(0xffffffffu, all.w, d);
            all.join(o);
            before += __shfl_xor_sync(0xffffffffu, before, d);
        }
        if (lane == 0) { part_s = all; before_cta = before; }
        if (lane == 0 && ctas == 1) lp_write(p, row, label, mine, all, before);
    }
    if (ENTRIES) {
        // (at least `top` entries of a row's only CTA; of a cluster's CTAs perhaps fewer)
        if (ctas > 1) {
            for (int i = threadIdx.x; i < LIST; i += LP_WARPS * 32) merged[i] = 0;
            __syncthreads();
        }
        for (int i = threadIdx.x; i < LP_WARPS * p.top; i += LP_WARPS * 32) {
            const unsigned long long x = shared.lists[i / p.top][i % p.top];
            const int at = x ? place(&shared.lists[0][0], LP_WARPS, x) : p.top;
            if (at < p.top) merged[at] = x;
        }
    }
    if (ctas == 1) {
        if (!ENTRIES) return;
        __syncthreads();
        if ((int)threadIdx.x < p.top) lp_write_top(p, row, threadIdx.x, merged[threadIdx.x], part_s);
        return;
    }
    auto cluster_sync = [] { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); };
    __syncwarp();
    cluster_sync();
    if (rank == 0) {
        auto there = [](const void* here, int r) {
            uint32_t a;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(here)), "r"(r));
            return a;
        };
        auto read = [](uint32_t a) {
            uint32_t x;
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(a) : "memory");
            return x;
        };
        if (ENTRIES)
            for (int i = threadIdx.x; i < ctas * p.top; i += LP_WARPS * 32) {
                unsigned long long x;
                asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(there(&merged[i % p.top], i / p.top)) : "memory");
                gathered[i / p.top * LIST + i % p.top] = x;
            }
        all = part_s;
        before = before_cta;
        Part o[LP_MAX_CLUSTER];
        unsigned c[LP_MAX_CLUSTER];
#pragma unroll
        for (int r = 1; r < LP_MAX_CLUSTER; r++)
            if (r < ctas) {
                const uint32_t a = there(&part_s, r);
                o[r] = Part{__uint_as_float(read(a)), __uint_as_float(read(a + 4)), __uint_as_float(read(a + 8))};
                c[r] = read(there(&before_cta, r));
            }
#pragma unroll
        for (int r = 1; r < LP_MAX_CLUSTER; r++)
            if (r < ctas) { all.join(o[r]); before += c[r]; }
        __syncthreads();
        if (threadIdx.x == 0) lp_write(p, row, label, mine, all, before);
        if (ENTRIES)
            for (int i = threadIdx.x; i < ctas * p.top; i += LP_WARPS * 32) {
                const unsigned long long x = gathered[i / p.top * LIST + i % p.top];
                const int at = x ? place(gathered, ctas, x) : p.top;
                if (at < p.top) lp_write_top(p, row, at, x, all);
            }
    }
    __syncwarp();
    cluster_sync();                                    // no CTA leaves while its part is being read
}

// Rows of one batch have a warp each; so do those of up to 4096 classes where every scheduler finds a row, and all where there
// are 16 rows for an SM (of 65536 bf16, top 8: 4096 rows 124 us with a warp each and 150 with a CTA, 2600 rows 95 and 99, 1900
// rows 85 and 74).
// Others a CTA, or as many CTAs (up to 8) as keep the SMs busy and find a batch for each of their warps: no more than three to an
// SM (100 rows of 50000 bf16: 14.2 us in four CTAs each, 15.7 in two, 22 in eight).
template <typename T, int ENTRIES>
static int lp_launch(const LogprobsParams& p, cudaStream_t stream) {
    if (p.classes <= 128 * Vec<T>::N || (p.classes <= 4096 && p.rows >= 4 * sm_count()) || p.rows >= 16 * sm_count()) {
        DABNN_CUDA_OK(launch_overlapped(logprobs_warp_kernel<T, ENTRIES>, dim3((unsigned)(((long long)p.rows + LP_ROWS - 1) / LP_ROWS)), dim3(LP_ROWS * 32), 0, stream, p));
        return DABNN_OK;
    }
    int ctas = 1;
    while (ctas < LP_MAX_CLUSTER && (long long)p.rows * ctas * 2 <= 3 * sm_count() && (long long)ctas * LP_WARPS * 128 * Vec<T>::N < p.classes) ctas *= 2;
    DABNN_REQUIRE((long long)p.rows * ctas <= INT_MAX, DABNN_ERR_SHAPE, "logprobs: too many rows");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p.rows * ctas));
    cfg.blockDim = dim3(LP_WARPS * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_overlap_launches ? 2 : 1;
    DABNN_CUDA_OK(cudaLaunchKernelEx(&cfg, logprobs_team_kernel<T, ENTRIES>, p, ctas));
    return DABNN_OK;
}

}  // namespace dabnn

using namespace dabnn;

extern "C" int dabnn_logprobs(const void* logits, int type, long long ld, const int64_t* labels, int rows, int classes, float* label_logprob,
                              int64_t* label_rank, float* entropy, float* top_logprob, int64_t* top_index, int top, dabnn_stream_t s) {
    return dabnn_logprobs_grouped(logits, type, ld, 0, labels, 0, rows > 0 ? rows : 1, rows, classes, label_logprob, label_rank, entropy, top_logprob, top_index, top, s);
}

extern "C" int dabnn_logprobs_grouped(const void* logits, int type, long long ld, long long ld_group, const int64_t* labels, long long label_group, int group_rows,
                                      int rows, int classes, float* label_logprob, int64_t* label_rank, float* entropy, float* top_logprob, int64_t* top_index,
                                      int top, dabnn_stream_t s) {
    DABNN_REQUIRE(type >= DABNN_F32 && type <= DABNN_BF16, DABNN_ERR_ARG, "logprobs: unknown type");
    DABNN_REQUIRE(rows >= 0 && classes >= 1 && group_rows >= 1, DABNN_ERR_ARG, "logprobs: bad dims");
    DABNN_REQUIRE(classes < INT_MAX / 2, DABNN_ERR_SHAPE, "logprobs: too many classes");
    DABNN_REQUIRE(top >= 0 && top <= DABNN_LOGPROBS_MAX_TOP && top <= classes, DABNN_ERR_ARG, "logprobs: top must be between 0 and the smaller of 64 and the classes");
    if (rows == 0) return DABNN_OK;
    DABNN_REQUIRE(labels || (!label_logprob && !label_rank), DABNN_ERR_ARG, "logprobs: a label's outputs without labels");
    DABNN_REQUIRE(top == 0 || (top_logprob && top_index), DABNN_ERR_ARG, "logprobs: null pointer");
    DABNN_REQUIRE(logits, DABNN_ERR_ARG, "logprobs: null pointer");
    DABNN_REQUIRE(ld >= classes || rows == 1 || group_rows == 1, DABNN_ERR_SHAPE, "logprobs: the row pitch is below the classes");
    DABNN_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (type == DABNN_F32 ? 3 : 1)) == 0, DABNN_ERR_ARG, "logprobs: misaligned pointer");
    const cudaStream_t stream = static_cast<cudaStream_t>(s);
    const LogprobsParams p{logits, ld, ld_group, labels, label_group, label_logprob, entropy, top_logprob, label_rank, top_index, group_rows, rows, classes, top};
    auto launch = [&](auto tag) {
        using T = decltype(tag);
        return top == 0 ? lp_launch<T, 0>(p, stream) : top <= 32 ? lp_launch<T, 1>(p, stream) : lp_launch<T, 2>(p, stream);
    };
    if (type == DABNN_F32) return launch(float{});
    if (type == DABNN_F16) return launch(__half{});
    return launch(__nv_bfloat16{});
}
