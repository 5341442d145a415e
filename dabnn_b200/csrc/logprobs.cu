// Scoring of rows of logits: log probability and rank of a given class, entropy, the top alternatives.
//
//   m = max x_j, d_j = x_j - m, S = sum e^d_j, W = sum d_j e^d_j
//   log p_j = d_j - ln S,   entropy = -sum p ln p = ln S - W / S
//
// Classes are ordered by value, larger first, equal ones (the two zeros are) by index, a NaN before everything.
#include <climits>

#include "common.cuh"
#include "kernels.h"
#include "scalar_types.cuh"

namespace dabnn {

// fp32 -> unsigned, order preserved; a NaN is the largest, the zeros are one value
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    if (x != x) return 0xffffffffu;
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

template <typename V, typename F>
__device__ V block_reduce(V v, F op, V* shared) {
    shared[threadIdx.x] = v;
    __syncthreads();
    for (int n = blockDim.x / 2; n; n >>= 1) {
        if ((int)threadIdx.x < n) shared[threadIdx.x] = op(shared[threadIdx.x], shared[threadIdx.x + n]);
        __syncthreads();
    }
    v = shared[0];
    __syncthreads();
    return v;
}

// one CTA per row
template <typename T>
__global__ void __launch_bounds__(256) logprobs_kernel(const T* __restrict__ logits, const long long ld, const int64_t* __restrict__ labels, const int classes,
                                                       float* label_logprob, int64_t* label_rank, float* entropy, float* top_logprob,
                                                       int64_t* top_index, const int top) {
    __shared__ float fs[256];
    __shared__ unsigned long long us[256];
    const long long row = blockIdx.x;
    const T* x = logits + row * ld;
    auto maxu = [](unsigned long long a, unsigned long long b) { return a > b ? a : b; };
    auto add = [](float a, float b) { return a + b; };
    float m = -INFINITY;
    for (int j = threadIdx.x; j < classes; j += 256) m = fmaxf(m, to_f32(x[j]));
    m = block_reduce(m, [](float a, float b) { return fmaxf(a, b); }, fs);
    const int64_t label = labels ? labels[row] : -1;
    const bool have = label >= 0 && label < classes;
    const float mine = have ? to_f32(x[label]) : 0.f;
    const uint32_t mykey = order_key(mine);
    float s = 0.f, w = 0.f;
    unsigned long long before = 0;
    for (int j = threadIdx.x; j < classes; j += 256) {
        const float v = to_f32(x[j]), d = v - m, e = expf(d);
        const uint32_t key = order_key(v);
        s += e;
        w += fmaxf(d, -3e38f) * e;
        before += key > mykey || (key == mykey && j < label);
    }
    s = block_reduce(s, add, fs);
    w = block_reduce(w, add, fs);
    before = block_reduce(before, [](unsigned long long a, unsigned long long b) { return a + b; }, us);
    const float ls = logf(s);
    unsigned long long best = 0;
    for (int j = threadIdx.x; j < classes; j += 256) best = maxu(best, ((unsigned long long)order_key(to_f32(x[j])) << 32) | (uint32_t)~j);
    best = block_reduce(best, maxu, us);
    const bool nothing = (uint32_t)(best >> 32) == order_key(-INFINITY);   // a row of -inf alone has no distribution
    if (threadIdx.x == 0) {
        if (labels) {
            if (label_logprob) label_logprob[row] = have ? (nothing ? -INFINITY : (mine - m) - ls) : label < 0 ? 0.f : __int_as_float(0x7fc00000);
            if (label_rank) label_rank[row] = have ? (int64_t)before : -1;
        }
        if (entropy) entropy[row] = nothing ? 0.f : ls - w / s;
    }
    for (int t = 0; t < top; t++) {
        if (threadIdx.x == 0) {
            const uint32_t key = (uint32_t)(best >> 32);
            const float v = key == 0xffffffffu ? __int_as_float(0x7fc00000) : key_value(key);
            if (top_logprob) top_logprob[row * top + t] = nothing ? -INFINITY : (v - m) - ls;
            if (top_index) top_index[row * top + t] = (int64_t)(uint32_t)~(uint32_t)best;
        }
        unsigned long long next = 0;
        for (int j = threadIdx.x; j < classes; j += 256) {
            const unsigned long long k = ((unsigned long long)order_key(to_f32(x[j])) << 32) | (uint32_t)~j;
            if (k < best) next = maxu(next, k);
        }
        best = block_reduce(next, maxu, us);
    }
}

}  // namespace dabnn

using namespace dabnn;

extern "C" int dabnn_logprobs(const void* logits, int type, long long ld, const int64_t* labels, int rows, int classes, float* label_logprob,
                              int64_t* label_rank, float* entropy, float* top_logprob, int64_t* top_index, int top, dabnn_stream_t s) {
    DABNN_REQUIRE(type >= DABNN_F32 && type <= DABNN_BF16, DABNN_ERR_ARG, "logprobs: unknown type");
    DABNN_REQUIRE(rows >= 0 && classes >= 1, DABNN_ERR_ARG, "logprobs: bad dims");
    DABNN_REQUIRE(top >= 0 && top <= DABNN_LOGPROBS_MAX_TOP && top <= classes, DABNN_ERR_ARG, "logprobs: top must be between 0 and the smaller of 64 and the classes");
    if (rows == 0) return DABNN_OK;
    DABNN_REQUIRE(labels || (!label_logprob && !label_rank), DABNN_ERR_ARG, "logprobs: a label's outputs without labels");
    DABNN_REQUIRE(top == 0 || (top_logprob && top_index), DABNN_ERR_ARG, "logprobs: null pointer");
    DABNN_REQUIRE(logits, DABNN_ERR_ARG, "logprobs: null pointer");
    DABNN_REQUIRE(ld >= classes || rows == 1, DABNN_ERR_SHAPE, "logprobs: the row pitch is below the classes");
    DABNN_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (type == DABNN_F32 ? 3 : 1)) == 0, DABNN_ERR_ARG, "logprobs: misaligned pointer");
    const cudaStream_t stream = static_cast<cudaStream_t>(s);
    auto launch = [&](auto tag) {
        using T = decltype(tag);
        logprobs_kernel<T><<<rows, 256, 0, stream>>>(static_cast<const T*>(logits), ld, labels, classes, label_logprob, label_rank, entropy, top_logprob, top_index, top);
    };
    if (type == DABNN_F32) launch(float{});
    else if (type == DABNN_F16) launch(__half{});
    else launch(__nv_bfloat16{});
    return check_launch("logprobs_kernel");
}
