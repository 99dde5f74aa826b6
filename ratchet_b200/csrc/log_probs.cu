// Log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits.
//
// With m = max v and S = sum e^(v - m): log p(t) = v_t - m - ln S and H = ln S - sum e^(v - m) (v - m) / S.
// A token's place in the order is one 64-bit number: the value's bits made monotone, then the id from above, so that equal
// values fall to the lower id and no two are equal.
#include "common.cuh"
#include "kernels.hpp"

namespace rt {

namespace {

constexpr int THREADS = 512;
using Order = unsigned long long;

// larger value = larger word; -0 counts as +0, NaN as the largest
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k == 0xffffffffu ? 0x7fc00000u : k ^ 0x80000000u) : ~k);
}
__device__ __forceinline__ Order order_of(float v, uint32_t id) { return (Order)order_bits(v) << 32 | (0xffffffffu - id); }

template <typename V, typename F> __device__ __forceinline__ V block_reduce(V v, V *red, F f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads(); // the slots may still be read from the last time
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < THREADS / 32; w++) v = f(v, red[w]);
    return v;
}

template <typename T> __global__ void __launch_bounds__(THREADS) log_probs_kernel(rt_log_probs p) {
    __shared__ float red[THREADS / 32];
    __shared__ Order best_of[THREADS / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long row = blockIdx.x;
    const T *v = (const T *)p.logits + row * p.ld;
    const int vocab = (int)p.vocab;
    float m = -INFINITY;
    Order mine = 0; // this thread's largest
    for (int i = threadIdx.x; i < vocab; i += THREADS) {
        const float a = to_f32(v[i]);
        m = fmaxf(m, a);
        const Order o = order_of(a, i);
        mine = o > mine ? o : mine;
    }
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    auto sum = [](float a, float b) { return a + b; };
    m = block_reduce(m, red, larger);
    float s = 0.f, w = 0.f;
    bool nan = false;
    for (int i = threadIdx.x; i < vocab; i += THREADS) {
        const float a = to_f32(v[i]), d = a - m, e = expf(d);
        nan = nan || a != a;
        s += e;
        if (e > 0.f) w = fmaf(e, d, w);
    }
    nan = __syncthreads_or(nan);
    s = block_reduce(s, red, sum);
    w = block_reduce(w, red, sum);
    const bool nothing = m == -INFINITY && !nan;
    const float log_s = nothing ? 0.f : nan ? NAN : logf(s);
    auto log_prob = [&](float a) { return nothing ? -INFINITY : a - m - log_s; };
    if (threadIdx.x == 0) {
        if (p.log_prob) {
            const int t = p.tokens[row];
            p.log_prob[row] = t >= 0 && t < vocab ? log_prob(to_f32(v[t])) : NAN;
        }
        if (p.entropy) p.entropy[row] = nothing ? 0.f : log_s - w / s;
    }
    for (int k = 0; k < p.top; k++) {
        const Order best = block_reduce(mine, best_of, [](Order a, Order b) { return a > b ? a : b; });
        if (threadIdx.x == 0) {
            p.top_ids[row * p.top + k] = (int)(0xffffffffu - (uint32_t)best);
            p.top_log_prob[row * p.top + k] = log_prob(order_value((uint32_t)(best >> 32)));
        }
        if (mine == best) { // this thread's next one
            mine = 0;
            for (int i = threadIdx.x; i < vocab; i += THREADS) {
                const Order o = order_of(to_f32(v[i]), i);
                if (o < best && o > mine) mine = o;
            }
        }
    }
}

} // namespace

cudaError_t launch_log_probs(const rt_log_probs &op, int, cudaStream_t stream) {
    switch (op.dt) {
    case RT_F32: return launch_pdl(log_probs_kernel<float>, dim3((unsigned)op.rows), dim3(THREADS), 0, stream, op);
    case RT_F16: return launch_pdl(log_probs_kernel<__half>, dim3((unsigned)op.rows), dim3(THREADS), 0, stream, op);
    case RT_BF16: return launch_pdl(log_probs_kernel<__nv_bfloat16>, dim3((unsigned)op.rows), dim3(THREADS), 0, stream, op);
    default: return cudaErrorInvalidValue;
    }
}

} // namespace rt
