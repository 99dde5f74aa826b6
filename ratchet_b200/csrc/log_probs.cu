// Log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits, in one pass over them.
//
// In powers of two, t = v log2(e) - c with any reference c near the row's largest: S = sum 2^t, W = sum t 2^t,
//     ln p(token) = ln 2 (t(token) - log2 S),   entropy = ln 2 (log2 S - W / S).
//  * A row belongs to a CTA, or with few rows to a cluster's CTAs.  A thread takes 16-byte chunks, keeps a reference of its own that
//    moves only when a chunk is 2^8 above it, and its largest value; the threads' sums meet at the end.
//  * A token's place in the order is one 64-bit number: the value's bits made monotone, then the id from above, so that equal values
//    fall to the lower id and no two are equal.  The `top` largest lie in threads whose largest value is no smaller than the
//    top-th largest of all threads' largest, and are no smaller themselves: a bound for that from the warps' largest few, then only
//    those threads read their chunks again (from L2) and collect what reaches it, a few more values than asked for.  Each counts
//    how many are larger, which is its place.  Rows with more ties than the collection holds take the values one by one.
//  * What is not finite: -inf adds nothing (t is held at -2000, a power of zero).  A row that has a NaN or +inf is known by its
//    largest value.  A row of nothing but -inf, or of values whose t overflows (f32's and bf16's lowest), has S = 0.
#include <algorithm>

#include "common.cuh"
#include "kernels.hpp"

namespace rt {

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int UNROLL = 4;          // chunks a thread has in flight
constexpr int LIST = 64;           // thread maxima that the bound is taken from
constexpr int MOST = THREADS;      // values collected
constexpr int MAX_RANKS = 8;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float NO_REFERENCE = -1e38f, LOW = -2000.f;
using Order = unsigned long long;

// larger value = larger word; -0 counts as +0, NaN as the largest; 0 is no value's word
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0xffffffffu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k == 0xffffffffu ? 0x7fc00000u : k ^ 0x80000000u) : ~k);
}
__device__ __forceinline__ Order order_of(uint32_t bits, uint32_t id) { return (Order)bits << 32 | (0xffffffffu - id); }
constexpr uint32_t INF_BITS = 0xff800000u, MINUS_INF_BITS = 0x007fffffu; // order_bits(+inf), order_bits(-inf)

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float exp2_approx(float t) {
    float d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(t));
    return d;
}

// A chunk's values; 16-bit types take the largest (NaN if there is one) two at a time.
template <typename T> struct Chunk;
template <> struct Chunk<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void values(const uint4 &r, float (&v)[N]) {
        v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ float largest(const uint4 &r) {
        return max_nan(max_nan(__uint_as_float(r.x), __uint_as_float(r.y)), max_nan(__uint_as_float(r.z), __uint_as_float(r.w)));
    }
};
template <> struct Chunk<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void values(const uint4 &r, float (&v)[N]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ float largest(const uint4 &r) {
        const __half2 a = __hmax2_nan(*reinterpret_cast<const __half2 *>(&r.x), *reinterpret_cast<const __half2 *>(&r.y));
        const __half2 b = __hmax2_nan(*reinterpret_cast<const __half2 *>(&r.z), *reinterpret_cast<const __half2 *>(&r.w));
        const float2 f = __half22float2(__hmax2_nan(a, b));
        return max_nan(f.x, f.y);
    }
};
template <> struct Chunk<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void values(const uint4 &r, float (&v)[N]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    static __device__ __forceinline__ float largest(const uint4 &r) {
        const __nv_bfloat162 a = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162 *>(&r.x), *reinterpret_cast<const __nv_bfloat162 *>(&r.y));
        const __nv_bfloat162 b = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162 *>(&r.z), *reinterpret_cast<const __nv_bfloat162 *>(&r.w));
        const __nv_bfloat162 m = __hmax2_nan(a, b);
        const uint32_t w = *reinterpret_cast<const uint32_t *>(&m);
        return max_nan(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory"); }
template <typename V> __device__ __forceinline__ V load_peer(const V *p, uint32_t rank) {
    const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
    uint32_t b;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
    V v;
    if (sizeof(V) == 8) {
        unsigned long long w;
        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(w) : "r"(b) : "memory");
        v = *reinterpret_cast<V *>(&w);
    } else {
        uint32_t w;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(b) : "memory");
        v = *reinterpret_cast<V *>(&w);
    }
    return v;
}

// A reference and the sums taken with it.
struct Sums {
    float c, s, w;
    __device__ __forceinline__ void move(float to) { // `to` >= c
        const float f = exp2_approx(c - to);
        w = f > 0.f ? f * fmaf(s, c - to, w) : 0.f;
        s *= f;
        c = to;
    }
};

template <typename T> __global__ void __launch_bounds__(THREADS, 2) log_probs_kernel(const __grid_constant__ rt_log_probs p, int ranks) {
    constexpr int N = Chunk<T>::N;
    __shared__ float red[2][WARPS], meet[4]; // what the CTAs of a cluster tell: c, s, w of the slice
    __shared__ uint32_t bits_of[WARPS], list[LIST], slice_bits, bound;
    __shared__ int count;
    __shared__ Order found[MOST], top[RT_LOG_PROBS_MAX_TOP], all[MAX_RANKS * RT_LOG_PROBS_MAX_TOP], best_of[WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = ranks > 1 ? (int)cluster_rank() : 0;
    const long long row = blockIdx.x / ranks;
    const int vocab = (int)p.vocab;
    const T *const v = (const T *)p.logits + row * p.ld;
    // chunks lie on 16-byte boundaries: chunk i has values i N - shift .. + N - 1 of the row; the first and the last may be partial
    const int shift = (int)(reinterpret_cast<uintptr_t>(v) % 16 / sizeof(T)), chunks = (int)(((long long)vocab + shift + N - 1) / N);
    const uint4 *const base = reinterpret_cast<const uint4 *>(v - shift);
    const int per = (chunks + ranks - 1) / ranks, begin = min(chunks, rank * per), end = min(chunks, begin + per);

    if (tid == 0) count = 0;
    float token_value = 0.f;
    bool token_there = false;
    if (tid == 0 && rank == 0 && p.log_prob) {
        const int t = p.tokens[row];
        token_there = t >= 0 && t < vocab;
        if (token_there) token_value = to_f32(v[t]);
    }

    // ---- one pass: sums and the thread's largest value
    auto partial = [&](int i) { return (i == 0 && shift > 0) || (i == chunks - 1 && (long long)chunks * N - shift > vocab); };
    auto guarded = [&](int i) { // values outside the row as -inf
        T raw[N];
#pragma unroll
        for (int k = 0; k < N; k++) {
            const long long at = (long long)i * N - shift + k;
            raw[k] = at >= 0 && at < vocab ? v[at] : from_f32<T>(-INFINITY);
        }
        uint4 r;
        memcpy(&r, raw, 16);
        return r;
    };
    Sums sum{NO_REFERENCE, 0.f, 0.f};
    float largest = -INFINITY;
    bool any = false;
    auto take = [&](const uint4 &r) {
        const float m = Chunk<T>::largest(r);
        largest = max_nan(largest, m);
        const float mc = m * LOG2E;
        if (mc > sum.c + 8.f) sum.move(mc);
        float f[N];
        Chunk<T>::values(r, f);
#pragma unroll
        for (int k = 0; k < N; k++) {
            const float t = fmaxf(fmaf(f[k], LOG2E, -sum.c), LOW), e = exp2_approx(t);
            sum.s += e;
            sum.w = fmaf(e, t, sum.w);
        }
    };
    const int first_whole = begin + (begin < end && partial(begin)), last_whole = end - (end > first_whole && partial(end - 1));
    int i = first_whole + tid;
    for (; i + (UNROLL - 1) * THREADS < last_whole; i += UNROLL * THREADS) {
        uint4 r[UNROLL];
#pragma unroll
        for (int k = 0; k < UNROLL; k++) r[k] = __ldg(base + i + k * THREADS);
#pragma unroll
        for (int k = 0; k < UNROLL; k++) take(r[k]);
        any = true;
    }
    for (; i < last_whole; i += THREADS) take(__ldg(base + i)), any = true;
    // the partial chunks: the first one is thread 0's, the last one thread 32's
    const int odd = tid == 0 && first_whole > begin ? begin : tid == 32 && last_whole < end ? end - 1 : -1;
    if (odd >= 0) take(guarded(odd)), any = true;

    // ---- the CTA's sums and largest value
    const uint32_t mine = any ? order_bits(largest) : 0u;
    uint32_t warp_bits = __reduce_max_sync(0xffffffffu, mine);
    float c = sum.c;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, o));
    if (lane == 0) red[0][warp] = c, bits_of[warp] = warp_bits;
    // the bound's list: the largest few thread maxima of each warp that has chunks
    const int busy = min(WARPS, (last_whole - first_whole + 31) / 32 + 1), few = busy >= WARPS ? LIST / WARPS : min(32, LIST / busy);
    const int listed = p.top ? min(LIST, busy * few) : 0;
    if (p.top && warp < busy) {
        uint32_t left = mine;
        for (int k = 0; k < few; k++) {
            if (k > 0) warp_bits = __reduce_max_sync(0xffffffffu, left);
            const uint32_t who = __ballot_sync(0xffffffffu, left == warp_bits);
            if (lane == __ffs(who) - 1) {
                if (warp * few + k < LIST) list[warp * few + k] = left;
                left = 0;
            }
        }
    }
    __syncthreads();
    c = red[0][lane % WARPS];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, o));
    sum.move(c);
    float s = sum.s, w = sum.w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), w += __shfl_xor_sync(0xffffffffu, w, o);
    // (red[0] was read by all before it is written again: the shuffles above wait for the warp, the barrier for the CTA)
    if (tid < listed) { // the top-th largest of the list; 0 where it is shorter
        const uint32_t me = list[tid];
        int above = 0;
        for (int k = 0; k < listed; k++) above += list[k] > me || (list[k] == me && k < tid);
        if (above == p.top - 1) bound = me;
    }
    if (tid == 0 && listed < p.top) bound = 0;
    __syncthreads();
    if (lane == 0) red[0][warp] = s, red[1][warp] = w;
    if (p.top) {
        const uint32_t least = max(bound, 1u);
        if (mine >= least) { // this thread has values that may be among the largest
            auto collect = [&](const uint4 &r, int at) {
                float f[N];
                Chunk<T>::values(r, f);
#pragma unroll
                for (int k = 0; k < N; k++) {
                    const uint32_t b = order_bits(f[k]);
                    const long long id = (long long)at * N - shift + k;
                    if (b >= least && id >= 0 && id < vocab) {
                        const int to = atomicAdd(&count, 1);
                        if (to < MOST) found[to] = order_of(b, (uint32_t)id);
                    }
                }
            };
            int j = first_whole + tid;
            for (; j + (UNROLL - 1) * THREADS < last_whole; j += UNROLL * THREADS) {
                uint4 r[UNROLL];
#pragma unroll
                for (int k = 0; k < UNROLL; k++) r[k] = __ldg(base + j + k * THREADS);
#pragma unroll
                for (int k = 0; k < UNROLL; k++)
                    if (order_bits(Chunk<T>::largest(r[k])) >= least) collect(r[k], j + k * THREADS);
            }
            for (; j < last_whole; j += THREADS) {
                const uint4 r = __ldg(base + j);
                if (order_bits(Chunk<T>::largest(r)) >= least) collect(r, j);
            }
            if (odd >= 0) collect(guarded(odd), odd);
        }
        if (tid < p.top) top[tid] = 0;
    }
    __syncthreads();
    s = red[0][lane % WARPS], w = red[1][lane % WARPS];
    uint32_t bits = bits_of[lane % WARPS];
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), w += __shfl_xor_sync(0xffffffffu, w, o);
    bits = __reduce_max_sync(0xffffffffu, bits);
    if (p.top) {
        const int n = count;
        if (n <= MOST) {
            if (tid < n) {
                const Order me = found[tid];
                int above = 0;
                for (int k = 0; k < n; k++) above += found[k] > me;
                if (above < p.top) top[above] = me;
            }
        } else { // many equal values: one after the other, each thread with its largest below the last one taken
            Order last = ~0ull;
            auto next = [&]() {
                Order o = 0;
                auto look = [&](const uint4 &r, int at) {
                    float f[N];
                    Chunk<T>::values(r, f);
                    for (int k = 0; k < N; k++) {
                        const long long id = (long long)at * N - shift + k;
                        if (id < 0 || id >= vocab) continue;
                        const Order q = order_of(order_bits(f[k]), (uint32_t)id);
                        if (q < last && q > o) o = q;
                    }
                };
                for (int j = first_whole + tid; j < last_whole; j += THREADS) look(__ldg(base + j), j);
                if (odd >= 0) look(guarded(odd), odd);
                return o;
            };
            Order own = next();
            for (int k = 0; k < p.top; k++) {
                Order o = own;
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) {
                    const Order other = __shfl_xor_sync(0xffffffffu, o, d);
                    o = other > o ? other : o;
                }
                __syncthreads();
                if (lane == 0) best_of[warp] = o;
                __syncthreads();
                o = best_of[0];
                for (int d = 1; d < WARPS; d++) o = best_of[d] > o ? best_of[d] : o;
                if (tid == 0) top[k] = o;
                last = o;
                if (own == o) own = next();
            }
        }
    }

    // ---- the cluster's
    if (ranks > 1) {
        if (tid == 0) meet[0] = c, meet[1] = s, meet[2] = w, slice_bits = bits;
        cluster_sync();
        if (rank == 0) {
            float cs = NO_REFERENCE;
            bits = 0;
            for (int r = 0; r < ranks; r++) cs = fmaxf(cs, load_peer(&meet[0], r)), bits = max(bits, load_peer(&slice_bits, r));
            s = w = 0.f;
            for (int r = 0; r < ranks; r++) {
                Sums part{load_peer(&meet[0], r), load_peer(&meet[1], r), load_peer(&meet[2], r)};
                part.move(cs);
                s += part.s, w += part.w;
            }
            c = cs;
            const int n = ranks * p.top;
            if (tid < n) all[tid] = load_peer(&top[tid % p.top], tid / p.top);
            __syncthreads();
            if (tid < n) {
                const Order me = all[tid];
                int above = 0;
                for (int k = 0; k < n; k++) above += all[k] > me || (all[k] == me && k < tid); // (slices without enough values have zeros)
                if (above < p.top) top[above] = me; // (the peers read none of rank 0's after the barrier below; its own were read above)
            }
        }
        cluster_sync(); // no CTA leaves while it may be read
        if (rank != 0) return;
    }
    __syncthreads();

    // ---- the row
    bool nothing = bits <= MINUS_INF_BITS;
    const bool broken = bits >= INF_BITS; // +inf or NaN
    if (!nothing && !broken && !(s > 0.f)) {
        // values whose t overflows: the lowest of f32 or bf16 and nothing above.  Differences to the largest are exact enough.
        const float m = order_value(bits);
        s = w = 0.f;
        for (int j = tid; j < vocab; j += THREADS) {
            const float t = fmaxf((to_f32(v[j]) - m) * LOG2E, LOW), e = exp2_approx(t);
            s += e;
            w = fmaf(e, t, w);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), w += __shfl_xor_sync(0xffffffffu, w, o);
        __syncthreads();
        if (lane == 0) red[0][warp] = s, red[1][warp] = w;
        __syncthreads();
        s = red[0][lane % WARPS], w = red[1][lane % WARPS];
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), w += __shfl_xor_sync(0xffffffffu, w, o);
        c = NAN; // the reference is m
    }
    // differences to the largest value keep their bits, however far from zero the row lies
    const float log_s = log2f(s), m = order_value(bits), above = LN2 * (log_s - (c == c ? fmaf(m, LOG2E, -c) : 0.f)); // ln sum e^(v - m)
    auto log_prob = [&](float x) { return broken ? NAN : nothing ? -INFINITY : (x - m) - above; };
    if (tid == 0) {
        if (p.log_prob) p.log_prob[row] = token_there ? log_prob(token_value) : NAN;
        if (p.entropy) p.entropy[row] = broken ? NAN : nothing ? 0.f : LN2 * (log_s - w / s);
    }
    if (tid < p.top) {
        const Order o = top[tid];
        p.top_ids[row * p.top + tid] = (int)(0xffffffffu - (uint32_t)o);
        p.top_log_prob[row * p.top + tid] = log_prob(order_value((uint32_t)(o >> 32)));
    }
}

template <typename T> cudaError_t launch_t(const rt_log_probs &op, int sm_count, cudaStream_t stream) {
    // few rows: a cluster to a row, as long as every thread of it gets a chunk
    int ranks = 1;
    while (ranks < MAX_RANKS && op.rows * ranks * 2 <= 2LL * sm_count && op.vocab / Chunk<T>::N >= 2LL * ranks * THREADS) ranks *= 2;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(op.rows * ranks));
    lc.blockDim = dim3(THREADS);
    lc.stream = stream;
    cudaLaunchAttribute a[2];
    a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a[0].val.programmaticStreamSerializationAllowed = 1;
    a[1].id = cudaLaunchAttributeClusterDimension;
    a[1].val.clusterDim.x = (unsigned)ranks;
    a[1].val.clusterDim.y = a[1].val.clusterDim.z = 1;
    lc.attrs = a;
    lc.numAttrs = ranks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&lc, log_probs_kernel<T>, op, ranks);
}

} // namespace

cudaError_t launch_log_probs(const rt_log_probs &op, int sm_count, cudaStream_t stream) {
    switch (op.dt) {
    case RT_F32: return launch_t<float>(op, sm_count, stream);
    case RT_F16: return launch_t<__half>(op, sm_count, stream);
    case RT_BF16: return launch_t<__nv_bfloat16>(op, sm_count, stream);
    default: return cudaErrorInvalidValue;
    }
}

} // namespace rt
