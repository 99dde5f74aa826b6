// Log probabilities of given tokens, the entropy and the likeliest tokens of rows of logits, in one pass over them.
//
// In powers of two, t = v log2(e) - c with any reference c near the row's largest: S = sum 2^t, W = sum t 2^t,
//     ln p(token) = ln 2 (t(token) - log2 S),   entropy = ln 2 (log2 S - W / S).
//  * A row belongs to a CTA, or with few long rows to a cluster's CTAs.  A thread takes 16-byte chunks, keeps a reference of its own that
//    moves only when a chunk is 2^8 above it, and its largest value; the threads' sums meet at the end.
//  * A token's place in the order is one 64-bit number: the value's bits made monotone, then the id from above, so that equal values
//    fall to the lower id and no two are equal.  The `top` largest lie in threads whose largest value is no smaller than the
//    top-th largest of all threads' largest, and are no smaller themselves: a bound for that from the warps' largest few, then only
//    those threads read their chunks again (from L2) and collect what reaches it, a few more values than asked for.  Each counts
//    how many are larger, which is its place.  Rows with more ties than the collection holds take the values one by one.
//  * What is not finite: -inf counts as the type's lowest or -1e38, a power of zero.  A row that has a NaN or +inf is known by its
//    largest value, a row of nothing but -inf too.
//  * c is rounded as v log2(e) is not.  Rows so far from zero that this shows, and rows that never reach the first reference (f32's and
//    bf16's lowest as a mask), take the differences v - max first, in a second pass.
//
// 2048 bf16 rows of 51865, 20 likeliest: 55 us, 3.9 TB/s, 11.5 instructions a value; without the likeliest 43.5, 4.9 TB/s, 8.9 at 2.8 a
// cycle and SM, of them one exponential at 16 a cycle.  One f16 row 6.7 us: 4000 of 12000 cycles are the pass of one SM, the rest steps that
// follow from one another (asking, sums and list, collecting from L2, ranking).  A pass for each of the maximum, the sums and every
// likeliest token took 686 and 30 us.  Times that compare two forms below are of inputs that follow one another and half stay in L2:
// 52 us for the first.
#include <algorithm>

#include "common.cuh"
#include "f32x2.cuh"
#include "kernels.hpp"

namespace rt {

namespace {

constexpr int GROUP = 2, GROUPS = 4; // chunks a thread asks for and works on together, and how many such groups are on their way
constexpr int SEGMENT = 256;         // such groups whose values are added one after the other, 4 or 8 of a group to each of a sum's two
constexpr int LIST = 64;             // thread maxima that the bound is taken from, at most
constexpr int MOST = 512;          // values collected
constexpr int MAX_RANKS = 8;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float LOWEST = -1e38f; // values below it count as it: their t is finite and 2^t is 0
using Order = unsigned long long;

// larger value = larger word; -0 counts as +0, NaN as the largest; 0 is no value's word, nor is the largest one: a token's Order lies
// below ~0
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0xfffffffeu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); // (NaN's is a NaN)
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

// A chunk's values, and its largest (NaN if there is one): `wide` words hold the places' largest so far, 16-bit types two places a
// word.  raised() is the chunk with values below LOWEST (and NaN) lifted to about that, or to the type's lowest; START is the reference
// before any value: so far above those that their powers are 0 from the first one on.
template <typename T> struct Chunk;
template <> struct Chunk<float> {
    static constexpr int N = 4;
    static constexpr float START = -1e38f;
    static __device__ __forceinline__ void values(const uint4 &r, float (&v)[N]) {
        v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint32_t wider(uint32_t a, uint32_t b) { return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float widest(uint32_t a) { return __uint_as_float(a); }
    static __device__ __forceinline__ uint32_t raised(uint32_t a) { return __float_as_uint(fmaxf(__uint_as_float(a), LOWEST)); }
};
template <> struct Chunk<__half> {
    static constexpr int N = 8;
    static constexpr float START = -94300.f; // the lowest's t: -204 (from -1e38 it was +inf, and every masked row went the long way below)
    static __device__ __forceinline__ void values(const uint4 &r, float (&v)[N]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint32_t wider(uint32_t a, uint32_t b) {
        return h2_as_u32(__hmax2_nan(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b)));
    }
    static __device__ __forceinline__ float widest(uint32_t a) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a));
        return max_nan(f.x, f.y);
    }
    static __device__ __forceinline__ uint32_t raised(uint32_t a) { // -65504
        const uint32_t low = 0xfbfffbffu;
        return h2_as_u32(__hmax2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&low)));
    }
};
template <> struct Chunk<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr float START = -1e38f;
    static __device__ __forceinline__ void values(const uint4 &r, float (&v)[N]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    static __device__ __forceinline__ uint32_t as_word(__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t *>(&v); }
    static __device__ __forceinline__ uint32_t wider(uint32_t a, uint32_t b) {
        return as_word(__hmax2_nan(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&b)));
    }
    static __device__ __forceinline__ float widest(uint32_t a) { return max_nan(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)); }
    static __device__ __forceinline__ uint32_t raised(uint32_t a) { // -9.97e37
        const uint32_t low = 0xfe96fe96u;
        return as_word(__hmax2(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&low)));
    }
};
template <typename T> __device__ __forceinline__ uint32_t wide_of(const uint4 &r) {
    return Chunk<T>::wider(Chunk<T>::wider(r.x, r.y), Chunk<T>::wider(r.z, r.w));
}

// 16 bytes from global to shared memory behind the thread's back, and the wait for all but the newest `GROUPS` groups of them
__device__ __forceinline__ void copy_async(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int GROUPS> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(GROUPS) : "memory"); }

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

// The values at and above `least` of a row's slice, one by one in falling order: for rows of many equal values, which the collection
// does not hold.
template <typename T, int TH, typename Each>
__device__ __noinline__ void take_one_by_one(Each each, int vocab, int n, Order *top, Order *best_of) {
    Order last = ~0ull; // above every token's
    auto next = [&]() { // this thread's largest below the last one taken
        Order o = 0;
        each([&](float f, long long id) {
            if (id < 0 || id >= vocab) return;
            const Order q = order_of(order_bits(f), (uint32_t)id);
            if (q < last && q > o) o = q;
        });
        return o;
    };
    Order own = next();
    for (int k = 0; k < n; k++) {
        Order o = own;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const Order other = __shfl_xor_sync(0xffffffffu, o, d);
            o = other > o ? other : o;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) best_of[threadIdx.x >> 5] = o;
        __syncthreads();
        o = best_of[0];
        for (int d = 1; d < TH / 32; d++) o = best_of[d] > o ? best_of[d] : o;
        if (threadIdx.x == 0) top[k] = o;
        last = o;
        if (own == o) own = next();
    }
}

// TH threads; `ranks` CTAs of a cluster to a row.  LONG: a thread has more than a segment, and its sums are put aside after each
template <typename T, int TH, bool LONG> __global__ void __launch_bounds__(TH, TH == 256 ? 5 : 2) log_probs_kernel(const __grid_constant__ rt_log_probs p, int ranks) {
    constexpr int N = Chunk<T>::N, WARPS = TH / 32;
    __shared__ float3 sums_of[WARPS];
    __shared__ float kept[3][LONG ? TH : 1]; // sums of a thread's earlier segments: c, s, w
    __shared__ float meet[3]; // what the CTAs of a cluster tell: c, s, w of the slice
    __shared__ uint32_t bits_of[WARPS], list[LIST], slice_bits, bound;
    __shared__ int count, marked, redo;
    __shared__ short mark[TH];
    extern __shared__ __align__(16) uint4 ring[]; // [GROUPS][GROUP][TH], a thread's own places: no barriers
    __shared__ __align__(16) Order found[MOST], all[MAX_RANKS * RT_LOG_PROBS_MAX_TOP];
    __shared__ Order top[RT_LOG_PROBS_MAX_TOP], best_of[WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = ranks > 1 ? (int)cluster_rank() : 0;
    const long long row = ranks > 1 ? blockIdx.x / ranks : blockIdx.x;
    const int vocab = (int)p.vocab;
    const T *const v = (const T *)p.logits + row * p.ld;
    // chunks lie on 16-byte boundaries: chunk i has values i N - shift .. + N - 1 of the row; the first and the last may be partial
    const int shift = (int)(reinterpret_cast<uintptr_t>(v) % 16 / sizeof(T)), chunks = (int)(((long long)vocab + shift + N - 1) / N);
    const uint4 *const base = reinterpret_cast<const uint4 *>(v - shift);
    const int per = ranks > 1 ? (chunks + ranks - 1) / ranks : chunks, begin = min(chunks, rank * per), end = min(chunks, begin + per);

    if (tid == 0) count = marked = 0, bound = 0xffffffffu;
    float token_value = 0.f;
    bool token_there = false;
    if (tid == 0 && rank == 0 && p.log_prob) {
        const int t = p.tokens[row];
        token_there = t >= 0 && t < vocab;
        if (token_there) token_value = to_f32(v[t]);
    }

    // ---- one pass: sums and the thread's largest value
    const bool partial0 = shift > 0, partial1 = (long long)chunks * N - shift > vocab;
    const int first_whole = begin + (begin == 0 && begin < end && (partial0 || (chunks == 1 && partial1))), last_whole = end - (end > first_whole && end == chunks && partial1);
    // the partial chunks: the first one is thread 0's, the last one thread 32's
    const int odd = tid == 0 && first_whole > begin ? begin : tid == 32 && last_whole < end ? end - 1 : -1;
    auto guarded = [=](int i) { // values outside the row as -inf
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
    // the largest values of the thread's best and second-best group of chunks (NaN above all), and where the best one begins
    float c = Chunk<T>::START, best = -INFINITY, second = -INFINITY;
    int best_at = 0;
    unsigned long long s2 = 0, w2 = 0; // pairs of sums
    const unsigned long long log2e2 = pack2f(LOG2E, LOG2E);
    auto raise = [&](float m) { // the largest of what comes next
        const float mc = m * LOG2E;
        if (mc > c + 8.f) {
            Sums sum{c, sum2(s2), sum2(w2)};
            sum.move(mc);
            c = mc, s2 = pack2f(sum.s, 0.f), w2 = pack2f(sum.w, 0.f);
        }
    };
    auto add = [&](const uint4 &r) {
        const unsigned long long minus_c = pack2f(-c, -c);
        float f[N];
        Chunk<T>::values(make_uint4(Chunk<T>::raised(r.x), Chunk<T>::raised(r.y), Chunk<T>::raised(r.z), Chunk<T>::raised(r.w)), f);
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const unsigned long long t = fma2(pack2f(f[k], f[k + 1]), log2e2, minus_c);
            float t0, t1;
            unpack2f(t, t0, t1);
            const unsigned long long e = pack2f(exp2_approx(t0), exp2_approx(t1));
            s2 = add2(s2, e);
            w2 = fma2(e, t, w2);
        }
    };
    const int mine_of = last_whole - first_whole - tid, my_chunks = mine_of > 0 ? (mine_of + TH - 1) / TH : 0;
    const uint4 *from = base + first_whole + tid; // chunk k of the thread: from + k TH
    uint4 *const place = ring + tid;
    int asked = 0;
    auto ask = [&](int part) {
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(place + part * GROUP * TH);
#pragma unroll
        for (int k = 0; k < GROUP; k++)
            if (asked + k < my_chunks) copy_async(to + k * TH * 16, from + k * TH);
        copy_commit();
        asked += GROUP, from += GROUP * TH;
    };
#pragma unroll
    for (int k = 0; k < GROUPS; k++) ask(k);
    auto rank_group = [&](float m, int at) { // (the maxima keep a NaN, the minimum leaves it behind for the other: NaN is the largest)
        const float larger = max_nan(best, m);
        best_at = __float_as_uint(larger) != __float_as_uint(best) ? at : best_at; // (max.NaN has one NaN only)
        second = max_nan(second, fminf(best, m));
        best = larger;
    };
    auto with_kept = [&]() {
        Sums sum{c, sum2(s2), sum2(w2)}, before{kept[0][tid], kept[1][tid], kept[2][tid]};
        before.move(c);
        sum.s += before.s, sum.w += before.w;
        return sum;
    };
    int left = my_chunks, part = 0;
    auto step = [&]() {
        copy_wait<GROUPS - 1>();
        uint4 r[GROUP];
#pragma unroll
        for (int k = 0; k < GROUP; k++) r[k] = place[(part * GROUP + k) * TH];
        uint32_t wide = wide_of<T>(r[0]);
#pragma unroll
        for (int k = 1; k < GROUP; k++) wide = Chunk<T>::wider(wide, wide_of<T>(r[k]));
        const float m = Chunk<T>::widest(wide);
        raise(m);
        rank_group(m, my_chunks - left);
        ask(part); // (into the places just read)
#pragma unroll
        for (int k = 0; k < GROUP; k++) add(r[k]);
        left -= GROUP, part = (part + 1) % GROUPS;
    };
    if constexpr (LONG) {
        while (left >= GROUP) {
            for (const int stop = max(left - SEGMENT * GROUP, GROUP - 1); left > stop;) step();
            if (left < GROUP) break;
            const Sums sum = left + SEGMENT * GROUP < my_chunks ? with_kept() : Sums{c, sum2(s2), sum2(w2)};
            kept[0][tid] = sum.c, kept[1][tid] = sum.s, kept[2][tid] = sum.w;
            s2 = w2 = 0;
        }
    } else {
        while (left >= GROUP) step();
    }
    copy_wait<0>();
    for (int k = 0; k < left; k++) {
        const uint4 r = place[(part * GROUP + k) * TH];
        const float m = Chunk<T>::widest(wide_of<T>(r));
        raise(m);
        rank_group(m, my_chunks - left + k);
        add(r);
    }
    float odd_largest = -INFINITY;
    if (odd >= 0) {
        const uint4 r = guarded(odd);
        odd_largest = Chunk<T>::widest(wide_of<T>(r));
        raise(odd_largest);
        add(r);
    }

    // ---- the warps' sums, and the list for the bound: the largest few thread maxima of each warp that has chunks
    const uint32_t mine = my_chunks > 0 || odd >= 0 ? order_bits(max_nan(best, odd_largest)) : 0u;
    uint32_t warp_bits = __reduce_max_sync(0xffffffffu, mine);
    Sums sum = LONG && my_chunks >= (SEGMENT + 1) * GROUP ? with_kept() : Sums{c, sum2(s2), sum2(w2)};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, o));
    sum.move(c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum.s += __shfl_xor_sync(0xffffffffu, sum.s, o), sum.w += __shfl_xor_sync(0xffffffffu, sum.w, o);
    if (lane == 0) sums_of[warp] = make_float3(c, sum.s, sum.w), bits_of[warp] = warp_bits;
    const int busy = min(WARPS, (last_whole - first_whole + 31) / 32 + 1), few = min(32, (p.top * 3 / 2 + busy - 1) / busy), listed = busy * few; // (LIST at most)
    if (warp < busy) {
        uint32_t rest = mine;
        for (int k = 0; k < few; k++) {
            if (k > 0) warp_bits = __reduce_max_sync(0xffffffffu, rest);
            const uint32_t who = __ballot_sync(0xffffffffu, rest == warp_bits);
            if (lane == __ffs(who) - 1) list[warp * few + k] = rest, rest = 0;
        }
    }
    __syncthreads();

    // ---- the slice's sums, in the first warp; the bound, by the next two
    float s = 0.f, w = 0.f;
    uint32_t bits = 0;
    if (warp == 0) {
        const float3 of = sums_of[lane % WARPS];
        sum = Sums{of.x, of.y, of.z};
        c = of.x;
        bits = __reduce_max_sync(0xffffffffu, bits_of[lane % WARPS]);
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) c = fmaxf(c, __shfl_xor_sync(0xffffffffu, c, o));
        sum.move(c);
        s = sum.s, w = sum.w;
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), w += __shfl_xor_sync(0xffffffffu, w, o);
    }
    if (p.top) {
        // the top-th largest of the list is the smallest that fewer than `top` are larger than; a list that is too short has none
        if (tid >= 32 && tid - 32 < listed) {
            const uint32_t me = list[tid - 32];
            int above = listed < p.top ? p.top : 0;
#pragma unroll 8
            for (int k = 0; k < listed; k++) above += list[k] > me;
            if (above < p.top) atomicMin(&bound, me);
        }
        if (tid == 0 && listed < p.top) bound = 0;
        if (tid < p.top) top[tid] = 0;
        __syncthreads();
        const uint32_t least = max(bound, 1u);
        auto push = [&](float f, uint32_t id) { // (an id before the row's first or behind its last is no less than vocab)
            const uint32_t b = order_bits(f);
            if (b >= least && id < (uint32_t)vocab) {
                const int to = atomicAdd(&count, 1);
                if (to < MOST) found[to] = order_of(b, id);
            }
        };
        // A thread that has some of the largest looks at its best group again; where the second-best has some too, it is marked, and
        // a warp goes over all of its chunks, a chunk a lane, and over a chunk that has some a value a lane.
        if (mine >= least) {
            if (order_bits(second) >= least) {
                mark[atomicAdd(&marked, 1)] = (short)tid;
            } else if (order_bits(best) >= least) {
#pragma unroll
                for (int g = 0; g < GROUP; g++) {
                    if (best_at + g >= my_chunks) break;
                    const int at = first_whole + tid + (best_at + g) * TH;
                    const uint4 r = __ldg(base + at);
                    float f[N];
                    Chunk<T>::values(r, f);
#pragma unroll
                    for (int k = 0; k < N; k++) push(f[k], (uint32_t)at * N - shift + k);
                }
            }
            if (odd >= 0) {
                float f[N];
                Chunk<T>::values(guarded(odd), f);
#pragma unroll
                for (int k = 0; k < N; k++) push(f[k], (uint32_t)odd * N - shift + k);
            }
        }
        __syncthreads();
        const int n_marked = marked;
        for (int m = warp; m < n_marked; m += WARPS)
            for (int at0 = first_whole + mark[m]; at0 < last_whole; at0 += 32 * TH) {
                const int at = at0 + lane * TH;
                uint4 r = make_uint4(0, 0, 0, 0);
                bool has = false;
                if (at < last_whole) {
                    r = __ldg(base + at);
                    has = order_bits(Chunk<T>::widest(wide_of<T>(r))) >= least;
                }
                for (uint32_t who = __ballot_sync(0xffffffffu, has); who; who &= who - 1) {
                    const int src = __ffs(who) - 1;
                    const uint4 u = make_uint4(__shfl_sync(0xffffffffu, r.x, src), __shfl_sync(0xffffffffu, r.y, src), __shfl_sync(0xffffffffu, r.z, src),
                                               __shfl_sync(0xffffffffu, r.w, src));
                    float f[N];
                    Chunk<T>::values(u, f);
                    float mine_of_it = f[0];
#pragma unroll
                    for (int k = 1; k < N; k++) mine_of_it = lane == k ? f[k] : mine_of_it;
                    if (lane < N) push(mine_of_it, (uint32_t)(at0 + src * TH) * N - shift + lane);
                }
            }
        __syncthreads();
        const int n = count;
        if (n <= MOST) {
            for (int e = tid; e < n; e += TH) {
                const Order me = found[e];
                int above = 0;
#pragma unroll 4
                for (int k = 0; k < n; k++) above += found[k] > me;
                if (above < p.top) top[above] = me;
            }
        } else {
            take_one_by_one<T, TH>([=](auto look) {
                auto values = [=](const uint4 &r, int at) {
                    float f[N];
                    Chunk<T>::values(r, f);
                    for (int k = 0; k < N; k++) look(f[k], (long long)at * N - shift + k);
                };
#pragma unroll 1
                for (int at = first_whole + tid; at < last_whole; at += TH) values(__ldg(base + at), at);
                if (odd >= 0) values(guarded(odd), odd);
            }, vocab, p.top, top, best_of);
        }
    }

    // ---- the cluster's
    if (ranks > 1) {
        if (tid == 0) meet[0] = c, meet[1] = s, meet[2] = w, slice_bits = bits;
        cluster_sync();
        if (rank == 0) {
            float cs = Chunk<T>::START;
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
            const int e = tid >> 1; // two threads to a value
            const Order me = e < n ? all[e] : 0;
            int above = 0;
#pragma unroll 4
            for (int k = tid & 1; k < n; k += 2) above += all[k] > me || (all[k] == me && k < e); // (slices without enough values have zeros)
            above += __shfl_xor_sync(0xffffffffu, above, 1);
            if (e < n && above < p.top) top[above] = me; // (nobody else reads this CTA's any more)
        }
        cluster_sync(); // no CTA leaves while it may be read
        if (rank != 0) return;
    }
    // ---- the row, in the first warp, which has c, s, w and the largest value's bits
    bool nothing = bits <= MINUS_INF_BITS;
    const bool broken = bits >= INF_BITS; // +inf or NaN
    // The reference serves where the largest value's power is an ordinary number: it lies 8 powers below the largest at most, and where it
    // does not, it was rounded (beyond 2^24) or is none of the row's.  Then, or where a t overflowed, the sums are taken again.
    if (tid == 0) redo = !nothing && !broken && !(fabsf(fmaf(order_value(bits), LOG2E, -c)) <= 9.f && w == w), slice_bits = bits;
    __syncthreads();
    if (redo) {
        // rows of the type's lowest and nothing above, of a finite mask over everything, of logits beyond 1e7: differences to the largest
        // are exact enough
        const float m = order_value(slice_bits);
        s = w = 0.f;
        for (uint32_t j = tid; j < (uint32_t)vocab;) { // (vocab + TH may pass 2^31)
            float ps = 0.f, pw = 0.f;
            const uint32_t stop = min((uint32_t)vocab, j + 8 * SEGMENT * TH);
#pragma unroll 4
            for (; j < stop; j += TH) {
                const float t = fmaxf((to_f32(v[j]) - m) * LOG2E, LOWEST), e = exp2_approx(t);
                ps += e;
                pw = fmaf(e, t, pw);
            }
            s += ps, w += pw;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), w += __shfl_xor_sync(0xffffffffu, w, o);
        if (lane == 0) sums_of[warp] = make_float3(0.f, s, w);
        __syncthreads();
        s = sums_of[lane % WARPS].y, w = sums_of[lane % WARPS].z;
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), w += __shfl_xor_sync(0xffffffffu, w, o);
        c = NAN; // the reference is m
    }
    if (warp > 0) return;
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

template <typename T, int TH, bool LONG> cudaError_t launch_kernel(const rt_log_probs &op, int ranks, cudaStream_t stream) {
    constexpr size_t RING = GROUPS * GROUP * TH * sizeof(uint4);
    static SmemAttr attr;
    cudaError_t e = attr.ensure(log_probs_kernel<T, TH, LONG>, RING);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(op.rows * ranks));
    lc.blockDim = dim3(TH);
    lc.dynamicSmemBytes = RING;
    lc.stream = stream;
    cudaLaunchAttribute a[2];
    a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a[0].val.programmaticStreamSerializationAllowed = 1;
    a[1].id = cudaLaunchAttributeClusterDimension;
    a[1].val.clusterDim.x = (unsigned)ranks;
    a[1].val.clusterDim.y = a[1].val.clusterDim.z = 1;
    lc.attrs = a;
    lc.numAttrs = ranks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&lc, log_probs_kernel<T, TH, LONG>, op, ranks);
}

// f32 sums of very many terms that are alike drift.  (Segments in every row: 2048 bf16 rows of 51865 52.9 us, 52.1 without; 16 f32 rows
// 10.0 and 9.9.)
template <typename T, int TH> cudaError_t launch_threads(const rt_log_probs &op, int ranks, cudaStream_t stream) {
    return op.vocab > (long long)SEGMENT * GROUP * Chunk<T>::N * TH * ranks ? launch_kernel<T, TH, true>(op, ranks, stream)
                                                                            : launch_kernel<T, TH, false>(op, ranks, stream);
}

template <typename T> cudaError_t launch_t(const rt_log_probs &op, int sm_count, cudaStream_t stream) {
    // Many rows: the work that a row costs beyond its values goes by its warps (2048 bf16 rows of 51865, 20 likeliest: 53 us with 256
    // threads, 74 with 512, before both gained 1; 200 f16 rows 17 and 12).  Few: more threads to a row, and a cluster's CTAs, then as many
    // as have some four chunks a thread, only where a thread alone would have more than 32: two cluster barriers cost more than they save
    // below that (a row of 51865 f16 7.1 us, 8.0 as two CTAs; of 160000 11.5 alone, 10.4 as two, 8.7 as eight; 16 f32 rows of 51865 10.0,
    // 11.8 as four).
    if (op.rows > 2LL * sm_count) return launch_threads<T, 256>(op, 1, stream);
    int ranks = 1;
    while (ranks < MAX_RANKS && op.rows * ranks * 2 <= 2LL * sm_count && op.vocab / Chunk<T>::N > (ranks == 1 ? 32LL : 4LL) * ranks * 512) ranks *= 2;
    return launch_threads<T, 512>(op, ranks, stream);
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
