// What stands between two blocks: h = a r + b g N_post(y), x = N_pre(h), in one pass over the rows.
//
// Memory-bound: r and y are read once, h and x written once.  Means and variances are taken in two passes over values that are at
// hand (centre first, then squares: no cancellation), in f32, the sums in a fixed order, and x comes from h before its rounding.
//  * Many rows: teams of threads stay and walk their rows, 16 values a thread in registers, the next rows on their way into shared
//    memory by bulk copies.  The gate and both norms' weights stay in registers from row to row, folded into one factor and one
//    summand for h and one of each for x, and the arithmetic goes by packed pairs.
//  * Few rows: a thread per 16 bytes of the row, which asks for gate and weights together with the row instead of one after the other.
//  * Longer rows: a CTA with more values a thread, or loops over the row, once per sum, that find it in L1 from the second pass on.
//
// 8192 bf16 rows of 2560, rms on both sides, a gate a sequence: 32.8 us, 5.1 TB/s (a CTA a row without the ring: 44; with means and
// biases 43.8, a gate behind them 46.6: four sums a row instead of two, 128 registers instead of 96).  What is left is instructions,
// 25 a value, 2.2 a cycle and SM with 20 warps, and the start.  Rows of 2561, all off the 16-byte boundary, with a sixth warp for one
// value: 52.5 us.  One row: 2.5 us, the launch.
#include <algorithm>
#include <cfloat>
#include <utility>

#include "common.cuh"
#include "f32x2.cuh"
#include "kernels.hpp"
#include "umma_gemv.cuh"

namespace rt {

namespace {

struct NormParams {
    int kind, f32; // rt_norm_kind; weight and bias are f32 (else the activations' type)
    float eps;
    const void *weight, *bias;
};

struct ResidualNormParams {
    const void *r, *y, *gate;
    void *h, *x;
    long long r_ld, y_ld, h_ld, x_ld;
    int rows, d, rows_per_gate; // 0: one gate for all rows
    float a, b, inv_d;
    NormParams post, pre;
};

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

// VEC values of T as they lie in memory: 16-byte accesses, or one value
template <typename T, int VEC> struct Values {
    static constexpr int WORDS = VEC * (int)sizeof(T) / 16;
    uint4 raw[WORDS];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < WORDS; i++) raw[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < WORDS; i++) raw[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    __device__ __forceinline__ void load_shared(uint32_t a) {
#pragma unroll
        for (int i = 0; i < WORDS; i++) raw[i] = lds128(a + 16 * i);
    }
    __device__ __forceinline__ void keep(int from, int to) { // 0 but for values from .. to - 1
        constexpr int PER = 4 / sizeof(T);
        uint32_t *const w = reinterpret_cast<uint32_t *>(raw);
#pragma unroll
        for (int k = 0; k < 4 * WORDS; k++) {
            const uint32_t low = k * PER >= from && k * PER < to ? PER == 2 ? 0xffffu : 0xffffffffu : 0u;
            const uint32_t high = PER == 2 && k * PER + 1 >= from && k * PER + 1 < to ? 0xffff0000u : 0u;
            w[k] &= low | high;
        }
    }
    __device__ __forceinline__ void get(float (&v)[VEC]) const {
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
            constexpr int PER = 4 / sizeof(T); // values of a word
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (sizeof(T) == 4) v[i * 4 + k] = __uint_as_float(w[k]);
                else if (cuda::std::is_same<T, __half>::value) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
                    v[(i * 4 + k) * PER] = f.x, v[(i * 4 + k) * PER + PER - 1] = f.y;
                } else {
                    v[(i * 4 + k) * PER] = __uint_as_float(w[k] << 16), v[(i * 4 + k) * PER + PER - 1] = __uint_as_float(w[k] & 0xffff0000u);
                }
            }
        }
    }
};
template <typename T> struct Values<T, 1> {
    T raw;
    __device__ __forceinline__ void clear() { raw = from_f32<T>(0.f); }
    __device__ __forceinline__ void load(const T *p) { raw = *p; }
    __device__ __forceinline__ void keep(int, int) {}
    __device__ __forceinline__ void load_shared(uint32_t a) {
        if constexpr (sizeof(T) == 4) {
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(raw) : "r"(a) : "memory");
        } else {
            unsigned short w;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(a) : "memory");
            raw = *reinterpret_cast<const T *>(&w);
        }
    }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = to_f32(raw); }
};

template <typename T, int VEC> __device__ __forceinline__ void store_values(T *p, const float *v) {
    if (VEC == 1) {
        *p = from_f32<T>(v[0]);
    } else {
        alignas(16) T raw[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) raw[i] = from_f32<T>(v[i]);
#pragma unroll
        for (int i = 0; i < (int)(VEC * sizeof(T) / 16); i++) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(raw)[i];
    }
}

// weight or bias, f32 or of the activations' type
template <typename T, int VEC> struct Param {
    Values<T, VEC> own;
    Values<float, VEC> f;
    __device__ __forceinline__ void load(const void *p, int f32, int i) {
        if (f32) f.load((const float *)p + i);
        else own.load((const T *)p + i);
    }
    __device__ __forceinline__ void get(int f32, float (&v)[VEC]) const {
        if (f32) f.get(v);
        else own.get(v);
    }
};

// Sum over the team, a warp or the CTA.  A CTA's warps meet in shared memory, each reduction of a row in a slot of its own (`slot`,
// zero past the last warp), so one barrier per reduction is enough; the order of the additions is fixed.
template <bool WARP> __device__ __forceinline__ float team_sum(float v, uint32_t slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (WARP) return v;
    if ((threadIdx.x & 31) == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(slot + threadIdx.x / 32 * 4), "f"(v) : "memory");
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < (int)blockDim.x; w += 128) {
        const uint4 f = lds128(slot + w / 8);
        v += (__uint_as_float(f.x) + __uint_as_float(f.y)) + (__uint_as_float(f.z) + __uint_as_float(f.w));
    }
    return v;
}
__device__ __forceinline__ void clear_sums(float (*red)[32], int slots) { // before a barrier
    for (int i = threadIdx.x; i < slots * 32; i += blockDim.x) red[0][i] = 0.f;
}

// A CTA per row, the row in registers.  VEC values per access, C accesses per thread and operand; thread t holds values
// (c * threads + t) * VEC .. in access c.  VEC divides d and every ld, so no access crosses a row's end.  EARLY: weights and gate are
// asked for with the row.
template <typename T, int VEC, int C, bool EARLY>
__global__ void __launch_bounds__(EARLY && (VEC == 1 || sizeof(T) == 4) ? 1024 : 512) residual_norm_kernel(const __grid_constant__ ResidualNormParams p) {
    __shared__ __align__(16) float red[4][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t red0 = umma_gemv::smem_u32(red);
    clear_sums(red, 4);
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int t = threadIdx.x, team = blockDim.x, row = blockIdx.x;
    const int d = p.d;
    Values<T, VEC> r[C], y[C];
    const T *const rp = (const T *)p.r + (long long)row * p.r_ld, *const yp = (const T *)p.y + (long long)row * p.y_ld;
    const T *const gate = p.gate ? (const T *)p.gate + (p.rows_per_gate ? (long long)((unsigned)row / (unsigned)p.rows_per_gate) * d : 0) : nullptr;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = (c * team + t) * VEC;
        r[c].clear(), y[c].clear();
        if (e >= d) continue;
        if (p.y) y[c].load(yp + e);
        if (p.r) r[c].load(rp + e);
    }
    constexpr int E = EARLY ? C : 1;
    Param<T, VEC> wpost[E], bpost[E], wpre[E], bpre[E];
    Values<T, VEC> gv[E];
    auto early = [&](int c, int e) {
        if (p.post.weight) wpost[c].load(p.post.weight, p.post.f32, e);
        if (p.post.bias) bpost[c].load(p.post.bias, p.post.f32, e);
        if (gate) gv[c].load(gate + e);
    };
    if (EARLY) {
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int e = (c * team + t) * VEC;
            if (e >= d) continue;
            early(c, e);
            if (p.pre.weight) wpre[c].load(p.pre.weight, p.pre.f32, e);
            if (p.pre.bias) bpre[c].load(p.pre.bias, p.pre.f32, e);
        }
    }

    // ---- the block's norm: its mean and scale
    float mean = 0.f, scale = 1.f;
    if (p.post.kind == RT_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            float u[VEC];
            y[c].get(u);
#pragma unroll
            for (int i = 0; i < VEC; i++) s += u[i]; // (0 past the row's end)
        }
        mean = team_sum<false>(s, red0 + 128 * 0) * p.inv_d;
    }
    if (p.post.kind != RT_NORM_NONE) {
        float q = 0.f;
#pragma unroll
        for (int c = 0; c < C; c++) {
            if ((c * team + t) * VEC >= d) continue;
            float u[VEC];
            y[c].get(u);
#pragma unroll
            for (int i = 0; i < VEC; i++) q = fmaf(u[i] - mean, u[i] - mean, q);
        }
        scale = rsqrtf(team_sum<false>(q, red0 + 128 * 1) * p.inv_d + p.post.eps);
    }

    // ---- h
    float h[C][VEC];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = (c * team + t) * VEC, k = EARLY ? c : 0;
#pragma unroll
        for (int i = 0; i < VEC; i++) h[c][i] = 0.f;
        if (e >= d) continue;
        if (!EARLY) early(0, e);
        float u[VEC], v[VEC];
        y[c].get(u);
#pragma unroll
        for (int i = 0; i < VEC; i++) u[i] = (u[i] - mean) * scale;
        if (p.post.weight) {
            wpost[k].get(p.post.f32, v);
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] *= v[i];
        }
        if (p.post.bias) {
            bpost[k].get(p.post.f32, v);
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] += v[i];
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) u[i] *= p.b;
        if (gate) {
            gv[k].get(v);
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] *= v[i];
        }
        if (p.r) {
            r[c].get(v);
#pragma unroll
            for (int i = 0; i < VEC; i++) h[c][i] = p.y ? fmaf(p.a, v[i], u[i]) : p.a * v[i];
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++) h[c][i] = u[i];
        }
        if (p.h) store_values<T, VEC>((T *)p.h + (long long)row * p.h_ld + e, h[c]);
    }
    if (p.pre.kind == RT_NORM_NONE) return;

    // ---- x
    if (p.pre.kind == RT_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) s += h[c][i];
        mean = team_sum<false>(s, red0 + 128 * 2) * p.inv_d;
#pragma unroll
        for (int c = 0; c < C; c++)
            if ((c * team + t) * VEC < d)
#pragma unroll
                for (int i = 0; i < VEC; i++) h[c][i] -= mean;
    }
    float q = 0.f;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < VEC; i++) q = fmaf(h[c][i], h[c][i], q);
    scale = rsqrtf(team_sum<false>(q, red0 + 128 * 3) * p.inv_d + p.pre.eps);
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = (c * team + t) * VEC, k = EARLY ? c : 0;
        if (e >= d) continue;
        if (!EARLY && p.pre.weight) wpre[0].load(p.pre.weight, p.pre.f32, e);
        if (!EARLY && p.pre.bias) bpre[0].load(p.pre.bias, p.pre.f32, e);
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) h[c][i] *= scale;
        if (p.pre.weight) {
            wpre[k].get(p.pre.f32, v);
#pragma unroll
            for (int i = 0; i < VEC; i++) h[c][i] *= v[i];
        }
        if (p.pre.bias) {
            bpre[k].get(p.pre.f32, v);
#pragma unroll
            for (int i = 0; i < VEC; i++) h[c][i] += v[i];
        }
        store_values<T, VEC>((T *)p.x + (long long)row * p.x_ld + e, h[c]);
    }
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Teams that walk rows, a warp each (blockDim.y of them in a CTA) or the CTA.  A team's rows are consecutive, `share` of them; each warp
// holds 32 N consecutive values of a row, of which a thread's are VEC every 32 VEC: all but the last warp go without predicates and
// with constant offsets.  `stages` rows are in shared memory or on their way there.
// SHIFT: rows start s values behind a 16-byte boundary, every operand's alike.  s is the same in every `period`-th row, so a team
// takes such rows only, and its threads' values sit at the same places in each: s values before those of an aligned row.  The
// 16-byte words that hold the row are copied, which in the first and the last row would reach outside the tensor: those are read where
// they are.  VEC = 1: the same copies for operands that differ in s, value by value.
// Form: PLAIN has no means and no biases, which leaves the registers for more teams; GATED a gate behind a bias, where an infinite gate
// may not be folded into both (8192 bf16 rows of 2560, layer norms, a gate a sequence: 46.8 us, 45.3 without that, in turn).
enum Form { PLAIN, MEANS, GATED };
constexpr int N = 16, MAX_STAGES = 4, MAX_TEAMS = 8, WALK_SMEM = 200 * 1024;
constexpr int MIN_WALK_D = 8; // 16 bytes: the words of a row that is neither first nor last lie in the tensor
template <Form F> constexpr int WALK_THREADS = F == PLAIN ? 640 : 512; // of an SM, at 96 or 128 registers

template <bool ALIGNED> __host__ __device__ constexpr int walk_operand_bytes(int row_bytes) { // of a stage
    return ALIGNED ? row_bytes : (row_bytes + 15) / 16 * 16 + 16;
}

template <typename T, int VEC, bool WARP, Form F, bool SHIFT>
__global__ void __launch_bounds__(WARP ? 32 * MAX_TEAMS : WALK_THREADS<F>, WARP ? 2 : 1) residual_norm_walk_kernel(const __grid_constant__ ResidualNormParams p, int share, int stages, int period) {
    constexpr int C = N / VEC;
    constexpr bool ALIGNED = VEC > 1 && !SHIFT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(16) float red[2][4][32]; // two rows' reductions: a warp may be one row ahead of another
    __shared__ __align__(8) unsigned long long bars[MAX_TEAMS][MAX_STAGES];
    __shared__ int abort_flag;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int t = threadIdx.x, y0 = WARP ? threadIdx.y : 0;
    const int d = p.d, row_bytes = d * (int)sizeof(T), op_bytes = walk_operand_bytes<ALIGNED>(row_bytes);
    const int stage_bytes = op_bytes * ((p.r != nullptr) + (p.y != nullptr));
    const int team = blockIdx.x * (WARP ? blockDim.y : 1) + y0, P = SHIFT ? period : 1; // the team's rows: first, first + P, ..
    const long long before = (long long)(team / P) * share, first = team % P + before * P;
    const int n = (int)max(0LL, min((long long)share, (p.rows - team % P + P - 1) / P - before));
    uint32_t bar0 = umma_gemv::smem_u32(&bars[y0][0]), ring0 = umma_gemv::smem_u32(smem) + y0 * stages * stage_bytes, red0 = umma_gemv::smem_u32(red);
    asm volatile("" : "+r"(bar0), "+r"(ring0), "+r"(red0)); // held, not worked out anew in each row
    if (!WARP) clear_sums(red[0], 8);
    if (t == 0) {
        if (y0 == 0) abort_flag = 0;
        for (int k = 0; k < stages; k++) umma_gemv::mbar_init(bar0 + 8 * k, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const T *const yp = (const T *)p.y + first * p.y_ld, *const rp = (const T *)p.r + first * p.r_ld;
    const long long y_step = p.y_ld * P, r_step = p.r_ld * P;
    auto row_of = [&](int i) { return first + (long long)i * P; };
    auto in_place = [&](int i) { return !ALIGNED && (row_of(i) == 0 || row_of(i) == p.rows - 1); };
    int asked = 0; // rows asked for, by thread 0 of the team
    auto ask = [&](int k) { // the next row, into stage k
        const uint32_t to = ring0 + k * stage_bytes, bar = bar0 + 8 * k;
        auto copy = [&](uint32_t dst, const T *src) {
            const uint32_t skip = (uint32_t)reinterpret_cast<uintptr_t>(src) & 15;
            bulk_load(dst, reinterpret_cast<const uint8_t *>(src) - skip, (skip + row_bytes + 15) & ~15u, bar);
        };
        if (in_place(asked)) {
            mbar_expect(bar, 0);
        } else {
            const T *const y = yp + asked * y_step, *const r = rp + asked * r_step;
            auto bytes = [&](const T *src) { return (((uint32_t)reinterpret_cast<uintptr_t>(src) & 15) + row_bytes + 15) & ~15u; };
            mbar_expect(bar, (p.y ? bytes(y) : 0) + (p.r ? bytes(r) : 0));
            if (p.y) copy(to, y);
            if (p.r) copy(to + (p.y ? op_bytes : 0), r);
        }
        asked++;
    };
    if (t == 0)
        for (int k = 0; k < min(n, stages); k++) ask(k);

    // h = mul (y - mean) scale + add + a r,  x = wx (h - mean) scale + bx
    float mul[N], add[N], wx[N], bx[N];
    float v[VEC];
    const int at0 = (t >> 5) * 32 * N + (t & 31) * VEC;
    const int s = SHIFT ? (int)((uint32_t)reinterpret_cast<uintptr_t>(p.y ? yp : rp) & 15) / (int)sizeof(T) : 0;
    const bool full = (t >> 5) * 32 * N >= s && (t >> 5) * 32 * N + 32 * N <= s + d; // the warp's part of the row
    auto at = [&](int c) { return at0 + c * 32 * VEC; };
    auto index = [&](int j) { return at(j / VEC) + j % VEC - s; }; // of value j in the row
    auto valid = [&](int j) { return SHIFT ? (unsigned)index(j) < (unsigned)d : at(j / VEC) < d; };
    auto take_param = [&](const void *from, bool f32, float(&to)[N]) { // all on their way before the first is used; past the row's end its last ones
        auto values = [&](auto *q, auto value) {
            constexpr int W = SHIFT ? 1 : VEC;
            decltype(value) raw[N / W];
#pragma unroll
            for (int c = 0; c < N / W; c++) raw[c].load(q + (SHIFT ? max(0, min(index(c), d - 1)) : min(at(c), d - VEC)));
#pragma unroll
            for (int c = 0; c < N / W; c++) {
                float of[W];
                raw[c].get(of);
#pragma unroll
                for (int j = 0; j < W; j++) to[c * W + j] = of[j];
            }
        };
        if (f32) values((const float *)from, Values<float, SHIFT ? 1 : VEC>());
        else values((const T *)from, Values<T, SHIFT ? 1 : VEC>());
    };
    auto fill = [&](float(&to)[N], float value) {
#pragma unroll
        for (int j = 0; j < N; j++) to[j] = value;
    };
    if (p.pre.weight) take_param(p.pre.weight, p.pre.f32, wx);
    else fill(wx, 1.f);
    if (F != PLAIN && p.pre.bias) take_param(p.pre.bias, p.pre.f32, bx);
    else fill(bx, 0.f);
    bool wild = false; // an infinite b g before a bias: the thread's values go by the formula's own order
    auto take_gate = [&](long long which) {
        float w[N];
        wild = false;
        if (p.post.weight) take_param(p.post.weight, p.post.f32, w);
        else fill(w, 1.f);
        if (F != PLAIN && p.post.bias) take_param(p.post.bias, p.post.f32, add);
        else fill(add, 0.f);
        if (p.gate) take_param((const T *)p.gate + which * d, sizeof(T) == 4, mul);
        else fill(mul, 1.f);
#pragma unroll
        for (int j = 0; j < N; j++) { // (past the row's end h stays 0)
            const float m = valid(j) ? p.b * mul[j] : 0.f;
            mul[j] = valid(j) ? m * w[j] : 0.f;
            if (F == PLAIN || !p.post.bias) continue; // (add is 0, whatever m is)
            if (F == GATED && !(fabsf(m) <= FLT_MAX)) wild = true;
            add[j] = valid(j) ? m * add[j] : 0.f;
        }
    };
    long long gate_end = 0; // first row of the gate behind the one in the registers
    T *hp = (T *)p.h + first * p.h_ld, *xp = (T *)p.x + first * p.x_ld;
    for (int i = 0, k = 0, phase = 0; i < n; i++, hp += p.h_ld * P, xp += p.x_ld * P) {
        if (row_of(i) >= gate_end) {
            const int which = p.rows_per_gate ? (int)row_of(i) / p.rows_per_gate : 0;
            gate_end = p.rows_per_gate ? (which + 1LL) * p.rows_per_gate : p.rows;
            take_gate(which);
        }
        Values<T, VEC> r[C], y[C];
        auto each = [&](auto &&live, auto &&dead) {
            if (full) {
#pragma unroll
                for (int c = 0; c < C; c++) live(c);
            } else {
#pragma unroll
                for (int c = 0; c < C; c++)
                    if (at(c) < s + d) live(c);
                    else dead(c);
            }
        };
        auto whole = [&](int c) { return !SHIFT || (index(c * VEC) >= 0 && index(c * VEC) + VEC <= d); }; // an access without a neighbour's values
        auto own = [&](Values<T, VEC> &of, int c) {
            if (!full && !whole(c)) of.keep(-index(c * VEC), d - index(c * VEC));
        };
        auto one_by_one = [&](const T *from, Values<T, VEC> &to, int c) { // an access's values that are the row's
            alignas(16) T of[VEC];
#pragma unroll
            for (int j = 0; j < VEC; j++) of[j] = valid(c * VEC + j) ? from[index(c * VEC + j)] : from_f32<T>(0.f);
            memcpy(&to.raw, of, sizeof(to.raw));
        };
        umma_gemv::mbar_wait_flag(bar0 + 8 * k, phase, &abort_flag, 1);
        const T *const ry = yp + i * y_step, *const rr = rp + i * r_step;
        if (in_place(i)) {
            if (p.y) each([&](int c) { one_by_one(ry, y[c], c); }, [&](int c) { y[c].clear(); });
            if (p.r) each([&](int c) { one_by_one(rr, r[c], c); }, [&](int c) { r[c].clear(); });
        } else {
            const uint32_t from = ring0 + k * stage_bytes + at0 * (int)sizeof(T);
            const uint32_t ys = from + (VEC > 1 ? 0 : (uint32_t)reinterpret_cast<uintptr_t>(ry) & 15);
            const uint32_t rs = from + (p.y ? op_bytes : 0) + (VEC > 1 ? 0 : (uint32_t)reinterpret_cast<uintptr_t>(rr) & 15);
            if (p.y) each([&](int c) { y[c].load_shared(ys + c * 32 * VEC * (int)sizeof(T)), own(y[c], c); }, [&](int c) { y[c].clear(); });
            if (p.r) each([&](int c) { r[c].load_shared(rs + c * 32 * VEC * (int)sizeof(T)), own(r[c], c); }, [&](int c) { r[c].clear(); });
        }
        auto refill = [&]() { // all of the team's reads of the stage come before
            if (WARP) __syncwarp();
            if (t == 0 && asked < n && !*(volatile int *)&abort_flag) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                ask(k);
            }
        };
        float u[N];
        const uint32_t sums = red0 + (i & 1) * 512;
        auto total = [&](bool squares, int slot) {
            unsigned long long s = 0;
#pragma unroll
            for (int j = 0; j < N; j += 2) {
                const unsigned long long w = pack2f(u[j], u[j + 1]);
                s = squares ? fma2(w, w, s) : add2(w, s);
            }
            return team_sum<WARP>(sum2(s), sums + slot * 128) * p.inv_d;
        };
        auto centre = [&](float mean) {
            const unsigned long long m = pack2f(-mean, -mean);
#pragma unroll
            for (int j = 0; j < N; j += 2) unpack2f(add2(pack2f(u[j], u[j + 1]), m), u[j], u[j + 1]);
            if (full) return;
#pragma unroll
            for (int c = 0; c < C; c++) // past the row's ends 0 again
                if (!whole(c) || at(c) >= d + s)
#pragma unroll
                    for (int j = c * VEC; j < (c + 1) * VEC; j++) u[j] = valid(j) ? u[j] : 0.f;
        };
        auto scaled = [&](float scale, const float(&m)[N], const float(&b)[N]) { // u = scale u m + b
            const unsigned long long sc = pack2f(scale, scale);
#pragma unroll
            for (int j = 0; j < N; j += 2)
                if (F == PLAIN) unpack2f(mul2(mul2(pack2f(u[j], u[j + 1]), sc), pack2f(m[j], m[j + 1])), u[j], u[j + 1]);
                else unpack2f(fma2(mul2(pack2f(u[j], u[j + 1]), sc), pack2f(m[j], m[j + 1]), pack2f(b[j], b[j + 1])), u[j], u[j + 1]);
        };
        auto store = [&](T *to) {
            T *const from = to + (at0 - s);
            each([&](int c) {
                if (full || whole(c)) {
                    store_values<T, VEC>(from + c * 32 * VEC, u + c * VEC);
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; j++)
                        if (valid(c * VEC + j)) to[index(c * VEC + j)] = from_f32<T>(u[c * VEC + j]);
                }
            }, [](int) {});
        };
        if (p.y) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                y[c].get(v);
#pragma unroll
                for (int j = 0; j < VEC; j++) u[c * VEC + j] = v[j];
            }
            if (F != PLAIN && p.post.kind == RT_NORM_LAYER) centre(total(false, 0));
            const float scale = p.post.kind != RT_NORM_NONE ? rsqrtf(total(true, 1) + p.post.eps) : 1.f;
            if (F == GATED && wild) {
                const long long which = p.rows_per_gate ? row_of(i) / p.rows_per_gate : 0;
                auto param = [&](const void *of, int f32, int at) { return f32 ? ((const float *)of)[at] : to_f32(((const T *)of)[at]); };
#pragma unroll
                for (int j = 0; j < N; j++) {
                    if (!valid(j)) continue; // (0)
                    const int at = index(j);
                    u[j] *= scale;
                    if (p.post.weight) u[j] *= param(p.post.weight, p.post.f32, at);
                    u[j] = (u[j] + param(p.post.bias, p.post.f32, at)) * p.b;
                    if (p.gate) u[j] *= to_f32(((const T *)p.gate)[which * d + at]);
                }
            } else {
                scaled(scale, mul, add);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) u[j] = -0.f; // (a r - 0 is a r)
        }
        if (p.r) {
            const unsigned long long a = pack2f(p.a, p.a);
            float w[N];
#pragma unroll
            for (int c = 0; c < C; c++) {
                r[c].get(v);
#pragma unroll
                for (int j = 0; j < VEC; j++) w[c * VEC + j] = v[j];
            }
#pragma unroll
            for (int j = 0; j < N; j += 2) unpack2f(fma2(a, pack2f(w[j], w[j + 1]), pack2f(u[j], u[j + 1])), u[j], u[j + 1]);
        }
        if (p.h) store(hp);
        if (p.pre.kind != RT_NORM_NONE) {
            if (F != PLAIN && p.pre.kind == RT_NORM_LAYER) centre(total(false, 2));
            const float scale = rsqrtf(total(true, 3) + p.pre.eps);
            refill();
            scaled(scale, wx, bx);
            store(xp);
        } else {
            if (!WARP) __syncthreads();
            refill();
        }
        if (++k == stages) k = 0, phase ^= 1;
    }
    if (abort_flag) { // a wait ran out: word of it, and no exit while a copy may still land here
        if (t == 0) {
            for (int i = max(0, asked - stages); i < asked; i++) {
                const unsigned long long t0 = umma_gemv::wait_clock();
                while (!umma_gemv::mbar_try_wait(bar0 + 8 * (i % stages), i / stages & 1) && umma_gemv::wait_clock() - t0 < umma_gemv::WAIT_LIMIT_CYCLES) {}
            }
            report_wait_error();
        }
        __syncthreads();
    }
}

// A CTA per row of any length: the row is read again for each sum.
template <typename T, int VEC> __global__ void __launch_bounds__(1024) residual_norm_loop_kernel(const __grid_constant__ ResidualNormParams p) {
    __shared__ __align__(16) float red[4][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t red0 = umma_gemv::smem_u32(red);
    clear_sums(red, 4);
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int d = p.d, row = blockIdx.x, step = blockDim.x * VEC;
    const T *const rp = (const T *)p.r + (long long)row * p.r_ld, *const yp = (const T *)p.y + (long long)row * p.y_ld;
    const T *const gate = p.gate ? (const T *)p.gate + (p.rows_per_gate ? (long long)(row / p.rows_per_gate) * d : 0) : nullptr;
    float mean = 0.f, scale = 1.f;
    auto each = [&](auto &&f) {
        for (int e = threadIdx.x * VEC; e < d; e += step) f(e);
    };
    auto block = [&](int e, float(&u)[VEC]) {
        Values<T, VEC> y;
        y.load(yp + e), y.get(u);
    };
    auto times = [&](float(&u)[VEC], const void *w, const void *b, int f32, int e) {
        Param<T, VEC> param;
        float v[VEC];
        if (w) {
            param.load(w, f32, e), param.get(f32, v);
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] *= v[i];
        }
        if (b) {
            param.load(b, f32, e), param.get(f32, v);
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] += v[i];
        }
    };
    if (p.post.kind == RT_NORM_LAYER) {
        float s = 0.f;
        each([&](int e) {
            float u[VEC];
            block(e, u);
#pragma unroll
            for (int i = 0; i < VEC; i++) s += u[i];
        });
        mean = team_sum<false>(s, red0 + 128 * 0) * p.inv_d;
    }
    if (p.post.kind != RT_NORM_NONE) {
        float q = 0.f;
        each([&](int e) {
            float u[VEC];
            block(e, u);
#pragma unroll
            for (int i = 0; i < VEC; i++) q = fmaf(u[i] - mean, u[i] - mean, q);
        });
        scale = rsqrtf(team_sum<false>(q, red0 + 128 * 1) * p.inv_d + p.post.eps);
    }
    const float block_mean = mean, block_scale = scale;
    auto sum = [&](int e, float(&u)[VEC]) { // h
        float v[VEC];
        if (p.y) {
            block(e, u);
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] = (u[i] - block_mean) * block_scale;
            times(u, p.post.weight, p.post.bias, p.post.f32, e);
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] *= p.b;
            times(u, gate, nullptr, 0, e);
        }
        if (p.r) {
            Values<T, VEC> r;
            r.load(rp + e), r.get(v);
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] = p.y ? fmaf(p.a, v[i], u[i]) : p.a * v[i];
        }
    };
    mean = 0.f;
    if (p.pre.kind == RT_NORM_LAYER) {
        float s = 0.f;
        each([&](int e) {
            float u[VEC];
            sum(e, u);
#pragma unroll
            for (int i = 0; i < VEC; i++) s += u[i];
        });
        mean = team_sum<false>(s, red0 + 128 * 2) * p.inv_d;
    }
    if (p.pre.kind != RT_NORM_NONE) {
        float q = 0.f;
        each([&](int e) {
            float u[VEC];
            sum(e, u);
#pragma unroll
            for (int i = 0; i < VEC; i++) q = fmaf(u[i] - mean, u[i] - mean, q);
        });
        scale = rsqrtf(team_sum<false>(q, red0 + 128 * 3) * p.inv_d + p.pre.eps);
    }
    each([&](int e) { // a thread reads what it overwrites before it does, and nobody else reads it any more
        float u[VEC];
        sum(e, u);
        if (p.h) store_values<T, VEC>((T *)p.h + (long long)row * p.h_ld + e, u);
        if (p.pre.kind == RT_NORM_NONE) return;
#pragma unroll
        for (int i = 0; i < VEC; i++) u[i] = (u[i] - mean) * scale;
        times(u, p.pre.weight, p.pre.bias, p.pre.f32, e);
        store_values<T, VEC>((T *)p.x + (long long)row * p.x_ld + e, u);
    });
}

template <typename T, int VEC, bool WARP, Form F, bool SHIFT> cudaError_t launch_walk(const ResidualNormParams &p, int period, int sm_count, cudaStream_t stream) {
    const auto kernel = residual_norm_walk_kernel<T, VEC, WARP, F, SHIFT>;
    const int threads = WARP ? 32 : (p.d + (SHIFT ? VEC - 1 : 0) + N * 32 - 1) / (N * 32) * 32, teams = WARP ? MAX_TEAMS : 1;
    const int stage = teams * walk_operand_bytes<(VEC > 1 && !SHIFT)>(p.d * (int)sizeof(T)) * ((p.r != nullptr) + (p.y != nullptr));
    const int per_sm = WALK_THREADS<F> / (threads * teams);
    const int stages = std::max(2, std::min(MAX_STAGES, WALK_SMEM / per_sm / stage));
    static SmemAttr attr;
    cudaError_t e = attr.ensure(kernel, (size_t)WALK_SMEM);
    if (e != cudaSuccess) return e;
    const long long rows = (p.rows + period - 1) / period; // of a kind
    const long long walkers = std::max(1, per_sm * sm_count * teams / period), share = (rows + walkers - 1) / walkers;
    const long long used = (rows + share - 1) / share * period;
    return launch_pdl(kernel, dim3((unsigned)((used + teams - 1) / teams)), dim3(threads, teams), (size_t)stages * stage, stream, p, (int)share, stages, period);
}

template <typename T, int VEC, Form F, bool SHIFT> cudaError_t launch_form(const ResidualNormParams &p, int period, int sm_count, cudaStream_t stream) {
    return p.d + (SHIFT ? VEC - 1 : 0) <= 32 * N ? launch_walk<T, VEC, true, F, SHIFT>(p, period, sm_count, stream)
                                                 : launch_walk<T, VEC, false, F, SHIFT>(p, period, sm_count, stream);
}

template <typename T, int VEC, bool SHIFT> cudaError_t launch_walks(const ResidualNormParams &p, Form form, int period, int sm_count, cudaStream_t stream) {
    return form == PLAIN   ? launch_form<T, VEC, PLAIN, SHIFT>(p, period, sm_count, stream)
           : form == MEANS ? launch_form<T, VEC, MEANS, SHIFT>(p, period, sm_count, stream)
                           : launch_form<T, VEC, GATED, SHIFT>(p, period, sm_count, stream);
}

template <typename T, int VEC, int C, bool EARLY> cudaError_t launch_row(const ResidualNormParams &p, cudaStream_t stream) {
    return launch_pdl(residual_norm_kernel<T, VEC, C, EARLY>, dim3(p.rows), dim3((p.d + C * VEC * 32 - 1) / (C * VEC * 32) * 32), 0, stream, p);
}

// Few rows: as many as are on the SMs at once, a CTA each (WAVE: threads of an SM at that kernel's registers), or with a warp to
// a row fewer than there are warps to walk: they have one round of loads, where a team that stays asks for its constants first.
// bf16, d = 2560, rms both sides: 77 rows 3.4 us a CTA each, 3.9 walked; 300 rows 4.7 and 4.0; 1500 rows 13.8 and 8.3.
// f32, d = 384, 1500 rows: 3.9 and 4.7.
template <typename T, int VEC> cudaError_t launch_t(const ResidualNormParams &p, int period, int sm_count, cudaStream_t stream) {
    constexpr int EARLY_C = VEC == 1 ? 4 : 1, WAVE = VEC == 1 ? 1024 : VEC == 4 ? 1344 : 704, WORD = 16 / (int)sizeof(T);
    const int threads = (p.d + 32 * VEC * EARLY_C - 1) / (32 * VEC * EARLY_C) * 32;
    const bool few = p.rows <= (long long)sm_count * (WAVE / threads) || (p.d <= 32 * N && p.rows <= 2 * MAX_TEAMS * sm_count);
    if (p.d <= 4096 && (few || p.d < MIN_WALK_D)) return launch_row<T, VEC, EARLY_C, true>(p, stream);
    const bool plain = p.post.kind != RT_NORM_LAYER && p.pre.kind != RT_NORM_LAYER && !p.post.bias && !p.pre.bias;
    const Form form = plain ? PLAIN : p.post.bias && (p.gate || !(fabsf(p.b) <= FLT_MAX)) ? GATED : MEANS;
    const int longest = (plain ? WALK_THREADS<PLAIN> : WALK_THREADS<MEANS>) * N;
    // operands that lie alike go by 16-byte words (8192 bf16 rows of 2561: 53 us, 71 value by value; 52000 rows of 383: 67 and 67, with
    // means and biases 93 and 102)
    if constexpr (VEC == 1)
        if (period && p.d + WORD - 1 <= longest) return launch_walks<T, WORD, true>(p, form, period, sm_count, stream);
    if (p.d <= longest) return launch_walks<T, VEC, false>(p, form, 1, sm_count, stream);
    // longer rows, 32 values a thread in registers while 512 threads hold them (2048 bf16 rows of 10240: 51 us, 103 with the loops;
    // value by value, rows of 9001, 282 and 128)
    if constexpr (VEC > 1)
        if (p.d <= 512 * 32) return launch_row<T, VEC, 32 / VEC, false>(p, stream);
    return launch_pdl(residual_norm_loop_kernel<T, VEC>, dim3(p.rows), dim3(1024), 0, stream, p);
}
// vec: every access on a 16-byte boundary; else the period in which rows lie the same way, or 0 where operands differ in that
template <typename T> cudaError_t launch_t(const ResidualNormParams &p, bool vec, int sm_count, cudaStream_t stream) {
    if (vec) return launch_t<T, 16 / (int)sizeof(T)>(p, 1, sm_count, stream);
    uintptr_t base = 0;
    long long pitch = 0;
    int period = 0;
    const std::pair<const void *, long long> operands[] = {{p.y, p.y_ld}, {p.r, p.r_ld}, {p.h, p.h_ld}, {p.x, p.x_ld}};
    for (const auto &o : operands) {
        if (!o.first) continue;
        const uintptr_t at = reinterpret_cast<uintptr_t>(o.first) % 16;
        const long long step = o.second * (long long)sizeof(T) % 16;
        if (period && (at != base || step != pitch)) return launch_t<T, 1>(p, 0, sm_count, stream);
        base = at, pitch = step, period = 1;
    }
    while (pitch * period % 16) period *= 2;
    return launch_t<T, 1>(p, period, sm_count, stream);
}

} // namespace

cudaError_t residual_norm_bind_wait_error(int *word) { return bind_wait_error(word); }

cudaError_t launch_residual_norm(const rt_residual_norm &op, int sm_count, cudaStream_t stream) {
    ResidualNormParams p{};
    p.r = op.residual; p.y = op.block; p.gate = op.gate; p.h = op.h; p.x = op.x;
    p.r_ld = op.residual_ld; p.y_ld = op.block_ld; p.h_ld = op.h_ld; p.x_ld = op.x_ld;
    p.rows = (int)op.rows; p.d = (int)op.d;
    p.rows_per_gate = op.gate && op.gate_rows > 1 ? (int)(op.rows / op.gate_rows) : 0;
    p.inv_d = 1.0f / (float)op.d;
    p.a = op.residual_scale; p.b = op.block_scale;
    auto norm = [](const rt_norm &n) { return NormParams{n.kind, n.dt == RT_F32, n.eps, n.kind ? n.weight : nullptr, n.kind ? n.bias : nullptr}; };
    p.post = norm(op.post); p.pre = norm(op.pre);
    // 16-byte accesses: every pointer on a 16-byte boundary, every row a whole number of them
    const int per = op.dt == RT_F32 ? 4 : 8;
    uintptr_t bits = 0;
    for (const void *q : {p.r, p.y, p.gate, (const void *)p.h, (const void *)p.x, p.post.weight, p.post.bias, p.pre.weight, p.pre.bias})
        bits |= reinterpret_cast<uintptr_t>(q);
    bool vec = bits % 16 == 0 && op.d % per == 0;
    if (p.r) vec = vec && p.r_ld % per == 0;
    if (p.y) vec = vec && p.y_ld % per == 0;
    if (p.h) vec = vec && p.h_ld % per == 0;
    if (p.x) vec = vec && p.x_ld % per == 0;
    switch (op.dt) {
    case RT_F32: return launch_t<float>(p, vec, sm_count, stream);
    case RT_F16: return launch_t<__half>(p, vec, sm_count, stream);
    case RT_BF16: return launch_t<__nv_bfloat16>(p, vec, sm_count, stream);
    default: return cudaErrorInvalidValue;
    }
}

} // namespace rt
