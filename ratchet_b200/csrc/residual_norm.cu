// What stands between two blocks: h = a r + b g N_post(y), x = N_pre(h), in one pass over the rows.
//
// Memory-bound: r and y are read once, h and x written once.  A row lives in the registers of a team of threads (a warp for
// short rows, a CTA for longer ones) as f32 from its loads to its stores; means and variances are taken from the registers in
// two passes (centre first, then squares: no cancellation), so nothing is read twice and an output may be an input's memory.
#include <algorithm>

#include "common.cuh"
#include "kernels.hpp"

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
    int rows, d, rows_per_gate;
    float a, b;
    NormParams post, pre;
};

// VEC values of T at p, as f32: one 16-byte access when VEC > 1
template <typename T, int VEC> __device__ __forceinline__ void load_values(const T *p, float *v) {
    if (VEC == 1) {
        v[0] = to_f32(*p);
    } else {
        alignas(16) T raw[VEC];
#pragma unroll
        for (int i = 0; i < (int)(VEC * sizeof(T) / 16); i++) reinterpret_cast<uint4 *>(raw)[i] = reinterpret_cast<const uint4 *>(p)[i];
#pragma unroll
        for (int i = 0; i < VEC; i++) v[i] = to_f32(raw[i]);
    }
}

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

template <typename T, int VEC> __device__ __forceinline__ void load_param(const void *p, int f32, int i, float *v) {
    if (f32) load_values<float, VEC>((const float *)p + i, v);
    else load_values<T, VEC>((const T *)p + i, v);
}

// Sum over the team.  A CTA's warps meet in shared memory, each reduction of a row in a slot of its own (`slot`), so one
// barrier per reduction is enough; the order of the additions is fixed.
template <bool WARP> __device__ __forceinline__ float team_sum(float v, float (*red)[32], int slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (WARP) return v;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) red[slot][warp] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? red[slot][lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// v <- N(v); `d` values in all, thread t of the team holds values ((c * team + t) * VEC ..) in chunk c
template <typename T, int VEC, int C, bool WARP>
__device__ __forceinline__ void normalise(float (*v)[VEC], const NormParams &n, int d, int t, int team, float (*red)[32], int slot) {
    if (n.kind == RT_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) s += v[c][i]; // (0 past the row's end)
        const float mean = team_sum<WARP>(s, red, slot) / (float)d;
#pragma unroll
        for (int c = 0; c < C; c++)
            if ((c * team + t) * VEC < d)
#pragma unroll
                for (int i = 0; i < VEC; i++) v[c][i] -= mean;
    }
    float q = 0.f;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < VEC; i++) q = fmaf(v[c][i], v[c][i], q);
    const float scale = rsqrtf(team_sum<WARP>(q, red, slot + 1) / (float)d + n.eps);
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = (c * team + t) * VEC;
        if (e >= d) continue;
        float w[VEC], b[VEC];
        if (n.weight) load_param<T, VEC>(n.weight, n.f32, e, w);
        if (n.bias) load_param<T, VEC>(n.bias, n.f32, e, b);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            float u = v[c][i] * scale;
            if (n.weight) u *= w[i];
            if (n.bias) u += b[i];
            v[c][i] = u;
        }
    }
}

// A team per row: a warp (blockDim.y of them in a CTA) or the CTA.  VEC values per access, C accesses per thread and operand;
// VEC divides d and every ld, so no access crosses a row's end.
template <typename T, int VEC, int C, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024) residual_norm_kernel(ResidualNormParams p) {
    __shared__ float red[4][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int t = threadIdx.x, team = blockDim.x;
    const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
    if (WARP && row >= p.rows) return; // whole warps; a CTA team always has a row
    float v[C][VEC], r[C][VEC];
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = (c * team + t) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; i++) v[c][i] = r[c][i] = 0.f;
        if (e >= p.d) continue;
        if (p.y) load_values<T, VEC>((const T *)p.y + row * p.y_ld + e, v[c]);
        if (p.r) load_values<T, VEC>((const T *)p.r + row * p.r_ld + e, r[c]);
    }
    if (p.post.kind != RT_NORM_NONE) normalise<T, VEC, C, WARP>(v, p.post, p.d, t, team, red, 0);
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = (c * team + t) * VEC;
        if (e >= p.d) continue;
        float g[VEC];
        if (p.gate) load_values<T, VEC>((const T *)p.gate + row / p.rows_per_gate * p.d + e, g);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            float add = p.y ? p.b * v[c][i] : 0.f;
            if (p.gate) add *= g[i];
            v[c][i] = p.r ? fmaf(p.a, r[c][i], add) : add;
        }
        if (p.h) store_values<T, VEC>((T *)p.h + row * p.h_ld + e, v[c]);
    }
    if (p.pre.kind == RT_NORM_NONE) return;
    normalise<T, VEC, C, WARP>(v, p.pre, p.d, t, team, red, 2);
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int e = (c * team + t) * VEC;
        if (e < p.d) store_values<T, VEC>((T *)p.x + row * p.x_ld + e, v[c]);
    }
}

template <typename T, int VEC, int C> cudaError_t launch_c(const ResidualNormParams &p, int threads, cudaStream_t stream) {
    if (threads <= 32) return launch_pdl(residual_norm_kernel<T, VEC, C, true>, dim3((p.rows + 7) / 8), dim3(32, 8), 0, stream, p);
    return launch_pdl(residual_norm_kernel<T, VEC, C, false>, dim3(p.rows), dim3(threads), 0, stream, p);
}

template <typename T> cudaError_t launch_t(const ResidualNormParams &p, bool vec, cudaStream_t stream) {
    constexpr int VEC = 16 / sizeof(T);
    auto threads = [&](int per) { return (p.d + per * 32 - 1) / (per * 32) * 32; };
    if (vec) {
        if (p.d <= 512 * VEC) return p.d <= 64 * VEC ? launch_c<T, VEC, 2>(p, 32, stream) : launch_c<T, VEC, 1>(p, threads(VEC), stream);
        if (p.d <= 1024 * 2 * VEC) return launch_c<T, VEC, 2>(p, threads(2 * VEC), stream);
        if (p.d <= 1024 * 4 * VEC) return launch_c<T, VEC, 4>(p, threads(4 * VEC), stream);
        return launch_c<T, VEC, 32 / VEC>(p, threads(32), stream);
    }
    if (p.d <= 4096) return launch_c<T, 1, 4>(p, threads(4), stream);
    return launch_c<T, 1, 32>(p, threads(32), stream);
}

} // namespace

cudaError_t launch_residual_norm(const rt_residual_norm &op, int, cudaStream_t stream) {
    ResidualNormParams p{};
    p.r = op.residual; p.y = op.block; p.gate = op.gate; p.h = op.h; p.x = op.x;
    p.r_ld = op.residual_ld; p.y_ld = op.block_ld; p.h_ld = op.h_ld; p.x_ld = op.x_ld;
    p.rows = (int)op.rows; p.d = (int)op.d;
    p.rows_per_gate = op.gate ? (int)(op.rows / op.gate_rows) : 1;
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
    case RT_F32: return launch_t<float>(p, vec, stream);
    case RT_F16: return launch_t<__half>(p, vec, stream);
    case RT_BF16: return launch_t<__nv_bfloat16>(p, vec, stream);
    default: return cudaErrorInvalidValue;
    }
}

} // namespace rt
