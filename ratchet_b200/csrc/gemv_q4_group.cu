// 4-bit group-scaled weights (Q4_G32 / G64 / G128) x f16 or bf16 activations, 1..16 vectors: y[n][m] = sum_k (q - z) s x[n][k].
//
// A decode step reads every weight once: half a byte a weight and 3 / group for its scale and zero point bound it, next to
// them the logic instructions that take the codes apart (half rate) and the warp MMAs (8 to 9 cycles each).
//  * A warp takes a 16-row tile and a part of K in steps of 128 values; a CTA has a few tiles, all of the machine's resident at
//    once where that is possible, and where rows are few its warps, then a cluster's CTAs, share K.  Codes go from global
//    memory to registers, AHEAD steps asked for in advance, the first ones for constant weights before the kernel waits for
//    its stream predecessor.
//  * Sums on the tensor cores (mma.sync m16n8k16; the sums of at most 16 columns do not need more).  Which values of k an MMA's 16
//    places hold is free as long as A and B agree, so a lane's own nibbles fill its places: lane t (of the four of a row) takes 16
//    code bytes, the 32 values from 32 t on, and the pairs (k, k + 4) of a word are masked out of it (below).
//  * A step holds G = 128 / group groups, whose sums must not mix before their scales come in.  For at most 8 / G vectors an MMA's
//    8 columns are G groups x 8 / G vectors, B being zero where a lane's values are of another group than the column's; a lane
//    ends up with the sums of just the group whose codes it took.  For more vectors the four lanes of a row exchange their words
//    first (SPREAD), so that a word's MMAs are of one group and the columns are vectors.
//  * Activations are staged in shared memory in the order the MMAs take them, with their sums by group; so are scales and zero
//    points, a word a group (read from global memory by the lanes that need them they would be more requests than the codes).
//  * f32 sums of a group times s, added in f32 over steps, warps and CTAs of the cluster in a fixed order.
//  * q x and z x are summed apart, so f32 roundings go with sum s (q + z) |x| and not with sum s |q - z| |x|: (K / 64 + 174) 2^-24 of it
//    at most by the count of additions, 2^-25 where it was looked for (codes at and next to zero points of 8 .. 31).  Beside f16's own
//    rounding that shows in outputs 2^14 times smaller than their terms; a group of codes equal to its zero point adds as much, not 0.
//
// One vector, 51200 rows of 2560: 15.4 us with groups of 128 (4.5 TB/s), 16.5 of 64, 18.2 of 32; 2560 x 2560 3.4, the launch and two
// trips to memory; 16 vectors 23.5 / 29 / 46: the epilogue of a group (FMAs by vectors, in pairs), the masking, and the B operands' 21
// thousand shared-memory wavefronts an SM bound those.  A CUDA-core product of the same layout took 5 to 90 times as long (2560 x 10240
// with 5 vectors: 841 us against 9.5).
#include <algorithm>

#include "common.cuh"
#include "f32x2.cuh"
#include "kernels.hpp"

namespace rt {

namespace {

constexpr int STEP = 128; // values of k per warp and step
constexpr int MAX_WARPS = 24; // of a CTA: 80 registers a thread (51200 x 2560, one vector: 15.2 us, with 32 warps at 64 registers and two steps ahead 17.3)

struct Q4GroupParams {
    MatmulParams p;
    int nv;       // vectors (columns of op(rhs), batches of them flattened)
    int rows;     // per CTA: rows of W, or gate | up pairs of them
    int steps;    // ceil(K / STEP)
    int ranks;    // CTAs of a cluster along K
    int per_rank; // steps of each
    int parts;    // warps of a row unit along K
    int per_part; // steps of each
    int stride;   // words between two rows' scales: 4 x an odd number (16-byte stores, and reads of a word of eight rows, without conflicts)
    int units;    // row units of a CTA
    int pair;     // gate | up rows: the output is their fold, [nv][M / 2]
    int lhs_constant;
    int fours;      // the groups of a row in a CTA's K range come in aligned fours
    uint32_t magic; // ceil(2^32 / n) for the number of these (or of groups) in a row
    uint32_t nv_magic; // and for nv
    uint32_t xsum_at, up_at, scales_at, part_at; // bytes into shared memory (activations at 0)
};

// The codes of a word as the values of an MMA's f16 A operand, without arithmetic: a nibble in the low bits of the mantissa under a
// zero exponent is q * 2^-24, four bits further up q * 2^-20 (subnormal numbers, which the tensor cores take exactly).  The two
// kinds go to sums of their own.  The zero point is taken off with the scale: z * (sum of the group's x), which one more MMA per B
// operand gives, with ones for A.  Pairs {k, k + 4}, k = 0 .. 3.
__device__ __forceinline__ void nibble_pairs(uint32_t w, uint32_t (&a)[4]) {
    const uint32_t hi = w >> 8;
    a[0] = w & 0x000f000fu;
    a[1] = w & 0x00f000f0u;
    a[2] = hi & 0x000f000fu;
    a[3] = hi & 0x00f000f0u;
}
// d = a b, or d += a b
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, bool add) {
    if (add)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// 16 bytes of codes, or 8 here and 8 bytes 32 further on
__device__ __forceinline__ void load_codes(uint32_t (&w)[4], const uint8_t *p) {
    asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
}
__device__ __forceinline__ void load_codes_halves(uint32_t (&w)[4], const uint8_t *p) {
    asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(w[2]), "=r"(w[3]) : "l"(p + 32));
}

// Two bf16 values of a 32-bit word times `scale` (a power of two) as f16
__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t w, float scale) {
    const float lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u);
    const __half2 h = __floats2half2_rn(lo * scale, hi * scale);
    return h2_as_u32(h);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_id() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}
// the float at `p` (shared memory) of CTA `rank` of this cluster
__device__ __forceinline__ float load_peer(const float *p, uint32_t rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), b;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(b) : "memory");
    return v;
}


// With groups of 32, lanes t and t ^ 2 of a row hold words of two groups: after the exchange w[j] is of group j in all four lanes
// (lane t has word 0, 2, 1, 3 of it).
__device__ __forceinline__ void spread_words(uint32_t (&w)[4], int t) {
    const bool upper = (t & 2) != 0;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? w[i] : w[i + 1], 2);
        if (upper) w[i] = got;
        else w[i + 1] = got;
    }
}

// The dot product of one row and one vector again, element by element: an infinity among the activations makes q x - z x a NaN that
// (q - z) x is not, so a NaN result is decided here by IEEE's rules for the plain sum.  One thread does it: a NaN in every vector takes
// 2560 x 2560 from 3.4 to 36 us, 51200 x 2560 with 16 vectors from 24 to 836.
template <typename T> __device__ __noinline__ float exact_row(const MatmulParams &p, long long row, const T *x) {
    float acc = 0.f;
#pragma unroll 1
    for (int k = 0; k < p.K; k += 32) {
        const long long at = row * p.K + k;
        const uint4 c = __ldg(reinterpret_cast<const uint4 *>((const uint8_t *)p.lhs + at / 2));
        const long long group = at >> p.lhs_group_shift;
        const float s = __half2float(((const __half *)p.lhs_scales)[group]);
        const int z = p.lhs_zeros[group] & 31;
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 32; i++) acc = fmaf((float)((int)(w[i >> 3] >> (4 * (i & 7)) & 15u) - z) * s, to_f32(x[k + i]), acc);
    }
    return acc;
}

// G groups in a step; NVS: vectors, rounded up to 1, 2, 4, 8 or 16
template <typename T, int G, int NVS>
__global__ void __launch_bounds__(MAX_WARPS * 32) q4_group_gemv_kernel(const __grid_constant__ Q4GroupParams q) {
    constexpr bool SPREAD = NVS > 8 / G;    // an MMA's columns are vectors, its values of one group
    constexpr int VP = SPREAD ? 8 : 8 / G;  // vectors per pass
    constexpr int P = (NVS + VP - 1) / VP;  // passes
    constexpr bool MIX = SPREAD && G > 1;   // (with one group a step there is nothing to keep apart)
    constexpr int XS = SPREAD ? G : 1;      // groups whose sums a lane gets: all with SPREAD, else its own
    constexpr int AHEAD = NVS > 8 ? 2 : 3;  // steps whose codes are asked for in advance (as many as the registers allow)
    constexpr bool BF16 = cuda::std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(16) uint8_t smem[];
    uint4 *const xs = reinterpret_cast<uint4 *>(smem);                          // [step][word][NVS][lane of a row]: 8 values
    float *const xsum = reinterpret_cast<float *>(smem + q.xsum_at);            // [step][group][NVS]
    float *const up = reinterpret_cast<float *>(smem + q.up_at);                // bf16: [step][NVS], the power of two taken out
    uint32_t *const scales = reinterpret_cast<uint32_t *>(smem + q.scales_at);  // [place][stride]: f16 s | f16 z << 16
    float *const part = reinterpret_cast<float *>(smem + q.part_at);            // [part][tile][NVS][16]
    const MatmulParams &p = q.p;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (!q.lhs_constant) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int rank = q.ranks > 1 ? (int)cluster_rank() : 0;
    const int row_base = (int)(q.ranks > 1 ? cluster_id() : blockIdx.x) * q.rows; // first row (pair) of the CTA
    const int batch = blockIdx.y;
    const int K = p.K, ff = p.M >> 1;
    const int have_rows = min(q.rows, (q.pair ? ff : p.M) - row_base); // rows (pairs) of this CTA
    const int unit = q.pair ? 8 : 16, tiles = (have_rows + unit - 1) / unit;
    const long long lhs_row = (long long)(p.lhs_stack == 1 ? 0 : batch) * p.M + row_base;
    const int first = rank * q.per_rank, n_steps = max(0, min(q.steps, first + q.per_rank) - first); // of this CTA
    const uint32_t row_bytes = (uint32_t)K >> 1;

    // ---- the warp's rows and steps; the first codes.  Rows that are not the CTA's are its last one again, with scales of 0.  The last
    // step of a row whose K is no multiple of 128 reads on into what lies behind it (the next row, or the scales); its scales and
    // activations are 0.
    const int kpart = q.parts > 1 ? warp % q.parts : 0, tile = q.parts > 1 ? warp / q.parts : warp;
    const int begin = min(n_steps, kpart * q.per_part), end = min(n_steps, begin + q.per_part); // within this CTA's steps
    const int row0 = min(tile * unit + g, have_rows - 1), row1 = q.pair ? row0 + ff : min(tile * unit + g + 8, have_rows - 1);
    const uint8_t *const codes = (const uint8_t *)p.lhs + (uint32_t)(first + begin) * (STEP / 2) + t * (MIX ? 8 : 16);
    const uint8_t *code0 = codes + (lhs_row + row0) * row_bytes;
    const long long half_bytes = (long long)(row1 - row0) * row_bytes;
    uint32_t code[AHEAD][2][4];
    auto load = [&](uint32_t (&c)[2][4], const uint8_t *at) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint8_t *from = at + (h ? half_bytes : 0);
            if (MIX) load_codes_halves(c[h], from);
            else load_codes(c[h], from);
        }
    };
#pragma unroll
    for (int a = 0; a < AHEAD; a++)
        if (begin + a < end) load(code[a], code0 + a * (STEP / 2));

    // ---- scales of the rows' groups in this K range, 0 (a group that adds nothing) past K: four groups of a row at a time where
    // their number allows it, FOURS of a thread asked for together, the first ones before it waits for the stream predecessor
    // (51200 x 2560, groups of 32, one vector: 19.1 us, 20.5 where the later ones came one by one)
    constexpr int FOURS = 4;
    const int row_groups = K >> p.lhs_group_shift, left = min(n_steps * G, row_groups - first * G);
    const long long scale0 = lhs_row * row_groups + first * G;
    const uint16_t *const s16 = (const uint16_t *)p.lhs_scales + scale0;
    const uint8_t *const z8 = p.lhs_zeros + scale0;
    const int per_row = q.per_rank * G >> (q.fours ? 2 : 0), n_units = tiles * 16 * per_row;
    auto place_of = [&](int e, int &i, bool &there) { // e -> place and fours (or group) i of its row
        const int place = per_row == 1 ? e : (int)__umulhi((uint32_t)e, q.magic), r = (place >> 4) * unit + (q.pair ? place & 7 : place & 15);
        i = e - place * per_row;
        there = r < have_rows;
        return place;
    };
    auto source = [&](int place) { return (long long)((place >> 4) * unit + (q.pair ? (place & 7) + (place & 8 ? ff : 0) : place & 15)) * row_groups; };
    auto put_four = [&](int place, int i, uint2 s, uint32_t z) { // words s | z as f16 << 16: 1024 + z less 1024
        z &= 0x1f1f1f1fu;
        uint32_t a = __byte_perm(z, 0x64646464u, 0x4140), b = __byte_perm(z, 0x64646464u, 0x4342);
        const __half2 k1024 = __float2half2_rn(1024.f);
        a = h2_as_u32(__hsub2(*reinterpret_cast<const __half2 *>(&a), k1024));
        b = h2_as_u32(__hsub2(*reinterpret_cast<const __half2 *>(&b), k1024));
        *reinterpret_cast<uint4 *>(scales + place * q.stride + 4 * i) =
            make_uint4(__byte_perm(s.x, a, 0x5410), __byte_perm(s.x, a, 0x7632), __byte_perm(s.y, b, 0x5410), __byte_perm(s.y, b, 0x7632));
    };
    uint2 s4[FOURS];
    uint32_t z4[FOURS];
    auto load_fours = [&](int from) {
#pragma unroll
        for (int k = 0; k < FOURS; k++) {
            const int e = from + k * (int)blockDim.x;
            s4[k] = make_uint2(0, 0), z4[k] = 0;
            if (e >= n_units) continue;
            int i;
            bool there;
            const int place = place_of(e, i, there);
            if (there && 4 * i < left) {
                const long long at = source(place) + 4 * i;
                s4[k] = __ldg(reinterpret_cast<const uint2 *>(s16 + at));
                z4[k] = __ldg(reinterpret_cast<const uint32_t *>(z8 + at));
            }
        }
    };
    if (q.fours) load_fours(tid);
    if (q.lhs_constant) asm volatile("griddepcontrol.wait;" ::: "memory");
    const T *const x = (const T *)p.rhs + (long long)(p.rhs_stack == 1 ? 0 : batch) * q.nv * K;
    constexpr int XA = NVS > 8 ? 3 : NVS > 1 ? 2 : 1; // asked for together
    const int n_x = n_steps * q.nv * 16; // eight values each
    auto step_of = [&](int sv) { return NVS <= 2 ? sv / NVS : (int)__umulhi((uint32_t)sv, q.nv_magic); }; // (nv = NVS up to 2)
    uint4 raw[XA];
    auto load_x = [&](int from) {
#pragma unroll
        for (int i = 0; i < XA; i++) {
            const int e = from + i * (int)blockDim.x, sv = e >> 4, step = step_of(sv), v = sv - step * q.nv, k = (first + step) * STEP + (e & 15) * 8;
            raw[i] = make_uint4(0, 0, 0, 0);
            if (e < n_x && k < K) raw[i] = *reinterpret_cast<const uint4 *>(x + ((uint32_t)v * (uint32_t)K + (uint32_t)k));
        }
    };
    load_x(tid);
    if (q.fours) {
        for (int from = tid;;) {
#pragma unroll
            for (int k = 0; k < FOURS; k++) {
                const int e = from + k * (int)blockDim.x;
                if (e >= n_units) continue;
                int i;
                bool there;
                const int place = place_of(e, i, there);
                put_four(place, i, s4[k], z4[k]);
            }
            from += FOURS * (int)blockDim.x;
            if (from >= n_units) break;
            load_fours(from);
        }
    } else {
#pragma unroll 4
        for (int e = tid; e < n_units; e += blockDim.x) {
            int i;
            bool there;
            const int place = place_of(e, i, there);
            uint32_t v = 0;
            if (there && i < left) {
                const long long at = source(place) + i;
                v = __ldg(s16 + at) | (uint32_t)__half_as_ushort(__ushort2half_rn((unsigned short)(__ldg(z8 + at) & 31))) << 16;
            }
            scales[place * q.stride + i] = v;
        }
    }

    // ---- activations: 16 threads take a step of one vector, 8 values each, XA of them asked for together (4096 x 8192, bf16, 5
    // vectors: 10.8 us, 11.5 one by one).  bf16 values come into f16's range with a power of two per step and vector, which the sums are multiplied by again: nothing saturates, and a value that loses bits is 2^-24 of
    // its step's largest or less.
    auto put_x = [&](int e, const uint4 &of) {
        const int u = e & 15, sv = e >> 4, step = step_of(sv), v = sv - step * q.nv;
        uint32_t w[4] = {of.x, of.y, of.z, of.w};
        if (BF16) {
            uint32_t top = 0; // the largest finite magnitude's bits
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t lo = (w[i] << 16) & 0x7fffffffu, hi = w[i] & 0x7fff0000u;
                if (lo < 0x7f800000u) top = max(top, lo);
                if (hi < 0x7f800000u) top = max(top, hi);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int sh = max((int)(top >> 23), 15) - 127 - 14; // the largest becomes 2^14 .. 2^15; exponents within f32's
            const float down = __uint_as_float((uint32_t)(127 - sh) << 23);
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = bf16x2_to_f16x2(w[i], down);
            if (u == 0 && e < n_x) up[step * NVS + v] = __uint_as_float((uint32_t)(127 + sh) << 23);
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            sum += f.x + f.y;
        }
#pragma unroll
        for (int o = 8 / G; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (e < n_x) {
            // the lane and word whose place these values have
            const int tt = !MIX ? u >> 2 : G == 2 ? u >> 1 & 3 : (u & 1) * 2 + (u >> 1 & 1), j = !MIX ? u & 3 : G == 2 ? (u >> 3) * 2 + (u & 1) : u >> 2;
            // pairs (0, 4) (2, 6) for the one kind of nibble, (1, 5) (3, 7) for the other
            xs[((step * 4 + j) * NVS + v) * 4 + tt] = make_uint4(__byte_perm(w[0], w[2], 0x5410), __byte_perm(w[1], w[3], 0x5410),
                                                                 __byte_perm(w[0], w[2], 0x7632), __byte_perm(w[1], w[3], 0x7632));
            if (u % (16 / G) == 0) xsum[(step * G + u / (16 / G)) * NVS + v] = sum;
        }
    };
    for (int from = tid;;) {
#pragma unroll
        for (int i = 0; i < XA; i++)
            if (from + i * (int)blockDim.x < (n_x + 31) / 32 * 32) put_x(from + i * (int)blockDim.x, raw[i]); // (whole warps, for the shuffles)
        from += XA * (int)blockDim.x;
        if (from >= (n_x + 31) / 32 * 32) break;
        load_x(from);
    }
    __syncthreads();

    unsigned long long sums[P][2]; // of the lane's two columns, a pair for row g and one for row g + 8
#pragma unroll
    for (int v = 0; v < P; v++) sums[v][0] = sums[v][1] = 0;
    // B operand: the lane's column is vector g (SPREAD; columns without a vector repeat the last one and are not stored), or vector
    // g % VP of group g / VP, zero where the lane's values are of another group
    const int own_group = SPREAD ? 0 : t * G / 4;
    const bool on = SPREAD || (g / VP == own_group && g % VP < q.nv);
    const uint4 *xb = xs + (size_t)begin * 4 * NVS * 4 + (SPREAD ? 0 : (on ? g % VP : 0) * 4) + t;
    int xv[P]; // SPREAD: offsets of the lane's vectors
#pragma unroll
    for (int i = 0; i < P; i++) xv[i] = SPREAD ? min(i * 8 + g, q.nv - 1) * 4 : 0;
    // the lane's two columns of D; those without a vector may be anything
    const int col = NVS == 1 ? 0 : SPREAD || G == 1 ? min(2 * t, NVS - 2) : min(2 * t % VP, NVS - 2);
    const float *xsum_at = xsum + (begin * G + own_group) * NVS + col, *up_at = up + begin * NVS + col;
    const uint32_t *sc = scales + (tile * 16 + g) * q.stride + begin * G + own_group;
    const int sc_half = 8 * q.stride;
    uint4 b0[4]; // without SPREAD: the step's B operands (lanes that are not on keep zeros)
#pragma unroll
    for (int j = 0; j < 4; j++) b0[j] = make_uint4(0, 0, 0, 0);
    auto pair_at = [](const float *at) {
        if (NVS == 1) return pack2f(*at, *at);
        return *reinterpret_cast<const unsigned long long *>(at);
    };
    const unsigned long long k16 = pack2f(16.f, 16.f), k20 = pack2f(1048576.f, 1048576.f);
    auto do_step = [&](uint32_t (&c)[2][4]) {
        if (!SPREAD && on) {
#pragma unroll
            for (int j = 0; j < 4; j++) b0[j] = xb[j * NVS * 4];
        }
        if (MIX && G == 4) spread_words(c[0], t), spread_words(c[1], t);
        unsigned long long back[P];
#pragma unroll
        for (int v = 0; v < P; v++) back[v] = BF16 ? pair_at(up_at + v * 8) : 0;
#pragma unroll
        for (int grp = 0; grp < XS; grp++) { // words 4 grp / XS .. of one group; without SPREAD the lane's own group
            float d[2][P][4];
#pragma unroll
            for (int j = 4 * grp / XS; j < 4 * (grp + 1) / XS; j++) {
                uint32_t a0[4], a1[4];
                nibble_pairs(c[0][j], a0);
                nibble_pairs(c[1][j], a1);
                const bool add = j > 4 * grp / XS;
#pragma unroll
                for (int v = 0; v < P; v++) { // one kind of nibble per MMA
                    const uint4 b = SPREAD ? xb[j * NVS * 4 + xv[v]] : b0[j];
                    mma_f16(d[0][v], a0[0], a1[0], a0[2], a1[2], b.x, b.y, add);
                    mma_f16(d[1][v], a0[1], a1[1], a0[3], a1[3], b.z, b.w, add);
                }
            }
#pragma unroll
            for (int v = 0; v < P; v++) {
                const unsigned long long sx = pair_at(xsum_at + grp * NVS + v * 8);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t e = sc[h * sc_half + grp];
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&e)); // s, z
                    unsigned long long &to = sums[v][h];
                    // 2^-20 times the sum of q x
                    const unsigned long long n = fma2(pack2f(d[0][v][2 * h], d[0][v][2 * h + 1]), k16, pack2f(d[1][v][2 * h], d[1][v][2 * h + 1]));
                    if (BF16) { // s and the power of two together: neither alone may be taken to the sum
                        to = fma2(mul2(pack2f(f.x, f.x), back[v]), fma2(n, k20, mul2(pack2f(-f.y, -f.y), sx)), to);
                    } else {
                        const float s20 = f.x * 1048576.f, sz = -f.x * f.y;
                        to = fma2(pack2f(sz, sz), sx, fma2(pack2f(s20, s20), n, to));
                    }
                }
            }
        }
        xb += 4 * NVS * 4;
        xsum_at += G * NVS;
        up_at += NVS;
        sc += G;
    };
    code0 += AHEAD * (STEP / 2);
    for (int step = begin; step < end; step += AHEAD) {
#pragma unroll
        for (int a = 0; a < AHEAD; a++) {
            if (step + a >= end) break;
            do_step(code[a]);
            if (step + a + AHEAD < end) load(code[a], code0 + a * (STEP / 2));
        }
        code0 += AHEAD * (STEP / 2);
    }

    constexpr int SLOT = NVS * 16; // a row unit's sums
    const int outs = q.units * SLOT;
    float *const mine_at = part + (kpart * q.units + tile) * SLOT;
#pragma unroll
    for (int v = 0; v < P; v++) {
        float acc[4];
        unpack2f(sums[v][0], acc[0], acc[1]);
        unpack2f(sums[v][1], acc[2], acc[3]);
#pragma unroll
        for (int j = 0; j < 4; j++) { // the groups of a vector are in lanes VP / 2 apart
            if (!SPREAD && G == 4) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], 1);
            if (!SPREAD && G >= 2) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], 2);
        }
        const int vec = v * VP + 2 * t;
        float *const at = mine_at + vec * 16 + g;
        if (2 * t < VP && vec < q.nv) at[0] = acc[0], at[8] = acc[2];
        if (2 * t < VP && vec + 1 < q.nv) at[16] = acc[1], at[24] = acc[3];
    }
    __syncthreads();
    auto sum_of = [&](int e) {
        float s = part[e];
#pragma unroll 4
        for (int k = 1; k < q.parts; k++) s += part[k * outs + e];
        return s;
    };
    const bool has_bias = p.bias_mode != BIAS_NONE;
    const int out_rows = q.pair ? ff : p.M;
    T *const out = (T *)p.out + (long long)batch * out_rows * q.nv;
    // output e (unit, vector, place): `sum` adds up what its warps or CTAs have
    auto finish = [&](int e, auto sum) {
        const int v = e % SLOT >> 4, place = e & 15, r = e / SLOT * unit + (q.pair ? place & 7 : place);
        if (v >= q.nv || r >= have_rows || (q.pair && (place & 8))) return; // the up rows: with their gate rows
        const int m = row_base + r;
        auto value = [&](int at, int behind) {
            float s = sum(at), bias = 0.f;
            if (s != s) s = exact_row<T>(p, lhs_row + r + behind, x + (long long)v * K);
            if (has_bias) bias = load_bias(p.bias, p.bias_dt, p.bias_mode == BIAS_PER_M ? m + behind : p.N == 1 ? 0 : v);
            return epilogue_value<T>(s, has_bias, bias, p.epilogue);
        };
        const T o = q.pair ? silu_mul_value<T>(value(e, 0), value(e + 8, ff)) : value(e, 0);
        out[p.trans_out ? (long long)v * out_rows + m : (long long)m * q.nv + v] = o;
    };
    if (q.ranks == 1) {
        for (int e = tid; e < outs; e += blockDim.x) finish(e, sum_of);
        return;
    }
    for (int e = tid; e < outs; e += blockDim.x) part[e] = sum_of(e);
    cluster_sync();
    for (int e = tid * q.ranks + rank; e < outs; e += blockDim.x * q.ranks)
        finish(e, [&](int at) {
            float s = 0.f;
            for (int c = 0; c < q.ranks; c++) s += load_peer(part + at, c);
            return s;
        });
    cluster_sync(); // no CTA leaves while its sums may be read
}

template <typename T, int G, int NVS>
cudaError_t launch_nv(const Q4GroupParams &q, const Q4GroupConfig &c, int batches, cudaStream_t stream) {
    const int out_rows = q.pair ? q.p.M / 2 : q.p.M;
    const auto kernel = q4_group_gemv_kernel<T, G, NVS>;
    static SmemAttr attr;
    cudaError_t e = attr.ensure(kernel, c.smem_bytes);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)((out_rows + q.rows - 1) / q.rows * c.ranks), (unsigned)batches);
    lc.blockDim = dim3((unsigned)(c.units * c.parts * 32));
    lc.dynamicSmemBytes = c.smem_bytes;
    lc.stream = stream;
    cudaLaunchAttribute a[2];
    a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a[0].val.programmaticStreamSerializationAllowed = 1;
    a[1].id = cudaLaunchAttributeClusterDimension;
    a[1].val.clusterDim.x = (unsigned)c.ranks;
    a[1].val.clusterDim.y = a[1].val.clusterDim.z = 1;
    lc.attrs = a;
    lc.numAttrs = c.ranks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&lc, kernel, q);
}

template <typename T, int G> cudaError_t launch_g(const Q4GroupParams &q, const Q4GroupConfig &c, int batches, cudaStream_t stream) {
    switch (c.nvs) {
    case 1: return launch_nv<T, G, 1>(q, c, batches, stream);
    case 2: return launch_nv<T, G, 2>(q, c, batches, stream);
    case 4: return launch_nv<T, G, 4>(q, c, batches, stream);
    case 8: return launch_nv<T, G, 8>(q, c, batches, stream);
    case 16: return launch_nv<T, G, 16>(q, c, batches, stream);
    default: return cudaErrorInvalidValue;
    }
}

template <typename T> cudaError_t launch_t(const Q4GroupParams &q, const Q4GroupConfig &c, int batches, cudaStream_t stream) {
    switch (q.p.lhs_group_shift) {
    case 5: return launch_g<T, 4>(q, c, batches, stream);
    case 6: return launch_g<T, 2>(q, c, batches, stream);
    case 7: return launch_g<T, 1>(q, c, batches, stream);
    default: return cudaErrorInvalidValue;
    }
}

constexpr size_t MOST_SMEM = 220u << 10, HALF_SMEM = 32u << 10; // for a CTA that has an SM to itself, or half of one

// The sizes that follow from units, parts and ranks; false when they do not fit.
bool complete(Q4GroupConfig &c, int M, int K, int group, int nv, bool pair) {
    const int steps = (K + STEP - 1) / STEP, g = STEP / group, out_rows = pair ? M / 2 : M, most = c.units * (pair ? 8 : 16);
    if (c.units * c.parts > MAX_WARPS) return false;
    const int ctas = (out_rows + most - 1) / most;
    c.rows = std::min(most, ((out_rows + ctas - 1) / ctas + 7) / 8 * 8);
    c.per_rank = (steps + c.ranks - 1) / c.ranks;
    c.per_part = (c.per_rank + c.parts - 1) / c.parts;
    c.stride = 4 * ((c.per_rank * g + 3) / 4 | 1);
    c.nvs = nv <= 2 ? nv : nv <= 4 ? 4 : nv <= 8 ? 8 : 16;
    auto up = [](size_t v) { return (v + 15) / 16 * 16; };
    size_t at = (size_t)c.per_rank * c.nvs * STEP * 2;
    c.xsum_at = (uint32_t)at;
    at = up(at + (size_t)c.per_rank * g * c.nvs * 4);
    c.up_at = (uint32_t)at;
    at = up(at + (size_t)c.per_rank * c.nvs * 4);
    c.scales_at = (uint32_t)at;
    at = up(at + (size_t)c.units * 16 * c.stride * 4);
    c.part_at = (uint32_t)at;
    at += (size_t)c.parts * c.units * c.nvs * 64;
    c.smem_bytes = at;
    return at <= MOST_SMEM;
}

} // namespace

// How rows and K are shared out.  Counted in steps of a tile (16 rows x 128 values) that an SM has to work off one after the
// other: with few rows the tiles do not divide evenly among the SMs, and a K range of the tiles shared by a cluster's CTAs does;
// activations that every CTA stages count as well, more where they take many rounds, and a cluster's start and two barriers as 55
// or 80 steps; the weights are fitted to what these products took.  2560 x 10240 with 8 vectors: 21.0 us without clusters, 12.3 in
// twos, 10.6 in fours; 2560 x 2560: 5.2, 5.2, 6.6; 20000 x 4096 with 16: 36 and 27 in twos.
// Clusters of eight are left out: with a CTA an SM few of them are resident (2560 x 2560, one vector: 18.7 us, 3.7 without).
bool q4_group_gemv_config(int M, int K, int group, int nv, int batches, bool pair, int sm_count, Q4GroupConfig *out) {
    const int steps = (K + STEP - 1) / STEP, nvs = nv <= 2 ? nv : nv <= 4 ? 4 : nv <= 8 ? 8 : 16;
    const long long tiles = (long long)(pair ? (M / 2 + 7) / 8 : (M + 15) / 16) * batches;
    bool found = false;
    double best = 0;
    for (int ranks = 1; ranks <= 4; ranks *= 2) {
        Q4GroupConfig c{};
        c.ranks = ranks;
        const int per = (steps + ranks - 1) / ranks;
        if (ranks > 1 && per * (ranks - 1) >= steps) break; // a CTA without steps
        const long long slots = ranks == 4 ? sm_count * 8 / 9 : sm_count; // (clusters of four leave some SMs of a GPC without a CTA)
        const long long per_sm = (tiles * ranks + slots - 1) / slots, waves = (per_sm + MAX_WARPS - 1) / MAX_WARPS;
        c.units = (int)((per_sm + waves - 1) / waves);
        c.parts = std::min(per, std::max(1, 20 / c.units));
        while (!complete(c, M, K, group, nv, pair) && c.units > 1) c.units = (c.units + 1) / 2, c.parts = std::min(per, std::max(1, 20 / c.units));
        if (!complete(c, M, K, group, nv, pair)) continue;
        const double staged = (double)per * nv * 16 / 640; // 16-byte pieces of activations a thread
        const double cost = (double)per_sm * per * (nvs > 8 ? 2 : 1) + 6 * staged + 8 * std::max(0.0, staged - (nvs > 8 ? 8 : 4)) +
                            (ranks == 4 ? 80 : ranks == 2 ? 55 : 0);
        if (found && cost >= best) continue;
        // two CTAs to an SM, of which one stages while the other works, where they stage little (51200 x 2560, groups of 128: one
        // vector 15.7 us, 16.4 as one CTA; 8 vectors, 55 KB each, 19.6 and 18.9; 16, 102 KB each, 31 and 25)
        if (c.units >= MAX_WARPS / 2 && ranks == 1) {
            Q4GroupConfig two = c;
            two.units = (c.units + 1) / 2;
            if (complete(two, M, K, group, nv, pair) && two.smem_bytes <= HALF_SMEM) c = two;
        }
        found = true, best = cost, *out = c;
    }
    return found;
}

cudaError_t launch_q4_group_gemv(const MatmulParams &p, rt_dtype act, int nv, int batches, const Q4GroupConfig &c, bool pair, bool lhs_constant,
                                 cudaStream_t stream) {
    Q4GroupParams q{};
    q.p = p;
    q.nv = nv;
    q.rows = c.rows;
    q.steps = (p.K + STEP - 1) / STEP;
    q.ranks = c.ranks;
    q.per_rank = c.per_rank;
    q.parts = c.parts;
    q.per_part = c.per_part;
    q.stride = c.stride;
    q.xsum_at = c.xsum_at;
    q.up_at = c.up_at;
    q.scales_at = c.scales_at;
    q.part_at = c.part_at;
    q.pair = pair;
    q.lhs_constant = lhs_constant;
    q.units = c.units;
    const int group = 1 << p.lhs_group_shift, per_row = c.per_rank * (STEP / group);
    q.fours = p.K / group % 4 == 0 && per_row % 4 == 0;
    const int n = q.fours ? per_row / 4 : per_row;
    q.magic = n > 1 ? (uint32_t)(((1ull << 32) + n - 1) / n) : 0u;
    q.nv_magic = nv > 1 ? (uint32_t)(((1ull << 32) + nv - 1) / nv) : 0u;
    return act == RT_F16 ? launch_t<__half>(q, c, batches, stream) : launch_t<__nv_bfloat16>(q, c, batches, stream);
}

} // namespace rt
