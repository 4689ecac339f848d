// mm16.h -- shared by the 16-bit matrix products (mm16_kernel.h, mm16_rows.hip) and their C entries (mm16.hip): argument
// blocks, the activations with their derivatives, and the epilogues on eight consecutive output columns.
#pragma once
#include "ga_common.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

enum { MM_KC = 0, MM_KS = 1 };   // operand element (row, k) lies at row * ld + k (K contiguous) / at k * ld + row (K strided)
// MM_ACT: y = act(v + bias) + residual, optionally v + bias kept.  MM_GATE: h = act(g + bg) * (u + bu), optionally both kept.
// MM_GATE_BWD: v = dh -> dg = dh u act'(g), du = dh act(g).  MM_PART: raw fp32 sums of one K range for mm_join.
enum { MM_ACT = 0, MM_GATE = 1, MM_GATE_BWD = 2, MM_PART = 3 };

enum { MM_S = 0, MM_L = 1, MM_D = 2, MM_R32 = 3, MM_R64 = 4 };   // tile configurations of mm16_kernel.h

constexpr int mm_wave_rows(int cfg) { return cfg == MM_D ? 4 : cfg == MM_R32 || cfg == MM_R64 ? 1 : 2; }     // waves of a tile along its rows

struct MmEpi {
    int act;
    const void *bias, *bias2;          // [N] in the operands' type, or null (bias2: of the second factor)
    const void* res; long long ldr;    // [M, N] or null
    void* out; long long ldo;          // MM_GATE_BWD: dg
    void* out2;                        // MM_GATE_BWD: du (row stride ldo)
    int npad;                          // >= N: columns N .. npad - 1 of out / out2 are written as zeros
    float *pre, *pre2; long long ldp;  // fp32 [M, ldp]: kept pre-activations (written by MM_ACT / MM_GATE, read by MM_GATE_BWD), or null
    float* part;                       // MM_PART: [splits][factors][M][ldpart]
    int ldpart;
    float* sums;                       // MM_GATE_BWD: null, or [tile rows x waves][2 npad]: column sums of dg and du before they are rounded
};

struct MmArgs {
    const char *q0, *q1;               // operand of the output's rows; q1: second K segment
    const char *p0, *p1;               // operand of the output's columns; p1: second K segment, or the second factor (DUAL)
    long long ldq, ldp;                // leading dimensions in BYTES
    int M, N;                          // output rows, columns (DUAL: of one factor)
    int Kq, Kp;                        // valid K of either operand in one segment; what lies beyond reads as zero
    int segs, splits;
    int ntm, ntn;
    MmEpi e;
};

// K steps of mm16_kernel.h
static inline int mm_steps(const MmArgs& a) { return a.segs * ((((a.Kq > a.Kp) ? a.Kq : a.Kp) + 63) / 64); }
int mm_launch_fwd(const MmArgs& a, bool bf, int epi, bool dual, int cfg, hipStream_t st);     // P, Q with K contiguous
int mm_launch_dgrad(const MmArgs& a, bool bf, int epi, int cfg, hipStream_t st);              // P with K strided
int mm_launch_wgrad(const MmArgs& a, bool bf, int epi, int cfg, hipStream_t st);              // both with K strided
// few rows: y / h of M <= ACMIL_FEW_ROWS rows straight from memory, any alignment of 2 bytes
int mm_launch_rows(const MmArgs& a, bool bf, bool dual, hipStream_t st);
int mm_rows_splits(int M, int cols, int K, bool dual);         // > 1: e.part receives the sums of each K range

// eight 16-bit values move in one piece from and to any address of theirs: the part's memory accesses of 16 bytes need no alignment (one by one,
// a product of 5000 x 200 x 3500, whose rows start on 8 bytes, took 50 us instead of 28)
typedef short mm_any8 __attribute__((ext_vector_type(8), aligned(2)));
template <bool BF> struct MmEl;
template <> struct MmEl<true> { typedef __bf16 T; typedef bf16x8 V; };
template <> struct MmEl<false> { typedef _Float16 T; typedef f16x8 V; };

// An epilogue evaluates these for every output, and on the vector unit of a CU that is no small part of a call: with the library's erff and an
// IEEE division a GELU layer of 768 rows took 3 us more than one without an activation, whatever its K.
// Sigmoid: one exponential, one reciprocal (1 ulp); exp overflows to inf for very negative z and the result is then exactly 0.
__device__ __forceinline__ float mm_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// Normal distribution function, e = exp(-z^2 / 2).  Phi(-x) = e P(t), t = 1 / (1 + 0.3 x): the form of Abramowitz and Stegun 7.1.26 with a
// degree-8 P fitted to least relative error over 0 <= x <= 14 (1.7e-7; in fp32: 6e-7 for x < 3, absolute 7e-8, and no loss in the lower tail).
__device__ __forceinline__ float mm_normal_cdf(float z, float& e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, fabsf(z), 1.0f));
    float p = 0.03567476198f;
    p = fmaf(p, t, -0.15720301867f);
    p = fmaf(p, t, 0.20635335147f);
    p = fmaf(p, t, -0.05368350446f);
    p = fmaf(p, t, 0.12856155634f);
    p = fmaf(p, t, 0.09991351516f);
    p = fmaf(p, t, 0.12075395882f);
    p = fmaf(p, t, 0.11962930113f);
    e = __expf(-0.5f * z * z);
    const float q = p * t * e;
    return z < 0.0f ? q : 1.0f - q;                                       // NaN stays NaN
}

__device__ __forceinline__ float mm_act(int act, float z) {
    switch (act) {
        case ACMIL_ACT_RELU: return z < 0.0f ? 0.0f : z;                 // NaN stays NaN
        case ACMIL_ACT_SILU: return z * mm_sigmoid(z);
        case ACMIL_ACT_GELU: { float e; return z * mm_normal_cdf(z, e); }
        case ACMIL_ACT_GELU_TANH: return z * mm_sigmoid(1.5957691216057308f * (z + 0.044715f * z * z * z));   // 0.5 z (1 + tanh t) = z sigmoid(2 t)
        case ACMIL_ACT_SIGMOID: return mm_sigmoid(z);
        default: return z;
    }
}

// act(z) and act'(z)
__device__ __forceinline__ float mm_act_slope(int act, float z, float& slope) {
    switch (act) {
        case ACMIL_ACT_RELU: slope = z > 0.0f ? 1.0f : 0.0f; return z < 0.0f ? 0.0f : z;
        case ACMIL_ACT_SILU: { const float s = mm_sigmoid(z); slope = s * (1.0f + z * (1.0f - s)); return z * s; }
        case ACMIL_ACT_GELU: {
            float e;
            const float c = mm_normal_cdf(z, e);
            slope = c + z * 0.39894228040143268f * e;
            return z * c;
        }
        case ACMIL_ACT_GELU_TANH: {
            const float s = mm_sigmoid(1.5957691216057308f * (z + 0.044715f * z * z * z));
            // (z^2 kept finite: beyond 5e19, which bf16 holds, 0.134145 z z is not, and the 0 in front of it would become NaN)
            slope = s + z * s * (1.0f - s) * 1.5957691216057308f * (1.0f + 0.134145f * fminf(z * z, 1e30f));
            return z * s;
        }
        case ACMIL_ACT_SIGMOID: { const float s = mm_sigmoid(z); slope = s * (1.0f - s); return s; }
        default: slope = 1.0f; return z;
    }
}

// eight at a time: one uniform branch on the activation, not one per element
#define MM_EACH_ACT(CASE) \
    switch (act) { \
        case ACMIL_ACT_RELU: CASE(ACMIL_ACT_RELU) break; \
        case ACMIL_ACT_SILU: CASE(ACMIL_ACT_SILU) break; \
        case ACMIL_ACT_GELU: CASE(ACMIL_ACT_GELU) break; \
        case ACMIL_ACT_GELU_TANH: CASE(ACMIL_ACT_GELU_TANH) break; \
        case ACMIL_ACT_SIGMOID: CASE(ACMIL_ACT_SIGMOID) break; \
        default: CASE(ACMIL_ACT_NONE) break; \
    }
__device__ __forceinline__ void mm_act8(int act, float* z) {
#define MM_CASE(A) { _Pragma("unroll") for (int j = 0; j < 8; ++j) z[j] = mm_act(A, z[j]); }
    MM_EACH_ACT(MM_CASE)
#undef MM_CASE
}
__device__ __forceinline__ void mm_act_slope8(int act, const float* z, float* a, float* slope) {
#define MM_CASE(A) { _Pragma("unroll") for (int j = 0; j < 8; ++j) a[j] = mm_act_slope(A, z[j], slope[j]); }
    MM_EACH_ACT(MM_CASE)
#undef MM_CASE
}

template <bool BF> __device__ __forceinline__ float mm_ld(const void* p, long long i) { return (float)((const typename MmEl<BF>::T*)p)[i]; }
template <bool BF> __device__ __forceinline__ void mm_ld8(const void* p, long long i, float* v) {
    const typename MmEl<BF>::V x = __builtin_bit_cast(typename MmEl<BF>::V, *(const mm_any8*)((const typename MmEl<BF>::T*)p + i));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)x[j];
}
template <bool BF> __device__ __forceinline__ void mm_st8(void* p, long long i, const float* v) {
    typename MmEl<BF>::V x;
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (typename MmEl<BF>::T)v[j];      // one rounding to the tensors' type, to nearest even
    *(mm_any8*)((typename MmEl<BF>::T*)p + i) = __builtin_bit_cast(mm_any8, x);
}
__device__ __forceinline__ void mm_ldf8(const float* p, float* v) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
}
__device__ __forceinline__ void mm_stf8(float* p, const float* v) {
    f32x4 a, b;
#pragma unroll
    for (int j = 0; j < 4; ++j) { a[j] = v[j]; b[j] = v[4 + j]; }
    *(f32x4*)p = a; *(f32x4*)(p + 4) = b;
}
// eight values of a [N] vector or of a row, from column n: nothing is read at or beyond N
template <bool BF> __device__ __forceinline__ void mm_row8(const void* p, long long base, int n, int N, float* v) {
    if (n + 8 <= N) { mm_ld8<BF>(p, base + n, v); return; }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = n + j < N ? mm_ld<BF>(p, base + n + j) : 0.0f;
}
// ... and their store; columns N .. npad - 1 become zero
template <bool BF> __device__ __forceinline__ void mm_put8(void* p, long long base, int n, int N, int npad, float* v) {
    if (n + 8 <= N) { mm_st8<BF>(p, base + n, v); return; }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (n + j < npad) ((typename MmEl<BF>::T*)p)[base + n + j] = (typename MmEl<BF>::T)(n + j < N ? v[j] : 0.0f);
}

// The epilogues: row m, columns n .. n + 7 (n a multiple of 8).  Kept pre-activations have ldp >= round8(N): all eight are written.
template <bool BF> __device__ __forceinline__ void mm_epi_act(const MmEpi& e, int m, int n, int N, float* v) {
    if (n >= e.npad) return;
    if (e.bias) {
        float b[8];
        mm_row8<BF>(e.bias, 0, n, N, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += b[j];
    }
    if (e.pre) mm_stf8(e.pre + m * e.ldp + n, v);
    mm_act8(e.act, v);
    if (e.res) {
        float r[8];
        mm_row8<BF>(e.res, m * e.ldr, n, N, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += r[j];
    }
    mm_put8<BF>(e.out, m * e.ldo, n, N, e.npad, v);
}

template <bool BF> __device__ __forceinline__ void mm_epi_gate(const MmEpi& e, int m, int n, int N, float* g, float* u) {
    if (n >= e.npad) return;
    if (e.bias) {
        float b[8];
        mm_row8<BF>(e.bias, 0, n, N, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] += b[j];
    }
    if (e.bias2) {
        float b[8];
        mm_row8<BF>(e.bias2, 0, n, N, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] += b[j];
    }
    if (e.pre) { mm_stf8(e.pre + m * e.ldp + n, g); mm_stf8(e.pre2 + m * e.ldp + n, u); }
    mm_act8(e.act, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] *= u[j];
    mm_put8<BF>(e.out, m * e.ldo, n, N, e.npad, g);
}

// sg, su: += dg, du as they are before they are rounded (a bias gradient sums them: with rounded ones it is off by half as much again)
template <bool BF> __device__ __forceinline__ void mm_epi_gate_bwd(const MmEpi& e, int m, int n, int N, float* v, float* sg, float* su) {
    if (n >= e.npad) return;
    float g[8], u[8], a[8], slope[8];
    mm_ldf8(e.pre + m * e.ldp + n, g);
    mm_ldf8(e.pre2 + m * e.ldp + n, u);
    mm_act_slope8(e.act, g, a, slope);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        g[j] = v[j] * u[j] * slope[j];
        u[j] = v[j] * a[j];
        sg[j] += n + j < N ? g[j] : 0.0f;
        su[j] += n + j < N ? u[j] : 0.0f;
    }
    mm_put8<BF>(e.out, m * e.ldo, n, N, e.npad, g);
    mm_put8<BF>(e.out2, m * e.ldo, n, N, e.npad, u);
}
