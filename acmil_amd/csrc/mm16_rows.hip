// mm16_rows.hip -- y = act(x W^T + b) + r and h = act(x Wg^T) * (x Wu^T) for FEW rows (a served token, a small batch of them).
//
// Such a call is bound by reading the weights once: 2 bytes per weight for 2 M flops.  So nothing goes through LDS on the way in: a
// workgroup of 8 waves owns 16 output columns, each wave an eighth of K, and a lane loads 16 bytes of "its" weight row straight into
// the A operand of v_mfma_f32_16x16x32 (a wave's load covers 64 contiguous bytes of 16 rows).  The batch of loads of the next steps
// is in flight while the present one multiplies.  The rows of x (padded to 16 with zeros that are never loaded) come from L2.  The 8 partial
// tiles meet in LDS, in a fixed order, and the epilogue stores whole 32-byte pieces.
// K, leading dimensions and base addresses may be anything the element type allows: 16-byte loads need no alignment here.
#include "mm16.h"

typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef s16x8 s16x8_any __attribute__((aligned(2)));

template <bool BF> __device__ __forceinline__ f32x4 mm_mfma16(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ s16x8 mm_load8(const short* p) { return *(const s16x8_any*)p; }
// the last chunk of a row: what lies at or beyond K reads as zero
__device__ __forceinline__ s16x8 mm_load_tail(const short* p, int k, int K) {
    s16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (k + j < K) v[j] = p[j];
    return v;
}

template <bool BF, int MT, bool DUAL>
__global__ __launch_bounds__(512) void mm16_rows_kernel(MmArgs a) {
    constexpr int NF = DUAL ? 2 : 1, U = MT * NF >= 4 ? 4 : 8;
    __shared__ __attribute__((aligned(16))) float red[8 * NF * MT * 256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16, r16 = lane & 15, kl = 8 * (lane >> 4), K = a.Kq;
    const int n = n0 + r16 < a.N ? n0 + r16 : a.N - 1;
    const short* p[2] = {(const short*)(a.p0 + (long long)n * a.ldp), (const short*)((DUAL ? a.p1 : a.p0) + (long long)n * a.ldp)};
    const short* q[MT];
    bool live[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        live[i] = r16 + 16 * i < a.M;
        q[i] = (const short*)(a.q0 + (long long)(live[i] ? r16 + 16 * i : 0) * a.ldq);
    }
    const int T = (K + 31) / 32, t0 = T * wave / 8, t1 = T * (wave + 1) / 8, full = K / 32;   // steps below `full` have all 32 k
    f32x4 acc[NF][MT];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[f][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    s16x8 pf[U][NF], qf[U][MT];
    const s16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
    int t = t0;
    auto load = [&](int tb) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (tb + u) * 32 + kl;
#pragma unroll
            for (int f = 0; f < NF; ++f) pf[u][f] = mm_load8(p[f] + k);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                qf[u][i] = zero;
                if (live[i]) qf[u][i] = mm_load8(q[i] + k);
            }
        }
    };
    auto mul = [&]() {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int f = 0; f < NF; ++f)
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[f][i] = mm_mfma16<BF>(pf[u][f], qf[u][i], acc[f][i]);
    };
    const int tf = t1 < full ? t1 : full;
    for (; t + U <= tf; t += U) { load(t); mul(); }
    for (; t < t1; ++t) {                                            // what is left: single steps, the last of them cut at K
        const int k = t * 32 + kl;
        s16x8 pv[NF], qv[MT];
#pragma unroll
        for (int f = 0; f < NF; ++f) pv[f] = k + 8 <= K ? mm_load8(p[f] + k) : mm_load_tail(p[f] + k, k, K);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            qv[i] = zero;
            if (live[i]) qv[i] = k + 8 <= K ? mm_load8(q[i] + k) : mm_load_tail(q[i] + k, k, K);
        }
#pragma unroll
        for (int f = 0; f < NF; ++f)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[f][i] = mm_mfma16<BF>(pv[f], qv[i], acc[f][i]);
    }
    // lane: row m = lane & 15, columns 4 (lane >> 4) .. + 3
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int i = 0; i < MT; ++i) *(f32x4*)(red + ((wave * NF + f) * MT + i) * 256 + r16 * 16 + 4 * (lane >> 4)) = acc[f][i];
    __syncthreads();
    const MmEpi& e = a.e;
    for (int x = threadIdx.x; x < MT * 256; x += 512) {
        const int m = x >> 4, c = n0 + (x & 15);
        float v[NF];
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            v[f] = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) v[f] += red[(w * NF + f) * MT * 256 + x];
        }
        if (m >= a.M || c >= e.npad) continue;
        typename MmEl<BF>::T* out = (typename MmEl<BF>::T*)e.out + m * e.ldo + c;
        if (c >= a.N) { *out = (typename MmEl<BF>::T)0.0f; continue; }
        if (e.bias) v[0] += mm_ld<BF>(e.bias, c);
        if (e.pre) e.pre[m * e.ldp + c] = v[0];
        float y = mm_act(e.act, v[0]);
        if constexpr (DUAL) {
            if (e.bias2) v[1] += mm_ld<BF>(e.bias2, c);
            if (e.pre) e.pre2[m * e.ldp + c] = v[1];
            y *= v[1];
        }
        if (e.res) y += mm_ld<BF>(e.res, m * e.ldr + c);
        *out = (typename MmEl<BF>::T)y;
    }
}

template <bool BF, int MT, bool DUAL> static int rows_go(const MmArgs& a, hipStream_t st) {
    const dim3 grid((a.e.npad + 15) / 16);
    hipLaunchKernelGGL((mm16_rows_kernel<BF, MT, DUAL>), grid, dim3(512), 0, st, a);
    return hipGetLastError() == hipSuccess ? ACMIL_OK : ACMIL_ERR_LAUNCH;
}
template <bool BF> static int rows_any(const MmArgs& a, bool dual, hipStream_t st) {
    if (a.M <= 16) return dual ? rows_go<BF, 1, true>(a, st) : rows_go<BF, 1, false>(a, st);
    return dual ? rows_go<BF, 2, true>(a, st) : rows_go<BF, 2, false>(a, st);
}
int mm_launch_rows(const MmArgs& a, bool bf, bool dual, hipStream_t st) {
    return bf ? rows_any<true>(a, dual, st) : rows_any<false>(a, dual, st);
}
