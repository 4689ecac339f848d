// mm16_rows.hip -- y = act(x W^T + b) + r and h = act(x Wg^T) * (x Wu^T) for FEW rows (a served token, a small batch of them).
//
// Such a call is bound by reading the weights once: 2 bytes per weight for 2 M flops.  So nothing goes through LDS on the way in: a
// workgroup of 8 waves owns 16 NT output columns (of both factors where there are two), each wave an eighth of K, and a lane loads 16
// bytes of "its" weight row straight into the A operand of v_mfma_f32_16x16x32 (a wave's load covers 64 contiguous bytes of 16 rows).  U
// steps of loads are always in flight: a step's registers are loaded again as soon as it has been multiplied.  The rows of x come from L2;
// the columns of the tile that stand for rows beyond M repeat a valid one and are never stored.
// x crosses the CU's L1 once per workgroup, next to the weights: with 16 columns a workgroup and 24 rows it is 1.5 times the weights, and
// the call slows to 2.6 TB/s.  So more rows get more columns per wave (NT), and where that leaves fewer workgroups than CUs, K is split
// over workgroups as well and joined behind.
// The 8 partial tiles meet in LDS, in a fixed order.  K, leading dimensions and base addresses may be anything the element type allows:
// 16-byte loads need no alignment here.
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

template <bool BF, int MT, bool DUAL, int NT>
__global__ __launch_bounds__(512) void mm16_rows_kernel(MmArgs a) {
    constexpr int NF = DUAL ? 2 : 1, W = 8, NP = NF * NT, U = NP + MT > 3 ? 4 : 8;      // up to 96 registers of loads
    __shared__ __attribute__((aligned(16))) float red[W * NP * MT * 256];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * 16 * NT, r16 = lane & 15, kl = 8 * (lane >> 4), K = a.Kq;
    const short* p[NP];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int n = n0 + 16 * j + r16 < a.N ? n0 + 16 * j + r16 : a.N - 1;
        p[j] = (const short*)(a.p0 + (long long)n * a.ldp);
        if constexpr (DUAL) p[NT + j] = (const short*)(a.p1 + (long long)n * a.ldp);
    }
    const short* q[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) q[i] = (const short*)(a.q0 + (long long)(r16 + 16 * i < a.M ? r16 + 16 * i : a.M - 1) * a.ldq);
    // Steps below `full` have all 32 k.  Up to 4 rows a wave takes a run of them (11008 -> 4096, 1 row: 19.3 us against 25.8 for steps in
    // turn); with more, the waves take them in turn and read whole lines of x together (4096 -> 11008 -> 4096, 24 rows: 88 us against 92).
    const int full = K / 32, parts = W * a.splits, part = blockIdx.y * W + wave;
    const bool turns = a.M > 4;
    const int t0 = turns ? part : (int)((long long)full * part / parts), by = turns ? parts : 1;
    const int tf = turns ? (full > part ? (full - part + parts - 1) / parts : 0) : (int)((long long)full * (part + 1) / parts) - t0;
    f32x4 acc[NP][MT];
#pragma unroll
    for (int f = 0; f < NP; ++f)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[f][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    s16x8 pf[U][NP], qf[U][MT];
    auto load = [&](int u, int t) __attribute__((always_inline)) {
        const int k = (t0 + t * by) * 32 + kl;
#pragma unroll
        for (int f = 0; f < NP; ++f) pf[u][f] = mm_load8(p[f] + k);
#pragma unroll
        for (int i = 0; i < MT; ++i) qf[u][i] = mm_load8(q[i] + k);
    };
    auto mul = [&](int u) __attribute__((always_inline)) {
#pragma unroll
        for (int f = 0; f < NP; ++f)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[f][i] = mm_mfma16<BF>(pf[u][f], qf[u][i], acc[f][i]);
    };
    int t = 0;
    if (t + U <= tf) {
#pragma unroll
        for (int u = 0; u < U; ++u) load(u, t + u);
        for (; t + 2 * U <= tf; t += U)
#pragma unroll
            for (int u = 0; u < U; ++u) {
                mul(u);
                load(u, t + U + u);
            }
#pragma unroll
        for (int u = 0; u < U; ++u) mul(u);
        t += U;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)                                      // fewer than U steps are left
        if (t + u < tf) load(u, t + u);
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (t + u < tf) mul(u);
    if (K % 32 != 0 && part == parts - 1) {                       // the one step that is cut at K
        const int k = full * 32 + kl;
        s16x8 pv[NP], qv[MT];
#pragma unroll
        for (int f = 0; f < NP; ++f) pv[f] = k + 8 <= K ? mm_load8(p[f] + k) : mm_load_tail(p[f] + k, k, K);
#pragma unroll
        for (int i = 0; i < MT; ++i) qv[i] = k + 8 <= K ? mm_load8(q[i] + k) : mm_load_tail(q[i] + k, k, K);
#pragma unroll
        for (int f = 0; f < NP; ++f)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[f][i] = mm_mfma16<BF>(pv[f], qv[i], acc[f][i]);
    }
    // lane: row m = lane & 15, columns 4 (lane >> 4) .. + 3
#pragma unroll
    for (int f = 0; f < NP; ++f)
#pragma unroll
        for (int i = 0; i < MT; ++i) *(f32x4*)(red + ((wave * NP + f) * MT + i) * 256 + r16 * 16 + 4 * (lane >> 4)) = acc[f][i];
    __syncthreads();
    const MmEpi& e = a.e;
    for (int y = threadIdx.x; y < NT * MT * 256; y += 512) {         // column tile j, row m, column of the tile
        const int j = y / (MT * 256), x = y - j * (MT * 256), m = x >> 4, c = n0 + 16 * j + (x & 15);
        float v[NF];
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            v[f] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) v[f] += red[(w * NP + f * NT + j) * MT * 256 + x];
        }
        if (m >= a.M) continue;
        if (e.part) {                                                // this K range's sums, for the join
            if (c < e.ldpart)
#pragma unroll
                for (int f = 0; f < NF; ++f) e.part[((size_t)(blockIdx.y * NF + f) * a.M + m) * e.ldpart + c] = v[f];
            continue;
        }
        if (c >= e.npad) continue;
        typename MmEl<BF>::T* out = (typename MmEl<BF>::T*)e.out + m * e.ldo + c;
        if (c >= a.N) { *out = (typename MmEl<BF>::T)0.0f; continue; }
        if (e.bias) v[0] += mm_ld<BF>(e.bias, c);
        if (e.pre) e.pre[m * e.ldp + c] = v[0];
        float o = mm_act(e.act, v[0]);
        if constexpr (DUAL) {
            if (e.bias2) v[1] += mm_ld<BF>(e.bias2, c);
            if (e.pre) e.pre2[m * e.ldp + c] = v[1];
            o *= v[1];
        }
        if (e.res) o += mm_ld<BF>(e.res, m * e.ldr + c);
        *out = (typename MmEl<BF>::T)o;
    }
}

// columns of a workgroup, and how many ways K is split over workgroups (at least 4 steps for each of the 8 waves)
static int rows_tiles(int M, bool dual) { return M <= 4 ? 1 : M <= 16 ? (dual ? 1 : 2) : dual ? 2 : 4; }
int mm_rows_splits(int M, int cols, int K, bool dual) {
    if (M <= 4) return 1;
    const int nt = rows_tiles(M, dual), grid = (cols + 16 * nt - 1) / (16 * nt), most = (K + 1023) / 1024;
    const int want = grid >= 256 ? 1 : (511 + grid) / grid;
    return want < most ? want : most;
}
template <bool BF, int MT, bool DUAL, int NT> static int rows_go(const MmArgs& a, hipStream_t st) {
    const int cols = a.e.part ? a.e.ldpart : a.e.npad;
    hipLaunchKernelGGL((mm16_rows_kernel<BF, MT, DUAL, NT>), dim3((cols + 16 * NT - 1) / (16 * NT), a.splits), dim3(512), 0, st, a);
    return hipGetLastError() == hipSuccess ? ACMIL_OK : ACMIL_ERR_LAUNCH;
}
template <bool BF> static int rows_any(const MmArgs& a, bool dual, hipStream_t st) {
    if (a.M <= 4) return dual ? rows_go<BF, 1, true, 1>(a, st) : rows_go<BF, 1, false, 1>(a, st);
    if (a.M <= 16) return dual ? rows_go<BF, 1, true, 1>(a, st) : rows_go<BF, 1, false, 2>(a, st);
    return dual ? rows_go<BF, 2, true, 2>(a, st) : rows_go<BF, 2, false, 4>(a, st);
}
int mm_launch_rows(const MmArgs& a, bool bf, bool dual, hipStream_t st) {
    return bf ? rows_any<true>(a, dual, st) : rows_any<false>(a, dual, st);
}
