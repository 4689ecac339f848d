// ortho.hip -- orthogonalisation of matrices by Newton-Schulz products: X = G / (|G|_F + eps), then `steps` times
//   A = X X^T;   B = b A + c A A;   X <- a X + B X        (on G^T where G has more rows than columns, so that A is the small Gram matrix).
// The odd polynomial a s + b s^3 + c s^5 acts on the singular values and drives them towards 1, whatever the singular vectors are.
//
// Arithmetic.  A single 16-bit product would not do: errors of the null directions are multiplied by a^steps (485 for 3.4445^5).  Every
// value is held as a pair of f16 halves, hi + lo, of 4096 times itself (|X|, |A|, |B| are bounded by the polynomial, checked on the host, and
// cannot overflow), and a product is hi hi + hi lo + lo hi on v_mfma_f32_16x16x32_f16 with fp32 accumulation, at a multiple of the rate of an fp32
// product.  What is held is off by at most 2^-22 of the value and 2^-37 of |G|_F: below 2^-15 of |G|_F the lo half is an f16 subnormal.  For a Gaussian
// matrix the result is as far from 64 bits as an fp32 iteration's; where that one is nearly exact, or one value outweighs the rest, it is further: 9
// times for an identity of 512 x 768 (4.9e-5 against 5.5e-6 of a norm of 22.6), and what is 1e-7 of |G|_F keeps 13 bits.
//
// Layout.  A row of K values lies as blocks of 32: 64 bytes of hi halves, then 64 bytes of lo halves.  A K step of 32 is then
// exactly one 128-byte row piece, and tiles move and lie in LDS like those of mm16_kernel.h, the first of a fragment's two halves being hi, the
// second lo.  K is padded to a multiple of 32 with zeros, so there is no tail.  All three products take both operands with K
// contiguous: X is kept in both orientations (its transpose twice, read and written alternately).  A and B are symmetric: only tiles on
// and below the diagonal are computed and each is written a second time, mirrored.
// All matrices of a call go through the same launches: 2 + 3 steps of them, whatever the number of matrices (up to NS_GROUP at a time); where
// all are small, one launch does everything (ns_tiny_kernel).
#include "mm16_kernel.h"

#include <cmath>

#define NS_GROUP 24
#define NS_SCALE 4096.0f          // |X| <= 3.9, |A|, |B| <= 15.5 (host check) stay below 65504

struct NsMat {
    const void* g; void* o; long long ldg, ldo;
    char *X, *XT0, *XT1, *A, *B;  // pair planes: X [s][t], XT [t][s], A and B [s][s]
    int s, t, tall, pad;          // s <= t; tall: G is [t][s]
};
struct NsArgs {
    int count, flip, last;        // flip: XT1 is the present transpose; last: X goes to o
    float a, b, c;
    float eps;
    const double* part;
    int first[NS_GROUP + 1];      // first workgroup of each matrix
    NsMat m[NS_GROUP];
};

enum { NS_GRAM = 0, NS_POLY = 1, NS_STEP = 2 };

__host__ __device__ static inline int ns_r32(int n) { return (n + 31) & ~31; }
__host__ __device__ static inline long long ns_ld(int k) { return ns_r32(k) * 4LL; }           // bytes of a row of k pairs
__device__ __forceinline__ long long ns_at(int k) { return (k >> 5) * 128LL + (k & 31) * 2; }  // byte of the hi half of column k; lo: + 64

__device__ __forceinline__ int ns_find(const NsArgs& a, int b) {
    int i = 0;
    while (i + 1 < a.count && b >= a.first[i + 1]) ++i;
    return i;
}

template <int DT> __device__ __forceinline__ float ns_load(const void* p, long long i) {
    if constexpr (DT == ACMIL_DTYPE_F32) return ((const float*)p)[i];
    else if constexpr (DT == ACMIL_DTYPE_F16) return (float)((const _Float16*)p)[i];
    else return (float)((const __bf16*)p)[i];
}
template <int DT> __device__ __forceinline__ void ns_store(void* p, long long i, float v) {
    if constexpr (DT == ACMIL_DTYPE_F32) ((float*)p)[i] = v;
    else if constexpr (DT == ACMIL_DTYPE_F16) ((_Float16*)p)[i] = (_Float16)v;
    else ((__bf16*)p)[i] = (__bf16)v;
}

// eight neighbouring values of a row, from column c (a multiple of 8); zeros at and beyond cols.  vec: rows start on 16 bytes
template <int DT> __device__ __forceinline__ void ns_load8(const void* p, long long row, int c, int cols, bool vec, float* v) {
    if (vec && c + 8 <= cols) {
        if constexpr (DT == ACMIL_DTYPE_F32) mm_ldf8((const float*)p + row + c, v);
        else mm_ld8<DT == ACMIL_DTYPE_BF16>(p, row + c, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? ns_load<DT>(p, row + c + j) : 0.0f;
}
template <int DT> __device__ __forceinline__ bool ns_on16(const void* g, long long ldg) {
    return ((size_t)g & 15) == 0 && ldg % (DT == ACMIL_DTYPE_F32 ? 4 : 8) == 0;
}

// sum of squares, in 64 bits (a gradient's squares leave the range of 32): NS_PARTS partial sums per matrix, fixed order
#define NS_PARTS 256
template <int DT> __global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs a, double* part) {
    const NsMat& m = a.m[blockIdx.y];
    const int rows = m.tall ? m.t : m.s, cols = m.tall ? m.s : m.t, cpr = (cols + 7) / 8;
    const bool vec = ns_on16<DT>(m.g, m.ldg);
    const long long total = (long long)rows * cpr, step = NS_PARTS * 256LL;
    double s = 0.0;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += 2 * step) {
        float v[2][8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {                                 // two chunks on their way at a time
            const long long k = i + h * step, r = k / cpr;
            if (k < total) ns_load8<DT>(m.g, r * m.ldg, (int)(k - r * cpr) * 8, cols, vec, v[h]);
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) v[h][j] = 0.0f;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += (double)v[h][j] * (double)v[h][j];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    __shared__ double red[4];
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * NS_PARTS + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

__device__ __forceinline__ void ns_put8(char* hi, const float* v) {          // eight scaled values -> their hi and lo halves
    unsigned h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) ga_split_pair_f16(v[2 * j], v[2 * j + 1], h[j], l[j]);
    *(u32x4*)hi = u32x4{h[0], h[1], h[2], h[3]};
    *(u32x4*)(hi + 64) = u32x4{l[0], l[1], l[2], l[3]};
}
__device__ __forceinline__ void ns_get8(const char* hi, float* v) {
    const f16x8 h = *(const f16x8*)hi, l = *(const f16x8*)(hi + 64);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)h[j] + (float)l[j];
}

// G / (|G|_F + eps) in both orientations, 64 x 64 values per workgroup turned through LDS
template <int DT> __global__ __launch_bounds__(256) void ns_split_kernel(NsArgs a) {
    __shared__ float tile[64][65];
    __shared__ double scale_s;                                        // in 64 bits: 1 / |G| may leave the range of 32
    const int mi = ns_find(a, blockIdx.x);
    const NsMat& m = a.m[mi];
    const int rows = m.tall ? m.t : m.s, cols = m.tall ? m.s : m.t;
    const int ct = (cols + 63) / 64, id = blockIdx.x - a.first[mi], r0 = id / ct * 64, c0 = id % ct * 64;
    float in[2][8];
    const bool vec = ns_on16<DT>(m.g, m.ldg);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = r0 + (threadIdx.x >> 3) + 32 * h, c = c0 + (threadIdx.x & 7) * 8;
        if (r < rows) ns_load8<DT>(m.g, r * m.ldg, c, cols, vec, in[h]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) in[h][j] = 0.0f;
    }
    if (threadIdx.x < 64) {                                           // every workgroup adds the partial sums up for itself, in one order
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < NS_PARTS / 64; ++i) s += a.part[mi * NS_PARTS + i * 64 + threadIdx.x];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (threadIdx.x == 0) scale_s = (double)NS_SCALE / (sqrt(s) + (double)a.eps);
    }
    __syncthreads();
    const double scale = scale_s;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[(threadIdx.x >> 3) + 32 * h][(threadIdx.x & 7) * 8 + j] = (float)((double)in[h][j] * scale);
    __syncthreads();
    char* direct = m.tall ? m.XT0 : m.X;      // [rows][cols]
    char* turned = m.tall ? m.X : m.XT0;      // [cols][rows]
#pragma unroll
    for (int i = threadIdx.x; i < 512; i += 256) {
        const int r = i >> 3, c = (i & 7) * 8;
        float v[8];
        if (r0 + r < rows && c0 + c < ns_r32(cols)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = tile[r][c + j];
            ns_put8(direct + (r0 + r) * ns_ld(cols) + ns_at(c0 + c), v);
        }
        if (c0 + r < cols && r0 + c < ns_r32(rows)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = tile[c + j][r];
            ns_put8(turned + (c0 + r) * ns_ld(rows) + ns_at(r0 + c), v);
        }
    }
}

// One product tile.  As in mm16_kernel.h, with 32 pairs a step and so one piece a step: the fragments of step t + 1 are read while those of
// step t multiply, and behind the barrier in front of step t both slots of its stage are free.  D steps are in flight or being read.
// KG groups of waves take a share of the steps each, with a ring of their own, and add up in LDS: where there are fewer tiles than CUs, one
// group spends most of a step waiting for its barrier and its fragments.
template <class C, int D, int KG, int KIND, int DT>
__global__ __launch_bounds__(C::WAVES * KG * 64) void ns_kernel(NsArgs a) {
    constexpr int MT = C::MT, NT = C::NT;
    constexpr int SLOT = C::QB, SLOTS = 2 * D + 1;
    static_assert(C::QB == C::PB && D >= 2, "either operand fits any slot");
    __shared__ __attribute__((aligned(128))) char smem[KG * SLOTS * SLOT];
    static_assert(MT % 2 == 0 && C::WAVES * 32 * 20 * 4 <= SLOTS * SLOT, "room for the turned tiles");
    static_assert((KG - 1) * C::WAVES * MT * NT * 1024 <= KG * SLOTS * SLOT, "room for the other groups' sums");
    const int lane = threadIdx.x & 63, wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = wave_all / C::WAVES, wave = wave_all % C::WAVES;
    const int wm = wave / C::WN, wn = wave % C::WN;
    int blk;
    {   // workgroup b runs on XCD b % 8: every XCD takes one contiguous run of tiles
        const int nt = gridDim.x, q = nt >> 3, r = nt & 7, x = blockIdx.x & 7, i = blockIdx.x >> 3;
        blk = x * q + (x < r ? x : r) + i;
    }
    const int mi = ns_find(a, blk);
    const NsMat& mat = a.m[mi];
    const int s = mat.s, t = mat.t, id = blk - a.first[mi];
    const int M = s, N = KIND == NS_STEP ? t : s, K = KIND == NS_GRAM ? t : s;
    int tm, tn;
    if (KIND == NS_STEP) {
        const int ntm = (M + C::BM - 1) / C::BM, ntn = (N + C::BN - 1) / C::BN;
        const int width = 4 * ntn, g = id / width, f = 4 * g, sz = ntm - f < 4 ? ntm - f : 4;
        tm = f + (id % width) % sz;
        tn = (id % width) / sz;
    } else {                                                          // row by row of the lower triangle
        static_assert(KIND == NS_STEP || C::BM == C::BN, "square tiles on the diagonal");
        tm = (int)((__builtin_sqrtf(8.0f * id + 1.0f) - 1.0f) * 0.5f);
        while ((tm + 1) * (tm + 2) / 2 <= id) ++tm;
        while (tm * (tm + 1) / 2 > id) --tm;
        tn = id - tm * (tm + 1) / 2;
    }
    const int m0 = tm * C::BM, n0 = tn * C::BN;
    const char* XT = a.flip ? mat.XT1 : mat.XT0;
    const char* qp = KIND == NS_GRAM ? mat.X : KIND == NS_POLY ? mat.A : mat.B;
    const char* pp = KIND == NS_GRAM ? mat.X : KIND == NS_POLY ? mat.A : XT;
    const long long ldk = ns_ld(K);
    MmLoad<MM_KC, C::BM, C::WAVES> lq;
    MmLoad<MM_KC, C::BN, C::WAVES> lp;
    lq.init(wave, lane, ldk, m0, M);
    lp.init(wave, lane, ldk, n0, N);
    qp += m0 * ldk;
    pp += n0 * ldk;
    const int all = ns_r32(K) / 32, t0 = all * group / KG, T = all * (group + 1) / KG - t0, most = (all + KG - 1) / KG;
    qp += t0 * 128LL;
    pp += t0 * 128LL;
    const unsigned smem0 = mm_lds_addr(smem) + group * SLOTS * SLOT;
    constexpr int NI = decltype(lq)::NI;
    auto fetch = [&](bool rows, int step, int slot, auto piece) MM_INLINE {
        constexpr int k = decltype(piece)::value;
        const long long at = (step < T ? step : T > 0 ? T - 1 : -t0) * 128LL;      // behind the last step it is fetched again, unused
        const unsigned lds = smem0 + slot * SLOT + (k * C::WAVES + wave) * 1024;
        if (rows) mm_dma_s(lq.off[k], qp + at, lds);
        else mm_dma_s(lp.off[k], pp + at, lds);
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    MmFrag<MM_KC, C::BM> fq;
    MmFrag<MM_KC, C::BN> fp;
    fq.init(lane, wm * C::TM);
    fp.init(lane, wn * C::TN);
    mm_lds* const ring = (mm_lds*)smem + group * SLOTS * SLOT;
    s16x8 ph[2][NT], pl[2][NT], qh[MT], ql[MT];
    auto read_p = [&](mm_lds* slot, auto set, auto kf) MM_INLINE {
        constexpr int x = decltype(set)::value, f = decltype(kf)::value;
        ph[x][f] = fp.get(slot, 16 * f, 0);
        pl[x][f] = fp.get(slot, 16 * f, 1);
    };
    auto read_q = [&](mm_lds* slot, auto kf) MM_INLINE {
        constexpr int f = decltype(kf)::value;
        qh[f] = fq.get(slot, 16 * f, 0);
        ql[f] = fq.get(slot, 16 * f, 1);
    };
    mm_for<0, SLOTS>([&](auto h) MM_INLINE {
        constexpr int k = decltype(h)::value;
        mm_for<0, NI>([&](auto d) MM_INLINE { fetch(k % 2 == 0, k / 2, k, d); });
    });
    mm_wait_dma<NI * (2 * D - 1)>();
    ga_lds_barrier();
    int qs = 0, ps = 1;                                               // slots of Q_t and P_t
    mm_for<0, NT>([&](auto f) MM_INLINE { read_p(ring + SLOT, std::integral_constant<int, 0>{}, f); });
    mm_for<0, MT>([&](auto f) MM_INLINE { read_q(ring, f); });
    auto step = [&](int t, auto set) MM_INLINE {
        constexpr int x = decltype(set)::value;
        mm_wait_dma<NI * (2 * D - 3)>();                              // stage t + 1 has landed, for everybody behind the barrier; stage t is read
        ga_lds_barrier();
        if (KG > 1 && t >= T) return;                                 // another group has one step more
        const int nq = qs >= SLOTS - 2 ? qs + 2 - SLOTS : qs + 2, np = ps >= SLOTS - 2 ? ps + 2 - SLOTS : ps + 2;
        mm_for<0, MT>([&](auto ki) MM_INLINE {
            constexpr int i = decltype(ki)::value;
            mm_for<i * NT / MT, (i + 1) * NT / MT>([&](auto f) MM_INLINE { read_p(ring + np * SLOT, std::integral_constant<int, 1 - x>{}, f); });
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mm_mfma<false>(pl[x][j], qh[i], acc[i][j]);          // the small products first
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mm_mfma<false>(ph[x][j], ql[i], acc[i][j]);
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = mm_mfma<false>(ph[x][j], qh[i], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
            read_q(ring + nq * SLOT, ki);
            mm_for<i * 2 * NI / MT, (i + 1) * 2 * NI / MT>([&](auto d) MM_INLINE {
                constexpr int k = decltype(d)::value;
                if constexpr (k < NI) fetch(false, t + D, qs, d);
                else fetch(true, t + D + 1, ps, std::integral_constant<int, k - NI>{});
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        qs = nq;
        ps = np;
    };
    for (int t = 0; t < most; t += 2) {
        step(t, std::integral_constant<int, 0>{});
        if (t + 1 < most) step(t + 1, std::integral_constant<int, 1>{});
    }
    mm_wait_dma<0>();
    ga_lds_barrier();
    if constexpr (KG > 1) {
        f32x4* sums = (f32x4*)smem;                                   // [group - 1][wave][tile][lane]
        if (group > 0)
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) sums[(((group - 1) * C::WAVES + wave) * MT * NT + i * NT + j) * 64 + lane] = acc[i][j];
        __syncthreads();
        if (group == 0)
#pragma unroll
            for (int g = 1; g < KG; ++g)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] += sums[(((g - 1) * C::WAVES + wave) * MT * NT + i * NT + j) * 64 + lane];
        __syncthreads();
        if (group > 0) return;
    }

    // Epilogue, 32 rows x 16 columns of a wave at a time: [m][n] with 8 consecutive n per lane, then [n][m] with 8 consecutive m.
    float* st = (float*)smem + wave * (32 * 20);
    char* XTn = a.flip ? mat.XT0 : mat.XT1;
    char* dst = KIND == NS_GRAM ? mat.A : KIND == NS_POLY ? mat.B : mat.X;
    const char* old = KIND == NS_POLY ? mat.A : mat.X;
    const long long ldn = ns_ld(N), ldm = ns_ld(M);
    const bool user = KIND == NS_STEP && a.last;
#pragma unroll
    for (int i = 0; i < MT / 2; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int ii = 0; ii < 2; ++ii) *(f32x4*)(st + (16 * ii + (lane & 15)) * 20 + 4 * (lane >> 4)) = acc[2 * i + ii][j];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const int mb = m0 + wm * C::TM + 32 * i, nb = n0 + wn * C::TN + 16 * j;
            {
                const int row = lane >> 1, c = (lane & 1) * 8, m = mb + row, n = nb + c;
                float v[8];
                mm_ldf8(st + row * 20 + c, v);
                if (m < M && n < ns_r32(N)) {
                    if (KIND == NS_GRAM) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] *= 1.0f / NS_SCALE;
                    } else {
                        float x[8];
                        ns_get8(old + m * ldn + ns_at(n), x);
                        const float ca = KIND == NS_POLY ? a.b : a.a, cc = KIND == NS_POLY ? a.c / NS_SCALE : 1.0f / NS_SCALE;
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = ca * x[e] + cc * v[e];
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = n + e < N ? v[e] : 0.0f;
                    if (!user) ns_put8(dst + m * ldn + ns_at(n), v);
                    else if (!mat.tall) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (n + e < N) ns_store<DT>(mat.o, m * mat.ldo + n + e, v[e] * (1.0f / NS_SCALE));
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = 0.0f;          // rows beyond the last are columns of zeros of the transpose
                }
                mm_stf8(st + row * 20 + c, v);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (KIND == NS_STEP ? (!user || mat.tall) : tm != tn) {
                char* tr = KIND == NS_STEP ? XTn : dst;
                const int mc = (lane >> 4) * 8, n = nb + (lane & 15), m = mb + mc;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = st[(mc + e) * 20 + (lane & 15)];
                if (n < N && m < ns_r32(M)) {
                    if (!user) ns_put8(tr + n * ldm + ns_at(m), v);
                    else {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (m + e < M) ns_store<DT>(mat.o, n * mat.ldo + m + e, v[e] * (1.0f / NS_SCALE));
                    }
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
}

// Small matrices, whole iterations in one workgroup.  Where X, both halves, and one s x s matrix fit the 160 KB of LDS (64 x 512, 128 x 160),
// a call of 2 + 3 steps dependent launches is nothing but their latencies.  Here a workgroup loads its matrix once (through registers: the norm is
// formed on the way), keeps X in LDS and multiplies there: A = X X^T from rows of X, B over A, X <- a X + B X in place (32 columns are a wave's
// own: it holds them as fragments before it writes).  X is its own transpose, read by ds_read_b64_tr_b16.  Rows are padded by 16 bytes: their
// length in banks is then an odd multiple of 4, and 16 rows of 16 bytes meet no bank twice.  Same arithmetic, same roundings as the tiles.
//
// (a on the diagonal of B would save reading X back, but rounds a X once more: 5 times the error of an fp32 iteration for a rank-one matrix.)
// A step of 64 x 512 takes about 10 us, half of it matrix instructions and LDS reads, half the epilogues' conversions.  Against the tiles:
// 16 x 16 11 us (65), 64 x 64 23 (73), 64 x 512 54 (87), 128 x 160 64 (90), sixty of 128 x 128 56 (325).
#define NS_TINY 60                // matrices of a launch: what the kernel arguments hold
#define NS_TINY_LDS (160 * 1024 - 64)
#define NS_TINY_CHUNKS 10         // of 8 values per thread: s t <= 40 000
#define NS_MAX_STEPS 64

struct NsTinyMat { const void* g; void* o; long long ldg, ldo; int s, t, tall, pad; };
struct NsTiny {
    int steps; float eps;
    float co[3 * NS_MAX_STEPS];
    NsTinyMat m[NS_TINY];
};
// bytes behind X: A, or the partial tiles of one round of a sum
__host__ __device__ constexpr long long ns_tiny_square(int S) { return S == 32 ? 12 * 1024 : S * (S + 8) * 4LL; }
__host__ __device__ static inline bool ns_tiny_fits(int s, int t) {
    const long long S = ns_r32(s), T = ns_r32(t);
    return S <= 128 && S * (T + 8) * 4 + ns_tiny_square((int)S) <= NS_TINY_LDS;
}
__device__ __forceinline__ void ns_tiny_put(short* h, short* l, f32x4 v) {
    unsigned hi[2], lo[2];
    ga_split_pair_f16(v[0], v[1], hi[0], lo[0]);
    ga_split_pair_f16(v[2], v[3], hi[1], lo[1]);
    *(uint2*)h = uint2{hi[0], hi[1]};
    *(uint2*)l = uint2{lo[0], lo[1]};
}
// acc += c (hi + lo)
__device__ __forceinline__ void ns_tiny_add(f32x4& acc, float c, const short* h, const short* l) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    const h4 x = *(const h4*)h, y = *(const h4*)l;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf((float)x[e], c, fmaf((float)y[e], c, acc[e]));
}

// the iterations; SK = padded s / 32
template <int DT, int SK> struct NsTinyRun {
    static constexpr int S = 32 * SK, LDA = S + 8, UNITS = SK * SK, PER_WAVE = (UNITS + 7) / 8;           // units of 32 x 32 of an s x s matrix
    static constexpr int KSPLIT = SK == 1 ? 4 : SK == 2 ? 2 : 1;      // ways K of X X^T is split over waves
    static_assert((KSPLIT - 1) * UNITS * 4096 <= ns_tiny_square(S), "partial sums lie over A");

    // A = X X^T, or (POLY; h, l are A) B = cb A + cc A A over A.  A is symmetric: its rows are its columns
    template <int KS, bool POLY> static __device__ __forceinline__ void square(const short* h, const short* l, int ld, int K, short* Ah, float cb, float cc) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, kg = lane >> 4, kq = KS == 1 ? 0 : wave / UNITS;
        short* Al = Ah + S * LDA;
        f32x4 acc[PER_WAVE][2][2] = {};
#pragma unroll
        for (int w = 0; w < PER_WAVE; ++w) {
            const int u = KS == 1 ? wave + 8 * w : wave % UNITS, m0 = u / SK * 32, n0 = u % SK * 32;
            if (u >= UNITS || kq >= KS) continue;
            const int q = (m0 + r) * ld + 8 * kg, p = (n0 + r) * ld + 8 * kg;
            for (int k = 32 * kq; k < K; k += 32 * KS) {
                s16x8 ph[2], pl[2], qh[2], ql[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    ph[i] = *(const s16x8*)(h + p + 16 * i * ld + k); pl[i] = *(const s16x8*)(l + p + 16 * i * ld + k);
                    qh[i] = *(const s16x8*)(h + q + 16 * i * ld + k); ql[i] = *(const s16x8*)(l + q + 16 * i * ld + k);
                }
#pragma unroll
                for (int o = 0; o < 3; ++o)                           // the small products first
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j) acc[w][i][j] = mm_mfma<false>(o == 0 ? pl[j] : ph[j], o == 1 ? ql[i] : qh[i], acc[w][i][j]);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int m = m0 + 16 * i + r, n = n0 + 16 * j + 4 * kg;
                    acc[w][i][j] *= POLY ? cc / NS_SCALE : 1.0f / NS_SCALE;
                    if (POLY) ns_tiny_add(acc[w][i][j], cb, Ah + m * LDA + n, Al + m * LDA + n);
                }
        }
        if (POLY) __syncthreads();                                    // everybody has read A
        if (KS > 1 && K > 32) {
            f32x4* part = (f32x4*)Ah + (wave % UNITS) * 256 + lane;   // [kq - 1][unit][tile][lane]
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (kq > 0 && kq < KS) part[((kq - 1) * UNITS * 4 + i) * 64] = acc[0][i >> 1][i & 1];
            __syncthreads();
#pragma unroll
            for (int k = 0; k + 1 < KS; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (kq == 0) acc[0][i >> 1][i & 1] += part[(k * UNITS * 4 + i) * 64];
            __syncthreads();
        }
#pragma unroll
        for (int w = 0; w < PER_WAVE; ++w) {
            const int u = KS == 1 ? wave + 8 * w : wave % UNITS, at = (u / SK * 32 + r) * LDA + u % SK * 32 + 4 * kg;
            if (u >= UNITS || kq > 0) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) ns_tiny_put(Ah + at + 16 * i * LDA + 16 * j, Al + at + 16 * i * LDA + 16 * j, acc[w][i][j]);
        }
        __syncthreads();
    }

    static __device__ __forceinline__ void run(const NsTiny& a, const NsTinyMat& m, char* smem) {
        const int T = ns_r32(m.t), ldx = T + 8, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, kg = lane >> 4;
        short *Xh = (short*)smem, *Xl = Xh + S * ldx, *Ah = Xl + S * ldx, *Al = Ah + S * LDA;
        mm_lds* const lds = (mm_lds*)smem;
        const unsigned xl = S * ldx * 2;
        const unsigned turn = ((8 * kg + (r >> 2)) * ldx + 4 * (lane & 3)) * 2;                  // of a K-strided fragment: MmFrag, without a permutation
        auto frag = [&](mm_lds* q) MM_INLINE {
            const s16x4 x = __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) mm_h4*)q));
            const s16x4 y = __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) mm_h4*)(q + 8 * ldx)));
            return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        };
        for (int step = 0; step < a.steps; ++step) {
            const float ca = a.co[3 * step];
            square<KSPLIT, false>(Xh, Xl, ldx, T, Ah, 0.0f, 0.0f);
            square<1, true>(Ah, Al, LDA, S, Ah, a.co[3 * step + 1], a.co[3 * step + 2]);
            // X <- a X + B X.  B, up to 64 x 64, is read once for all columns of a wave
            constexpr bool HELD = SK <= 2;
            s16x8 qh[HELD ? 2 * SK : 1][SK], ql[HELD ? 2 * SK : 1][SK];
            if constexpr (HELD)
#pragma unroll
                for (int i = 0; i < 2 * SK; ++i)
#pragma unroll
                    for (int k = 0; k < SK; ++k) {
                        qh[i][k] = *(const s16x8*)(Ah + (16 * i + r) * LDA + 32 * k + 8 * kg);
                        ql[i][k] = *(const s16x8*)(Al + (16 * i + r) * LDA + 32 * k + 8 * kg);
                    }
            // (the last step, with its bounds on what is stored, is a copy of its own: branches between the tiles keep them from overlapping)
            auto columns = [&](int n0, auto last) MM_INLINE {
                s16x8 ph[SK][2], pl[SK][2];
#pragma unroll
                for (int k = 0; k < SK; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        mm_lds* p = lds + turn + (32 * k * ldx + n0 + 16 * j) * 2;
                        ph[k][j] = frag(p);
                        pl[k][j] = frag(p + xl);
                    }
                auto rows = [&](int i, const s16x8* bh, const s16x8* bl) MM_INLINE {
                    f32x4 acc[2] = {};
#pragma unroll
                    for (int k = 0; k < SK; ++k)
#pragma unroll
                        for (int p = 0; p < 3; ++p)
#pragma unroll
                            for (int j = 0; j < 2; ++j) acc[j] = mm_mfma<false>(p == 0 ? pl[k][j] : ph[k][j], p == 1 ? bl[k] : bh[k], acc[j]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int mr = 16 * i + r, n = n0 + 16 * j + 4 * kg, at = mr * ldx + n;
                        f32x4 v = acc[j] * (1.0f / NS_SCALE);
                        ns_tiny_add(v, ca, Xh + at, Xl + at);
                        if constexpr (!decltype(last)::value) ns_tiny_put(Xh + at, Xl + at, v);
                        else if (mr < m.s)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (n + e < m.t) ns_store<DT>(m.o, m.tall ? (n + e) * m.ldo + mr : mr * m.ldo + n + e, v[e] * (1.0f / NS_SCALE));
                    }
                };
                if constexpr (HELD) {
#pragma unroll
                    for (int i = 0; i < 2 * SK; ++i) rows(i, qh[i], ql[i]);
                } else {
                    for (int i = 0; i < 2 * SK; ++i) {
#pragma unroll
                        for (int k = 0; k < SK; ++k) {
                            qh[0][k] = *(const s16x8*)(Ah + (16 * i + r) * LDA + 32 * k + 8 * kg);
                            ql[0][k] = *(const s16x8*)(Al + (16 * i + r) * LDA + 32 * k + 8 * kg);
                        }
                        rows(i, qh[0], ql[0]);
                    }
                }
            };
            if (step + 1 < a.steps)
                for (int n0 = wave * 32; n0 < T; n0 += 256) columns(n0, std::false_type());
            else
                for (int n0 = wave * 32; n0 < T; n0 += 256) columns(n0, std::true_type());
            __syncthreads();
        }
    }
};

template <int DT> __global__ __launch_bounds__(512, 2) void ns_tiny_kernel(NsTiny a) {
    __shared__ __attribute__((aligned(128))) char smem[NS_TINY_LDS];
    __shared__ double red[8];
    const NsTinyMat& m = a.m[blockIdx.x];
    const int S = ns_r32(m.s), T = ns_r32(m.t), ldx = T + 8, total = S * T / 8;
    const int rows = m.tall ? m.t : m.s, cols = m.tall ? m.s : m.t, cpr = (m.tall ? S : T) / 8;
    const bool vec = ns_on16<DT>(m.g, m.ldg);
    float v[NS_TINY_CHUNKS][8];
    double sum = 0.0;
#pragma unroll
    for (int h = 0; h < NS_TINY_CHUNKS; ++h) {
        const int i = threadIdx.x + 512 * h, q = i / cpr, c = (i - q * cpr) * 8;
        if (i < total && q < rows && c < cols) ns_load8<DT>(m.g, q * m.ldg, c, cols, vec, v[h]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[h][j] = 0.0f;
    }
#pragma unroll
    for (int h = 0; h < NS_TINY_CHUNKS; ++h)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += (double)v[h][j] * (double)v[h][j];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = ((red[0] + red[1]) + (red[2] + red[3])) + ((red[4] + red[5]) + (red[6] + red[7]));
    const double scale = (double)NS_SCALE / (sqrt(sum) + (double)a.eps);
    short *Xh = (short*)smem, *Xl = Xh + S * ldx;
#pragma unroll
    for (int h = 0; h < NS_TINY_CHUNKS; ++h) {
        const int i = threadIdx.x + 512 * h, q = i / cpr, c = (i - q * cpr) * 8;
        if (i < total) {
            unsigned hi[4], lo[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) ga_split_pair_f16((float)((double)v[h][2 * j] * scale), (float)((double)v[h][2 * j + 1] * scale), hi[j], lo[j]);
            if (!m.tall) {
                *(u32x4*)(Xh + q * ldx + c) = u32x4{hi[0], hi[1], hi[2], hi[3]};
                *(u32x4*)(Xl + q * ldx + c) = u32x4{lo[0], lo[1], lo[2], lo[3]};
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    Xh[(c + j) * ldx + q] = (short)(hi[j >> 1] >> (16 * (j & 1)));
                    Xl[(c + j) * ldx + q] = (short)(lo[j >> 1] >> (16 * (j & 1)));
                }
            }
        }
    }
    __syncthreads();
    if (S == 32) NsTinyRun<DT, 1>::run(a, m, smem);
    else if (S == 64) NsTinyRun<DT, 2>::run(a, m, smem);
    else if (S == 96) NsTinyRun<DT, 3>::run(a, m, smem);
    else NsTinyRun<DT, 4>::run(a, m, smem);
}

namespace {

typedef MmGeom<64, 64, 4, 2> NsT;
typedef MmGeom<128, 128, 8, 4> NsS;
typedef MmGeom<192, 192, 8, 4> NsM;      // (two waves a SIMD: with one, more than 256 registers, and moves between their halves in the loop)

size_t al(size_t n) { return (n + 255) & ~(size_t)255; }

// one matrix's planes; base may be null (only the size is wanted)
size_t ns_planes(NsMat* m, char* base, int s, int t) {
    const size_t x = al((size_t)s * ns_ld(t)), xt = al((size_t)t * ns_ld(s)), g = al((size_t)s * ns_ld(s));
    if (m) { m->X = base; m->XT0 = base + x; m->XT1 = m->XT0 + xt; m->A = m->XT1 + xt; m->B = m->A + g; }
    return x + 2 * xt + 2 * g;
}

long long tri(long long n) { return n * (n + 1) / 2; }

// tiles of all matrices of the group for one product
template <class C> int ns_tiles(NsArgs& a, int kind) {
    long long at = 0;
    for (int i = 0; i < a.count; ++i) {
        a.first[i] = (int)at;
        const long long r = (a.m[i].s + C::BM - 1) / C::BM, c = (a.m[i].t + C::BN - 1) / C::BN;
        at += kind == NS_STEP ? r * c : tri(r);
    }
    a.first[a.count] = (int)at;
    return (int)at;
}

template <class C, int D, int KG, int KIND, int DT> int ns_go(NsArgs& a, hipStream_t st) {
    const int tiles = ns_tiles<C>(a, KIND);
    hipLaunchKernelGGL((ns_kernel<C, D, KG, KIND, DT>), dim3(tiles), dim3(C::WAVES * KG * 64), 0, st, a);
    return hipGetLastError() == hipSuccess ? ACMIL_OK : ACMIL_ERR_LAUNCH;
}

template <int KIND, int DT> int ns_product(NsArgs& a, hipStream_t st) {
    // The largest tile that still gives most CUs work: larger tiles read less of LDS and L2 per flop.  From 160 tiles on instead of 200: 1500 x 1500
    // 413 -> 419 us, 1536 x 2048 472 -> 460; from 130 on: 1024 x 4096 375 -> 445, 2048 x 2048 681 -> 725.
    if (ns_tiles<NsM>(a, KIND) >= 200) return ns_go<NsM, 2, 1, KIND, DT>(a, st);
    if (ns_tiles<NsS>(a, KIND) >= 200) return ns_go<NsS, 2, 1, KIND, DT>(a, st);
    const int small = ns_tiles<NsT>(a, KIND);
    if (small <= 256) return ns_go<NsT, 4, 2, KIND, DT>(a, st);       // one workgroup of two groups per CU, three steps ahead
    if (small <= 512) return ns_go<NsT, 4, 1, KIND, DT>(a, st);       // two workgroups of one
    return ns_go<NsT, 2, 1, KIND, DT>(a, st);
}

// all matrices small: one launch for NS_TINY of them (beside a larger one they would add a launch to those that they can share)
bool ns_tiny_call(int count, const acmil_ortho_mat* mats) {
    for (int i = 0; i < count; ++i)
        if (!ns_tiny_fits(mats[i].m < mats[i].n ? mats[i].m : mats[i].n, mats[i].m < mats[i].n ? mats[i].n : mats[i].m)) return false;
    return true;
}
template <int DT> int ns_tiny_go(int count, const acmil_ortho_mat* mats, int steps, const float* co, float eps, hipStream_t st) {
    for (int at = 0; at < count; at += NS_TINY) {
        NsTiny a = {};
        const int n = count - at < NS_TINY ? count - at : NS_TINY;
        a.steps = steps;
        a.eps = eps;
        for (int k = 0; k < 3 * steps; ++k) a.co[k] = co[k];
        for (int i = 0; i < n; ++i) {
            const acmil_ortho_mat& u = mats[at + i];
            const int tall = u.m > u.n;
            a.m[i] = {u.g, u.o, u.ldg, u.ldo, tall ? u.n : u.m, tall ? u.m : u.n, tall, 0};
        }
        hipLaunchKernelGGL((ns_tiny_kernel<DT>), dim3(n), dim3(512), 0, st, a);
        if (hipGetLastError() != hipSuccess) return ACMIL_ERR_LAUNCH;
    }
    return ACMIL_OK;
}

template <int DT> int ns_run(int count, const acmil_ortho_mat* mats, int steps, const float* co, float eps, char* ws, hipStream_t st) {
    if (ns_tiny_call(count, mats)) return ns_tiny_go<DT>(count, mats, steps, co, eps, st);
    for (int at = 0; at < count; at += NS_GROUP) {                   // groups reuse the workspace: stream order
        NsArgs a = {};
        a.count = count - at < NS_GROUP ? count - at : NS_GROUP;
        a.eps = eps;
        double* part = (double*)ws;
        a.part = part;
        char* p = ws + al((size_t)NS_GROUP * NS_PARTS * 8);
        long long blocks = 0;
        for (int i = 0; i < a.count; ++i) {
            const acmil_ortho_mat& u = mats[at + i];
            NsMat& m = a.m[i];
            m.g = u.g; m.o = u.o; m.ldg = u.ldg; m.ldo = u.ldo;
            m.tall = u.m > u.n;
            m.s = m.tall ? u.n : u.m; m.t = m.tall ? u.m : u.n;
            p += ns_planes(&m, p, m.s, m.t);
            a.first[i] = (int)blocks;
            blocks += (long long)((u.m + 63) / 64) * ((u.n + 63) / 64);
        }
        a.first[a.count] = (int)blocks;
        hipLaunchKernelGGL((ns_norm_kernel<DT>), dim3(NS_PARTS, a.count), dim3(256), 0, st, a, part);
        hipLaunchKernelGGL((ns_split_kernel<DT>), dim3((unsigned)blocks), dim3(256), 0, st, a);
        if (hipGetLastError() != hipSuccess) return ACMIL_ERR_LAUNCH;
        for (int k = 0; k < steps; ++k) {
            a.a = co[3 * k]; a.b = co[3 * k + 1]; a.c = co[3 * k + 2];
            a.flip = k & 1;
            a.last = k == steps - 1;
            int rc = ns_product<NS_GRAM, ACMIL_DTYPE_F32>(a, st);
            if (rc == ACMIL_OK) rc = ns_product<NS_POLY, ACMIL_DTYPE_F32>(a, st);
            if (rc == ACMIL_OK) rc = ns_product<NS_STEP, DT>(a, st);
            if (rc != ACMIL_OK) return rc;
        }
    }
    return ACMIL_OK;
}

const int NS_MAX_DIM = 1 << 16;

int ns_check(int count, const acmil_ortho_mat* mats, int dtype) {
    if (!mats) return ACMIL_ERR_NULL;
    if (count <= 0) return ACMIL_ERR_SHAPE;
    if (dtype != ACMIL_DTYPE_F32 && dtype != ACMIL_DTYPE_F16 && dtype != ACMIL_DTYPE_BF16) return ACMIL_ERR_UNSUPPORTED;
    for (int i = 0; i < count; ++i) {
        if (mats[i].m <= 0 || mats[i].n <= 0 || mats[i].m > NS_MAX_DIM || mats[i].n > NS_MAX_DIM) return ACMIL_ERR_SHAPE;
        if (mats[i].ldg < mats[i].n || mats[i].ldo < mats[i].n) return ACMIL_ERR_SHAPE;
    }
    return ACMIL_OK;
}

// Do the polynomials keep the singular values, which start in [0, 1], where the scaled f16 halves can hold X, A and B?  In x = s^2 the extrema of
// a s + b s^3 + c s^5 lie at 5 c x^2 + 3 b x + a = 0, that of b x + c x^2 at x = -b / 2c, and either can lie at the end of [0, u^2].  (Samples of
// [0, u] step over a peak, and 2049 of them for each of five steps took 20 us and more of a call's host time: 64 x 64 38 us against 23.)
bool ns_coeffs_ok(int steps, const float* co) {
    double end = 1.0;                                                // u^2
    for (int k = 0; k < steps; ++k) {
        const double a = co[3 * k], b = co[3 * k + 1], c = co[3 * k + 2];
        if (!std::isfinite(a + b + c)) return false;
        // both roots without cancellation; where one does not exist (c = 0, or no real root) it is an infinity or NaN, and outside
        const double q = -0.5 * (3.0 * b + std::copysign(std::sqrt(9.0 * b * b - 20.0 * a * c), b));
        const double at[3] = {end, q / (5.0 * c), a / q}, top = -b / (2.0 * c);
        double up = 0.0;
        for (double x : at)
            if (x > 0.0 && x <= end) up = std::fmax(up, std::sqrt(x) * std::fabs(a + x * (b + x * c)));
        double bp = end * std::fabs(b + end * c);
        if (top > 0.0 && top <= end) bp = std::fmax(bp, top * std::fabs(b + top * c));
        if (!(up <= 3.9) || !(bp <= 15.5)) return false;
        end = up * up;
    }
    return true;
}

}  // namespace

extern "C" size_t acmil_orthogonalize_workspace_bytes(int count, const acmil_ortho_mat* mats, int dtype) {
    if (ns_check(count, mats, dtype) != ACMIL_OK) return 0;
    size_t most = 0;
    for (int at = 0; at < count; at += NS_GROUP) {
        size_t n = 0;
        for (int i = at; i < count && i < at + NS_GROUP; ++i) {
            const bool tall = mats[i].m > mats[i].n;
            n += ns_planes(nullptr, nullptr, tall ? mats[i].n : mats[i].m, tall ? mats[i].m : mats[i].n);
        }
        if (n > most) most = n;
    }
    return al((size_t)NS_GROUP * NS_PARTS * 8) + most;
}

extern "C" int acmil_orthogonalize(int count, const acmil_ortho_mat* mats, int dtype, int steps, const float* coeffs, float eps, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    const int rc = ns_check(count, mats, dtype);
    if (rc != ACMIL_OK) return rc;
    if (!coeffs) return ACMIL_ERR_NULL;
    for (int i = 0; i < count; ++i)
        if (!mats[i].g || !mats[i].o) return ACMIL_ERR_NULL;
    if (steps < 1 || steps > NS_MAX_STEPS || !(eps >= 0.0f) || !ns_coeffs_ok(steps, coeffs)) return ACMIL_ERR_SHAPE;
    if (!workspace) return ACMIL_ERR_NULL;
    if (((size_t)workspace & 255) != 0 || workspace_bytes < acmil_orthogonalize_workspace_bytes(count, mats, dtype)) return ACMIL_ERR_SHAPE;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ACMIL_DTYPE_F32) return ns_run<ACMIL_DTYPE_F32>(count, mats, steps, coeffs, eps, (char*)workspace, st);
    if (dtype == ACMIL_DTYPE_F16) return ns_run<ACMIL_DTYPE_F16>(count, mats, steps, coeffs, eps, (char*)workspace, st);
    return ns_run<ACMIL_DTYPE_BF16>(count, mats, steps, coeffs, eps, (char*)workspace, st);
}
