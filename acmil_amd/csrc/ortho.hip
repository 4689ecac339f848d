// ortho.hip -- orthogonalisation of matrices by Newton-Schulz products: X = G / (|G|_F + eps), then `steps` times
//   A = X X^T;   B = b A + c A A;   X <- a X + B X        (on G^T where G has more rows than columns, so that A is the small Gram matrix).
// The odd polynomial a s + b s^3 + c s^5 acts on the singular values and drives them towards 1, whatever the singular vectors are.
//
// Arithmetic.  A single 16-bit product would not do: errors of the null directions are multiplied by a^steps (485 for 3.4445^5).  Every
// value is held as a pair of f16 halves, hi + lo (22 bits and a common power-of-two scale, so that nothing is lost to the narrow
// exponent: |X|, |A|, |B| are bounded by the polynomial, checked on the host), and a product is hi hi + hi lo + lo hi on
// v_mfma_f32_16x16x32_f16 with fp32 accumulation -- as exact as an fp32 product at a multiple of its rate.
//
// Layout.  A row of K values lies as blocks of 32: 64 bytes of hi halves, then 64 bytes of lo halves.  A K step of 32 is then
// exactly one 128-byte row piece, and tiles move and lie in LDS like those of mm16_kernel.h, the first of a fragment's two halves being hi, the
// second lo.  K is padded to a multiple of 32 with zeros, so there is no tail.  All three products take both operands with K
// contiguous: X is kept in both orientations (its transpose twice, read and written alternately).  A and B are symmetric: only tiles on
// and below the diagonal are computed and each is written a second time, mirrored.
// All matrices of a call go through the same launches: 2 + 3 steps of them, whatever the number of matrices (up to NS_GROUP at a time).
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
    const double* part; int nparts;
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
template <int DT> __device__ __forceinline__ bool ns_on16(const NsMat& m) {
    return ((size_t)m.g & 15) == 0 && m.ldg % (DT == ACMIL_DTYPE_F32 ? 4 : 8) == 0;
}

// sum of squares, in 64 bits (a gradient's squares leave the range of 32): NS_PARTS partial sums per matrix, fixed order
#define NS_PARTS 256
template <int DT> __global__ __launch_bounds__(256) void ns_norm_kernel(NsArgs a, double* part) {
    const NsMat& m = a.m[blockIdx.y];
    const int rows = m.tall ? m.t : m.s, cols = m.tall ? m.s : m.t, cpr = (cols + 7) / 8;
    const bool vec = ns_on16<DT>(m);
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
    const bool vec = ns_on16<DT>(m);
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
    // the largest tile that still gives most CUs work: larger tiles read less of LDS and L2 per flop
    if (ns_tiles<NsM>(a, KIND) >= 200) return ns_go<NsM, 2, 1, KIND, DT>(a, st);
    if (ns_tiles<NsS>(a, KIND) >= 200) return ns_go<NsS, 2, 1, KIND, DT>(a, st);
    const int small = ns_tiles<NsT>(a, KIND);
    if (small <= 256) return ns_go<NsT, 4, 2, KIND, DT>(a, st);       // one workgroup of two groups per CU, three steps ahead
    if (small <= 512) return ns_go<NsT, 4, 1, KIND, DT>(a, st);       // two workgroups of one
    return ns_go<NsT, 2, 1, KIND, DT>(a, st);
}

template <int DT> int ns_run(int count, const acmil_ortho_mat* mats, int steps, const float* co, float eps, char* ws, hipStream_t st) {
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

const int NS_MAX_DIM = 1 << 16, NS_MAX_STEPS = 64;

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

// Do the polynomials keep the singular values, which start in [0, 1], where the scaled f16 halves can hold X, A and B?
bool ns_coeffs_ok(int steps, const float* co) {
    double u = 1.0;
    for (int k = 0; k < steps; ++k) {
        const double a = co[3 * k], b = co[3 * k + 1], c = co[3 * k + 2];
        if (!std::isfinite(a + b + c)) return false;
        double up = 0.0, bp = 0.0;
        for (int i = 0; i <= 2048; ++i) {
            const double s = u * i / 2048.0, q = b * s * s + c * s * s * s * s;
            up = fmax(up, fabs(a * s + q * s));
            bp = fmax(bp, fabs(q));
        }
        if (!(up <= 3.9) || !(bp <= 15.5)) return false;
        u = up;
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
    if (!coeffs || !workspace) return ACMIL_ERR_NULL;
    for (int i = 0; i < count; ++i)
        if (!mats[i].g || !mats[i].o) return ACMIL_ERR_NULL;
    if (steps < 1 || steps > NS_MAX_STEPS || !(eps >= 0.0f) || !ns_coeffs_ok(steps, coeffs)) return ACMIL_ERR_SHAPE;
    if (((size_t)workspace & 255) != 0 || workspace_bytes < acmil_orthogonalize_workspace_bytes(count, mats, dtype)) return ACMIL_ERR_SHAPE;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == ACMIL_DTYPE_F32) return ns_run<ACMIL_DTYPE_F32>(count, mats, steps, coeffs, eps, (char*)workspace, st);
    if (dtype == ACMIL_DTYPE_F16) return ns_run<ACMIL_DTYPE_F16>(count, mats, steps, coeffs, eps, (char*)workspace, st);
    return ns_run<ACMIL_DTYPE_BF16>(count, mats, steps, coeffs, eps, (char*)workspace, st);
}
