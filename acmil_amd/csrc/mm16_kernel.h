// mm16_kernel.h -- out[M, N] = sum_k Q(m, k) P(n, k) of fp16 / bf16 operands on v_mfma_f32_32x32x16, fp32 accumulation.
//
// Every product of a linear layer and of a gated feed-forward block is this one with another choice of which dimension is
// contiguous (MM_KC / MM_KS):   y = x W^T: P = W (KC), Q = x (KC);   dx = dz W: P = W (KS), Q = dz (KC);
// dW = dz^T x: P = x (KS), Q = dz (KS).  DUAL multiplies the same Q by two P (gate and up projection) so that one wave holds both
// factors of an output element in its accumulators and the product needs no second pass.
//
// Layout.  A K step is 64 wide.  Tiles travel global -> LDS by 16-byte LDS-DMA (no registers), two stages, one barrier a step: the
// DMA of step t + 1 runs under the matrix instructions of step t.  The LDS image is linear in the DMA's lane order, so bank
// conflicts are avoided by permuting which 16-byte chunk of its row each LANE FETCHES.  K-strided tiles lie in LDS as they lie in
// memory ([k][row]) and are read by ds_read_b64_tr_b16, which hands every lane four consecutive k of its row: no transposed copy of
// an operand is ever made.  P feeds the A side of the instruction: a lane then owns 4 consecutive COLUMNS of an output row.
// The epilogue turns the accumulators through LDS (fp32, 68-float rows: conflict-free both ways) into 8 consecutive columns per
// lane, so bias, residual, saved values and the result move in 16-byte pieces, 128 bytes a row.
#pragma once
#include "mm16.h"

typedef __fp16 mm_h4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char mm_lds;

static __device__ __attribute__((aligned(16))) unsigned mm_zero[4];     // what a lane fetches in place of a chunk beyond K

// tile geometry: WAVES waves, WN of them along the columns, each with MT x NT accumulator tiles of 32 x 32
template <int BM_, int BN_, int WAVES_, int WN_> struct MmGeom {
    static constexpr int BM = BM_, BN = BN_, WAVES = WAVES_, WN = WN_;
    static constexpr int TM = BM / (WAVES / WN), TN = BN / WN, MT = TM / 32, NT = TN / 32;
    static constexpr int QB = BM * 128, PB = BN * 128, STAGE = QB + PB;
};
// LARGE: one 8-wave workgroup per CU (128 KB of LDS), else two 4-wave workgroups per CU
template <bool LARGE> struct MmCfg;
template <> struct MmCfg<true> : MmGeom<256, 256, 8, 4> {};
template <> struct MmCfg<false> : MmGeom<128, 128, 4, 2> {};

__device__ __forceinline__ unsigned mm_lds_addr(const void* p) { return (unsigned)(size_t)(const __attribute__((address_space(3))) void*)p; }

// 64 lanes x 16 bytes: lane l's bytes at sbase + voff land at LDS byte lds + 16 l (lds uniform)
__device__ __forceinline__ void mm_dma_s(unsigned voff, const char* sbase, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 2\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(sbase), "s"(lds) : "memory");
}
__device__ __forceinline__ void mm_dma_v(const char* src, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 2\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(src), "s"(lds) : "memory");
}
__device__ __forceinline__ void mm_wait_dma() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// chunk permutations: conflict-free for 8 lanes over 128 bytes and for 16 lanes over 256 bytes
__device__ __forceinline__ int mm_swz_kc(int row) { return (row & 7) ^ ((row >> 3) & 1); }
__device__ __forceinline__ int mm_swz_ks(int k) { return 2 * (k & 3) + 8 * (k & 1); }

// One operand tile of R rows x 64 k: where a lane fetches from
template <int KIND, int R, int WAVES> struct MmLoad {
    static constexpr int NI = R * 128 / (WAVES * 1024);             // DMA instructions per wave and stage
    static constexpr int CPR = R / 8;                               // KS: 16-byte chunks per k row
    unsigned off[NI];                                               // byte offset from the tile's base at k = 0
    __device__ __forceinline__ void init(int wave, int lane, long long ld, int row0, int rows) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int piece = i * WAVES + wave;
            if (KIND == MM_KC) {
                const int r = piece * 8 + (lane >> 3), c = (lane & 7) ^ mm_swz_kc(r);
                const int rr = row0 + r < rows ? r : (rows - 1 - row0 > 0 ? rows - 1 - row0 : 0);   // rows beyond the last repeat it; never stored
                off[i] = (unsigned)(rr * ld) + c * 16;
            } else {
                const int k = piece * (64 / CPR) + lane / CPR, c = (lane % CPR) ^ mm_swz_ks(k);
                const int last = (rows - row0 + 7) / 8 - 1;
                off[i] = (unsigned)(k * ld) + (c < last ? c : last) * 16;
            }
        }
    }
    // k index (KC: of the chunk's first element) that instruction i of this lane fetches, relative to the step
    __device__ __forceinline__ static int k_of(int i, int wave, int lane) {
        const int piece = i * WAVES + wave;
        if (KIND == MM_KC) return 8 * ((lane & 7) ^ mm_swz_kc(piece * 8 + (lane >> 3)));
        return piece * (64 / CPR) + lane / CPR;
    }
};

template <int KIND, int R> struct MmFrag {                           // reading a 32-row x 16-k fragment out of LDS
    unsigned base;
    int swz, lane;
    __device__ __forceinline__ void init(int l) {
        lane = l;
        if (KIND == MM_KC) {
            const int r = l & 31;
            base = r * 128 + ((((l >> 5)) ^ mm_swz_kc(r)) << 4);
        } else {
            const int k = 8 * (l >> 5) + ((l & 15) >> 2);
            base = k * (R * 2) + (l & 1) * 8;
            swz = mm_swz_ks(k);
        }
    }
    // KS: byte offset of the lane's chunk for the 32-row tile that starts at row
    __device__ __forceinline__ unsigned tile(int row) const {
        if (KIND == MM_KC) return row * 128;
        return (((row >> 3) + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ swz) << 4;
    }
    __device__ __forceinline__ s16x8 get(mm_lds* sm, unsigned tile_off, int s) const {
        if (KIND == MM_KC) return *(const __attribute__((address_space(3))) s16x8*)(sm + (base ^ (s << 5)) + tile_off);
        mm_lds* p = sm + base + tile_off + s * 16 * (R * 2);
        const s16x4 lo = __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) mm_h4*)p));
        const s16x4 hi = __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) mm_h4*)(p + 4 * (R * 2))));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

template <bool BF> __device__ __forceinline__ f32x16 mm_mfma(s16x8 a, s16x8 b, f32x16 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF, int PK, int QK, int EPI, bool DUAL, bool LARGE>
__global__ __launch_bounds__(MmCfg<LARGE>::WAVES * 64, 2) void mm16_kernel(MmArgs a) {
    using C = MmCfg<LARGE>;
    constexpr int MT = C::MT, NT = C::NT;
    __shared__ __attribute__((aligned(128))) char smem[2 * C::STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / C::WN, wn = wave % C::WN;

    // Workgroup b runs on XCD b % 8.  Each XCD takes one contiguous run of tiles, in groups of 8 row tiles by all column tiles, so
    // that the tiles its 32 CUs work on together share operand rows and columns in its L2.
    int tm, tn;
    {
        const int nt = a.ntm * a.ntn, q = nt >> 3, r = nt & 7, x = blockIdx.x & 7, i = blockIdx.x >> 3;
        const int id = x * q + (x < r ? x : r) + i;
        const int width = 8 * a.ntn, g = id / width, first = 8 * g, sz = a.ntm - first < 8 ? a.ntm - first : 8;
        tm = first + (id % width) % sz;
        tn = (id % width) / sz;
    }
    constexpr int BNF = DUAL ? C::BN / 2 : C::BN;                    // columns of one factor in this tile
    const int m0 = tm * C::BM, n0 = tn * BNF;

    MmLoad<QK, C::BM, C::WAVES> lq;
    MmLoad<PK, C::BN, C::WAVES> lp;
    lq.init(wave, lane, a.ldq, m0, a.M);
    if constexpr (!DUAL) lp.init(wave, lane, a.ldp, n0, a.N);
    else {                                                           // LDS rows 0 .. BN/2 - 1 from the first factor, the others from the second
        static_assert(!DUAL || PK == MM_KC, "two factors: K contiguous");
#pragma unroll
        for (int i = 0; i < lp.NI; ++i) {
            const int piece = i * C::WAVES + wave, r = piece * 8 + (lane >> 3), rf = r & (BNF - 1);
            const int rr = n0 + rf < a.N ? rf : a.N - 1 - n0;
            lp.off[i] = (unsigned)(rr * a.ldp) + ((lane & 7) ^ mm_swz_kc(r)) * 16;
        }
    }
    const long long qbase = QK == MM_KC ? m0 * a.ldq : m0 * 2LL, pbase = PK == MM_KC ? n0 * a.ldp : n0 * 2LL;
    const long long qstep = QK == MM_KC ? 128 : 64 * a.ldq, pstep = PK == MM_KC ? 128 : 64 * a.ldp;
    const int kmax = a.Kq > a.Kp ? a.Kq : a.Kp, kmin = a.Kq < a.Kp ? a.Kq : a.Kp, tseg = (kmax + 63) >> 6, T = a.segs * tseg;
    const int t0 = (int)((long long)T * blockIdx.y / a.splits), t1 = (int)((long long)T * (blockIdx.y + 1) / a.splits);
    const unsigned smem0 = mm_lds_addr(smem);

    auto issue = [&](int t, int buf) {
        const bool s1 = t >= tseg;                                   // segs <= 2
        const int tt = s1 ? t - tseg : t;
        const char* qb = (s1 ? a.q1 : a.q0) + qbase + tt * qstep;
        const char* pb = (s1 && !DUAL ? a.p1 : a.p0) + pbase + tt * pstep;
        const char* pb2 = DUAL ? a.p1 + pbase + tt * pstep : pb;
        const unsigned lds = smem0 + buf * C::STAGE + wave * 1024;
        if (tt * 64 + 64 <= kmin) {
#pragma unroll
            for (int i = 0; i < lq.NI; ++i) mm_dma_s(lq.off[i], qb, lds + i * C::WAVES * 1024);
#pragma unroll
            for (int i = 0; i < lp.NI; ++i) mm_dma_s(lp.off[i], DUAL && i >= lp.NI / 2 ? pb2 : pb, lds + C::QB + i * C::WAVES * 1024);
        } else {                                                     // the last step of a segment: chunks beyond K come from the zero block
            const char* z = (const char*)mm_zero;
#pragma unroll
            for (int i = 0; i < lq.NI; ++i)
                mm_dma_v(tt * 64 + lq.k_of(i, wave, lane) < a.Kq ? qb + lq.off[i] : z, lds + i * C::WAVES * 1024);
#pragma unroll
            for (int i = 0; i < lp.NI; ++i)
                mm_dma_v(tt * 64 + lp.k_of(i, wave, lane) < a.Kp ? (DUAL && i >= lp.NI / 2 ? pb2 : pb) + lp.off[i] : z,
                         lds + C::QB + i * C::WAVES * 1024);
        }
    };

    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    MmFrag<QK, C::BM> fq;
    MmFrag<PK, C::BN> fp;
    fq.init(lane);
    fp.init(lane);
    unsigned qt[MT], pt[NT];
#pragma unroll
    for (int i = 0; i < MT; ++i) qt[i] = fq.tile(wm * C::TM + 32 * i);
#pragma unroll
    for (int j = 0; j < NT; ++j) pt[j] = C::QB + fp.tile(DUAL ? j * BNF + wn * 32 : wn * 64 + 32 * j);

    if (t0 < t1) issue(t0, 0);
    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        mm_wait_dma();                                               // this wave's share of step t has landed ...
        ga_lds_barrier();                                            // ... and everybody's; everybody is done reading step t - 1
        if (t + 1 < t1) issue(t + 1, buf ^ 1);
        mm_lds* sm = (mm_lds*)smem + buf * C::STAGE;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            s16x8 p[NT], q[MT];
#pragma unroll
            for (int j = 0; j < NT; ++j) p[j] = fp.get(sm, pt[j], s);
#pragma unroll
            for (int i = 0; i < MT; ++i) q[i] = fq.get(sm, qt[i], s);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = mm_mfma<BF>(p[j], q[i], acc[i][j]);
        }
    }
    ga_lds_barrier();                                                // the stages are free: the epilogue turns its tiles there

    float* st = (float*)smem + wave * (32 * 68);
    const int mrow = m0 + wm * C::TM;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *(f32x4*)(st + (lane & 31) * 68 + 32 * j + 8 * r + 4 * (lane >> 5)) =
                    f32x4{acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // a wave turns its own tile: its LDS operations are in order
        if constexpr (!DUAL) {
#pragma unroll 1
            for (int it = 0; it < 4; ++it) {
                const int row = it * 8 + (lane >> 3), c = (lane & 7) * 8, m = mrow + 32 * i + row, n = n0 + wn * 64 + c;
                float v[8];
                mm_ldf8(st + row * 68 + c, v);
                if (m < a.M) {
                    if constexpr (EPI == MM_ACT) mm_epi_act<BF>(a.e, m, n, a.N, v);
                    else if constexpr (EPI == MM_GATE_BWD) mm_epi_gate_bwd<BF>(a.e, m, n, a.N, v);
                    else if (n < a.e.ldpart) mm_stf8(a.e.part + ((size_t)blockIdx.y * a.M + m) * a.e.ldpart + n, v);
                }
            }
        } else {
#pragma unroll 1
            for (int it = 0; it < 2; ++it) {
                const int row = it * 16 + (lane >> 2), c = (lane & 3) * 8, m = mrow + 32 * i + row, n = n0 + wn * 32 + c;
                float g[8], u[8];
                mm_ldf8(st + row * 68 + c, g);
                mm_ldf8(st + row * 68 + 32 + c, u);
                if (m < a.M) {
                    if constexpr (EPI == MM_GATE) mm_epi_gate<BF>(a.e, m, n, a.N, g, u);
                    else if (n < a.e.ldpart) {
                        float* o = a.e.part + ((size_t)blockIdx.y * 2 * a.M + m) * a.e.ldpart + n;
                        mm_stf8(o, g);
                        mm_stf8(o + (size_t)a.M * a.e.ldpart, u);
                    }
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

template <bool BF, int PK, int QK, int EPI, bool DUAL, bool LARGE> static inline int mm_go(const MmArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((mm16_kernel<BF, PK, QK, EPI, DUAL, LARGE>), dim3(a.ntm * a.ntn, a.splits), dim3(MmCfg<LARGE>::WAVES * 64), 0, st, a);
    return hipGetLastError() == hipSuccess ? ACMIL_OK : ACMIL_ERR_LAUNCH;
}
template <int PK, int QK, int EPI, bool DUAL> static inline int mm_go_any(const MmArgs& a, bool bf, bool large, hipStream_t st) {
    if (bf) return large ? mm_go<true, PK, QK, EPI, DUAL, true>(a, st) : mm_go<true, PK, QK, EPI, DUAL, false>(a, st);
    return large ? mm_go<false, PK, QK, EPI, DUAL, true>(a, st) : mm_go<false, PK, QK, EPI, DUAL, false>(a, st);
}
