// mm16_kernel.h -- out[M, N] = sum_k Q(m, k) P(n, k) of fp16 / bf16 operands on v_mfma_f32_16x16x32, fp32 accumulation.
//
// Every product of a linear layer and of a gated feed-forward block is this one with another choice of which dimension is
// contiguous (MM_KC / MM_KS):   y = x W^T: P = W (KC), Q = x (KC);   dx = dz W: P = W (KS), Q = dz (KC);
// dW = dz^T x: P = x (KS), Q = dz (KS).  DUAL multiplies the same Q by two P (gate and up projection) so that one wave holds both
// factors of an output element in its accumulators and the product needs no second pass.
//
// Layout.  A K step is 64 wide.  Tiles travel global -> LDS by 16-byte LDS-DMA (no registers) through a ring, one barrier a step.  The
// LDS image is linear in the DMA's lane order, so bank conflicts are avoided by permuting which 16-byte chunk of its row each LANE
// FETCHES.  K-strided tiles lie in LDS as they lie in memory ([k][row]) and are read by ds_read_b64_tr_b16, which hands every lane four
// consecutive k of its row: no transposed copy of an operand is ever made.  P feeds the A side of the instruction: a lane then owns 4
// consecutive COLUMNS of an output row.
// The epilogue turns the accumulators through LDS (fp32, 68-float rows: conflict-free both ways) into 8 consecutive columns per
// lane, so bias, residual, saved values and the result move in 16-byte pieces, 128 bytes a row.
//
// Bound: large products by the card's power (8192 x 4096 x 11008 training block 5.3 ms, 1.25 PFLOP/s over its nine products and its
// element-wise work; a library product of 4096^3 1.45), small ones by latency: a call of 768 x 2816 outputs takes 6 us for K = 64 and 0.45 us for
// every further step, an activation 1 to 2 us.
#pragma once
#include "mm16.h"

#include <utility>

#define MM_INLINE __attribute__((always_inline))
// f(0), f(1), ... f(N - 1) with constant arguments: register arrays must never be indexed by a variable
template <class F, int... I> __device__ __forceinline__ void mm_for_(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int A, int B, class F> __device__ __forceinline__ void mm_for(F f) {
    if constexpr (A < B) mm_for_([&](auto i) MM_INLINE { f(std::integral_constant<int, A + decltype(i)::value>{}); }, std::make_integer_sequence<int, B - A>{});
}

typedef __fp16 mm_h4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char mm_lds;

static __device__ __attribute__((aligned(16))) unsigned mm_zero[4];     // what a lane fetches in place of a chunk beyond K

// Tile geometry: WAVES waves, WN of them along the columns, each with MT x NT accumulator tiles of 16 x 16.  One operand of one K step is
// 128 bytes of every row (64 values, or 32 pairs of ortho.hip) and fills one slot of LDS.
template <int BM_, int BN_, int WAVES_, int WN_> struct MmGeom {
    static constexpr int BM = BM_, BN = BN_, WAVES = WAVES_, WN = WN_;
    static constexpr int TM = BM / (WAVES / WN), TN = BN / WN, MT = TM / 16, NT = TN / 16;
    static constexpr int QB = BM * 128, PB = BN * 128;
};
// MM_L: one 8-wave workgroup per CU.  MM_S: two 4-wave workgroups per CU.  MM_D: where there is one workgroup per CU or less, 8 waves and three
// steps ahead instead of 4 waves and one (1 to 10 % faster than MM_S for 64 to 2000 rows of 768 to 4096 features).  MM_R32, MM_R64: few rows
// by many columns, for products that are bound by streaming P.  D: steps of the ring, D + 1 slots of Q and D of P: 80 or up to 160 KB of LDS.
template <int CFG> struct MmCfg;
template <> struct MmCfg<MM_L> : MmGeom<256, 256, 8, 4> { static constexpr int D = 2, PER_SIMD = 2; };
template <> struct MmCfg<MM_S> : MmGeom<128, 128, 4, 2> { static constexpr int D = 2, PER_SIMD = 2; };
template <> struct MmCfg<MM_R32> : MmGeom<32, 256, 4, 4> { static constexpr int D = 4, PER_SIMD = 1; };
template <> struct MmCfg<MM_R64> : MmGeom<64, 256, 4, 4> { static constexpr int D = 3, PER_SIMD = 1; };
template <> struct MmCfg<MM_D> : MmGeom<128, 128, 8, 2> { static constexpr int D = 4, PER_SIMD = 2; };

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
template <int N> __device__ __forceinline__ void mm_wait_dma() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// chunk permutations: conflict-free for 8 lanes over 128 bytes and for 16 lanes over 256 bytes
__device__ __forceinline__ int mm_swz_kc(int row) { return (row >> 1) & 7; }
__device__ __forceinline__ int mm_swz_ks(int k) { return 2 * (k & 3) + 8 * ((k >> 3) & 1); }

// One operand tile of R rows x one K step: where a lane fetches from
template <int KIND, int R, int WAVES> struct MmLoad {
    static constexpr int NI = R * 128 / (WAVES * 1024);             // DMA instructions per wave and step
    static constexpr int CPR = KIND == MM_KC ? 8 : R / 8;           // 16-byte chunks per row (KC: of one row, KS: of one k)
    unsigned off[NI];                                               // byte offset from the tile's base at k = 0
    __device__ __forceinline__ static int row_of(int i, int wave, int lane) { return (i * WAVES + wave) * (64 / CPR) + lane / CPR; }
    __device__ __forceinline__ void init(int wave, int lane, long long ld, int row0, int rows) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = row_of(i, wave, lane);
            if (KIND == MM_KC) {
                const int c = (lane % CPR) ^ mm_swz_kc(r);
                const int rr = row0 + r < rows ? r : rows - 1 - row0;                        // rows beyond the last repeat it; never stored
                off[i] = (unsigned)(rr * ld) + c * 16;
            } else {
                const int c = (lane % CPR) ^ mm_swz_ks(r), last = (rows - row0 + 7) / 8 - 1;
                off[i] = (unsigned)(r * ld) + (c < last ? c : last) * 16;
            }
        }
    }
    // k index (KC: of the chunk's first element) that instruction i of this lane fetches, relative to the step
    __device__ __forceinline__ static int k_of(int i, int wave, int lane) {
        const int r = row_of(i, wave, lane);
        return KIND == MM_KC ? 8 * ((lane % CPR) ^ mm_swz_kc(r)) : r;
    }
};

template <int KIND, int R> struct MmFrag {                           // reading 16-row x 32-k fragments of a wave out of LDS
    unsigned base;
    __device__ __forceinline__ void init(int l, int row0) {          // row0: the wave's first row, a multiple of 32
        if (KIND == MM_KC) {
            const int r = l & 15;
            base = (row0 + r) * 128 + (((l >> 4) ^ mm_swz_kc(r)) << 4);
        } else {                                                     // the chunk permutation commutes with the (even) chunk a 16-row tile starts at
            const int k = 8 * (l >> 4) + ((l & 15) >> 2);
            base = k * (R * 2) + (((((l & 3) >> 1) ^ mm_swz_ks(k)) << 4) ^ (row0 * 2)) + (l & 1) * 8;
        }
    }
    // rows row0 + row .. + 15, the s-th 32 k of the step (pairs of ortho.hip: 0 the hi halves, 1 the lo halves)
    __device__ __forceinline__ s16x8 get(mm_lds* sm, int row, int s) const {
        if (KIND == MM_KC) return *(const __attribute__((address_space(3))) s16x8*)(sm + (base ^ (s << 6)) + row * 128);
        mm_lds* p = sm + (base ^ (row * 2)) + s * 32 * (R * 2);
        const s16x4 lo = __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) mm_h4*)p));
        const s16x4 hi = __builtin_bit_cast(s16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) mm_h4*)(p + 4 * (R * 2))));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
};

// The 16 x 16 x 32 form moves half the accumulator bytes per flop of the 32 x 32 x 16 one.  That is what counts: a loop of nothing
// but these instructions runs into the power limit, at 2.02 PFLOP/s against 1.82 for the larger form (bf16, 256 CUs).
template <bool BF> __device__ __forceinline__ f32x4 mm_mfma(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <bool BF, int PK, int QK, int EPI, bool DUAL, int CFG>
__global__ __launch_bounds__(MmCfg<CFG>::WAVES * 64, MmCfg<CFG>::PER_SIMD) void mm16_kernel(MmArgs a) {
    using C = MmCfg<CFG>;
    constexpr int MT = C::MT, NT = C::NT;
    constexpr int D = C::D, RINGP = (D + 1) * C::QB;                 // D + 1 slots of Q, behind them D of P
    __shared__ __attribute__((aligned(128))) char smem[RINGP + D * C::PB];
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
            const int r = lp.row_of(i, wave, lane), rf = r & (BNF - 1);
            const int rr = n0 + rf < a.N ? rf : a.N - 1 - n0;
            lp.off[i] = (unsigned)(rr * a.ldp) + ((lane % lp.CPR) ^ mm_swz_kc(r)) * 16;
        }
    }
    const long long qbase = QK == MM_KC ? m0 * a.ldq : m0 * 2LL, pbase = PK == MM_KC ? n0 * a.ldp : n0 * 2LL;
    constexpr int BK = 64;                                           // K of a step
    const long long qstep = QK == MM_KC ? 128 : BK * a.ldq, pstep = PK == MM_KC ? 128 : BK * a.ldp;
    const int kmax = a.Kq > a.Kp ? a.Kq : a.Kp, kmin = a.Kq < a.Kp ? a.Kq : a.Kp, tseg = (kmax + BK - 1) / BK, T = a.segs * tseg;
    const int t0 = (int)((long long)T * blockIdx.y / a.splits), t1 = (int)((long long)T * (blockIdx.y + 1) / a.splits);
    const unsigned smem0 = mm_lds_addr(smem);

    // Fetching one operand of one step in NI pieces.  Fetches are never skipped, so that their count is a constant: behind the last step
    // it is fetched again, unused.  tail (a K that is no multiple of 64): chunks beyond K come from the zero block.
    constexpr int NIQ = decltype(lq)::NI, NIP = decltype(lp)::NI;
    struct Half { const char *from, *from2; unsigned lds; int k; };  // k: how much of K is left
    auto half_of = [&](int t, int slot, bool rows) MM_INLINE {
        t = t < t1 ? t : t1 - 1;
        const bool s1 = t >= tseg;                                   // segs <= 2
        const int tt = s1 ? t - tseg : t;
        Half h;
        h.from = rows ? (s1 ? a.q1 : a.q0) + qbase + tt * qstep : (s1 && !DUAL ? a.p1 : a.p0) + pbase + tt * pstep;
        h.from2 = DUAL && !rows ? a.p1 + pbase + tt * pstep : h.from;
        h.lds = smem0 + (rows ? slot * C::QB : RINGP + slot * C::PB) + wave * 1024;
        h.k = (rows ? a.Kq : a.Kp) - tt * BK;
        return h;
    };
    auto fetch_q = [&](const Half& x, auto piece, auto tail) MM_INLINE {
        constexpr int i = decltype(piece)::value;
        const unsigned lds = x.lds + i * C::WAVES * 1024;
        if constexpr (!decltype(tail)::value) mm_dma_s(lq.off[i], x.from, lds);
        else mm_dma_v(lq.k_of(i, wave, lane) < x.k ? x.from + lq.off[i] : (const char*)mm_zero, lds);
    };
    auto fetch_p = [&](const Half& x, auto piece, auto tail) MM_INLINE {
        constexpr int i = decltype(piece)::value;
        const unsigned lds = x.lds + i * C::WAVES * 1024;
        const char* from = DUAL && i >= NIP / 2 ? x.from2 : x.from;
        if constexpr (!decltype(tail)::value) mm_dma_s(lp.off[i], from, lds);
        else mm_dma_v(lp.k_of(i, wave, lane) < x.k ? from + lp.off[i] : (const char*)mm_zero, lds);
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    MmFrag<QK, C::BM> fq;
    MmFrag<PK, C::BN> fp;
    fq.init(lane, wm * C::TM);
    fp.init(lane, wn * (DUAL ? C::TN / 2 : C::TN));

    // The ring.  A step is two pieces of 32 k.  A piece goes row tile by row tile: NT matrix
    // instructions, then the row fragment just used is read again for the next piece (the column fragments, which every row tile needs,
    // have two register sets).  Between the pieces of step t a wave has read all it needs of Q_t and P_t, and its share of Q_(t+1) and
    // P_(t+1) has landed: behind the one barrier of the step the first fragments of step t + 1 are read.  Q_(t+D) is fetched during the
    // first piece, into the slot of Q_(t-1), and P_(t+D) during the second, into that of P_t.  Fetches are spread over the step because
    // one that finds the address unit busy holds its wave up, with its matrix instructions: sent out in one burst behind the barrier
    // they cost 18 % more cycles.
    s16x8 p[2][NT], q[MT];
    auto read_p = [&](mm_lds* slot, auto ks, auto kf) MM_INLINE {
        constexpr int sub = decltype(ks)::value, f = decltype(kf)::value;
        p[sub][f] = fp.get(slot, DUAL ? (f / (NT / 2)) * BNF + (f % (NT / 2)) * 16 : 16 * f, sub);
    };
    auto read_q = [&](mm_lds* slot, auto ks, auto kf) MM_INLINE {
        constexpr int sub = decltype(ks)::value, f = decltype(kf)::value;
        q[f] = fq.get(slot, 16 * f, sub);
    };
    mm_lds* const ring = (mm_lds*)smem;
    int qs = 0, ps = 0;                                              // slots of Q_t and P_t
    auto start = [&](auto tail) MM_INLINE {
        mm_for<0, D>([&](auto i) MM_INLINE {
            const Half hq = half_of(t0 + i, i, true), hp = half_of(t0 + i, i, false);
            mm_for<0, NIQ>([&](auto d) MM_INLINE { fetch_q(hq, d, tail); });
            mm_for<0, NIP>([&](auto d) MM_INLINE { fetch_p(hp, d, tail); });
        });
    };
    auto steps = [&](int from, int to, auto tail) MM_INLINE {
        // piece `sub` multiplies; fragments of the other piece are read from the given slots
        auto piece = [&](auto ks, mm_lds* qslot, mm_lds* pslot, const Half& h) MM_INLINE {
            constexpr int sub = decltype(ks)::value;
            using Other = std::integral_constant<int, 1 - sub>;
            mm_for<0, MT>([&](auto ki) MM_INLINE {
                constexpr int i = decltype(ki)::value;
                mm_for<i * NT / MT, (i + 1) * NT / MT>([&](auto f) MM_INLINE { read_p(pslot, Other{}, f); });
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = mm_mfma<BF>(p[sub][j], q[i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);                   // else the read goes first, into registers that are not there
                read_q(qslot, Other{}, ki);
                if constexpr (sub == 0) mm_for<i * NIQ / MT, (i + 1) * NIQ / MT>([&](auto d) MM_INLINE { fetch_q(h, d, tail); });
                else mm_for<i * NIP / MT, (i + 1) * NIP / MT>([&](auto d) MM_INLINE { fetch_p(h, d, tail); });
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        for (int t = from; t < to; ++t) {
            const Half hq = half_of(t + D, qs == 0 ? D : qs - 1, true), hp = half_of(t + D, ps, false);
            piece(std::integral_constant<int, 0>{}, ring + qs * C::QB, ring + RINGP + ps * C::PB, hq);
            mm_wait_dma<(D - 1) * NIQ + (D - 2) * NIP>();            // younger steps may still be on their way
            ga_lds_barrier();
            qs = qs == D ? 0 : qs + 1;
            ps = ps == D - 1 ? 0 : ps + 1;
            piece(std::integral_constant<int, 1>{}, ring + qs * C::QB, ring + RINGP + ps * C::PB, hp);
        }
    };
    // The first step that holds the end of K.  Steps that fetch only what lies in front of it take the plain loop: chunk by chunk comparisons
    // cost the training of a block of 3001 x 767 x 2047 219 us against 208.
    const int cut = t0 < tseg ? tseg - 1 : 2 * tseg - 1, split = kmin == kmax && kmin % BK == 0 ? t1 : cut < t1 ? (cut - D > t0 ? cut - D : t0) : t1;
    if (split == t1) start(std::false_type{});
    else start(std::true_type{});
    mm_wait_dma<(D - 1) * (NIQ + NIP)>();
    ga_lds_barrier();
    mm_for<0, NT>([&](auto f) MM_INLINE { read_p(ring + RINGP, std::integral_constant<int, 0>{}, f); });
    mm_for<0, MT>([&](auto f) MM_INLINE { read_q(ring, std::integral_constant<int, 0>{}, f); });
    steps(t0, split, std::false_type{});
    steps(split, t1, std::true_type{});
    mm_wait_dma<0>();
    ga_lds_barrier();                                                // the stages are free: the epilogue turns its tiles there

    // The epilogue's code is long (six activations, ragged columns) and a workgroup runs through it once.  So there are as few copies as
    // LDS allows, 64 rows a time, and its inner loop stays rolled: unrolled, 50000 x 1536 x 768 took 196 us against 125.
    constexpr int HB = MT < 4 ? MT : 4;                              // 16-row tiles a time
    static_assert(C::TN == 64 && MT % HB == 0, "a wave's columns: 64 (DUAL: 32 of both factors)");
    static_assert(C::WAVES * HB * 16 * 68 * 4 <= RINGP + D * C::PB, "room for the turned tiles");
    float* st = (float*)smem + wave * (HB * 16 * 68);
    const int mrow = m0 + wm * C::TM;
    float sg[8] = {}, su[8] = {};                                    // MM_GATE_BWD: sums over this wave's rows
#pragma unroll
    for (int i = 0; i < MT / HB; ++i) {
#pragma unroll
        for (int ii = 0; ii < HB; ++ii)
#pragma unroll
            for (int j = 0; j < NT; ++j) *(f32x4*)(st + (16 * ii + (lane & 15)) * 68 + 16 * j + 4 * (lane >> 4)) = acc[HB * i + ii][j];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");           // a wave turns its own tile: its LDS operations are in order
        if constexpr (!DUAL) {
#pragma unroll 1
            for (int it = 0; it < 2 * HB; ++it) {
                const int row = it * 8 + (lane >> 3), c = (lane & 7) * 8, m = mrow + 16 * HB * i + row, n = n0 + wn * 64 + c;
                float v[8];
                mm_ldf8(st + row * 68 + c, v);
                if (m < a.M) {
                    if constexpr (EPI == MM_ACT) mm_epi_act<BF>(a.e, m, n, a.N, v);
                    else if constexpr (EPI == MM_GATE_BWD) mm_epi_gate_bwd<BF>(a.e, m, n, a.N, v, sg, su);
                    else if (n < a.e.ldpart) mm_stf8(a.e.part + ((size_t)blockIdx.y * a.M + m) * a.e.ldpart + n, v);
                }
            }
        } else {
#pragma unroll 1
            for (int it = 0; it < HB; ++it) {
                const int row = it * 16 + (lane >> 2), c = (lane & 3) * 8, m = mrow + 16 * HB * i + row, n = n0 + wn * 32 + c;
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
    if constexpr (EPI == MM_GATE_BWD) {
        const int n = n0 + wn * 64 + (lane & 7) * 8;
        if (a.e.sums) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int o = 8; o < 64; o <<= 1) {
                    sg[j] += __shfl_xor(sg[j], o);
                    su[j] += __shfl_xor(su[j], o);
                }
            if (lane < 8 && n < a.e.npad) {
                float* to = a.e.sums + (size_t)(tm * (C::BM / C::TM) + wm) * 2 * a.e.npad + n;
                mm_stf8(to, sg);
                mm_stf8(to + a.e.npad, su);
            }
        }
    }
}

template <bool BF, int PK, int QK, int EPI, bool DUAL, int CFG> static inline int mm_go(const MmArgs& a, hipStream_t st) {
    static_assert(MmCfg<CFG>::BM / MmCfg<CFG>::TM == mm_wave_rows(CFG), "rows of MmEpi::sums");
    hipLaunchKernelGGL((mm16_kernel<BF, PK, QK, EPI, DUAL, CFG>), dim3(a.ntm * a.ntn, a.splits), dim3(MmCfg<CFG>::WAVES * 64), 0, st, a);
    return hipGetLastError() == hipSuccess ? ACMIL_OK : ACMIL_ERR_LAUNCH;
}
template <bool BF, int PK, int QK, int EPI, bool DUAL> static inline int mm_go_cfg(const MmArgs& a, int cfg, hipStream_t st) {
    // (K is never split where the large tiles fill the chip)
    if constexpr (EPI != MM_PART) if (cfg == MM_L) return mm_go<BF, PK, QK, EPI, DUAL, MM_L>(a, st);
    if constexpr (QK == MM_KC) {                                      // few rows: not for weight gradients, whose rows are features
        if (cfg == MM_R32) return mm_go<BF, PK, QK, EPI, DUAL, MM_R32>(a, st);
        if (cfg == MM_R64) return mm_go<BF, PK, QK, EPI, DUAL, MM_R64>(a, st);
    }
    return cfg == MM_D ? mm_go<BF, PK, QK, EPI, DUAL, MM_D>(a, st) : mm_go<BF, PK, QK, EPI, DUAL, MM_S>(a, st);
}
template <int PK, int QK, int EPI, bool DUAL> static inline int mm_go_any(const MmArgs& a, bool bf, int cfg, hipStream_t st) {
    return bf ? mm_go_cfg<true, PK, QK, EPI, DUAL>(a, cfg, st) : mm_go_cfg<false, PK, QK, EPI, DUAL>(a, cfg, st);
}
