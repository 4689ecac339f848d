// mm16.hip -- C entries of the 16-bit linear layer with a fused epilogue and of the gated feed-forward block, forward and
// backward: shape and alignment handling, choice of tile and K split, and the small kernels around the products (padding copy,
// dz = dy act'(z), column sums, the join of a split product).
#include "mm16.h"

// ------------------------------------------------------------------------------------------------ small kernels
// Up to MM_PADS matrices src [rows, cols] (any leading dimension, any alignment of 2 bytes) -> dst [rows, ldd], ldd = round8(cols),
// zero-filled: the one shape whose rows the LDS-DMA can fetch in 16-byte chunks.  Only matrices that are not already so pass through here, all
// of a call in one launch: a training step of odd sizes is bound by its launches.
#define MM_PADS 5
struct MmPads {
    int count;
    struct { const short* src; short* dst; long long lds, first; int rows, cols, ldd; } m[MM_PADS];     // first: chunks of the matrices in front
    long long total;
};
__global__ __launch_bounds__(256) void mm_pad_kernel(MmPads a) {
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < a.total; i += (long long)gridDim.x * 256) {
        int k = 0;
#pragma unroll
        for (int j = 1; j < MM_PADS; ++j) k += j < a.count && i >= a.m[j].first;
        const int cols = a.m[k].cols, ldd = a.m[k].ldd, cpr = ldd / 8;
        const long long q = i - a.m[k].first;
        const int r = (int)(q / cpr), c = (int)(q - (long long)r * cpr) * 8;
        const short* s = a.m[k].src + r * a.m[k].lds + c;
        mm_any8 v;
        if (c + 8 <= cols) v = *(const mm_any8*)s;
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? s[j] : (short)0;
        *(mm_any8*)(a.m[k].dst + (long long)r * ldd + c) = v;
    }
}

// Column sums, and dz on the way.  DZ: dz = dy act'(z) with z kept in fp32, stored as [rows][cols8] with zeros behind column cols - 1, and the
// sums (if wanted) are those of its values before they are rounded; else: x [rows][cols8] as it lies.  A workgroup takes a run of rows of
// 8 << lcx columns, 256 >> lcx rows a time.  Sums go to part [gridDim.y][cols8], or straight to out where one workgroup has all rows: two
// passes of fixed order, no atomics.  Bound by its bytes: 8 a value with dz, 2 without.
template <bool BF, bool DZ>
__global__ __launch_bounds__(256) void mm_colsum_kernel(const void* __restrict__ x, long long ld, int rows, int cols, int cols8, int lcx,
                                                        const float* __restrict__ z, int act, void* __restrict__ dz, float* __restrict__ part,
                                                        void* __restrict__ out) {
    __shared__ float red[256][9];
    const int cx = threadIdx.x & ((1 << lcx) - 1), ry = threadIdx.x >> lcx, lanes = 256 >> lcx, c = ((blockIdx.x << lcx) + cx) * 8;
    const int per = (rows + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = r0 + per < rows ? r0 + per : rows;
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (c < cols8)
        for (int r = r0 + ry; r < r1; r += lanes) {
            float v[8];
            if constexpr (DZ) {
                float p[8], a[8], slope[8];
                mm_row8<BF>(x, r * ld, c, cols, v);
                mm_ldf8(z + (long long)r * cols8 + c, p);
                mm_act_slope8(act, p, a, slope);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] *= slope[j];
                mm_put8<BF>(dz, (long long)r * cols8, c, cols, cols8, v);
            } else mm_ld8<BF>(x, r * ld + c, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) s[j] += v[j];
        }
    if (!part && !out) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[threadIdx.x][j] = s[j];
    __syncthreads();
    const int own = threadIdx.x, col = (blockIdx.x << lcx) * 8 + own;
    if (own >= (8 << lcx) || col >= cols8) return;
    float t = 0.0f;
    for (int k = 0; k < lanes; ++k) t += red[(k << lcx) + (own >> 3)][own & 7];
    if (part) part[(size_t)blockIdx.y * cols8 + col] = t;
    else if (col < cols) ((typename MmEl<BF>::T*)out)[col] = (typename MmEl<BF>::T)t;
}
// 32 columns a workgroup, 8 lanes a column
template <bool BF> __global__ __launch_bounds__(256) void mm_colsum_join_kernel(const float* __restrict__ part, int n, int cols8, int cols, void* __restrict__ out) {
    __shared__ float red[8][33];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
    float t = 0.0f;
    if (c < cols)
        for (int k = ry; k < n; k += 8) t += part[(size_t)k * cols8 + c];
    red[ry][cx] = t;
    __syncthreads();
    if (ry != 0 || c >= cols) return;
#pragma unroll
    for (int k = 1; k < 8; ++k) t += red[k][cx];
    ((typename MmEl<BF>::T*)out)[c] = (typename MmEl<BF>::T)t;
}

// the K ranges of a split product, added in their order
template <int NF> __device__ __forceinline__ void mm_join8(const MmArgs& a, int m, int n, float (*v)[8]) {
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[f][j] = 0.0f;
    const size_t plane = (size_t)a.M * a.e.ldpart;
    for (int s = 0; s < a.splits; ++s)
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            float w[8];
            mm_ldf8(a.e.part + (size_t)(s * NF + f) * plane + (size_t)m * a.e.ldpart + n, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[f][j] += w[j];
        }
}
// ... and the epilogue
template <bool BF, int EPI>
__global__ __launch_bounds__(256) void mm_join_kernel(MmArgs a) {
    const int cpr = a.e.ldpart / 8;
    const long long total = (long long)a.M * cpr;
    const long long i = blockIdx.x * 256LL + threadIdx.x;
    if (i >= total) return;
    const int m = (int)(i / cpr), n = (int)(i - (long long)m * cpr) * 8;
    constexpr int NF = EPI == MM_GATE ? 2 : 1;
    float v[NF][8];
    mm_join8<NF>(a, m, n, v);
    if constexpr (EPI == MM_GATE) mm_epi_gate<BF>(a.e, m, n, a.N, v[0], v[1]);
    else mm_epi_act<BF>(a.e, m, n, a.N, v[0]);
}
// ... and the gate's backward, with the column sums (e.sums [gridDim.y][2 npad]): a run of rows of 256 columns a workgroup, 8 rows a time
template <bool BF> __global__ __launch_bounds__(256) void mm_join_gate_bwd_kernel(MmArgs a) {
    __shared__ float red[8][32][17];
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, n = (blockIdx.x * 32 + cx) * 8;
    const int per = (a.M + gridDim.y - 1) / gridDim.y, r0 = blockIdx.y * per, r1 = r0 + per < a.M ? r0 + per : a.M;
    float sums[16] = {};
    if (n < a.e.npad)
        for (int m = r0 + ry; m < r1; m += 8) {
            float v[1][8];
            mm_join8<1>(a, m, n, v);
            mm_epi_gate_bwd<BF>(a.e, m, n, a.N, v[0], sums, sums + 8);
        }
    if (!a.e.sums) return;
#pragma unroll
    for (int j = 0; j < 16; ++j) red[ry][cx][j] = sums[j];
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += 256) {                   // factor, column
        const int f = i >> 8, c = i & 255, col = blockIdx.x * 256 + c;
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += red[k][c >> 3][8 * f + (c & 7)];
        if (col < a.e.npad) a.e.sums[(size_t)blockIdx.y * 2 * a.e.npad + f * a.e.npad + col] = t;
    }
}

// ------------------------------------------------------------------------------------------------ host
namespace {

inline int r8(int n) { return (n + 7) & ~7; }

// Hands out the caller's workspace; with a null base it only adds up what the same calls would take.
struct Arena {
    char* base; size_t cap, off = 0, peak = 0;
    bool dry() const { return base == nullptr; }
    void* take(size_t bytes) {
        off = (off + 255) & ~(size_t)255;
        void* p = base ? base + off : nullptr;
        off += bytes;
        if (off > peak) peak = off;
        return p;
    }
    bool full() const { return base && peak > cap; }
};

struct Ctx {
    Arena& ar; bool bf; hipStream_t st; int rc = ACMIL_OK;
    MmPads pads = {};                                                // asked for, not yet launched
    bool go() const { return rc == ACMIL_OK && !ar.dry(); }
    void launched() { if (hipGetLastError() != hipSuccess) rc = ACMIL_ERR_LAUNCH; }
    bool room() { if (ar.full()) { if (rc == ACMIL_OK) rc = ACMIL_ERR_SHAPE; return false; } return true; }
};

struct Mat { const void* p; long long ld; int rows, cols; };

inline bool on16(const void* p) { return ((size_t)p & 15) == 0; }
inline unsigned grid_of(long long items) { const long long g = (items + 255) / 256; return (unsigned)(g < 1 ? 1 : g > 65536 ? 65536 : g); }

// launch the padding copies asked for so far: in front of the first kernel that reads one
void flush(Ctx& c) {
    if (c.pads.count == 0) return;
    if (c.room() && c.go()) {
        hipLaunchKernelGGL(mm_pad_kernel, dim3(grid_of(c.pads.total)), dim3(256), 0, c.st, c.pads);
        c.launched();
    }
    c.pads.count = 0;
    c.pads.total = 0;
}
// m as the products take it: rows on 16 bytes, a multiple of 8 columns (zeros behind the last)
Mat aligned(Ctx& c, const Mat& m, bool force = false) {
    if (!force && on16(m.p) && m.ld % 8 == 0 && m.cols % 8 == 0) return m;
    const int ldd = r8(m.cols);
    short* d = (short*)c.ar.take((size_t)m.rows * ldd * 2);
    if (c.pads.count == MM_PADS) flush(c);
    c.pads.m[c.pads.count++] = {(const short*)m.p, d, m.ld, c.pads.total, m.rows, m.cols, ldd};
    c.pads.total += (long long)m.rows * (ldd / 8);
    return Mat{d, ldd, m.rows, ldd};
}
// two matrices that one product addresses with one leading dimension
void aligned_pair(Ctx& c, Mat& a, Mat& b) {
    Mat x = aligned(c, a), y = aligned(c, b);
    if (x.ld != y.ld) {
        if (x.p == a.p && x.ld != r8(a.cols)) x = aligned(c, a, true);
        if (y.p == b.p && y.ld != r8(b.cols)) y = aligned(c, b, true);
    }
    a = x; b = y;
}

enum { FWD, DGRAD, WGRAD };

// runs of rows of mm_join_gate_bwd_kernel: at least 8 rows each, up to 2048 workgroups
int join_gate_rows(const MmArgs& a) {
    const int gx = (a.e.npad + 255) / 256, most = gx >= 256 ? 8 : 2048 / gx, gy = (a.M + 7) / 8;
    return gy > most ? most : gy;
}

void join(Ctx& c, const MmArgs& a, int epi) {
    const dim3 g((unsigned)(((long long)a.M * (a.e.ldpart / 8) + 255) / 256));
#define JOIN(B, E) hipLaunchKernelGGL((mm_join_kernel<B, E>), g, dim3(256), 0, c.st, a)
    if (epi == MM_GATE_BWD) {
        const dim3 gb((a.e.npad + 255) / 256, join_gate_rows(a));
        if (c.bf) hipLaunchKernelGGL((mm_join_gate_bwd_kernel<true>), gb, dim3(256), 0, c.st, a);
        else hipLaunchKernelGGL((mm_join_gate_bwd_kernel<false>), gb, dim3(256), 0, c.st, a);
    } else if (epi == MM_GATE) { if (c.bf) JOIN(true, MM_GATE); else JOIN(false, MM_GATE); }
    else { if (c.bf) JOIN(true, MM_ACT); else JOIN(false, MM_ACT); }
#undef JOIN
    c.launched();
}

// How many ways to split K of a product of 128 x 128 tiles.  A step of one tile takes about 0.55 us alone on its CU and 1.0 us beside
// another; a split costs a join launch and 8 bytes of partial sums per output and part, written and read at about 4 TB/s.  The rule without
// these costs, as many parts as fill 512 workgroups, took 20.2 us for 2000 x 768 x 768 against 11.2, and 19.4 for 64 x 4096 x 4096 against 15.4.
int mm_splits(long long tiles, int steps, double outputs, double* cost = nullptr) {
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 64 && s * 4 <= (steps > 4 ? steps : 4); ++s) {
        const long long wgs = tiles * s, rounds = (wgs + 511) / 512, rest = wgs - 512 * (rounds - 1);
        const double step = (rounds - 1) * 1.0 + (rest > 256 ? 1.0 : 0.55);
        const double us = ((steps + s - 1) / s) * step + (s > 1 ? 2.5 + s * outputs * 8.0 / 4e6 : 0.0);
        if (us < least) { least = us; best = s; }
    }
    if (cost) *cost = least;
    return best;
}

// ... and of a product of up to 64 rows in 256-column tiles: a step streams 32 KB of P and the rows of Q, at 37 GB/s and CU (a workgroup
// waits for memory alone) and at 5 TB/s altogether
int slim_splits(long long tiles, int steps, int bm, double outputs) {
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 64 && s * 4 <= (steps > 4 ? steps : 4) && tiles * s <= 256; ++s) {
        const double bytes = 128.0 * (256 + bm), all = (double)tiles * s * bytes / 5e6, one = bytes / 37e3;
        const double us = ((steps + s - 1) / s) * (all > one ? all : one) + (s > 1 ? 2.5 + s * outputs * 8.0 / 4e6 : 0.0);
        if (us < least) { least = us; best = s; }
    }
    return best;
}

template <bool BF> void colsum_join(Ctx& c, const float* part, int n, int cols8, int cols, void* out) {
    hipLaunchKernelGGL((mm_colsum_join_kernel<BF>), dim3((cols + 31) / 32), dim3(256), 0, c.st, part, n, cols8, cols, out);
}

// rows from .. from + count - 1 of a product
MmArgs rows_of(MmArgs a, int kind, int from, int count) {
    const long long q = kind == WGRAD ? from * 2LL : from * a.ldq, o = from * a.e.ldo * 2;
    a.q0 += q; a.q1 += q;
    a.e.out = (char*)a.e.out + o;
    if (a.e.out2) a.e.out2 = (char*)a.e.out2 + o;
    if (a.e.res) a.e.res = (const char*)a.e.res + from * a.e.ldr * 2;
    if (a.e.pre) a.e.pre += from * a.e.ldp;
    if (a.e.pre2) a.e.pre2 += from * a.e.ldp;
    a.M = count;
    return a;
}

// One product: tile, K split, launch, join.  sums (MM_GATE_BWD): null, or [2 npad] for the column sums of dg and du.  whole: rows stay in one launch.
void product(Ctx& c, int kind, MmArgs a, int epi, void* sums = nullptr, bool whole = false) {
    const bool dual = epi == MM_GATE;
    const int n_eff = dual ? 2 * a.N : a.N, steps = mm_steps(a);
    const long long tl = (long long)((a.M + 255) / 256) * ((n_eff + 255) / 256);
    // 256 x 256 tiles need half the LDS reads and fetches per flop of 128 x 128 ones, but only one fits a CU: taken where they fill
    // most of the 256 CUs
    const bool large = tl >= 160;
    // (Not where column sums are formed on the way, the gated block's backward with bias gradients: they are laid out by the row tiles of one launch.)
    if (large && tl > 256 && tl % 256 != 0 && !sums && !whole) {
        // The last round of large tiles leaves CUs without work.  A full round takes about 10 us and 1.4 us a step; where its rows take less as a
        // product of their own, by 128 x 128 tiles (6 us for the launch), they become one: 5000 x 2048 x 3500 123 -> 97 us, 10000 x 2048 x 2048
        // 97 -> 79, 50000 x 1536 x 768 140 -> 135; 7000 x 1024 x 4096, which the rule takes too, 65 -> 66.
        const long long row = (n_eff + 255) / 256, kept = (tl - tl % 256) / row * 256;
        if (kept > 0 && kept < a.M) {
            double cost;
            const int rest = a.M - (int)kept;
            mm_splits((long long)((rest + 127) / 128) * ((n_eff + 127) / 128), steps, (double)rest * r8(a.e.npad) * (dual ? 2 : 1), &cost);
            if (cost + 6.0 < 10.0 + 1.4 * steps) {
                product(c, kind, rows_of(a, kind, 0, (int)kept), epi, nullptr, true);
                product(c, kind, rows_of(a, kind, (int)kept, rest), epi, nullptr, true);
                return;
            }
        }
    }
    // up to 64 rows: tiles of as many rows where the weights have to be streamed (below 64 MB the 128-row tiles take 16 us for 64 x 4096 x 4096
    // against 19, and 8.5 for 64 x 1024 x 1024 against 10.3)
    const bool slim = !large && kind != WGRAD && a.M <= 64 && (double)n_eff * steps * 64 >= 33554432.0;
    const int bm = large ? 256 : slim ? (a.M <= 32 ? 32 : 64) : 128, bn = large || slim ? 256 : 128;
    a.ntm = (a.M + bm - 1) / bm;
    a.ntn = (n_eff + bn - 1) / bn;
    const long long tiles = (long long)a.ntm * a.ntn;
    const double outputs = (double)a.M * r8(a.e.npad) * (dual ? 2 : 1);
    a.splits = large ? 1 : slim ? slim_splits(tiles, steps, bm, outputs) : mm_splits(tiles, steps, outputs);
    const size_t mark = c.ar.off;
    if (a.splits > 1) {
        a.e.ldpart = r8(a.e.npad);
        a.e.part = (float*)c.ar.take((size_t)a.splits * (dual ? 2 : 1) * a.M * a.e.ldpart * 4);
    }
    const int cfg = large ? MM_L : slim ? (bm == 32 ? MM_R32 : MM_R64) : tiles * a.splits <= 256 ? MM_D : MM_S;
    const int rows = a.splits > 1 ? join_gate_rows(a) : a.ntm * mm_wave_rows(cfg);
    if (sums) a.e.sums = (float*)c.ar.take((size_t)rows * 2 * a.e.npad * 4);
    flush(c);
    if (c.room() && c.go()) {
        const int e = a.splits > 1 ? MM_PART : epi;
        c.rc = kind == FWD ? mm_launch_fwd(a, c.bf, e, dual, cfg, c.st) : kind == DGRAD ? mm_launch_dgrad(a, c.bf, e, cfg, c.st)
                                                                             : mm_launch_wgrad(a, c.bf, e, cfg, c.st);
        if (a.splits > 1 && c.rc == ACMIL_OK) join(c, a, epi);
        if (sums && c.rc == ACMIL_OK) {
            if (c.bf) colsum_join<true>(c, a.e.sums, rows, 2 * a.e.npad, 2 * a.e.npad, sums);
            else colsum_join<false>(c, a.e.sums, rows, 2 * a.e.npad, 2 * a.e.npad, sums);
            c.launched();
        }
    }
    c.ar.off = mark;                                                 // the partial sums are dead behind the join: stream order
}

MmArgs operands(const Mat& q, const Mat& p, int M, int N, int Kq, int Kp) {
    MmArgs a = {};
    a.q0 = a.q1 = (const char*)q.p; a.p0 = a.p1 = (const char*)p.p;
    a.ldq = q.ld * 2; a.ldp = p.ld * 2;
    a.M = M; a.N = N; a.Kq = Kq; a.Kp = Kp; a.segs = 1; a.splits = 1;
    a.e.act = ACMIL_ACT_NONE;
    return a;
}
void output(MmArgs& a, void* out, long long ldo, const void* bias = nullptr, const void* res = nullptr, long long ldr = 0) {
    a.e.out = out; a.e.ldo = ldo; a.e.bias = bias; a.e.res = res; a.e.ldr = ldr; a.e.npad = a.N;
}

// out [cols] = column sums of x (null: none wanted); with z, x is dy and dz [rows][round8(cols)] receives dy act'(z)
void colsum(Ctx& c, const Mat& x, int rows, int cols, void* out, const float* z = nullptr, int act = ACMIL_ACT_NONE, void* dz = nullptr) {
    const size_t mark = c.ar.off;
    const int c8 = r8(cols);
    int lcx = 0;
    while (lcx < 5 && (8 << lcx) < c8) ++lcx;
    const int gx = (c8 + (8 << lcx) - 1) / (8 << lcx), lanes = 256 >> lcx, most = gx >= 256 ? 8 : 2048 / gx;
    int gy = rows / (2 * lanes);                                     // enough workgroups to keep the memory busy, and at least two rows a lane
    gy = rows <= 8 * lanes ? 1 : gy > most ? most : gy;
    gy = gy > 256 ? 256 : gy;
    float* part = out && gy > 1 ? (float*)c.ar.take((size_t)gy * c8 * 4) : nullptr;
    flush(c);
    if (c.room() && c.go()) {
        const dim3 g(gx, gy);
#define COLSUM(B, Z) hipLaunchKernelGGL((mm_colsum_kernel<B, Z>), g, dim3(256), 0, c.st, x.p, x.ld, rows, cols, c8, lcx, z, act, dz, part, out)
        if (z) { if (c.bf) COLSUM(true, true); else COLSUM(false, true); }
        else { if (c.bf) COLSUM(true, false); else COLSUM(false, false); }
#undef COLSUM
        if (part && c.bf) colsum_join<true>(c, part, gy, c8, cols, out);
        else if (part) colsum_join<false>(c, part, gy, c8, cols, out);
        c.launched();
    }
    c.ar.off = mark;
}

// 32-bit byte offsets inside a tile: 256 rows (64 k rows) of the largest leading dimension; 31-bit row, column and tile counts
const long long MAX_LD = 1LL << 22;
const int MAX_DIM = 1 << 22, MAX_ROWS = 1 << 30;
const double MAX_OUT = 274877906944.0;       // 2^38 outputs, more than the memory holds: at most 2^23 tiles, 2^32 threads

bool same_dtype_ok(int dtype) { return dtype == ACMIL_DTYPE_F16 || dtype == ACMIL_DTYPE_BF16; }
bool act_ok(int act) { return act >= ACMIL_ACT_NONE && act <= ACMIL_ACT_SIGMOID; }
bool ld_ok(const void* p, long long ld, int cols) { return !p || (ld >= 0 && ld <= MAX_LD && (ld >= cols || ld == 0)); }

void few_rows(Ctx& c, MmArgs a, bool dual) {
    const size_t mark = c.ar.off;
    flush(c);
    a.splits = mm_rows_splits(a.M, a.e.npad, a.Kq, dual);
    if (a.splits > 1) {
        a.e.ldpart = r8(a.e.npad);
        a.e.part = (float*)c.ar.take((size_t)a.splits * (dual ? 2 : 1) * a.M * a.e.ldpart * 4);
    }
    if (c.room() && c.go()) {
        c.rc = mm_launch_rows(a, c.bf, dual, c.st);
        if (a.splits > 1 && c.rc == ACMIL_OK) join(c, a, dual ? MM_GATE : MM_ACT);
    }
    c.ar.off = mark;
}

int linear_check(const acmil_linear_args* a, bool backward) {
    if (!a) return ACMIL_ERR_NULL;
    if (!same_dtype_ok(a->dtype)) return ACMIL_ERR_UNSUPPORTED;
    if (!act_ok(a->act) || a->M <= 0 || a->K <= 0 || a->N <= 0 || a->M > MAX_ROWS || a->K > MAX_DIM || a->N > MAX_DIM) return ACMIL_ERR_SHAPE;
    if ((double)a->M * a->N > MAX_OUT || (double)a->M * a->K > MAX_OUT) return ACMIL_ERR_SHAPE;
    if (!a->x || !a->W) return ACMIL_ERR_NULL;
    if (!ld_ok(a->x, a->ldx, a->K) || !ld_ok(a->W, a->ldw, a->K)) return ACMIL_ERR_SHAPE;
    if (!backward) {
        if (!a->y) return ACMIL_ERR_NULL;
        if (a->ldy < a->N || !ld_ok(a->res, a->ldr, a->N)) return ACMIL_ERR_SHAPE;
        if (a->pre && !on16(a->pre)) return ACMIL_ERR_SHAPE;
        return ACMIL_OK;
    }
    if (!a->dy || (a->act != ACMIL_ACT_NONE && !a->pre)) return ACMIL_ERR_NULL;
    if (!ld_ok(a->dy, a->lddy, a->N) || (a->pre && !on16(a->pre))) return ACMIL_ERR_SHAPE;
    return ACMIL_OK;
}

bool plain(const Mat& m) { return on16(m.p) && m.ld % 8 == 0 && m.cols % 8 == 0; }

// The kernel of mm16_rows.hip, or tiles of 32 rows?  The former reads x once per 16 to 64 columns beside the weights (3.1 TB/s at 24 rows
// against 4.0), the latter takes two launches and rows on 16 bytes: worth it for 64 MB of weights and more (32 rows 4096 -> 4096: 15 us both).
bool few_rows_wanted(const Mat& x, const Mat& w, int factors) {
    if (x.rows > ACMIL_FEW_ROWS) return false;
    return x.rows <= 4 || !plain(x) || !plain(w) || (double)factors * w.rows * w.cols < 33554432.0;
}

int linear_fwd(const acmil_linear_args& a, Ctx& c) {
    Mat x{a.x, a.ldx, a.M, a.K}, w{a.W, a.ldw, a.N, a.K};
    const bool few = few_rows_wanted(x, w, 1);
    if (!few) { x = aligned(c, x); w = aligned(c, w); }
    MmArgs p = operands(x, w, a.M, a.N, x.cols, w.cols);
    output(p, a.y, a.ldy, a.bias, a.res, a.ldr);
    p.e.act = a.act; p.e.pre = a.pre; p.e.ldp = r8(a.N);
    if (few) few_rows(c, p, false); else product(c, FWD, p, MM_ACT);
    return c.rc;
}

int linear_bwd(const acmil_linear_args& a, Ctx& c) {
    const Mat dy{a.dy, a.lddy, a.M, a.N};
    Mat dz;
    if (a.act == ACMIL_ACT_NONE) dz = aligned(c, dy);
    else {
        const int ldz = r8(a.N);
        void* z = c.ar.take((size_t)a.M * ldz * 2);
        colsum(c, dy, a.M, a.N, a.db, a.pre, a.act, z);
        dz = Mat{z, ldz, a.M, ldz};
    }
    Mat w{a.W, a.ldw, a.N, a.K}, x{a.x, a.ldx, a.M, a.K};
    if (a.dx) w = aligned(c, w);
    if (a.dW) x = aligned(c, x);
    if (a.dx) {
        MmArgs p = operands(dz, w, a.M, a.K, dz.cols, a.N);
        output(p, a.dx, a.K);
        product(c, DGRAD, p, MM_ACT);
    }
    if (a.dW) {
        MmArgs p = operands(dz, x, a.N, a.K, a.M, a.M);
        output(p, a.dW, a.K);
        product(c, WGRAD, p, MM_ACT);
    }
    if (a.db && a.act == ACMIL_ACT_NONE) colsum(c, dz, a.M, a.N, a.db);
    return c.rc;
}

int ffn_check(const acmil_ffn_args* a, bool backward) {
    if (!a) return ACMIL_ERR_NULL;
    if (!same_dtype_ok(a->dtype)) return ACMIL_ERR_UNSUPPORTED;
    if (!act_ok(a->act) || a->M <= 0 || a->D <= 0 || a->F <= 0 || a->M > MAX_ROWS || a->D > MAX_DIM || a->F > MAX_DIM / 2) return ACMIL_ERR_SHAPE;
    if ((double)a->M * a->D > MAX_OUT || (double)a->M * a->F > MAX_OUT / 2) return ACMIL_ERR_SHAPE;
    if (!a->x || !a->Wg || !a->Wu || !a->Wd) return ACMIL_ERR_NULL;
    if (!ld_ok(a->x, a->ldx, a->D) || !ld_ok(a->Wg, a->ldwg, a->D) || !ld_ok(a->Wu, a->ldwu, a->D) || !ld_ok(a->Wd, a->ldwd, a->F)) return ACMIL_ERR_SHAPE;
    const int saved = (a->g != nullptr) + (a->u != nullptr) + (a->h != nullptr);
    if (saved != 0 && saved != 3) return ACMIL_ERR_NULL;
    if (!on16(a->g) || !on16(a->u) || !on16(a->h)) return ACMIL_ERR_SHAPE;
    if (!backward) {
        if (!a->y) return ACMIL_ERR_NULL;
        return a->ldy < a->D || !ld_ok(a->res, a->ldr, a->D) ? ACMIL_ERR_SHAPE : ACMIL_OK;
    }
    if (!a->dy || saved != 3) return ACMIL_ERR_NULL;
    return ld_ok(a->dy, a->lddy, a->D) ? ACMIL_OK : ACMIL_ERR_SHAPE;
}

int ffn_fwd(const acmil_ffn_args& a, Ctx& c) {
    const int F8 = r8(a.F);
    Mat x{a.x, a.ldx, a.M, a.D}, wg{a.Wg, a.ldwg, a.F, a.D}, wu{a.Wu, a.ldwu, a.F, a.D}, wd{a.Wd, a.ldwd, a.D, a.F};
    const bool few = few_rows_wanted(x, wg, 2) || (a.M <= ACMIL_FEW_ROWS && !plain(wu));
    if (!few) { x = aligned(c, x); aligned_pair(c, wg, wu); }
    else if (wg.ld != wu.ld) aligned_pair(c, wg, wu);                // one leading dimension for both
    Mat h{a.h ? a.h : c.ar.take((size_t)a.M * F8 * 2), F8, a.M, F8};
    const bool few_down = few_rows_wanted(h, wd, 1);
    if (!few_down) wd = aligned(c, wd);
    if (!c.room()) return c.rc;
    MmArgs p = operands(x, wg, a.M, a.F, few ? a.D : x.cols, few ? a.D : wg.cols);
    p.p1 = (const char*)wu.p;
    output(p, (void*)h.p, F8, a.bg);
    p.e.bias2 = a.bu; p.e.npad = F8; p.e.act = a.act;
    p.e.pre = a.g; p.e.pre2 = a.u; p.e.ldp = F8;
    if (few) few_rows(c, p, true); else product(c, FWD, p, MM_GATE);
    MmArgs d = operands(h, wd, a.M, a.D, few_down ? a.F : F8, few_down ? a.F : wd.cols);
    output(d, a.y, a.ldy, a.bd, a.res, a.ldr);
    if (few_down) few_rows(c, d, false); else product(c, FWD, d, MM_ACT);
    return c.rc;
}

int ffn_bwd(const acmil_ffn_args& a, Ctx& c) {
    const int F8 = r8(a.F);
    const Mat dy = aligned(c, Mat{a.dy, a.lddy, a.M, a.D}), h{a.h, F8, a.M, F8};
    Mat x{a.x, a.ldx, a.M, a.D}, wg{a.Wg, a.ldwg, a.F, a.D}, wu{a.Wu, a.ldwu, a.F, a.D}, wd{a.Wd, a.ldwd, a.D, a.F};
    Mat dgu{nullptr, 2LL * F8, a.M, 2 * F8};                         // [dg | du], each with zeros behind column F
    if (a.dx || a.dWgu || a.dbgu) wd = aligned(c, wd);
    if (a.dx) aligned_pair(c, wg, wu);
    if (a.dWgu) x = aligned(c, x);
    if (a.dx || a.dWgu || a.dbgu) {
        dgu.p = c.ar.take((size_t)a.M * 2 * F8 * 2);
        if (!c.room()) return c.rc;
        MmArgs p = operands(dy, wd, a.M, a.F, dy.cols, a.D);
        output(p, (void*)dgu.p, 2LL * F8);
        p.e.out2 = (short*)dgu.p + F8; p.e.npad = F8; p.e.act = a.act;
        p.e.pre = a.g; p.e.pre2 = a.u; p.e.ldp = F8;
        product(c, DGRAD, p, MM_GATE_BWD, a.dbgu);
    }
    if (a.dx) {
        MmArgs p = operands(dgu, wg, a.M, a.D, F8, a.F);             // dg Wg + du Wu: two K segments of one product
        p.segs = 2;
        p.q1 = p.q0 + 2LL * F8; p.p1 = (const char*)wu.p;
        output(p, a.dx, a.D);
        product(c, DGRAD, p, MM_ACT);
    }
    if (a.dWgu) {
        MmArgs p = operands(dgu, x, 2 * F8, a.D, a.M, a.M);
        output(p, a.dWgu, a.D);
        product(c, WGRAD, p, MM_ACT);
    }
    if (a.dWd) {
        MmArgs p = operands(dy, h, a.D, a.F, a.M, a.M);
        output(p, a.dWd, a.F);
        product(c, WGRAD, p, MM_ACT);
    }
    if (a.dbd) colsum(c, dy, a.M, a.D, a.dbd);
    return c.rc;
}

const size_t NOTHING = 256;      // what a call that takes no workspace answers to the query (0 = refused)
template <class A> size_t need(const A* a, int rc, int (*f)(const A&, Ctx&)) {
    if (rc != ACMIL_OK) return 0;
    Arena ar{nullptr, 0};
    Ctx c{ar, a->dtype == ACMIL_DTYPE_BF16, nullptr};
    f(*a, c);
    return ((ar.peak + 255) & ~(size_t)255) + NOTHING;
}
template <class A> int go(const A* a, int rc, int (*f)(const A&, Ctx&), void* ws, size_t bytes, void* stream) {
    if (rc != ACMIL_OK) return rc;
    if (((size_t)ws & 255) != 0) return ACMIL_ERR_SHAPE;
    const size_t want = need(a, rc, f);                              // before anything is launched
    if (want > NOTHING && !ws) return ACMIL_ERR_NULL;
    if (want > NOTHING && bytes < want) return ACMIL_ERR_SHAPE;
    Arena ar{ws ? (char*)ws : (char*)256, bytes};                    // (nothing is taken from a workspace that is not needed)
    Ctx c{ar, a->dtype == ACMIL_DTYPE_BF16, (hipStream_t)stream};
    return f(*a, c);
}

}  // namespace

extern "C" size_t acmil_linear_act_workspace_bytes(const acmil_linear_args* a) { return need(a, linear_check(a, false), linear_fwd); }
extern "C" int acmil_linear_act(const acmil_linear_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    return go(a, linear_check(a, false), linear_fwd, workspace, workspace_bytes, stream);
}
extern "C" size_t acmil_linear_act_bwd_workspace_bytes(const acmil_linear_args* a) { return need(a, linear_check(a, true), linear_bwd); }
extern "C" int acmil_linear_act_bwd(const acmil_linear_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    return go(a, linear_check(a, true), linear_bwd, workspace, workspace_bytes, stream);
}
extern "C" size_t acmil_gated_ffn_workspace_bytes(const acmil_ffn_args* a) { return need(a, ffn_check(a, false), ffn_fwd); }
extern "C" int acmil_gated_ffn(const acmil_ffn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    return go(a, ffn_check(a, false), ffn_fwd, workspace, workspace_bytes, stream);
}
extern "C" size_t acmil_gated_ffn_bwd_workspace_bytes(const acmil_ffn_args* a) { return need(a, ffn_check(a, true), ffn_bwd); }
extern "C" int acmil_gated_ffn_bwd(const acmil_ffn_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    return go(a, ffn_check(a, true), ffn_bwd, workspace, workspace_bytes, stream);
}
