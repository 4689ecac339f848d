// muon.hip -- The two element-wise passes around acmil_orthogonalize in an optimizer step over flat buffers: momentum in front, the step itself
// behind.  Both are bound by their bytes (12 + 4 and 8 + 4 per element): inside a step 4096 x 4096 takes 55 and 49 us, 4.9 and 4.1 TB/s, and the three
// matrices of the gated-attention aggregator 4 us each, an empty launch.  The matrices of a model are segments of the flat buffers, up to MUON_SEGS
// of them per launch, and an element finds its segment by bisection in the kernel arguments.
#include "ga_common.h"

#define MUON_SEGS 64
struct MuonSegs {
    int count;
    long long off[MUON_SEGS];         // where segment i starts in the flat parameter / gradient / momentum buffers
    long long at[MUON_SEGS + 1];      // ... and in the packed update buffer (ascending; the launch covers at[0] .. at[count])
    float scale[MUON_SEGS];
};

__device__ __forceinline__ int muon_seg(const MuonSegs& s, long long i) {
    int lo = 0, hi = s.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (i >= s.at[mid]) lo = mid; else hi = mid;
    }
    return lo;
}

// buf = mu buf + g;  upd = nesterov ? g + mu buf : buf.  A raised flag leaves buf as it is (and upd undefined: muon_apply skips as well).
__global__ __launch_bounds__(256) void muon_momentum_kernel(MuonSegs s, const float* __restrict__ g, float* __restrict__ buf, float* __restrict__ upd,
                                                           float mu, int nesterov, const float* __restrict__ skip_flag, float* __restrict__ flag_report) {
    if (flag_report && blockIdx.x == 0 && threadIdx.x == 0) __builtin_nontemporal_store(skip_flag ? skip_flag[0] : 0.0f, flag_report);
    if (skip_flag && !(skip_flag[0] == 0.0f)) return;
    const long long end = s.at[s.count];
    for (long long i = s.at[0] + blockIdx.x * 256LL + threadIdx.x; i < end; i += (long long)gridDim.x * 256) {
        const int k = muon_seg(s, i);
        const long long f = s.off[k] + (i - s.at[k]);
        const float gi = g[f], b = mu * buf[f] + gi;
        buf[f] = b;
        upd[i] = nesterov ? gi + mu * b : b;
    }
}

// p = p (1 - lr wd) - lr scale upd
__global__ __launch_bounds__(256) void muon_apply_kernel(MuonSegs s, float* __restrict__ p, const float* __restrict__ upd, float lr, float wd,
                                                        const float* __restrict__ skip_flag) {
    if (skip_flag && !(skip_flag[0] == 0.0f)) return;
    const long long end = s.at[s.count];
    for (long long i = s.at[0] + blockIdx.x * 256LL + threadIdx.x; i < end; i += (long long)gridDim.x * 256) {
        const int k = muon_seg(s, i);
        const long long f = s.off[k] + (i - s.at[k]);
        p[f] = p[f] * (1.0f - lr * wd) - lr * s.scale[k] * upd[i];
    }
}

static int muon_check(int count, const acmil_muon_seg* segs) {
    if (!segs) return ACMIL_ERR_NULL;
    if (count <= 0) return ACMIL_ERR_SHAPE;
    for (int i = 0; i < count; ++i)
        if (segs[i].offset < 0 || segs[i].numel <= 0) return ACMIL_ERR_SHAPE;
    return ACMIL_OK;
}
template <class F> static int muon_groups(int count, const acmil_muon_seg* segs, F launch) {
    long long at = 0;
    for (int b = 0; b < count; b += MUON_SEGS) {
        MuonSegs s = {};
        s.count = count - b < MUON_SEGS ? count - b : MUON_SEGS;
        s.at[0] = at;
        for (int i = 0; i < s.count; ++i) {
            s.off[i] = segs[b + i].offset;
            s.scale[i] = segs[b + i].scale;
            at += segs[b + i].numel;
            s.at[i + 1] = at;
        }
        const long long n = at - s.at[0], blocks = (n + 255) / 256;
        launch(s, (unsigned)(blocks < 2048 ? blocks : 2048));
        if (hipGetLastError() != hipSuccess) return ACMIL_ERR_LAUNCH;
    }
    return ACMIL_OK;
}

extern "C" int acmil_muon_momentum(int count, const acmil_muon_seg* segs, const float* grads, float* momentum, float* update, float mu, int nesterov,
                                   const float* skip_flag, float* flag_report, void* stream) {
    const int rc = muon_check(count, segs);
    if (rc != ACMIL_OK) return rc;
    if (!(mu >= 0.0f && mu < 1.0f)) return ACMIL_ERR_SHAPE;
    if (!grads || !momentum || !update) return ACMIL_ERR_NULL;
    return muon_groups(count, segs, [&](const MuonSegs& s, unsigned blocks) {
        hipLaunchKernelGGL(muon_momentum_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, s, grads, momentum, update, mu, nesterov, skip_flag,
                           flag_report);
    });
}

extern "C" int acmil_muon_apply(int count, const acmil_muon_seg* segs, float* params, const float* update, float lr, float weight_decay,
                                const float* skip_flag, void* stream) {
    const int rc = muon_check(count, segs);
    if (rc != ACMIL_OK) return rc;
    if (!params || !update) return ACMIL_ERR_NULL;
    return muon_groups(count, segs, [&](const MuonSegs& s, unsigned blocks) {
        hipLaunchKernelGGL(muon_apply_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, s, params, update, lr, weight_decay, skip_flag);
    });
}
