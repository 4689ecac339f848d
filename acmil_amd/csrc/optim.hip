// optim.hip -- AdamW over ONE flat fp32 parameter buffer (torch.optim.AdamW semantics, decoupled weight decay), one launch.
// Replaces the optimizer.step() of the reference's loop (Step3_WSI_classification_ACMIL.py:139,219: torch.optim.AdamW over
// 26 small tensors = 10 foreach launches, or 38 us in torch's fused variant); the training step is launch-bound at small
// bags, and parameters / gradients / moments already live in flat buffers (slide-level DP all-reduces one flat bucket).
//   p *= 1 - lr * wd ;  m = b1 m + (1-b1) g ;  v = b2 v + (1-b2) g^2 ;  p -= (lr / bc1) * m / (sqrt(v) / sqrt(bc2) + eps)
// with bc1 = 1 - b1^t, bc2 = 1 - b2^t formed on the device in double (t = the caller's launch ordinal minus the skipped launches).
#include "ga_common.h"
#include "optim_kernel.h"

__global__ __launch_bounds__(256) void adamw_flat_kernel(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
                                                        float* __restrict__ v, long long n, float lr, double beta1, double beta2, float eps,
                                                        float wd, long long launch, const float* __restrict__ skip_flag,
                                                        int* __restrict__ skipped, float* __restrict__ flag_report) {
    // device-side skip (like an AMP overflow skip): a non-zero / NaN flag -- the all-reduced range flag of a split-f16 training
    // step, csrc/ga_step.hip -- leaves parameters and moments untouched and is counted in *skipped; the host learns about it
    // later (optim.py).  The step number of the bias corrections is the launch ordinal minus the launches skipped so far, so
    // the update stays torch.optim.AdamW's for the steps that are applied.
    __shared__ float s_bc[2];
    // the flag, reported to the host without a copy on the stream: one lane stores it to a device-visible address (pinned host
    // memory); the host reads it after the event it records behind this launch
    if (flag_report && blockIdx.x == 0 && threadIdx.x == 0) __builtin_nontemporal_store(skip_flag ? skip_flag[0] : 0.0f, flag_report);
    if (skip_flag && !(skip_flag[0] == 0.0f)) {
        if (skipped && blockIdx.x == 0 && threadIdx.x == 0) atomicAdd(skipped, 1);
        return;
    }
    if (threadIdx.x == 0) {
        const long long t = launch - (skipped ? (long long)*skipped : 0);
        adamw_bias(beta1, beta2, t, s_bc[0], s_bc[1]);
    }
    __syncthreads();
    const float inv_bc1 = s_bc[0], inv_sqrt_bc2 = s_bc[1];
    const float b1 = (float)beta1, b2 = (float)beta2;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float pi = p[i], mi = m[i], vi = v[i];
        adamw_update(pi, g[i], mi, vi, lr, wd, inv_bc1, inv_sqrt_bc2, eps, b1, b2);
        m[i] = mi; v[i] = vi; p[i] = pi;
    }
}

extern "C" int acmil_adamw_step_report(float* params, const float* grads, float* exp_avg, float* exp_avg_sq, long long n, float lr,
                                       double beta1, double beta2, float eps, float weight_decay, long long step, const float* skip_flag,
                                       int* skipped, float* flag_report, void* stream) {
    if (n <= 0 || step < 1 || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return ACMIL_ERR_SHAPE;
    if (!params || !grads || !exp_avg || !exp_avg_sq) return ACMIL_ERR_NULL;
    const unsigned blocks = (unsigned)((n + 255) / 256 < 2048 ? (n + 255) / 256 : 2048);
    hipLaunchKernelGGL(adamw_flat_kernel, dim3(blocks), dim3(256), 0, (hipStream_t)stream, params, grads, exp_avg, exp_avg_sq, n, lr,
                       beta1, beta2, eps, weight_decay, step, skip_flag, skipped, flag_report);
    return hipGetLastError() == hipSuccess ? ACMIL_OK : ACMIL_ERR_LAUNCH;
}

extern "C" int acmil_adamw_step(float* params, const float* grads, float* exp_avg, float* exp_avg_sq, long long n, float lr,
                                double beta1, double beta2, float eps, float weight_decay, long long step, const float* skip_flag,
                                int* skipped, void* stream) {
    return acmil_adamw_step_report(params, grads, exp_avg, exp_avg_sq, n, lr, beta1, beta2, eps, weight_decay, step, skip_flag, skipped,
                                   nullptr, stream);
}

// ---------------------------------------------------------------------------------------------------
// The two element-wise passes around acmil_orthogonalize in an optimizer step over flat buffers: momentum in front, the step itself
// behind.  Both are bound by their bytes (12 + 4 and 8 + 4 per element); the matrices of a model are segments of the flat buffers,
// up to MUON_SEGS of them per launch, and an element finds its segment by bisection in the kernel arguments.
// ---------------------------------------------------------------------------------------------------
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
