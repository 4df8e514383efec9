// Fused AdamW step (decoupled weight decay) over a set of tensors.
//     m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;  p = (1 - lr wd) p - (lr / (1 - b1^t)) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// HBM-bound: 28 B per parameter (read p, g, m, v; write p, m, v): all of PSPNet-R50's, 1.44 GB, in 283 us = 5.1 TB/s, above what a copy reaches
// (4.7).  Up to 56 tensors travel as kernel arguments, so nothing is uploaded when gradients move from step to step (the host makes
// their descriptors anew: 0.88 instead of 0.13 ms of its time for those 187 tensors); a workgroup finds its tensor with one load and a ballot
// over the tensors' first workgroups.
#include "segmi_common.h"
#include <cmath>

namespace {

constexpr int MAX_GROUPS = 8;
constexpr int BATCH = 56;            // 56 B a tensor: with the hyper-parameters below the 4 KiB of kernel arguments
static_assert(BATCH <= 64, "a lane looks at a tensor");
constexpr int CHUNK = 4096;          // elements per workgroup: four 16-byte vectors per thread and stream

struct AdamTensor {
    float *p, *m, *v;
    const float* g;
    long count;
    unsigned first;
    int group;
    float lr1, rbc2;                 // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
};
// a group's numbers as the kernels use them, rounded once from 64 bits (1 - b2 and 1 - b2^t lose all their digits otherwise)
struct AdamHyper {
    float keep, b1, b2, eps, c1, c2;
    __host__ __device__ static AdamHyper from(const double* q) {      // lr, wd, b1, b2, eps
        return AdamHyper{(float)(1.0 - q[0] * q[1]), (float)q[2], (float)q[3], (float)q[4], (float)(1.0 - q[2]), (float)(1.0 - q[3])};
    }
};
struct AdamBatch {
    int count;
    AdamTensor t[BATCH];
    AdamHyper h[MAX_GROUPS];
};
static_assert(sizeof(AdamTensor) == 56 && sizeof(AdamBatch) + 2 * sizeof(void*) < 4096, "kernel arguments");

__device__ __forceinline__ float adam_one(float p, float g, float& m, float& v, const AdamHyper& h, float lr1, float rbc2) {
    m = fmaf(h.b1, m, h.c1 * g);
    v = fmaf(h.b2, v, h.c2 * g * g);
    return fmaf(h.keep, p, -lr1 * (m / fmaf(sqrtf(v), rbc2, h.eps)));
}

// coef: the two bias corrections per tensor from device memory (graphs), else from the arguments
__global__ __launch_bounds__(256) void adamw_kernel(AdamBatch b, const double* __restrict__ hd, const float2* __restrict__ coef) {
    const int lane = threadIdx.x & 63;
    const unsigned first = lane < b.count ? b.t[lane].first : 0xFFFFFFFFu;
    const int it = __builtin_amdgcn_readfirstlane((int)__popcll(__ballot(first <= blockIdx.x)) - 1);
    const AdamTensor t = b.t[it];
    const AdamHyper h = hd ? AdamHyper::from(hd + t.group * SEGMI_ADAMW_HYPER) : b.h[t.group];
    const float lr1 = coef ? coef[it].x : t.lr1, rbc2 = coef ? coef[it].y : t.rbc2;
    const long at = (long)(blockIdx.x - t.first) * CHUNK;
    const long n = t.count - at < CHUNK ? t.count - at : CHUNK;
    float* __restrict__ const p = t.p + at;
    float* __restrict__ const m = t.m + at;
    float* __restrict__ const v = t.v + at;
    const float* __restrict__ const g = t.g + at;
    const bool vec = ((((size_t)t.p | (size_t)t.m | (size_t)t.v | (size_t)t.g) & 15) == 0);
    const long n4 = vec ? n & ~3L : 0;
    for (long i = threadIdx.x * 4; i < n4; i += 1024) {
        float4 pv = ld4(p + i), mv = ld4(m + i), vv = ld4(v + i);
        const float4 gv = ld4(g + i);
        pv.x = adam_one(pv.x, gv.x, mv.x, vv.x, h, lr1, rbc2);
        pv.y = adam_one(pv.y, gv.y, mv.y, vv.y, h, lr1, rbc2);
        pv.z = adam_one(pv.z, gv.z, mv.z, vv.z, h, lr1, rbc2);
        pv.w = adam_one(pv.w, gv.w, mv.w, vv.w, h, lr1, rbc2);
        st4(p + i, pv);
        st4(m + i, mv);
        st4(v + i, vv);
    }
    for (long i = n4 + threadIdx.x; i < n; i += 256) {
        float mv = m[i], vv = v[i];
        p[i] = adam_one(p[i], g[i], mv, vv, h, lr1, rbc2);
        m[i] = mv;
        v[i] = vv;
    }
}

struct AdamSteps {
    int count;
    float* step[BATCH];
    int group[BATCH];
};

// graphs: every tensor's step number lives on the device; one launch advances all of them and leaves their bias corrections
__global__ void adamw_advance(AdamSteps s, const double* __restrict__ hd, float2* __restrict__ coef) {
    const int i = threadIdx.x;
    if (i >= s.count) return;
    const double* const q = hd + s.group[i] * SEGMI_ADAMW_HYPER;
    const float t = *s.step[i] + 1.f;
    *s.step[i] = t;
    coef[i] = make_float2((float)(q[0] / (1.0 - pow(q[2], (double)t))), (float)(1.0 / sqrt(1.0 - pow(q[3], (double)t))));
}

}  // namespace

extern "C" {

int segmi_adamw_step(const segmi_adamw_tensor* tensors_host, int count, const double* hyper_host, int ngroups, const double* hyper_dev,
                     void* workspace, size_t workspace_bytes, segmi_stream_t stream) {
    if (!tensors_host || count <= 0 || ngroups <= 0 || ngroups > MAX_GROUPS || (!hyper_dev && !hyper_host)) return SEGMI_ERR_BADARG;
    if (hyper_dev && (!workspace || workspace_bytes < (size_t)count * 8)) return SEGMI_ERR_WORKSPACE;
    for (int i = 0; i < count; ++i) {
        const segmi_adamw_tensor& a = tensors_host[i];
        if (!a.param || !a.grad || !a.exp_avg || !a.exp_avg_sq || a.count <= 0 || a.count > ((long)1 << 40) || a.group < 0 || a.group >= ngroups)
            return SEGMI_ERR_BADARG;
        if (hyper_dev ? !a.step_dev : !(a.step >= 1.0)) return SEGMI_ERR_BADARG;
    }
    for (int at = 0; at < count; at += BATCH) {
        AdamBatch b{};
        AdamSteps s{};
        b.count = s.count = count - at < BATCH ? count - at : BATCH;
        if (!hyper_dev)
            for (int i = 0; i < ngroups; ++i) b.h[i] = AdamHyper::from(hyper_host + i * SEGMI_ADAMW_HYPER);
        unsigned grid = 0;
        for (int i = 0; i < b.count; ++i) {
            const segmi_adamw_tensor& a = tensors_host[at + i];
            AdamTensor& t = b.t[i];
            t = AdamTensor{a.param, a.exp_avg, a.exp_avg_sq, a.grad, a.count, grid, a.group, 0.f, 0.f};
            if (!hyper_dev) {
                const double* const q = hyper_host + a.group * SEGMI_ADAMW_HYPER;
                t.lr1 = (float)(q[0] / (1.0 - std::pow(q[2], a.step)));
                t.rbc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(q[3], a.step)));
            }
            s.step[i] = a.step_dev;
            s.group[i] = a.group;
            grid += (unsigned)segmi_cdiv(a.count, CHUNK);
        }
        float2* const coef = hyper_dev ? static_cast<float2*>(workspace) + at : nullptr;
        if (hyper_dev) hipLaunchKernelGGL(adamw_advance, dim3(1), dim3(64), 0, (hipStream_t)stream, s, hyper_dev, coef);
        hipLaunchKernelGGL(adamw_kernel, dim3(grid), dim3(256), 0, (hipStream_t)stream, b, hyper_dev, coef);
    }
    return segmi_launch_status();
}

}  // extern "C"
