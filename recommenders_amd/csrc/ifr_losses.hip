// ifr_losses.hip -- what a factor model learns from: the preference loss on paired log ratios and the clipped policy loss with
// a KL term, each with its gradient in the same call (contracts: include/ifr.h).
#include <hip/hip_runtime.h>

#include "ifr_losses.h"

namespace ifr {

namespace {

dim3 grid_of_rows(int64_t n) { return dim3((uint32_t)(n < (1 << 22) ? n : (1 << 22))); }

__device__ __forceinline__ double wave_sum(double v)
{
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ int wave_sum(int v)
{
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// sum over the 256 threads, the same bits in every thread
template <typename T>
__device__ __forceinline__ T block_sum(T v, T *lds)
{
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

__device__ __forceinline__ float sigmoid(float x)
{
    const float e = expf(-fabsf(x));
    return (x >= 0.f ? 1.f : e) / (1.f + e);
}

// loss and its slope in h (a NaN in h stays one: fmaxf would drop it)
__device__ __forceinline__ void preference_of(const ifr_preference &p, float h, float *loss, float *slope)
{
    if (h != h) { *loss = h; *slope = h; return; }
    if (p.kind == IFR_PREFERENCE_LOGISTIC) {
        const float e = (float)p.label_smoothing;
        *loss = (1.f - e) * softplus(-h) + (e > 0.f ? e * softplus(h) : 0.f);
        *slope = e * sigmoid(h) - (1.f - e) * sigmoid(-h);
    } else if (p.kind == IFR_PREFERENCE_HINGE) {
        *loss = fmaxf(1.f - h, 0.f);
        *slope = h < 1.f ? -1.f : 0.f;
    } else {
        const float b = (float)p.beta, d = (h - 0.5f) / b;
        *loss = d * d;
        *slope = 2.f * d / b;
    }
}

}  // namespace

// One workgroup a pair: sums of both slates in 64 bits (without a reference the two sums are large and near each other), the
// loss, and the gradient, which is one number per slate.
__global__ __launch_bounds__(256) void preference_kernel(ifr_preference p)
{
    __shared__ double lds[4];
    __shared__ int ldsn[4];
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
        double sum[2];
        int count[2];
        for (int side = 0; side < 2; ++side) {
            const float *x = side ? p.rejected + row * p.ld_rejected : p.chosen + row * p.ld_chosen;
            const float *ref = side ? p.ref_rejected : p.ref_chosen;
            if (ref) ref += row * (side ? p.ld_ref_rejected : p.ld_ref_chosen);
            const uint8_t *mask = side ? p.mask_rejected : p.mask_chosen;
            if (mask) mask += row * (side ? p.ld_mask_rejected : p.ld_mask_chosen);
            const int len = side ? p.len_rejected : p.len_chosen;
            double s = 0.0;
            int c = 0;
            for (int t = threadIdx.x; t < len; t += 256) {
                if (mask && !mask[t]) continue;
                s += (double)x[t] - (ref ? (double)ref[t] : 0.0);
                ++c;
            }
            sum[side] = block_sum(s, lds);
            count[side] = p.average ? max(block_sum(c, ldsn), 1) : 1;
        }
        const float h = (float)(p.beta * (sum[0] / count[0] - sum[1] / count[1]) - p.margin);
        float loss, slope;
        preference_of(p, h, &loss, &slope);
        const float g = (p.weight ? p.weight[row] : 1.f) * slope * (float)p.beta;
        if (threadIdx.x == 0) {
            if (p.loss) p.loss[row] = loss;
            if (p.h) p.h[row] = h;
        }
        for (int side = 0; side < 2; ++side) {
            float *out = side ? p.d_rejected : p.d_chosen;
            if (!out) continue;
            out += row * (side ? p.ld_d_rejected : p.ld_d_chosen);
            const uint8_t *mask = side ? p.mask_rejected : p.mask_chosen;
            if (mask) mask += row * (side ? p.ld_mask_rejected : p.ld_mask_chosen);
            const int len = side ? p.len_rejected : p.len_chosen;
            const float v = (side ? -g : g) / (float)count[side];
            for (int t = threadIdx.x; t < len; t += 256) out[t] = mask && !mask[t] ? 0.f : v;
        }
    }
}

int launch_preference(const ifr_preference &p, hipStream_t s)
{
    hipLaunchKernelGGL(preference_kernel, grid_of_rows(p.n), dim3(256), 0, s, p);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// ---------------------------------------------------------------------------- policy

// exp(q) - q - 1: the series where the difference would cancel
__device__ __forceinline__ float kl_term(float q)
{
    if (fabsf(q) < 0.5f) {
        float s = 2.7557319e-7f;                      // 1 / 10!
        s = fmaf(s, q, 2.7557319e-6f);
        s = fmaf(s, q, 2.4801587e-5f);
        s = fmaf(s, q, 1.9841270e-4f);
        s = fmaf(s, q, 1.3888889e-3f);
        s = fmaf(s, q, 8.3333333e-3f);
        s = fmaf(s, q, 4.1666667e-2f);
        s = fmaf(s, q, 1.6666667e-1f);
        s = fmaf(s, q, 0.5f);
        return s * q * q;
    }
    return expm1f(q) - q;
}

enum { COUNT_BLOCKS = 1024 };

// masked elements of the batch, one partial count a workgroup (whole numbers: any order gives the same total)
__global__ __launch_bounds__(256) void policy_count_kernel(ifr_policy p, int64_t *part)
{
    __shared__ int lds[4];
    int64_t total = 0;
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
        const uint8_t *mask = p.mask + row * p.ld_mask;
        int c = 0;
        for (int t = threadIdx.x; t < p.len; t += 256) c += mask[t] != 0;
        total += block_sum(c, lds);
    }
    if (threadIdx.x == 0) part[blockIdx.x] = total;
}

__global__ __launch_bounds__(256) void policy_kernel(ifr_policy p, const int64_t *part, int n_part, float hi, float lo)
{
    __shared__ double lds[4];
    __shared__ int ldsn[4];
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
        const uint8_t *mask = p.mask ? p.mask + row * p.ld_mask : nullptr;
        int count = p.len;
        if (mask) {
            int c = 0;
            for (int t = threadIdx.x; t < p.len; t += 256) c += mask[t] != 0;
            count = block_sum(c, ldsn);
        }
        float scale = p.weight ? p.weight[row] : 1.f;
        if (p.reduction == IFR_POLICY_ROW) scale /= (float)max(count, 1);
        else if (p.reduction == IFR_POLICY_BATCH) {
            double all = 0.0;                             // counts below 2^53: exact
            if (part) {
                for (int i = threadIdx.x; i < n_part; i += 256) all += (double)part[i];
                all = block_sum(all, lds);
            } else {
                all = (double)p.n * p.len;
            }
            scale = (float)((double)scale / (all > 1.0 ? all : 1.0));
        }
        const float A = p.advantages[row], kl_coef = (float)p.kl_coef;
        const float most = (float)(1.0 + p.clip_high), least = (float)(1.0 - p.clip_low);
        const float *logp = p.logp + row * p.ld_logp, *old = p.old_logp + row * p.ld_old;
        const float *ref = p.ref_logp ? p.ref_logp + row * p.ld_ref : nullptr;
        float *out = p.d_logp ? p.d_logp + row * p.ld_d_logp : nullptr;
        double loss = 0.0, kl = 0.0;
        int clipped = 0;
        for (int t = threadIdx.x; t < p.len; t += 256) {
            float g = 0.f;
            if (!mask || mask[t]) {
                const float d = logp[t] - old[t];
                const bool over = A > 0.f && d > hi, under = A < 0.f && d < lo;
                float term;
                if (over || under) {
                    term = -A * (over ? most : least);
                    ++clipped;
                } else {
                    g = -A * expf(d);
                    term = g;
                }
                if (ref) {
                    const float q = ref[t] - logp[t], m = kl_term(q);
                    kl += m;
                    term += kl_coef * m;
                    g -= kl_coef * expm1f(q);
                }
                loss += term;
                g *= scale;
            }
            if (out) out[t] = g;
        }
        loss = block_sum(loss, lds);
        if (threadIdx.x == 0 && p.loss) p.loss[row] = (float)(loss * scale);
        if (p.kl) {
            kl = block_sum(kl, lds);
            if (threadIdx.x == 0) p.kl[row] = (float)(kl / max(count, 1));
        }
        clipped = block_sum(clipped, ldsn);
        if (threadIdx.x == 0 && p.clipped) p.clipped[row] = clipped;
    }
}

size_t policy_workspace(const ifr_policy &p) { return p.mask && p.reduction == IFR_POLICY_BATCH ? sizeof(int64_t) * COUNT_BLOCKS : 0; }

int launch_policy(const ifr_policy &p, void *ws, hipStream_t s)
{
    int64_t *part = nullptr;
    int n_part = 0;
    if (policy_workspace(p)) {
        part = (int64_t *)ws;
        n_part = (int)(p.n < COUNT_BLOCKS ? p.n : COUNT_BLOCKS);
        hipLaunchKernelGGL(policy_count_kernel, dim3(n_part), dim3(256), 0, s, p, part);
    }
    // the clip borders as logarithms, rounded once: log p - log p_old is compared with them
    hipLaunchKernelGGL(policy_kernel, grid_of_rows(p.n), dim3(256), 0, s, p, part, n_part, (float)log1p(p.clip_high),
                       (float)log1p(-p.clip_low));
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace ifr
