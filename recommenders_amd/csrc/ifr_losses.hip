// ifr_losses.hip -- what a factor model learns from: the preference loss on paired log ratios and the clipped policy loss with
// a KL term, each with its gradient in the same call (contracts: include/ifr.h).
//
// Both are bound by memory: every element is read once, its gradient written once.  A row belongs to a group of 16, 64, 256 or 1024
// threads by its length (short rows would leave most of a workgroup idle), which takes it four elements a thread at a time.
#include <hip/hip_runtime.h>

#include "ifr_losses.h"

namespace ifr {

namespace {

constexpr int64_t MAX_GRID = 1 << 20;  // workgroups of one launch; rows beyond come round again

// sum over the GROUP threads of a row, the same bits in each of them (GROUP <= 64: lanes of one wave)
template <int GROUP, typename T>
__device__ __forceinline__ T group_sum(T v, T *lds)
{
    for (int o = (GROUP < 64 ? GROUP : 64) / 2; o; o >>= 1) v += __shfl_xor(v, o);
    if (GROUP <= 64) return v;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    T s = lds[0];
    for (int w = 1; w < GROUP / 64; ++w) s += lds[w];
    return s;
}

// Four neighbouring elements of rows of several arrays at once.  Where all rows begin at the same place modulo four elements, the
// pieces lie at 16-byte borders (the first and the last may be partial); otherwise, and at the ends, elements are taken one by one.
struct Pieces {
    int phase, len;                    // elements of the first piece before the row
    bool whole;                        // pieces may be taken at once
    __device__ int count() const { return (len + phase + 3) >> 2; }
    __device__ int at(int piece) const { return 4 * piece - phase; }
    __device__ bool full(int t) const { return whole && t >= 0 && t + 4 <= len; }
};

__device__ __forceinline__ int phase_of(const float *p) { return (int)(((uintptr_t)p >> 2) & 3); }
__device__ __forceinline__ int phase_of(const uint8_t *p) { return (int)((uintptr_t)p & 3); }

template <typename... P>
__device__ __forceinline__ Pieces pieces_of(int len, const float *first, P... others)
{
    Pieces r;
    r.len = len;
    const int f = phase_of(first);
    r.whole = ((others == nullptr || phase_of(others) == f) && ...);
    r.phase = r.whole ? f : 0;
    return r;
}

__device__ __forceinline__ void take(const Pieces &r, const float *row, int t, float v[4])
{
    if (r.full(t)) {
        const float4 a = *(const float4 *)(row + t);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
        for (int j = 0; j < 4; ++j) v[j] = t + j >= 0 && t + j < r.len ? row[t + j] : 0.f;
    }
}

// bit j: element j lies in the row and its mask (null: every place) is set
__device__ __forceinline__ uint32_t take_mask(const Pieces &r, const uint8_t *row, int t)
{
    if (r.full(t)) {
        if (!row) return 15u;
        const uint32_t w = *(const uint32_t *)(row + t);
        return (w & 0xffu ? 1u : 0u) | (w & 0xff00u ? 2u : 0u) | (w & 0xff0000u ? 4u : 0u) | (w & 0xff000000u ? 8u : 0u);
    }
    uint32_t m = 0;
    for (int j = 0; j < 4; ++j)
        if (t + j >= 0 && t + j < r.len && (!row || row[t + j])) m |= 1u << j;
    return m;
}

__device__ __forceinline__ void put(const Pieces &r, float *row, int t, const float v[4])
{
    if (r.full(t)) {
        *(float4 *)(row + t) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
        for (int j = 0; j < 4; ++j)
            if (t + j >= 0 && t + j < r.len) row[t + j] = v[j];
    }
}

__device__ __forceinline__ float softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

__device__ __forceinline__ float sigmoid(float x)
{
    const float e = expf(-fabsf(x));
    return (x >= 0.f ? 1.f : e) / (1.f + e);
}

// loss, and slope times factor = its slope in h times beta (a NaN in h stays one: fmaxf would drop it).  Squared: the slope 2 (h - 1/2) / beta^2
// leaves fp32 where beta is far from 1, its product with beta does not
__device__ __forceinline__ void preference_of(const ifr_preference &p, float h, float *loss, float *slope, float *factor)
{
    *factor = (float)p.beta;
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
        *slope = 2.f * d;
        *factor = 1.f;
    }
}

}  // namespace

// A group of threads a pair (16 384 pairs of 500 + 1000 with masks and a reference, 319 MB: 77 us, 4.1 TB/s; 64 pairs of 10 + 10: 8 us under the
// profiler, all latency): the sums of both slates in 64 bits (without a reference the two are large and near each other), the loss, and
// the gradient, which is one number per slate.
template <int GROUP>
__global__ __launch_bounds__(GROUP < 256 ? 256 : GROUP) void preference_kernel(ifr_preference p)
{
    constexpr int BLOCK = GROUP < 256 ? 256 : GROUP, ROWS = BLOCK / GROUP;
    __shared__ double lds[16];
    __shared__ int ldsn[16];
    const int me = threadIdx.x % GROUP;
    for (int64_t first = (int64_t)blockIdx.x * ROWS; first < p.n; first += (int64_t)gridDim.x * ROWS) {
        const int64_t row = first + threadIdx.x / GROUP;
        if (row >= p.n) return;                       // groups within a wave or whole workgroups: nobody waits for this one
        double sum[2];
        int count[2];
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const float *x = side ? p.rejected + row * p.ld_rejected : p.chosen + row * p.ld_chosen;
            const float *ref = side ? p.ref_rejected : p.ref_chosen;
            if (ref) ref += row * (side ? p.ld_ref_rejected : p.ld_ref_chosen);
            const uint8_t *mask = side ? p.mask_rejected : p.mask_chosen;
            if (mask) mask += row * (side ? p.ld_mask_rejected : p.ld_mask_chosen);
            const Pieces r = pieces_of(side ? p.len_rejected : p.len_chosen, x, ref, mask);
            double s = 0.0;
            int c = 0;
#pragma unroll 2
            for (int q = me; q < r.count(); q += GROUP) {
                const int t = r.at(q);
                const uint32_t m = take_mask(r, mask, t);
                float a[4], b[4] = {0.f, 0.f, 0.f, 0.f};
                take(r, x, t, a);
                if (ref) take(r, ref, t, b);
                for (int j = 0; j < 4; ++j)
                    if (m >> j & 1) s += (double)a[j] - (double)b[j];
                c += __popc(m);
            }
            sum[side] = group_sum<GROUP>(s, lds);
            count[side] = p.average ? max(group_sum<GROUP>(c, ldsn), 1) : 1;
        }
        const float h = (float)(p.beta * (sum[0] / count[0] - sum[1] / count[1]) - p.margin);
        float loss, slope, factor;
        preference_of(p, h, &loss, &slope, &factor);
        const float g = (p.weight ? p.weight[row] : 1.f) * slope * factor;
        if (me == 0) {
            if (p.loss) p.loss[row] = loss;
            if (p.h) p.h[row] = h;
        }
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            float *out = side ? p.d_rejected : p.d_chosen;
            if (!out) continue;
            out += row * (side ? p.ld_d_rejected : p.ld_d_chosen);
            const uint8_t *mask = side ? p.mask_rejected : p.mask_chosen;
            if (mask) mask += row * (side ? p.ld_mask_rejected : p.ld_mask_chosen);
            const Pieces r = pieces_of(side ? p.len_rejected : p.len_chosen, out, mask);
            const float v = (side ? -g : g) / (float)count[side];
            for (int q = me; q < r.count(); q += GROUP) {
                const int t = r.at(q);
                const uint32_t m = take_mask(r, mask, t);
                const float o[4] = {m & 1 ? v : 0.f, m & 2 ? v : 0.f, m & 4 ? v : 0.f, m & 8 ? v : 0.f};
                put(r, out, t, o);
            }
        }
    }
}

namespace {

// Threads of a row, by what a launch takes in units of one trip to memory: rounds of the 8192 waves that the chip holds, times the trips
// that a row makes (four elements a thread each), six for what a row costs besides, three more where a workgroup has to meet.
// (16 384 pairs of 500 + 1000: 64 threads 82 us, 256 threads 107 us; 31 455 pairs of 35 + 122: 64 threads 61 us, 16 threads 33 us.)
int group_of(int64_t len, int64_t n)
{
    int best = 16;
    double least = 0;
    for (int g = 16; g <= 1024; g *= 4) {
        const double waves = (double)n * g / 64, rounds = waves <= 8192 ? 1 : waves / 8192;
        const double cost = rounds * ((double)((len + 4 * g - 1) / (4 * g)) + 6 + (g > 64 ? 3 : 0));
        if (g == 16 || cost < least) { best = g; least = cost; }
    }
    return best;
}

dim3 grid_of(int64_t n, int group)
{
    const int64_t rows = group < 256 ? 256 / group : 1, want = (n + rows - 1) / rows;
    return dim3((uint32_t)(want < MAX_GRID ? want : MAX_GRID));
}

}  // namespace

int launch_preference(const ifr_preference &p, hipStream_t s)
{
    const int group = group_of(p.len_chosen > p.len_rejected ? p.len_chosen : p.len_rejected, p.n);
    const dim3 grid = grid_of(p.n, group);
    if (group == 16) hipLaunchKernelGGL(preference_kernel<16>, grid, dim3(256), 0, s, p);
    else if (group == 64) hipLaunchKernelGGL(preference_kernel<64>, grid, dim3(256), 0, s, p);
    else if (group == 256) hipLaunchKernelGGL(preference_kernel<256>, grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL(preference_kernel<1024>, grid, dim3(1024), 0, s, p);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

// ---------------------------------------------------------------------------- policy

// exp(q) - 1 and exp(q) - 1 - q: below 1 by the series of the second, where the difference would cancel
__device__ __forceinline__ void exp_terms(float q, float *m1, float *kl)
{
    if (fabsf(q) < 1.f) {
        float s = 2.0876757e-9f;                      // 1 / 12!
        s = fmaf(s, q, 2.5052108e-8f);
        s = fmaf(s, q, 2.7557319e-7f);
        s = fmaf(s, q, 2.7557319e-6f);
        s = fmaf(s, q, 2.4801587e-5f);
        s = fmaf(s, q, 1.9841270e-4f);
        s = fmaf(s, q, 1.3888889e-3f);
        s = fmaf(s, q, 8.3333333e-3f);
        s = fmaf(s, q, 4.1666667e-2f);
        s = fmaf(s, q, 1.6666667e-1f);
        s = fmaf(s, q, 0.5f);
        *kl = s * q * q;
        *m1 = *kl + q;
    } else {
        *m1 = expm1f(q);
        *kl = *m1 - q;
    }
}

enum { COUNT_BLOCKS = 1024 };

__device__ __forceinline__ int set_bytes(uint32_t w) { return __popc((((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) & 0x80808080u); }

// places of the batch, one partial count a workgroup (whole numbers: any order gives the same total)
__global__ __launch_bounds__(256) void policy_count_kernel(ifr_policy p, int64_t *part)
{
    __shared__ int64_t lds[4];
    int64_t total = 0;
    const int64_t me = (int64_t)blockIdx.x * 256 + threadIdx.x, all = (int64_t)gridDim.x * 256;
    if (p.ld_mask == p.len || p.n == 1) {             // one row of bytes
        const int64_t bytes = p.n * p.len;
        const int64_t head = min((int64_t)((16 - ((uintptr_t)p.mask & 15)) & 15), bytes), body = (bytes - head) / 16;
        for (int64_t i = me; i < body; i += all) {
            const uint4 w = ((const uint4 *)(p.mask + head))[i];
            total += set_bytes(w.x) + set_bytes(w.y) + set_bytes(w.z) + set_bytes(w.w);
        }
        if (me < head) total += p.mask[me] != 0;
        if (me < bytes - head - body * 16) total += p.mask[head + body * 16 + me] != 0;
    } else {
        for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x)
            for (int t = threadIdx.x; t < p.len; t += 256) total += p.mask[row * p.ld_mask + t] != 0;
    }
    total = group_sum<256>(total, lds);
    if (threadIdx.x == 0) part[blockIdx.x] = total;
}

// A group of threads a row; the count of the row's places comes first where the scale needs it (the mask alone is read twice, from the caches).
// 4096 rows of 8191, 570 MB: 133 us, 4.3 TB/s, where a copy reaches 4.73; before it 7.5 us for the count of the batch's places.
template <int GROUP>
__global__ __launch_bounds__(GROUP < 256 ? 256 : GROUP) void policy_kernel(ifr_policy p, const int64_t *part, int n_part, float hi, float lo)
{
    constexpr int BLOCK = GROUP < 256 ? 256 : GROUP, ROWS = BLOCK / GROUP;
    __shared__ double lds[16];
    __shared__ int ldsn[16];
    __shared__ int64_t ldsl[16];
    const int me = threadIdx.x % GROUP;
    const float most = (float)(1.0 + p.clip_high), least = (float)(1.0 - p.clip_low), kl_coef = (float)p.kl_coef;
    double all = 1.0;
    if (p.reduction == IFR_POLICY_BATCH) {
        int64_t c = (int64_t)p.n * p.len;
        if (part) {
            c = 0;
            for (int i = threadIdx.x; i < n_part; i += BLOCK) c += part[i];
            c = group_sum<BLOCK>(c, ldsl);
        }
        all = c > 1 ? (double)c : 1.0;
    }
    for (int64_t first = (int64_t)blockIdx.x * ROWS; first < p.n; first += (int64_t)gridDim.x * ROWS) {
        const int64_t row = first + threadIdx.x / GROUP;
        if (row >= p.n) return;
        const uint8_t *mask = p.mask ? p.mask + row * p.ld_mask : nullptr;
        const float *logp = p.logp + row * p.ld_logp, *old = p.old_logp + row * p.ld_old;
        const float *ref = p.ref_logp ? p.ref_logp + row * p.ld_ref : nullptr;
        float *out = p.d_logp ? p.d_logp + row * p.ld_d_logp : nullptr;
        const Pieces r = pieces_of(p.len, logp, old, ref, (const float *)out, mask);
        const float weight = p.weight ? p.weight[row] : 1.f, A = p.advantages[row];
        int count = p.len;
        if (mask && p.reduction == IFR_POLICY_ROW) {
            int c = 0;
            for (int q = me; q < r.count(); q += GROUP) c += __popc(take_mask(r, mask, r.at(q)));
            count = group_sum<GROUP>(c, ldsn);
        }
        const float scale = p.reduction == IFR_POLICY_SUM ? weight : p.reduction == IFR_POLICY_ROW ? weight / (float)max(count, 1) : (float)(weight / all);
        double loss = 0.0, kl = 0.0;
        int clipped = 0, places = 0;
        for (int q = me; q < r.count(); q += GROUP) {
            const int t = r.at(q);
            const uint32_t m = take_mask(r, mask, t);
            float a[4], b[4], c[4], g[4];
            take(r, logp, t, a);
            take(r, old, t, b);
            if (ref) take(r, ref, t, c);
            float loss4 = 0.f, kl4 = 0.f;
            for (int j = 0; j < 4; ++j) {
                g[j] = 0.f;
                if (!(m >> j & 1)) continue;
                const float d = a[j] - b[j];
                const bool over = A > 0.f && d > hi, under = A < 0.f && d < lo;
                float term;
                if (over || under) {
                    term = -A * (over ? most : least);
                    ++clipped;
                } else {
                    g[j] = -A * expf(d);
                    term = g[j];
                }
                if (ref) {
                    float m1, k;
                    exp_terms(c[j] - a[j], &m1, &k);
                    kl4 += k;
                    term = fmaf(kl_coef, k, term);
                    g[j] -= kl_coef * m1;
                }
                loss4 += term;
                g[j] *= scale;
            }
            loss += loss4;
            kl += kl4;
            places += __popc(m);
            if (out) put(r, out, t, g);
        }
        loss = group_sum<GROUP>(loss, lds);
        if (me == 0 && p.loss) p.loss[row] = (float)(loss * scale);
        if (p.kl) {
            kl = group_sum<GROUP>(kl, lds);
            places = group_sum<GROUP>(places, ldsn);
            if (me == 0) p.kl[row] = (float)(kl / max(places, 1));
        }
        clipped = group_sum<GROUP>(clipped, ldsn);
        if (me == 0 && p.clipped) p.clipped[row] = clipped;
    }
}

size_t policy_workspace(const ifr_policy &p) { return p.mask && p.reduction == IFR_POLICY_BATCH ? sizeof(int64_t) * COUNT_BLOCKS : 0; }

int launch_policy(const ifr_policy &p, void *ws, hipStream_t s)
{
    int64_t *part = nullptr;
    int n_part = 0;
    if (policy_workspace(p)) {
        const int64_t want = (p.n * p.len + 4095) / 4096;
        part = (int64_t *)ws;
        n_part = (int)(want < 1 ? 1 : want < COUNT_BLOCKS ? want : COUNT_BLOCKS);
        hipLaunchKernelGGL(policy_count_kernel, dim3(n_part), dim3(256), 0, s, p, part);
    }
    // the clip borders as logarithms, rounded once: log p - log p_old is compared with them
    const float hi = (float)log1p(p.clip_high), lo = (float)log1p(-p.clip_low);
    const int group = group_of(p.len, p.n);
    const dim3 grid = grid_of(p.n, group);
    if (group == 16) hipLaunchKernelGGL(policy_kernel<16>, grid, dim3(256), 0, s, p, part, n_part, hi, lo);
    else if (group == 64) hipLaunchKernelGGL(policy_kernel<64>, grid, dim3(256), 0, s, p, part, n_part, hi, lo);
    else if (group == 256) hipLaunchKernelGGL(policy_kernel<256>, grid, dim3(256), 0, s, p, part, n_part, hi, lo);
    else hipLaunchKernelGGL(policy_kernel<1024>, grid, dim3(1024), 0, s, p, part, n_part, hi, lo);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace ifr
