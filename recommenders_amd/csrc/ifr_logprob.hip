// ifr_logprob.hip -- log-probabilities of items under the softmax over the whole catalogue, and their gradient.
//
//   z[u][i] = scale (x_u . v_i + b_i);  lse[u] = log sum_i exp z;  logp[u][j] = z[u][id_j] - lse[u]
//   dX = scale (T_x - G P V),  dV = scale (T_v - P^T (G X)),  db = scale (t_b - P^T G),   P = exp(z - lse),
// G[u] the sum of the user's upstream gradients and T_x, T_v, t_b the parts of the named items (sparse sums).
//
// Scores are not stored: forward and each of the two products of the gradient walk the catalogue (or the users) in tiles of 32
// rows, form a 32 x 32 block of scores on the matrix cores, and use it in registers.  One kernel serves the three: S, the rows
// that stay (32 a wave, in registers as the B operand), and T, the rows that stream past (the A operand).
// D[t][s] of a 32 x 32 block has its column s in lane % 32, so a lane owns one S row: running maximum and sum need no exchange
// between lanes, and the block of probabilities already is the B operand of the second product, whose contraction runs over t in
// the order the block's registers hold (t = 16 c + 8 (j / 4) + 4 (lane / 32) + j % 4 for element j of step c).
//
// Operands in 16 bits: bf16 as it is.  fp32 is split into two fp16 parts after scaling by a power of two that brings the largest
// magnitude to [2^14, 2^15): hi + lo keeps 22 bits of values near the maximum and an absolute step of 2^-39 of the maximum below,
// and three products (hi hi, hi lo, lo hi) leave out lo lo, at most 2^-24 of a term.  Three fp16 products at 16 times the
// rate of the fp32 matrix instruction cost a fifth of it.
#include <hip/hip_runtime.h>

#include <math.h>

#include "ifr_logprob.h"

namespace ifr {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v8i __attribute__((ext_vector_type(8)));

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr double LN2 = 0.6931471805599453;
constexpr int S_ROWS = 128;            // S rows of a workgroup: 4 waves of 32
constexpr int AMAX_BLOCKS = 256;
constexpr int64_t MAX_GRID = 1 << 22;  // workgroups of 256 in one launch (the grid counts work items in 32 bits)

int pad_factors(int k) { return k <= 64 ? 64 : k <= 128 ? 128 : k <= 192 ? 192 : 256; }
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__bf16 v) { return (float)v; }

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// exponent e with max * 2^e in [2^14, 2^15) from the partial maxima (bit patterns) of amax_kernel; 0 for an all-zero matrix
__device__ __forceinline__ int split_exponent(const uint32_t *part)
{
    uint32_t m = 0;
    for (int i = 0; i < AMAX_BLOCKS; i += 64) m = max(m, part[i + (threadIdx.x & 63)]);
    for (int o = 32; o; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    if (m == 0) return 0;
    // a subnormal maximum counts as 2^-126: it is scaled to at most 2^14, which is as exact
    const int e = m < 0x00800000u ? -126 : (int)(m >> 23) - 127;
    return 14 - e;
}

// v * 2^e for any e in [-113, 140]
__device__ __forceinline__ float scale_pow2(float v, int e) { return ldexpf(v, e); }

}  // namespace

// ---------------------------------------------------------------------------- preparation

// Largest finite magnitude of a matrix, one partial maximum a workgroup; `row_factor` multiplies each row (G x).
template <typename T>
__global__ __launch_bounds__(256) void amax_kernel(const T *src, int64_t rows, int k, int64_t ld, const float *row_factor, uint32_t *part)
{
    __shared__ uint32_t lds[4];
    uint32_t m = 0;
    const int lane = threadIdx.x & 63;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    for (int64_t r = wave; r < rows; r += (int64_t)AMAX_BLOCKS * 4) {
        const float f = row_factor ? row_factor[r] : 1.f;
        for (int c = lane; c < k; c += 64) {
            const uint32_t b = __float_as_uint(as_f32(src[r * ld + c]) * f) & 0x7fffffffu;
            if (b < 0x7f800000u) m = max(m, b);
        }
    }
    for (int o = 32; o; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
    if (lane == 0) lds[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.x] = max(max(lds[0], lds[1]), max(lds[2], lds[3]));
}

// A matrix in the order the matrix instructions read it, 32 rows a workgroup, zeros behind the last row and column:
//   f1 [tile][part][KP / 16][lane][8]: row lane % 32, columns 16 s + 8 (lane / 32) + 0..7                 (first product)
//   f2 [tile][part][KP / 32][2][lane][8]: column 32 kb + lane % 32, rows 16 c + 8 (j / 4) + 4 (lane / 32) + j % 4   (second)
template <typename T, int NS>
__global__ __launch_bounds__(256) void fragments_kernel(const T *src, int64_t rows, int k, int64_t ld, const float *row_factor,
                                                        const uint32_t *amax, int KP, uint4 *f1, uint4 *f2)
{
    extern __shared__ float tile[];                   // [32][KP + 1]
    const int W = KP + 1;
    const int64_t r0 = (int64_t)blockIdx.x * 32;
    const int e = NS == 2 ? split_exponent(amax) : 0;
    for (int i = threadIdx.x; i < 32 * KP; i += 256) {
        const int r = i / KP, c = i - r * KP;
        float v = 0.f;
        if (r0 + r < rows && c < k) {
            v = as_f32(src[(r0 + r) * ld + c]);
            if (row_factor) v *= row_factor[r0 + r];
            if (NS == 2) v = scale_pow2(v, e);
        }
        tile[r * W + c] = v;
    }
    __syncthreads();
    for (int which = 0; which < 2; ++which) {
        uint4 *f = which ? f2 : f1;
        if (!f) continue;
        const int per = KP / 16 * 64;                 // 16-byte pieces of one part of a tile
        for (int i = threadIdx.x; i < per; i += 256) {
            const int lane = i & 63, s = i >> 6, q = lane & 31, h = lane >> 5;
            float v[8];
            for (int j = 0; j < 8; ++j) {
                const int r = which ? 16 * (s & 1) + 8 * (j >> 2) + 4 * h + (j & 3) : q;
                const int c = which ? 32 * (s >> 1) + q : 16 * s + 8 * h + j;
                v[j] = tile[r * W + c];
            }
            if (NS == 1) {
                b8 o;
                for (int j = 0; j < 8; ++j) o[j] = (__bf16)v[j];
                f[(int64_t)blockIdx.x * per + i] = __builtin_bit_cast(uint4, o);
            } else {
                h8 hi, lo;
                for (int j = 0; j < 8; ++j) {
                    hi[j] = (_Float16)v[j];
                    lo[j] = (_Float16)(v[j] - (float)hi[j]);
                }
                f[((int64_t)blockIdx.x * 2) * per + i] = __builtin_bit_cast(uint4, hi);
                f[((int64_t)blockIdx.x * 2 + 1) * per + i] = __builtin_bit_cast(uint4, lo);
            }
        }
    }
}

// Per-row terms in powers of two: the item side scale log2(e) b_i, the user side -log2(e) lse_u; -inf behind the last row.
__global__ __launch_bounds__(256) void item_terms_kernel(const float *ibase, int64_t n, int64_t padded, float c, float *out)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < padded) out[i] = i < n ? (ibase ? ibase[i] * c : 0.f) : -INFINITY;
}

// ... and G, the sum of a user's upstream gradients over the places that hold an item (in place order)
__global__ __launch_bounds__(256) void user_terms_kernel(const float *lse, const int32_t *ids, int64_t m, int64_t ld_ids, const float *dlogp,
                                                         int64_t ld_dlogp, int64_t n, int64_t padded, float *term, float *G)
{
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= padded) return;
    float t = -INFINITY, g = 0.f;
    if (u < n) {
        t = lse[u] == -INFINITY ? -INFINITY : -lse[u] * LOG2E;      // no probabilities: every exponential is 0
        for (int64_t j = 0; j < m; ++j)
            if (ids[u * ld_ids + j] >= 0) g += dlogp[u * ld_dlogp + j];
    }
    term[u] = t;
    G[u] = g;
}

// ---------------------------------------------------------------------------- the walk

enum { WALK_STATS = 0, WALK_GRAD = 1 };

struct WalkParams {
    const uint4 *s_f1, *t_f1, *t_f2;
    const float *s_term, *t_term;      // powers of two added to the score (see item_terms_kernel, user_terms_kernel)
    const float *t_factor;             // WALK_GRAD: sum_t factor P -> out_b, or null
    const uint32_t *s_amax, *t_amax;   // split operands: their exponents
    float c;                           // scale log2(e)
    int t_tiles, tiles_per_split;
    int64_t s_padded;
    float *out_m, *out_s;              // WALK_STATS: [splits][s_padded]
    float *out_acc;                    // WALK_GRAD: [splits][s_padded][KP]
    float *out_b;                      // ... [splits][s_padded]
};

template <int NS>
__device__ __forceinline__ v16f product(uint4 a, uint4 b, v16f d)
{
    if (NS == 1) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), d, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), d, 0, 0, 0);
}

template <int KP, int NS, int MODE>
__global__ __launch_bounds__(256, KP * NS <= 256 ? 2 : 1) void walk_kernel(WalkParams p)
{
    constexpr int STEPS = KP / 16;
    constexpr int PART = STEPS * 64;                  // 16-byte pieces of a part of a tile
    constexpr int TILE = PART * NS * (MODE == WALK_GRAD ? 2 : 1);
    __shared__ uint4 lds[TILE];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int64_t s_tile = (int64_t)blockIdx.x * 4 + wave;
    const int64_t s_row = s_tile * 32 + (lane & 31);

    uint4 sf[NS][STEPS];
    for (int q = 0; q < NS; ++q)
        for (int s = 0; s < STEPS; ++s) sf[q][s] = p.s_f1[(s_tile * NS + q) * PART + s * 64 + lane];
    float c = p.c;
    if (NS == 2) c = fminf(ldexpf(c, -split_exponent(p.s_amax) - split_exponent(p.t_amax)), 3.402823466e38f);
    // split probabilities sit at 2^15: fp16 then holds them down to 2^-39 of 1
    const float s_term = (p.s_term ? p.s_term[s_row] : 0.f) + (MODE == WALK_GRAD && NS == 2 ? 15.f : 0.f);

    v16f acc[MODE == WALK_GRAD ? KP / 32 : 1] = {};
    float m = -3.402823466e38f, sum = 0.f, b_sum = 0.f;

    const int first = blockIdx.y * p.tiles_per_split, last = min(first + p.tiles_per_split, p.t_tiles);
    for (int t = first; t < last; ++t) {
        __syncthreads();
        for (int i = threadIdx.x; i < PART * NS; i += 256) lds[i] = p.t_f1[(int64_t)t * PART * NS + i];
        if (MODE == WALK_GRAD)
            for (int i = threadIdx.x; i < PART * NS; i += 256) lds[PART * NS + i] = p.t_f2[(int64_t)t * PART * NS + i];
        __syncthreads();
        v16f d = {};
        for (int s = 0; s < STEPS; ++s) {
            const uint4 a = lds[s * 64 + lane];
            d = product<NS>(a, sf[0][s], d);
            if (NS == 2) {
                d = product<NS>(a, sf[NS - 1][s], d);
                d = product<NS>(lds[PART + s * 64 + lane], sf[0][s], d);
            }
        }
        float z[16];
        for (int q = 0; q < 4; ++q) {
            const float4 tt = *(const float4 *)(p.t_term + (int64_t)t * 32 + 8 * q + 4 * h);
            z[4 * q] = fmaf(d[4 * q], c, tt.x); z[4 * q + 1] = fmaf(d[4 * q + 1], c, tt.y);
            z[4 * q + 2] = fmaf(d[4 * q + 2], c, tt.z); z[4 * q + 3] = fmaf(d[4 * q + 3], c, tt.w);
        }
        if (MODE == WALK_STATS) {
            float top = m;
            for (int r = 0; r < 16; ++r) top = fmaxf(top, z[r]);
            float add = 0.f;
            for (int r = 0; r < 16; ++r) add += exp2_raw(z[r] - top);
            sum = fmaf(sum, exp2_raw(m - top), add);
            m = top;
        } else {
            float P[16];
            for (int r = 0; r < 16; ++r) P[r] = exp2_raw(z[r] + s_term);
            if (p.t_factor)
                for (int q = 0; q < 4; ++q) {
                    const float4 g = *(const float4 *)(p.t_factor + (int64_t)t * 32 + 8 * q + 4 * h);
                    b_sum = fmaf(P[4 * q], g.x, b_sum); b_sum = fmaf(P[4 * q + 1], g.y, b_sum);
                    b_sum = fmaf(P[4 * q + 2], g.z, b_sum); b_sum = fmaf(P[4 * q + 3], g.w, b_sum);
                }
            uint4 pf[NS][2];
            for (int e = 0; e < 2; ++e) {
                if (NS == 1) {
                    b8 o;
                    for (int j = 0; j < 8; ++j) o[j] = (__bf16)P[8 * e + j];
                    pf[0][e] = __builtin_bit_cast(uint4, o);
                } else {
                    h8 hi, lo;
                    for (int j = 0; j < 8; ++j) {
                        hi[j] = (_Float16)P[8 * e + j];
                        lo[j] = (_Float16)(P[8 * e + j] - (float)hi[j]);
                    }
                    pf[0][e] = __builtin_bit_cast(uint4, hi);
                    pf[NS - 1][e] = __builtin_bit_cast(uint4, lo);
                }
            }
            const uint4 *l2 = lds + PART * NS;
            for (int kb = 0; kb < KP / 32; ++kb)
                for (int e = 0; e < 2; ++e) {
                    const uint4 a = l2[(kb * 2 + e) * 64 + lane];
                    acc[kb] = product<NS>(a, pf[0][e], acc[kb]);
                    if (NS == 2) {
                        acc[kb] = product<NS>(a, pf[NS - 1][e], acc[kb]);
                        acc[kb] = product<NS>(l2[PART + (kb * 2 + e) * 64 + lane], pf[0][e], acc[kb]);
                    }
                }
        }
    }
    const int64_t at = (int64_t)blockIdx.y * p.s_padded + s_row;
    if (MODE == WALK_STATS) {
        // lane and lane + 32 hold the same S row
        const float m2 = __shfl_xor(m, 32), s2 = __shfl_xor(sum, 32), top = fmaxf(m, m2);
        sum = sum * exp2_raw(m - top) + s2 * exp2_raw(m2 - top);
        if (h == 0) { p.out_m[at] = top; p.out_s[at] = sum; }
    } else {
        float unit = 1.f;
        if (NS == 2) unit = ldexpf(1.f, -15);
        if (p.out_b) {
            b_sum += __shfl_xor(b_sum, 32);
            if (h == 0) p.out_b[at] = b_sum * unit;
        }
        for (int kb = 0; kb < KP / 32; ++kb)
            for (int q = 0; q < 4; ++q)
                *(float4 *)(p.out_acc + at * KP + kb * 32 + 8 * q + 4 * h) =
                    make_float4(acc[kb][4 * q] * unit, acc[kb][4 * q + 1] * unit, acc[kb][4 * q + 2] * unit, acc[kb][4 * q + 3] * unit);
    }
}

// The same statistics from 4-bit operands: a lane of the instruction reads one block of 32 and its scale from memory.
__global__ __launch_bounds__(256) void walk_mx_kernel(const uint8_t *xc, const uint8_t *xs, int64_t n, const uint8_t *vc, const uint8_t *vs, int64_t n_items,
                                                      int kb, const float *t_term, float c, int t_tiles, int tiles_per_split, int64_t s_padded,
                                                      float *out_m, float *out_s)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    const int64_t s_row = ((int64_t)blockIdx.x * 4 + wave) * 32 + (lane & 31);
    const int64_t u = min(s_row, n - 1);
    const int steps = (kb + 1) / 2;
    float m = -3.402823466e38f, sum = 0.f;
    const int first = blockIdx.y * tiles_per_split, last = min(first + tiles_per_split, t_tiles);
    for (int t = first; t < last; ++t) {
        const int64_t item = min((int64_t)t * 32 + (lane & 31), n_items - 1);
        v16f d = {};
        for (int s = 0; s < steps; ++s) {
            const int b = 2 * s + h;
            v8i a = {}, w = {};
            int sa = 127, sw = 127;
            if (b < kb) {
                const uint4 ca = *(const uint4 *)(vc + (item * kb + b) * 16), cw = *(const uint4 *)(xc + (u * kb + b) * 16);
                a[0] = ca.x; a[1] = ca.y; a[2] = ca.z; a[3] = ca.w;
                w[0] = cw.x; w[1] = cw.y; w[2] = cw.z; w[3] = cw.w;
                sa = vs[item * kb + b];
                sw = xs[u * kb + b];
            }
            d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, w, d, 4, 4, 0, sa, 0, sw);
        }
        float z[16], top = m;
        for (int q = 0; q < 4; ++q) {
            const float4 tt = *(const float4 *)(t_term + (int64_t)t * 32 + 8 * q + 4 * h);
            z[4 * q] = fmaf(d[4 * q], c, tt.x); z[4 * q + 1] = fmaf(d[4 * q + 1], c, tt.y);
            z[4 * q + 2] = fmaf(d[4 * q + 2], c, tt.z); z[4 * q + 3] = fmaf(d[4 * q + 3], c, tt.w);
        }
        for (int r = 0; r < 16; ++r) top = fmaxf(top, z[r]);
        float add = 0.f;
        for (int r = 0; r < 16; ++r) add += exp2_raw(z[r] - top);
        sum = fmaf(sum, exp2_raw(m - top), add);
        m = top;
    }
    const float m2 = __shfl_xor(m, 32), s2 = __shfl_xor(sum, 32), top = fmaxf(m, m2);
    sum = sum * exp2_raw(m - top) + s2 * exp2_raw(m2 - top);
    if (h == 0) { out_m[(int64_t)blockIdx.y * s_padded + s_row] = top; out_s[(int64_t)blockIdx.y * s_padded + s_row] = sum; }
}

// ---------------------------------------------------------------------------- joins

// lse from the splits' maxima and sums
__global__ __launch_bounds__(256) void join_lse_kernel(const float *m, const float *s, int splits, int64_t n, int64_t s_padded, float *lse)
{
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= n) return;
    float top = -3.402823466e38f, sum = 0.f;
    bool nan = false;
    for (int q = 0; q < splits; ++q) {
        const float b = s[q * s_padded + u];
        nan |= b != b;
        top = fmaxf(top, m[q * s_padded + u]);
    }
    for (int q = 0; q < splits; ++q) sum += s[q * s_padded + u] * exp2f(m[q * s_padded + u] - top);
    lse[u] = nan ? __uint_as_float(0x7fc00000u) : (float)(((double)top + (double)log2f(sum)) * LN2);
}

// logp of the named items: 16 lanes a place, the score as one fp32 sum over the factors
template <typename T>
__global__ __launch_bounds__(256) void targets_kernel(const T *X, int64_t ldx, const T *V, int64_t ldv, const float *ibase, int k, int64_t n_items, float scale,
                                                      const int32_t *ids, int64_t n, int64_t m, int64_t ld_ids, const float *lse, float *logp, int64_t ld_logp)
{
    const int l = threadIdx.x & 15;
    for (int64_t g = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4; g < n * m; g += (int64_t)gridDim.x * 16) {
        const int64_t u = g / m, j = g - u * m;
        const int32_t id = ids[u * ld_ids + j];
        float out = 0.f;
        if (id >= n_items) out = __uint_as_float(0x7fc00000u);
        else if (id >= 0) {
            float d = 0.f;
            for (int c = l; c < k; c += 16) d = fmaf(as_f32(X[u * ldx + c]), as_f32(V[id * ldv + c]), d);
            for (int o = 8; o; o >>= 1) d += __shfl_xor(d, o);
            const float z = scale * (d + (ibase ? ibase[id] : 0.f));
            const float l0 = lse[u];
            out = z == -INFINITY && l0 == -INFINITY ? z : z - l0;
        }
        if (l == 0) logp[u * ld_logp + j] = out;
    }
}

__device__ __forceinline__ float mx_unit(uint32_t byte)
{
    return byte == 255 ? __uint_as_float(0x7fc00000u) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// ... of a 4-bit model: 8 columns a lane and step
__global__ __launch_bounds__(256) void targets_mx_kernel(const uint8_t *xc, const uint8_t *xs, const uint8_t *vc, const uint8_t *vs, const float *ibase, int kb,
                                                         int64_t n_items, float scale, const int32_t *ids, int64_t n, int64_t m, int64_t ld_ids,
                                                         const float *lse, float *logp, int64_t ld_logp)
{
    const int l = threadIdx.x & 15;
    for (int64_t g = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4; g < n * m; g += (int64_t)gridDim.x * 16) {
        const int64_t u = g / m, j = g - u * m;
        const int32_t id = ids[u * ld_ids + j];
        float out = 0.f;
        if (id >= n_items) out = __uint_as_float(0x7fc00000u);
        else if (id >= 0) {
            float d = 0.f;
            for (int c = l; c < kb * 4; c += 16) {
                const uint32_t a = ((const uint32_t *)xc)[u * kb * 4 + c], b = ((const uint32_t *)vc)[(int64_t)id * kb * 4 + c];
                const v2f a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 1.0f, 0), b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 0);
                const v2f a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 1.0f, 1), b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 1);
                const v2f a2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 1.0f, 2), b2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 2);
                const v2f a3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 1.0f, 3), b3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 3);
                // sums of products of the grid are exact; the scales are powers of two
                const float e = a0[0] * b0[0] + a0[1] * b0[1] + a1[0] * b1[0] + a1[1] * b1[1] + a2[0] * b2[0] + a2[1] * b2[1] + a3[0] * b3[0] + a3[1] * b3[1];
                d += e * mx_unit(xs[u * kb + (c >> 2)]) * mx_unit(vs[(int64_t)id * kb + (c >> 2)]);
            }
            for (int o = 8; o; o >>= 1) d += __shfl_xor(d, o);
            const float z = scale * (d + (ibase ? ibase[id] : 0.f));
            const float l0 = lse[u];
            out = z == -INFINITY && l0 == -INFINITY ? z : z - l0;
        }
        if (l == 0) logp[u * ld_logp + j] = out;
    }
}

// dX = scale (sum over the places of g v - G acc 2^-e): a wave a user
template <typename T>
__global__ __launch_bounds__(256) void join_dx_kernel(const float *acc, int splits, int64_t s_padded, int KP, const uint32_t *v_amax, const float *G,
                                                      const T *V, int64_t ldv, int64_t n_items, int k, float scale, const int32_t *ids, int64_t m,
                                                      int64_t ld_ids, const float *dlogp, int64_t ld_dlogp, int64_t n, T *dX, int64_t ld_dx)
{
    const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int e = v_amax ? split_exponent(v_amax) : 0;
    if (u >= n) return;
    for (int c = lane; c < k; c += 64) {
        float a = 0.f;
        for (int q = 0; q < splits; ++q) a += acc[((int64_t)q * s_padded + u) * KP + c];
        float r = -G[u] * ldexpf(a, -e);
        for (int64_t j = 0; j < m; ++j) {
            const int32_t id = ids[u * ld_ids + j];
            if (id >= 0 && id < n_items) r = fmaf(dlogp[u * ld_dlogp + j], as_f32(V[id * ldv + c]), r);
        }
        dX[u * ld_dx + c] = (T)(scale * r);
    }
}

// dV = scale (sum over the places that name the item of g x - acc 2^-e), db likewise: 32 items a workgroup.  The workgroup scans
// all places in order and keeps those that name one of its items; each column of an item is summed by one thread in that order,
// so no sum depends on scheduling.
constexpr int JOIN_ITEMS = 32, JOIN_LIST = 1024;

template <typename T>
__global__ __launch_bounds__(256) void join_dv_kernel(const float *acc, const float *acc_b, int splits, int64_t s_padded, int KP, const uint32_t *x_amax,
                                                      const T *X, int64_t ldx, int64_t n_items, int k, float scale, const int32_t *ids, int64_t n, int64_t m,
                                                      int64_t ld_ids, const float *dlogp, int64_t ld_dlogp, T *dV, int64_t ld_dv, float *db)
{
    extern __shared__ float tile[];                   // [32][KP], then [32] for db
    __shared__ int list_at[JOIN_LIST];                // item of the tile in the low 5 bits, place above ... row kept apart
    __shared__ int list_row[JOIN_LIST];
    __shared__ float list_g[JOIN_LIST];
    __shared__ int wave_hits[4];
    const int64_t i0 = (int64_t)blockIdx.x * JOIN_ITEMS;
    const int e = x_amax ? split_exponent(x_amax) : 0;
    float *tile_b = tile + JOIN_ITEMS * KP;
    for (int i = threadIdx.x; i < JOIN_ITEMS * KP + JOIN_ITEMS; i += 256) tile[i] = 0.f;
    __syncthreads();
    const int64_t places = n * m;
    const int groups = 256 / KP > 0 ? 256 / KP : 1;
    const int col = threadIdx.x % KP, group = threadIdx.x / KP;
    int held = 0;
    for (int64_t b = 0; b < places || held; b += 256) {
        bool hit = false;
        int local = 0, row = 0;
        float g = 0.f;
        if (b < places) {
            const int64_t at = b + threadIdx.x;
            if (at < places) {
                const int64_t u = at / m, j = at - u * m;
                const int64_t id = (int64_t)ids[u * ld_ids + j] - i0;
                hit = id >= 0 && id < JOIN_ITEMS && i0 + id < n_items;
                if (hit) { local = (int)id; row = (int)u; g = dlogp[u * ld_dlogp + j]; }
            }
        }
        const unsigned long long votes = __ballot(hit);
        if ((threadIdx.x & 63) == 0) wave_hits[threadIdx.x >> 6] = __popcll(votes);
        __syncthreads();
        int at = held;
        for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) at += wave_hits[w];
        at += __popcll(votes & ((1ull << (threadIdx.x & 63)) - 1));
        if (hit) { list_at[at] = local; list_row[at] = row; list_g[at] = g; }
        held += wave_hits[0] + wave_hits[1] + wave_hits[2] + wave_hits[3];
        __syncthreads();
        if (held > JOIN_LIST - 256 || b + 256 >= places) {
            if (group < groups) {
                for (int q = 0; q < held; ++q) {
                    const int li = list_at[q];
                    if (li % groups != group) continue;
                    if (col < k) tile[li * KP + col] = fmaf(list_g[q], as_f32(X[(int64_t)list_row[q] * ldx + col]), tile[li * KP + col]);
                    if (col == 0) tile_b[li] += list_g[q];
                }
            }
            held = 0;
            __syncthreads();
        }
    }
    __syncthreads();
    if (dV)
        for (int i = threadIdx.x; i < JOIN_ITEMS * k; i += 256) {
            const int li = i / k, c = i - li * k;
            if (i0 + li >= n_items) break;
            float a = 0.f;
            for (int q = 0; q < splits; ++q) a += acc[((int64_t)q * s_padded + i0 + li) * KP + c];
            dV[(i0 + li) * ld_dv + c] = (T)(scale * (tile[li * KP + c] - ldexpf(a, -e)));
        }
    if (db)
        for (int li = threadIdx.x; li < JOIN_ITEMS; li += 256) {
            if (i0 + li >= n_items) break;
            float a = 0.f;
            for (int q = 0; q < splits; ++q) a += acc_b[(int64_t)q * s_padded + i0 + li];
            db[i0 + li] = scale * (tile_b[li] - a);
        }
}

// ---------------------------------------------------------------------------- launches

namespace {

// a workspace as a row of aligned pieces; with base null it only counts
struct Pieces {
    char *base;
    size_t used = 0;
    template <typename T>
    T *take(int64_t count)
    {
        if (!count) return nullptr;
        T *p = base ? (T *)(base + used) : nullptr;
        used += (size_t)up((int64_t)sizeof(T) * count, 256);
        return p;
    }
};

// splits of the T axis: enough workgroups for the chip, none shorter than 4 tiles
int split_count(int64_t s_blocks, int64_t t_tiles)
{
    const int64_t want = (1024 + s_blocks - 1) / s_blocks;
    const int64_t most = t_tiles / 4 > 0 ? t_tiles / 4 : 1;
    const int64_t n = want < most ? want : most;
    const int64_t per = (t_tiles + n - 1) / n;
    return (int)((t_tiles + per - 1) / per);
}

struct Side {                          // one matrix in fragment order
    int64_t rows, tiles, padded;       // tiles of 32 rows; padded: rows up to whole S blocks
    uint32_t *amax;
    uint4 *f1, *f2;
};

Side side(Pieces &w, int64_t rows, int KP, int NS, bool want1, bool want2)
{
    Side s;
    s.rows = rows;
    s.padded = up(rows, S_ROWS);
    s.tiles = s.padded / 32;
    s.amax = w.take<uint32_t>(NS == 2 ? AMAX_BLOCKS : 0);
    const int64_t n = s.tiles * NS * (KP / 16) * 64;
    s.f1 = want1 ? w.take<uint4>(n) : nullptr;
    s.f2 = want2 ? w.take<uint4>(n) : nullptr;
    return s;
}

template <typename T>
void fill_side(const Side &d, const T *src, int k, int64_t ld, const float *row_factor, int KP, hipStream_t s)
{
    constexpr int NS = sizeof(T) == 4 ? 2 : 1;
    if (NS == 2) hipLaunchKernelGGL((amax_kernel<T>), dim3(AMAX_BLOCKS), dim3(256), 0, s, src, d.rows, k, ld, row_factor, d.amax);
    hipLaunchKernelGGL((fragments_kernel<T, NS>), dim3((uint32_t)d.tiles), dim3(256), 32 * (KP + 1) * sizeof(float), s, src, d.rows, k, ld, row_factor,
                       d.amax, KP, d.f1, d.f2);
}

template <int NS, int MODE>
void launch_walk(const WalkParams &p, int KP, dim3 grid, hipStream_t s)
{
    if (KP == 64) hipLaunchKernelGGL((walk_kernel<64, NS, MODE>), grid, dim3(256), 0, s, p);
    else if (KP == 128) hipLaunchKernelGGL((walk_kernel<128, NS, MODE>), grid, dim3(256), 0, s, p);
    else if (KP == 192) hipLaunchKernelGGL((walk_kernel<192, NS, MODE>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((walk_kernel<256, NS, MODE>), grid, dim3(256), 0, s, p);
}

struct ForwardPlan {
    Side x, v;
    float *term, *lse, *out_m, *out_s;
    int splits, per;
    int64_t s_padded, t_tiles;
};

ForwardPlan forward_plan(Pieces &w, const ifr_catalogue &c)
{
    ForwardPlan p = {};
    const int KP = pad_factors(c.k), NS = c.dtype == IFR_F32 ? 2 : 1;
    p.s_padded = up(c.n, S_ROWS);
    p.t_tiles = (c.n_items + 31) / 32;
    if (c.dtype != IFR_MXFP4) {
        p.x = side(w, c.n, KP, NS, true, false);
        p.v = side(w, c.n_items, KP, NS, true, false);
    }
    p.splits = split_count(p.s_padded / S_ROWS, p.t_tiles);
    p.per = (int)((p.t_tiles + p.splits - 1) / p.splits);
    p.term = w.take<float>(p.t_tiles * 32);
    p.lse = w.take<float>(c.n);
    p.out_m = w.take<float>(p.splits * p.s_padded);
    p.out_s = w.take<float>(p.splits * p.s_padded);
    return p;
}

struct BackwardPlan {
    Side x, v, xg;                     // xg: rows times G, second product of dV
    float *item_term, *user_term, *G, *acc, *acc_b;
    int splits_x, per_x, splits_v, per_v;
};

BackwardPlan backward_plan(Pieces &w, const ifr_catalogue &c, bool dx, bool dv, bool db)
{
    BackwardPlan p = {};
    const int KP = pad_factors(c.k), NS = c.dtype == IFR_F32 ? 2 : 1;
    p.x = side(w, c.n, KP, NS, true, false);
    p.v = side(w, c.n_items, KP, NS, true, dx);
    p.xg = side(w, c.n, KP, NS, false, dv || db);
    p.item_term = w.take<float>(p.v.padded);
    p.user_term = w.take<float>(p.x.padded);
    p.G = w.take<float>(p.x.padded);
    const int64_t tv = (c.n_items + 31) / 32, tx = (c.n + 31) / 32;
    p.splits_x = split_count(p.x.padded / S_ROWS, tv);
    p.per_x = (int)((tv + p.splits_x - 1) / p.splits_x);
    p.splits_v = split_count(p.v.padded / S_ROWS, tx);
    p.per_v = (int)((tx + p.splits_v - 1) / p.splits_v);
    const int64_t ax = dx ? p.splits_x * p.x.padded * KP : 0, av = dv || db ? p.splits_v * p.v.padded * KP : 0;
    p.acc = w.take<float>(ax > av ? ax : av);         // dX is joined before dV is begun
    p.acc_b = w.take<float>(db ? p.splits_v * p.v.padded : 0);
    return p;
}

}  // namespace

size_t logprob_workspace(const ifr_catalogue &c)
{
    Pieces w{nullptr};
    forward_plan(w, c);
    return w.used;
}

size_t logprob_backward_workspace(const ifr_catalogue &c, bool want_dx, bool want_dv, bool want_db)
{
    Pieces w{nullptr};
    backward_plan(w, c, want_dx, want_dv, want_db);
    return w.used;
}

template <typename T>
static void forward_typed(const ifr_catalogue &c, const ForwardPlan &p, hipStream_t s)
{
    constexpr int NS = sizeof(T) == 4 ? 2 : 1;
    const int KP = pad_factors(c.k);
    fill_side<T>(p.x, (const T *)c.X, c.k, c.ldx, nullptr, KP, s);
    fill_side<T>(p.v, (const T *)c.V, c.k, c.ldv, nullptr, KP, s);
    WalkParams w = {};
    w.s_f1 = p.x.f1; w.t_f1 = p.v.f1; w.t_term = p.term; w.s_amax = p.x.amax; w.t_amax = p.v.amax;
    w.c = (float)(c.scale / LN2); w.t_tiles = (int)p.t_tiles; w.tiles_per_split = p.per; w.s_padded = p.s_padded;
    w.out_m = p.out_m; w.out_s = p.out_s;
    launch_walk<NS, WALK_STATS>(w, KP, dim3((uint32_t)(p.s_padded / S_ROWS), p.splits), s);
}

int launch_logprob(const ifr_catalogue &c, const int32_t *ids, int64_t m, int64_t ld_ids, float *logp, int64_t ld_logp, float *lse,
                   void *ws, hipStream_t s)
{
    Pieces w{(char *)ws};
    const ForwardPlan p = forward_plan(w, c);
    const float cc = (float)(c.scale / LN2);
    hipLaunchKernelGGL(item_terms_kernel, dim3((uint32_t)((p.t_tiles * 32 + 255) / 256)), dim3(256), 0, s, c.ibase, c.n_items, p.t_tiles * 32, cc, p.term);
    const int kb = (c.k + 31) / 32;
    if (c.dtype == IFR_MXFP4)
        hipLaunchKernelGGL(walk_mx_kernel, dim3((uint32_t)(p.s_padded / S_ROWS), p.splits), dim3(256), 0, s, (const uint8_t *)c.X, c.x_scales, c.n,
                           (const uint8_t *)c.V, c.v_scales, c.n_items, kb, p.term, cc, (int)p.t_tiles, p.per, p.s_padded, p.out_m, p.out_s);
    else if (c.dtype == IFR_F32) forward_typed<float>(c, p, s);
    else forward_typed<__bf16>(c, p, s);
    float *l = lse ? lse : p.lse;
    hipLaunchKernelGGL(join_lse_kernel, dim3((uint32_t)((c.n + 255) / 256)), dim3(256), 0, s, p.out_m, p.out_s, p.splits, c.n, p.s_padded, l);
    if (m > 0) {
        const int64_t want = (c.n * m + 15) / 16;
        const dim3 grid((uint32_t)(want < MAX_GRID ? want : MAX_GRID));
        const float sc = (float)c.scale;
        if (c.dtype == IFR_MXFP4)
            hipLaunchKernelGGL(targets_mx_kernel, grid, dim3(256), 0, s, (const uint8_t *)c.X, c.x_scales, (const uint8_t *)c.V, c.v_scales, c.ibase, kb,
                               c.n_items, sc, ids, c.n, m, ld_ids, l, logp, ld_logp);
        else if (c.dtype == IFR_F32)
            hipLaunchKernelGGL((targets_kernel<float>), grid, dim3(256), 0, s, (const float *)c.X, c.ldx, (const float *)c.V, c.ldv, c.ibase, c.k, c.n_items, sc,
                               ids, c.n, m, ld_ids, l, logp, ld_logp);
        else
            hipLaunchKernelGGL((targets_kernel<__bf16>), grid, dim3(256), 0, s, (const __bf16 *)c.X, c.ldx, (const __bf16 *)c.V, c.ldv, c.ibase, c.k, c.n_items,
                               sc, ids, c.n, m, ld_ids, l, logp, ld_logp);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <typename T>
static void backward_typed(const ifr_catalogue &c, const int32_t *ids, int64_t m, int64_t ld_ids, const LogprobGrad &g, const BackwardPlan &p, hipStream_t s)
{
    constexpr int NS = sizeof(T) == 4 ? 2 : 1;
    const int KP = pad_factors(c.k);
    const float cc = (float)(c.scale / LN2), sc = (float)c.scale;
    const T *X = (const T *)c.X, *V = (const T *)c.V;
    hipLaunchKernelGGL(item_terms_kernel, dim3((uint32_t)((p.v.padded + 255) / 256)), dim3(256), 0, s, c.ibase, c.n_items, p.v.padded, cc, p.item_term);
    hipLaunchKernelGGL(user_terms_kernel, dim3((uint32_t)((p.x.padded + 255) / 256)), dim3(256), 0, s, g.lse, ids, m, ld_ids, g.dlogp, g.ld_dlogp, c.n,
                       p.x.padded, p.user_term, p.G);
    fill_side<T>(p.x, X, c.k, c.ldx, nullptr, KP, s);
    fill_side<T>(p.v, V, c.k, c.ldv, nullptr, KP, s);
    WalkParams w = {};
    w.c = cc;
    if (g.dX) {
        w.s_f1 = p.x.f1; w.t_f1 = p.v.f1; w.t_f2 = p.v.f2; w.s_term = p.user_term; w.t_term = p.item_term;
        w.s_amax = p.x.amax; w.t_amax = p.v.amax;
        w.t_tiles = (int)((c.n_items + 31) / 32); w.tiles_per_split = p.per_x; w.s_padded = p.x.padded; w.out_acc = p.acc;
        launch_walk<NS, WALK_GRAD>(w, KP, dim3((uint32_t)(p.x.padded / S_ROWS), p.splits_x), s);
        hipLaunchKernelGGL((join_dx_kernel<T>), dim3((uint32_t)((c.n + 3) / 4)), dim3(256), 0, s, p.acc, p.splits_x, p.x.padded, KP, p.v.amax, p.G, V, c.ldv,
                           c.n_items, c.k, sc, ids, m, ld_ids, g.dlogp, g.ld_dlogp, c.n, (T *)g.dX, g.ld_dx);
    }
    if (g.dV || g.dibase) {
        fill_side<T>(p.xg, X, c.k, c.ldx, p.G, KP, s);
        w.s_f1 = p.v.f1; w.t_f1 = p.x.f1; w.t_f2 = p.xg.f2; w.s_term = p.item_term; w.t_term = p.user_term;
        w.s_amax = p.v.amax; w.t_amax = p.x.amax; w.t_factor = g.dibase ? p.G : nullptr;
        w.t_tiles = (int)((c.n + 31) / 32); w.tiles_per_split = p.per_v; w.s_padded = p.v.padded; w.out_acc = p.acc; w.out_b = g.dibase ? p.acc_b : nullptr;
        launch_walk<NS, WALK_GRAD>(w, KP, dim3((uint32_t)(p.v.padded / S_ROWS), p.splits_v), s);
        hipLaunchKernelGGL((join_dv_kernel<T>), dim3((uint32_t)((c.n_items + JOIN_ITEMS - 1) / JOIN_ITEMS)), dim3(256), (JOIN_ITEMS * KP + JOIN_ITEMS) * sizeof(float), s,
                           p.acc, p.acc_b, p.splits_v, p.v.padded, KP, p.xg.amax, X, c.ldx, c.n_items, c.k, sc, ids, c.n, m, ld_ids, g.dlogp, g.ld_dlogp,
                           (T *)g.dV, g.ld_dv, g.dibase);
    }
}

int launch_logprob_backward(const ifr_catalogue &c, const int32_t *ids, int64_t m, int64_t ld_ids, const LogprobGrad &g, void *ws,
                            hipStream_t s)
{
    Pieces w{(char *)ws};
    const BackwardPlan p = backward_plan(w, c, g.dX != nullptr, g.dV != nullptr, g.dibase != nullptr);
    if (c.dtype == IFR_F32) backward_typed<float>(c, ids, m, ld_ids, g, p, s);
    else backward_typed<__bf16>(c, ids, m, ld_ids, g, p, s);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace ifr
