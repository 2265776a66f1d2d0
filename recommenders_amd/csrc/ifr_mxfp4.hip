// ifr_mxfp4.hip -- a catalogue in 4-bit microscaled floating point: quantisation, its inverse and the product that yields
// score rows (layout: ifr_mxfp4.h).
#include <hip/hip_runtime.h>

#include "ifr_mxfp4.h"

namespace ifr {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

namespace {

__device__ __forceinline__ float load_f32(const float *p) { return *p; }
__device__ __forceinline__ float load_f32(const __bf16 *p) { return (float)*p; }

// 8 consecutive elements of a row, zeros behind its end
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *row, int64_t col, int64_t k, float v[8])
{
    if (VEC) {                                        // 16-byte aligned rows, k a multiple of 8
        if (col >= k) {
            for (int j = 0; j < 8; ++j) v[j] = 0.f;
        } else if (sizeof(T) == 4) {
            const float4 a = ((const float4 *)(row + col))[0], b = ((const float4 *)(row + col))[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 a = *(const uint4 *)(row + col);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    } else {
        for (int j = 0; j < 8; ++j) v[j] = col + j < k ? load_f32(row + col + j) : 0.f;
    }
}

}  // namespace

// One lane takes 8 columns of a row, four neighbouring lanes a block: e = floor(log2 max|v|) - 2 is the exponent field of the
// largest magnitude less 2 (subnormal maxima clamp to 2^-127), v / 2^e is exact, and the conversion rounds to the nearest of the
// grid, ties to the even code, at most 6 in magnitude.  HBM-bound: 4 bytes read and 17/32 written an
// element (1 000 000 x 128: 580 MB in 100 us, 5.8 TB/s, where a large copy reaches 4.73 and a fill 6.9).
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T *X, int64_t n, int64_t k, int64_t ld, int kb, uint8_t *codes, uint8_t *scales)
{
    const int64_t g = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = g / (kb * 4);
    const int c8 = (int)(g - row * (kb * 4));         // which 8 columns of the row
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (row < n) load8<T, VEC>(X + row * ld, (int64_t)c8 * 8, k, v);
    uint32_t top = 0;
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    top = max(top, (uint32_t)__shfl_xor((int)top, 1));
    top = max(top, (uint32_t)__shfl_xor((int)top, 2));
    if (row >= n) return;
    const uint32_t field = top >> 23;
    const uint32_t byte = field == 255 ? 255u : (field > 2 ? field - 2 : 0u);
    // 2^(127 - byte): byte <= 252, so the exponent field 254 - byte is at least 2
    const float inv = byte == 255 ? 0.f : __uint_as_float((254u - byte) << 23);
    uint32_t c = 0;
    if (byte != 255) {
        for (int j = 0; j < 8; ++j) v[j] = fminf(fmaxf(v[j] * inv, -6.f), 6.f);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], 1.0f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], 1.0f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], 1.0f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], 1.0f, 3);
    }
    ((uint32_t *)codes)[row * (kb * 4) + c8] = c;
    if ((c8 & 3) == 0) scales[row * kb + (c8 >> 2)] = (uint8_t)byte;
}

// 2^(byte - 127), NaN for 255 (2^-127 is the subnormal 0x400000)
__device__ __forceinline__ float mx_scale(uint32_t byte)
{
    return byte == 255 ? __uint_as_float(0x7fc00000u) : byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// A lane takes four columns, so that a wave stores 1024 bytes in one piece, past the caches: bound by that store (1 000 000 x 128: 580 MB in
// 101 us, 5.8 TB/s).  With eight columns a lane, two pieces of 16 bytes, the store past the
// caches was slower than the one through them, since neither of the two fills a line.
template <bool VEC>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t *codes, const uint8_t *scales, int64_t n, int64_t k, int kb, float *out, int64_t ld)
{
    const int64_t g = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = g / (kb * 8);
    const int c4 = (int)(g - row * (kb * 8));         // which 4 columns of the row
    if (row >= n || (int64_t)c4 * 4 >= k) return;
    const uint32_t c = ((const uint16_t *)codes)[row * (kb * 8) + c4];
    const float s = mx_scale(scales[row * kb + (c4 >> 3)]);
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    const f4 v = {a[0] * s, a[1] * s, b[0] * s, b[1] * s};
    float *o = out + row * ld + (int64_t)c4 * 4;
    if (VEC) {
        __builtin_nontemporal_store(v, (f4 *)o);
    } else {
        for (int j = 0; j < 4; ++j)
            if ((int64_t)c4 * 4 + j < k) o[j] = v[j];
    }
}

// ---------------------------------------------------------------------------- product

// what the lanes of a wave wrote to its strip may be read by the others (LDS serves a wave in order: only the compiler has to keep it)
__device__ __forceinline__ void strip_ready()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Score rows by v_mfma_scale_f32_32x32x64 with both operands in E2M1.  A lane of that instruction holds one block of 32 of one row and
// that block's scale, which is the layout in memory, so nothing is rearranged.  A wave keeps IT tiles of 32 items in registers (A
// operand) and walks query tiles of 32 (B operand): D[item][query], four neighbouring items of one query a lane and quad, which go
// through a strip of LDS of the wave's own so that rows are stored in long pieces.  Bound by the store of the scores for k <= 256: 1000 x
// 1 000 000 in bf16, 2.0 GB, 378 us = 5.3 TB/s, where filling as much reaches 6.9 (stores straight from the registers, 8 bytes of a row
// a lane: 792 us with the quantisation of X; strips through the caches 457, past them 380).
template <int STEPS, int IT, typename OUT>
__global__ __launch_bounds__(256, 2) void mx_scores_kernel(MxScoreParams p, int kb, int64_t q_tiles, int64_t q_per_block, int vec)
{
    constexpr int COLS = IT * 32, PITCH = COLS + 16 / sizeof(OUT);      // a row further by one 16-byte piece: fewer bank conflicts
    __shared__ __align__(16) OUT strips[4][32 * PITCH];
    __shared__ __align__(16) float bases[4][COLS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    OUT *strip = strips[wave];
    const int64_t i0 = ((int64_t)blockIdx.x * 4 + wave) * COLS;
    if (i0 >= p.v.n) return;                          // waves work alone: no barrier below
    v8i a[IT][STEPS];
    int sa[IT][STEPS];
    auto block_of = [&](const MxMatrix &m, int64_t row, int s, v8i *to, int *scale) {
        const int b = 2 * s + h;
        v8i v = {0};
        *scale = 127;
        if (b < kb) {
            const uint4 c = *(const uint4 *)(m.codes + (row * kb + b) * 16);
            v[0] = c.x; v[1] = c.y; v[2] = c.z; v[3] = c.w;
            *scale = m.scales[row * kb + b];
        }
        *to = v;
    };
#pragma unroll
    for (int t = 0; t < IT; ++t)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) block_of(p.v, min(i0 + t * 32 + r, p.v.n - 1), s, &a[t][s], &sa[t][s]);
    for (int c = lane; c < COLS; c += 64) bases[wave][c] = p.ibase && i0 + c < p.v.n ? p.ibase[i0 + c] : 0.f;
    const int64_t first = (int64_t)blockIdx.y * q_per_block, last = min(first + q_per_block, q_tiles);
    const int cols = (int)min((int64_t)COLS, p.v.n - i0);
    for (int64_t qt = first; qt < last; ++qt) {
        const int64_t q = min(qt * 32 + r, p.x.n - 1);
        v8i x[STEPS];
        int sx[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) block_of(p.x, q, s, &x[s], &sx[s]);
        const float ub = p.ubase ? p.ubase[q] : 0.f;
        strip_ready();
#pragma unroll
        for (int t = 0; t < IT; ++t) {
            v16f d = {0};
#pragma unroll
            for (int s = 0; s < STEPS; ++s) d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a[t][s], x[s], d, 4, 4, 0, sa[t][s], 0, sx[s]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4 b = *(const float4 *)&bases[wave][t * 32 + 8 * e + 4 * h];
                const float v0 = d[4 * e] + (b.x + ub), v1 = d[4 * e + 1] + (b.y + ub), v2 = d[4 * e + 2] + (b.z + ub), v3 = d[4 * e + 3] + (b.w + ub);
                OUT *to = strip + r * PITCH + t * 32 + 8 * e + 4 * h;
                to[0] = (OUT)v0; to[1] = (OUT)v1; to[2] = (OUT)v2; to[3] = (OUT)v3;
            }
        }
        strip_ready();
        OUT *out = (OUT *)p.out + qt * 32 * p.ld + i0;
        const int rows = (int)min((int64_t)32, p.x.n - qt * 32);
        if (vec && cols == COLS) {
            constexpr int PIECE = 16 / sizeof(OUT), ROW = COLS / PIECE;          // 16-byte pieces of a row
#pragma unroll
            for (int i = 0; i < 32 * ROW / 64; ++i) {
                const int at = i * 64 + lane, row = at / ROW, c = (at - row * ROW) * PIECE;
                if (row < rows) __builtin_nontemporal_store(*(const u4 *)(strip + row * PITCH + c), (u4 *)(out + row * p.ld + c));
            }
        } else {
            for (int row = 0; row < rows; ++row)
                for (int c = lane; c < cols; c += 64) out[row * p.ld + c] = strip[row * PITCH + c];
        }
    }
}

// ---------------------------------------------------------------------------- launches

namespace {
// the grid counts work items in 32 bits: more than 2^22 workgroups go into a second dimension
dim3 grid_of(int64_t blocks)
{
    const int64_t x = blocks < (1 << 22) ? blocks : (1 << 22);
    return dim3((uint32_t)x, (uint32_t)((blocks + x - 1) / x));
}

bool aligned16(const void *p, int64_t row_bytes) { return ((uintptr_t)p & 15) == 0 && row_bytes % 16 == 0; }
}  // namespace

int launch_mx_quantize(const void *X, int bf16, int64_t n, int64_t k, int64_t ld, uint8_t *codes, uint8_t *scales, hipStream_t s)
{
    const int kb = (int)((k + 31) / 32);
    const dim3 grid = grid_of((n * kb * 4 + 255) / 256);
    const bool vec = k % 8 == 0 && aligned16(X, ld * (bf16 ? 2 : 4));
    if (bf16) {
        if (vec) hipLaunchKernelGGL((mx_quantize_kernel<__bf16, true>), grid, dim3(256), 0, s, (const __bf16 *)X, n, k, ld, kb, codes, scales);
        else hipLaunchKernelGGL((mx_quantize_kernel<__bf16, false>), grid, dim3(256), 0, s, (const __bf16 *)X, n, k, ld, kb, codes, scales);
    } else {
        if (vec) hipLaunchKernelGGL((mx_quantize_kernel<float, true>), grid, dim3(256), 0, s, (const float *)X, n, k, ld, kb, codes, scales);
        else hipLaunchKernelGGL((mx_quantize_kernel<float, false>), grid, dim3(256), 0, s, (const float *)X, n, k, ld, kb, codes, scales);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int launch_mx_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t n, int64_t k, float *out, int64_t ld, hipStream_t s)
{
    const int kb = (int)((k + 31) / 32);
    const dim3 grid = grid_of((n * kb * 8 + 255) / 256);
    if (k % 4 == 0 && aligned16(out, ld * 4)) hipLaunchKernelGGL(mx_dequantize_kernel<true>, grid, dim3(256), 0, s, codes, scales, n, k, kb, out, ld);
    else hipLaunchKernelGGL(mx_dequantize_kernel<false>, grid, dim3(256), 0, s, codes, scales, n, k, kb, out, ld);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <int STEPS, typename OUT>
static void launch_mx_scores_typed(const MxScoreParams &p, int kb, hipStream_t s)
{
    const int64_t qt = (p.x.n + 31) / 32, it = (p.v.n + 31) / 32;
    const int vec = aligned16(p.out, p.ld * (int64_t)sizeof(OUT));
    // few scores: 32 items a wave fill the chip; many: 128 (bf16: 256), which read X as much less often and store rows of 512 bytes.  16 384
    // tiles are four for each wave that the chip holds
    const bool wide = it * qt >= 16384;
    constexpr int IT = sizeof(OUT) == 2 ? 8 : 4;
    const int64_t gx = wide ? (it + 4 * IT - 1) / (4 * IT) : (it + 3) / 4;
    int64_t gy = (4096 + gx - 1) / gx;
    gy = gy < qt ? gy : qt;
    const int64_t per = (qt + gy - 1) / gy;
    gy = (qt + per - 1) / per;
    const dim3 grid((uint32_t)gx, (uint32_t)gy);
    if (wide) hipLaunchKernelGGL((mx_scores_kernel<STEPS, IT, OUT>), grid, dim3(256), 0, s, p, kb, qt, per, vec);
    else hipLaunchKernelGGL((mx_scores_kernel<STEPS, 1, OUT>), grid, dim3(256), 0, s, p, kb, qt, per, vec);
}

int launch_mx_scores(const MxScoreParams &p, hipStream_t s)
{
    const int kb = (p.k + 31) / 32;
#define IFR_SCORES(STEPS)                                                                                  \
    p.out_bf16 ? launch_mx_scores_typed<STEPS, __bf16>(p, kb, s) : launch_mx_scores_typed<STEPS, float>(p, kb, s)
    if (kb <= 2) IFR_SCORES(1);
    else if (kb <= 4) IFR_SCORES(2);
    else if (kb <= 6) IFR_SCORES(3);
    else IFR_SCORES(4);
#undef IFR_SCORES
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace ifr
