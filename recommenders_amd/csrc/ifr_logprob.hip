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
// Operands in 16 bits: bf16 as it is.  fp32 is split into two fp16 parts after scaling each row by the power of two that
// brings its largest magnitude to [2^14, 2^15): hi + lo keeps 22 bits of values down to 2^-17 of the row's maximum and an absolute step of
// 2^-39 of the maximum below, and three products (hi hi, hi lo, lo hi) leave out lo lo, at most 2^-22 of a term.  Three fp16 products at 16
// times the rate of the fp32 matrix instruction cost a fifth of it.
#include <hip/hip_runtime.h>

#include <math.h>
#include <type_traits>

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
constexpr int64_t DEAL_FROM = 65536;
constexpr int BUCKETS = 64, CHUNK = 4096;      // of places: see deal_kernel
constexpr int64_t MAX_GRID = 1 << 22;  // workgroups of 256 in one launch (the grid counts work items in 32 bits)

int pad_factors(int k) { return (k + 31) / 32 * 32; }
int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__bf16 v) { return (float)v; }

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }

// exponent e with max * 2^e in [2^14, 2^15) for a row's largest finite magnitude (a subnormal one counts as 2^-126: scaled to at most 2^14, which is as
// exact), a row of zeros too
__device__ __forceinline__ int split_exponent(float top)
{
    const uint32_t m = __float_as_uint(top);
    if (m == 0) return 140;
    return 14 - (m < 0x00800000u ? -126 : (int)(m >> 23) - 127);
}

// One block of sums d (16 of a lane's own S row) into the running maximum m (of c d) and the sum of 2^(c d - m); c > 0, so the
// largest d gives the largest exponent.
__device__ __forceinline__ void online(const v16f &d, float c, float &m, float &sum)
{
    float high = d[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) high = fmaxf(high, d[r]);
    // at least the lowest finite number, so that a block of -inf adds zeros; NaN in d reaches the sum through its own exponential
    const float top = fmaxf(m, high * c);
    float add = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) add += exp2_raw(fmaf(d[r], c, -top));
    sum = fmaf(sum, exp2_raw(m - top), add);
    m = top;
}

}  // namespace

// ---------------------------------------------------------------------------- preparation

// A matrix in the order the walks read it, by tiles of 32 rows, zeros behind the last row and column:
//   frag [tile][part][KP / 16][64][8]: columns 16 s + 8 h + 0..7 of a row are the 16-byte piece piece_at(s, row, h)
//   units [row]: 2^(-24 - e) of the row's exponent e (split operands); infinities and NaN do not count for it and stay what they are
// A bf16 V whose rows are whole, aligned pieces (k = KP) is read as it lies: v_frag is null then, and x_frag where lse is.  For the gradient
// X is always put in order: users without an item (a batch's padding) become rows of zeros, so that nothing in them reaches dV.
struct PrepParams {
    const void *V, *X;
    int64_t ldv, ldx, n_items, n, v_blocks, v_padded;
    int k, KP;
    float *v_unit, *x_unit;
    uint4 *v_frag, *x_frag;
    const float *ibase;
    // terms of split operands are powers of two, to be added to the exponent; those of bf16 operands are in units of <x, v>, to begin
    // its sum with.  item_term = base_unit ibase, user_term = lse_unit lse; -inf behind the last item and user
    float base_unit, lse_unit;
    float *item_term;
    // gradient only (lse null otherwise)
    const float *lse, *dlogp;
    const int32_t *ids;
    int64_t m, ld_ids, ld_dlogp, places_padded;
    float *user_term, *G, *G_scaled;   // G: the sum of a user's upstream gradients; split: also times 2^24
    int32_t *places;                   // the items named in (user, place) order, -1 behind the last place; null: not wanted
    uint8_t *named;                    // [items / 64], cleared before: set where an item is named; or null
};

// Where a tile keeps the piece of columns 16 s + 8 h + 0..7 of a row: a row's two pieces of a step side by side, so that memory is read in
// 32 bytes; the rows of odd steps and the order of the two are turned so that 16 rows of one h (first product) and four rows of two
// steps (second product) fall on all 64 banks of LDS.  Without the turns a third of the LDS cycles were conflicts.
__host__ __device__ constexpr int piece_at(int s, int row, int h)
{
    const int r = row ^ (s & 1) * 4;
    return s * 64 + r * 2 + (h ^ (r >> 3 & 1));
}

// LDS tile [32][W] -> pieces
template <int NS>
__device__ __forceinline__ void store_fragments(const float *tile, int W, int KP, const int *e, int64_t at, uint4 *f)
{
    const int per = KP / 16 * 64;                     // 16-byte pieces of one part of a tile
    for (int i = threadIdx.x; i < per; i += 256) {
        const int step = i >> 6, r = i >> 1 & 31, row = r ^ (step & 1) * 4, h = (i & 1) ^ (r >> 3 & 1);      // piece_at turned round
        const float *v = tile + row * W + step * 16 + h * 8;
        if (NS == 1) {
            b8 o;
            for (int j = 0; j < 8; ++j) o[j] = (__bf16)v[j];
            f[at * per + i] = __builtin_bit_cast(uint4, o);
        } else {
            h8 hi, lo;
            for (int j = 0; j < 8; ++j) {
                const float x = ldexpf(v[j], e[row]);
                hi[j] = (_Float16)x;
                lo[j] = (_Float16)(x - (float)hi[j]);
            }
            f[at * 2 * per + i] = __builtin_bit_cast(uint4, hi);
            f[(at * 2 + 1) * per + i] = __builtin_bit_cast(uint4, lo);
        }
    }
}

// Everything the walks read, a workgroup a tile of 32 rows of V (or 256 of its terms, where it needs no other order) or X.  One read, one
// write, through LDS since a piece is eight columns of one row; short, so bound by the latency of its loads (eight under way a thread).
// fp32 2048 + 26 744 rows of 200: 16 us (23 MB in, 26 MB out).
template <typename T, int NS>
__global__ __launch_bounds__(256) void prepare_kernel(PrepParams p)
{
    extern __shared__ float tile[];                   // [32][KP + 1]
    __shared__ float sums[256];
    __shared__ int exps[32], holds[32];
    const int W = p.KP + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool of_v = blockIdx.x < p.v_blocks;
    const int64_t at = of_v ? blockIdx.x : blockIdx.x - p.v_blocks, r0 = at * 32;
    uint4 *frag = of_v ? p.v_frag : p.x_frag;
    auto item_term = [&](int64_t i) {
        if (i < p.v_padded) p.item_term[i] = i < p.n_items ? (p.ibase ? p.ibase[i] * p.base_unit : 0.f) : -INFINITY;
    };
    if (of_v && !frag) {
        item_term(at * 256 + threadIdx.x);
        return;
    }
    if (!of_v && p.lse) {   // G over the places that hold an item: eight threads a user, their sums added in their order
        const int r = threadIdx.x >> 3;
        const int64_t u = r0 + r;
        float g = 0.f;
        int held = 0;
        if (u < p.n)
            for (int64_t j = threadIdx.x & 7; j < p.m; j += 8)
                if (p.ids[u * p.ld_ids + j] >= 0) { g += p.dlogp[u * p.ld_dlogp + j]; held = 1; }
        sums[threadIdx.x] = g;
        for (int o = 4; o; o >>= 1) held |= __shfl_xor(held, o);
        if ((threadIdx.x & 7) == 0) holds[r] = held;
        __syncthreads();
    }
    if (frag) {
        const T *src = (const T *)(of_v ? p.V : p.X);
        const int64_t rows = of_v ? p.n_items : p.n, ld = of_v ? p.ldv : p.ldx;
        float top[8] = {};
        for (int c = lane; c < p.KP; c += 64) {
            float v[8];                               // eight loads under way at once
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int r = wave + 4 * q;
                v[q] = r0 + r < rows && c < p.k && (of_v || !p.lse || holds[r]) ? as_f32(src[(r0 + r) * ld + c]) : 0.f;
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                tile[(wave + 4 * q) * W + c] = v[q];
                if (NS == 2 && fabsf(v[q]) < INFINITY) top[q] = fmaxf(top[q], fabsf(v[q]));
            }
        }
        if (NS == 2) {
            // eight rows at once: a lane gives half of what it holds to the lane that keeps those rows, until eight lanes hold one row
#pragma unroll
            for (int w = 4, o = 32; w; w >>= 1, o >>= 1)
#pragma unroll
                for (int q = 0; q < w; ++q) {
                    const float give = lane & o ? top[q] : top[q + w], keep = lane & o ? top[q + w] : top[q];
                    top[q] = fmaxf(keep, __shfl_xor(give, o));
                }
            for (int o = 4; o; o >>= 1) top[0] = fmaxf(top[0], __shfl_xor(top[0], o));
            if ((lane & 7) == 0) {
                const int r = wave + 4 * (lane >> 3), e = split_exponent(top[0]);
                exps[r] = e;
                (of_v ? p.v_unit : p.x_unit)[r0 + r] = ldexpf(1.f, -24 - e);
            }
        }
        __syncthreads();
        store_fragments<NS>(tile, W, p.KP, exps, at, frag);
    }
    if (of_v) {
        if (threadIdx.x < 32) item_term(r0 + threadIdx.x);
        return;
    }
    if (!p.lse) return;
    if (threadIdx.x < 32) {
        const int64_t u = r0 + threadIdx.x;
        float g = 0.f;
        for (int q = 0; q < 8; ++q) g += sums[threadIdx.x * 8 + q];
        p.G[u] = g;
        if (NS == 2) p.G_scaled[u] = g * 16777216.f;
        // no probabilities where lse is -inf, and none that matter where no item is named: every exponential is 0
        p.user_term[u] = u < p.n && holds[threadIdx.x] && p.lse[u] != -INFINITY ? p.lse[u] * p.lse_unit : -INFINITY;
    }
    if (p.places) {
        const int64_t all = p.n * p.m;
        const int64_t from = min(r0 * p.m, all), to = r0 + 32 >= p.n ? (r0 < p.n ? p.places_padded : from) : (r0 + 32) * p.m;
        for (int64_t i = from + threadIdx.x; i < to; i += 256) {
            int32_t id = -1;
            if (i < all) {
                const int32_t r = (int32_t)((i - from) / (int32_t)p.m);          // below 32 m, at most 2^25
                id = p.ids[(r0 + r) * p.ld_ids + (i - from - (int64_t)r * p.m)];
                if (p.named && id >= 0 && id < p.n_items) p.named[id >> 6] = 1;
            }
            p.places[i] = id;
        }
    }
}

__global__ __launch_bounds__(256) void clear_kernel(uint32_t *p, int64_t n)
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

// Places in the order of 64 buckets of items (whole S blocks each), so that a workgroup that finishes rows of dV looks through its
// bucket's only.  A stable counting sort: a workgroup takes 4096 places, a thread 16 neighbouring ones, and each (bucket, thread) has a
// byte of its own in LDS, so no order depends on scheduling.  Empty places and those behind the catalogue are left out.  Latency-bound:
// three short launches.
struct Deal {
    const int32_t *places;
    int64_t chunks, n_items, bucket_items;
    uint32_t *counts;                  // [BUCKETS][chunks], then their exclusive sums
    uint32_t *bounds;                  // [BUCKETS + 1]
    int32_t *to;                       // the items again, -1 up to the next 1024
    uint32_t *place_of;
};

template <bool WRITE>
__global__ __launch_bounds__(256) void deal_kernel(Deal d)
{
    __shared__ uint32_t held[64 * 64];                // [bucket][thread], bytes
    uint8_t *mine = (uint8_t *)held + threadIdx.x;
    const int64_t chunk = blockIdx.x, at = chunk * CHUNK + threadIdx.x * 16;
    for (int i = threadIdx.x; i < 64 * 64; i += 256) held[i] = 0;
    int32_t id[16];
    uint8_t bucket[16];
    for (int q = 0; q < 16; q += 4) *(int4 *)(id + q) = *(const int4 *)(d.places + at + q);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const bool in = id[q] >= 0 && id[q] < d.n_items;
        bucket[q] = in ? (uint8_t)(id[q] / (int32_t)d.bucket_items) : 255;
        if (in) ++mine[bucket[q] * 256];
    }
    __syncthreads();
    // four threads a bucket, 64 of the bytes each
    const int b = threadIdx.x >> 2, quarter = threadIdx.x & 3;
    uint32_t sum = 0;
    for (int i = 0; i < 16; ++i) {
        const uint32_t w = held[b * 64 + quarter * 16 + i];
        sum += (w & 255) + (w >> 8 & 255) + (w >> 16 & 255) + (w >> 24);
    }
    uint32_t before = 0, all = sum;
    for (int o = 1; o < 4; ++o) {
        const uint32_t other = __shfl_xor(sum, o);
        all += other;
        if ((quarter ^ o) < quarter) before += other;
    }
    if (!WRITE) {
        if (quarter == 0) d.counts[b * d.chunks + chunk] = all;
        return;
    }
    // where the places of each thread and bucket go: sixteen bits beside the chunk's begin
    __shared__ uint16_t first[64 * 256];
    uint32_t run = before;
    for (int i = 0; i < 64; ++i) {
        first[b * 256 + quarter * 64 + i] = (uint16_t)run;
        run += ((const uint8_t *)held)[b * 256 + quarter * 64 + i];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 16; ++q)
        if (bucket[q] != 255) {
            const uint32_t to = d.counts[bucket[q] * d.chunks + chunk] + first[bucket[q] * 256 + threadIdx.x]++;
            d.to[to] = id[q];
            d.place_of[to] = (uint32_t)(at + q);
        }
    if (chunk == 0) {
        const uint32_t total = d.bounds[BUCKETS];
        for (uint32_t i = total + threadIdx.x; i < (total + 1023) / 1024 * 1024; i += 256) d.to[i] = -1;
    }
}

// exclusive sums of the counts, one workgroup
__global__ __launch_bounds__(1024) void deal_sums_kernel(Deal d)
{
    __shared__ uint32_t waves[16];
    const int64_t all = BUCKETS * d.chunks;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (int64_t i0 = 0; i0 < all; i0 += 1024) {
        const int64_t i = i0 + threadIdx.x;
        const uint32_t v = i < all ? d.counts[i] : 0;
        uint32_t sum = v;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t other = __shfl_up(sum, o);
            if (lane >= o) sum += other;
        }
        if (lane == 63) waves[wave] = sum;
        __syncthreads();
        uint32_t before = carry;
        for (int w = 0; w < 16; ++w) {
            if (w < wave) before += waves[w];
            carry += waves[w];
        }
        before += sum - v;
        if (i < all) {
            d.counts[i] = before;
            if (i % d.chunks == 0) d.bounds[i / d.chunks] = before;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) d.bounds[BUCKETS] = carry;
}

// ---------------------------------------------------------------------------- the walk

// lse; the sums of dX (S users, T items); those of dV (S items, T users), and of dV and db
enum { WALK_STATS = 0, WALK_USERS = 1, WALK_ITEMS = 2, WALK_ITEMS_BASE = 3 };

// What the gradient of V needs to finish its rows in the kernel that summed them (one split): see find_places.
struct Finish {
    const int32_t *places;             // [n_places, padded to 1024]: items named, in (user, place) order
    const uint8_t *named;              // [n_items / 64]: whether one of 64 items is, or null
    const void *X;                     // [n][ldx]
    const float *dlogp;
    void *dV;                          // [n_items][ld_dv] or null
    float *db;                         // [n_items] or null
    const uint32_t *place_of;          // places dealt into buckets: the number of each, or null: as they are
    const uint32_t *bounds;            // [BUCKETS + 1]: a bucket's first place
    int64_t bucket_items;              // items of a bucket
    int64_t n_places, m, ldx, ld_dlogp, ld_dv, n_items;
    int k;
    float scale;
    int vec_x, vec_dv;                 // rows of X, of dV are aligned for four columns at once, k a multiple of four
};

struct WalkParams {
    const uint4 *s_frag, *t_frag;      // null: bf16 rows as they lie
    const __bf16 *s_rows, *t_rows;
    int64_t s_ld, t_ld, s_n, t_n;
    const float *s_term, *t_term;      // item_term, user_term of prepare_kernel
    const float *t_factor;             // WALK_ITEMS...: G (split: times 2^24)
    const float *s_unit, *t_unit;      // split operands: powers of two of their rows
    float c;                           // scale log2(e)
    int s_blocks, splits, t_tiles, tiles_per_split;
    int64_t s_padded;
    float *out_m, *out_s;              // WALK_STATS: [splits][s_padded]
    float *out_acc;                    // else: [splits][s_padded][KP], or null: finish
    float *out_b;                      // WALK_ITEMS_BASE: [splits][s_padded]: sums of factor P, or null
    Finish f;
};

// two times four rows of this lane's column (see at2 in walk_kernel)
__device__ __forceinline__ uint4 turned(const char *low, const char *high)
{
    typedef short s4 __attribute__((ext_vector_type(4)));
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)low);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)high);
    const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
    return make_uint4(a.x, a.y, b.x, b.y);
}

template <int NS>
__device__ __forceinline__ v16f product(uint4 a, uint4 b, v16f d)
{
    if (NS == 1) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), d, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), d, 0, 0, 0);
}

// 64 floats (one wave), and PIECES 16-byte pieces, from memory to LDS without a stop in registers; the caller waits for them
__device__ __forceinline__ void fetch_row(const float *from, float *to)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from + (threadIdx.x & 63)),
                                     (__attribute__((address_space(3))) void *)to, 4, 0, 0);
}

template <int PIECES>
__device__ __forceinline__ void fetch(const uint4 *from, uint4 *to)
{
    static_assert(PIECES % 64 == 0, "whole waves");
#pragma unroll
    for (int i = 0; i < (PIECES + 255) / 256; ++i) {
        const int at = i * 256 + (int)(threadIdx.x & ~63u);
        if (PIECES % 256 == 0 || at < PIECES)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from + at + (threadIdx.x & 63)),
                                             (__attribute__((address_space(3))) void *)(to + at), 16, 0, 0);
    }
}

// asks the scheduler for LDS reads six ahead of the matrix instructions that use them
template <int READS, int PRODUCTS>
__device__ __forceinline__ void reads_ahead()
{
    __builtin_amdgcn_sched_group_barrier(0x100, READS < 6 ? READS : 6, 0);
#pragma unroll
    for (int i = 6; i < READS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS / READS, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, PRODUCTS, 0);
}

// places a workgroup keeps of those it looks through: their users, gradients and sorted order, 12 bytes each, fit a stage of walk_kernel
constexpr int list_length(int KP) { return KP >= 192 ? 4096 : KP >= 96 ? 2048 : KP >= 64 ? 1024 : 512; }

// four columns of a row, zeros behind its end
template <typename T>
__device__ __forceinline__ void load4(const T *row, int c, int k, bool vec, float v[4])
{
    if (vec) {
        if (sizeof(T) == 4) {
            const float4 a = *(const float4 *)(row + c);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        } else {
            const uint2 a = *(const uint2 *)(row + c);
            v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
            v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
        }
    } else {
        for (int j = 0; j < 4; ++j) {                 // no branch: the last column again behind it
            const float a = as_f32(row[min(c + j, k - 1)]);
            v[j] = c + j < k ? a : 0.f;
        }
    }
}

// The last steps of dV: rows of sums lie in LDS as rows[local][KP], 64 at a time; g x of every place that names one of the items is added,
// the rows are scaled, rounded and stored.  Nothing depends on scheduling.
//
// find_places: each wave looks through a quarter of the places [from, to) -- those of the users that the workgroup walked -- and lists
// those that name one of `count` (at most 128) items, until its list is full or the quarter is done (`step` keeps where it is); the
// lists are sorted by item.  Returns how many, `more`: come again.
template <int KP>
__device__ __forceinline__ int find_places(const Finish &f, uint32_t *list, int *counts, uint8_t *item_of, int64_t i0, int count, int64_t from, int64_t to,
                                           int64_t &step, bool &more)
{
    constexpr int LIST = list_length(KP), CAP = LIST / 4, EACH = CAP / 64;
    uint32_t *order = list + 2 * LIST;
    float *gs = (float *)(list + LIST);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (f.place_of) {                                 // what lies beside them in the first and last step names other items
        const int64_t b = i0 / f.bucket_items;
        from = f.bounds[b] / (64 * EACH) * (64 * EACH);
        to = (f.bounds[b + 1] + 64 * EACH - 1) / (64 * EACH) * (64 * EACH);
    }
    const int64_t begin = from / (64 * EACH), steps = (to + 64 * EACH - 1) / (64 * EACH) - begin;
    const int64_t end = begin + steps * (wave + 1) / 4;
    if (step < 0) step = begin + steps * wave / 4;
    int held = 0;
    int32_t id[EACH], next[EACH];
    auto load = [&](int64_t at, int32_t *to) {
        if (EACH >= 4) {
            const int4 *src = (const int4 *)f.places + at * 64 * (EACH / 4) + lane;
#pragma unroll
            for (int q = 0; q < EACH / 4; ++q) *(int4 *)(to + 4 * q) = src[q * 64];
        } else {
#pragma unroll
            for (int q = 0; q < EACH; ++q) to[q] = f.places[(at * EACH + q) * 64 + lane];
        }
    };
    if (step < end) load(step, id);
    while (step < end) {
        if (step + 1 < end) load(step + 1, next);
        int mine = 0;
        const bool edge = step * 64 * EACH < from || (step + 1) * 64 * EACH > to;
#pragma unroll
        for (int q = 0; q < EACH; ++q) {
            if (id[q] >= f.n_items) id[q] = -1;       // behind the catalogue: no row takes it
            if (edge) {
                const int64_t at = step * 64 * EACH + (EACH >= 4 ? (q >> 2) * 256 + lane * 4 + (q & 3) : q * 64 + lane);
                if (at < from || at >= to) id[q] = -1;
            }
            mine += (uint64_t)((int64_t)id[q] - i0) < (uint64_t)count;
        }
        if (__ballot(mine)) {
            int before = mine;
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(before, o);
                if (lane >= o) before += v;
            }
            const int all = __shfl(before, 63);
            if (held + all > CAP) break;              // next time: a step alone always fits
            before += held - mine;
            if (mine) {
#pragma unroll
                for (int q = 0; q < EACH; ++q) {
                    const int64_t local = (int64_t)id[q] - i0;
                    if ((uint64_t)local < (uint64_t)count) {
                        const int in = EACH >= 4 ? (q >> 2) * 256 + lane * 4 + (q & 3) : q * 64 + lane;
                        const int to = wave * CAP + before++;
                        item_of[to] = (uint8_t)local;
                        list[to] = (uint32_t)(step * 64 * EACH + in);                     // at most 2^32 places
                    }
                }
            }
            held += all;
        }
        ++step;
#pragma unroll
        for (int q = 0; q < EACH; ++q) id[q] = next[q];
    }
    if (lane == 0) counts[wave] = held;
    more = __syncthreads_or(step < end);
    int total = 0, offset = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < wave) offset += counts[w];
        total += counts[w];
    }
    for (int q = lane; q < held; q += 64) {           // places to users and gradients, each by one lane
        const int at = wave * CAP + q;
        const uint32_t place = f.place_of ? f.place_of[list[at]] : list[at], u = place / (uint32_t)f.m;
        order[offset + q] = (uint32_t)item_of[at] << 12 | (uint32_t)at;
        list[at] = u;
        gs[at] = f.dlogp[(int64_t)u * f.ld_dlogp + (place - u * (uint32_t)f.m)];
    }
    int size = 1;
    while (size < total) size <<= 1;
    for (int q = total + tid; q < size; q += 256) order[q] = ~0u;
    __syncthreads();
    for (int w = 2; w <= size; w <<= 1)               // bitonic: keys are unique (item, position)
        for (int d = w >> 1; d; d >>= 1) {
            for (int q = tid; q < size / 2; q += 256) {
                const int lo = 2 * q - (q & (d - 1)), hi = lo + d;
                const uint32_t x = order[lo], y = order[hi];
                if ((x > y) == !(lo & w)) { order[lo] = y; order[hi] = x; }
            }
            __syncthreads();
        }
    return total;
}

// threads of a group in add_places: those of a row (four columns each), rounded up so that a wave holds whole groups
constexpr int group_threads(int KP) { return KP > 128 ? 64 : KP > 64 ? 32 : KP > 32 ? 16 : 8; }

// The found places [from, to) in their sorted order, of items whose local number is 64 at a time from `local0`.  The groups of threads
// (four columns a thread) take equal parts, so that an item that everybody names does not fall to one group; an item's first run in a
// part goes to a row set aside, which is added after the others, in the parts' order.  A run is summed in registers.  Short code on purpose: it runs once a
// workgroup, and what it costs is the fetching of its instructions as much as that of the rows.
template <typename T, int KP>
__device__ __forceinline__ void add_places(const Finish &f, float *rows, float *row_b, const uint32_t *list, float *aside, int *aside_item, int local0, int from,
                                           int to)
{
    constexpr int COLS = group_threads(KP), GROUPS = 256 / COLS, BATCH = 16;
    const uint32_t *order = list + 2 * list_length(KP);
    const float *gs = (const float *)(list + list_length(KP));
    const int tid = threadIdx.x, group = tid / COLS, c4 = (tid % COLS) * 4;
    const T *X = (const T *)f.X;
    const int part = (to - from + GROUPS - 1) / GROUPS, begin = from + group * part, end = min(begin + part, to);
    const bool in = c4 < KP, vec = f.vec_x && c4 < f.k;
    const int first = begin < end ? (int)(order[begin] >> 12) - local0 : -1;
    if (c4 == 0) { aside_item[group] = first; aside[GROUPS * KP + group] = 0.f; }
    if (in) *(float4 *)(aside + group * KP + c4) = make_float4(0.f, 0.f, 0.f, 0.f);
    int cur = -1;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum_b = 0.f;
    auto row_of = [&](int at) { return at == first ? aside + group * KP : rows + at * KP; };
    auto flush = [&]() {
        *(float4 *)(row_of(cur) + c4) = sum;
        if (c4 == 0) *(cur == first ? aside + GROUPS * KP + group : row_b + cur) += sum_b;
    };
    for (int q0 = begin; q0 < end; q0 += BATCH) {
        // all keys, then all users, then all rows: sixteen gathers are under way at once
        uint32_t key[BATCH], u[BATCH];
        float x[BATCH][4], g[BATCH];
#pragma unroll
        for (int q = 0; q < BATCH; ++q) key[q] = order[min(q0 + q, end - 1)];
#pragma unroll
        for (int q = 0; q < BATCH; ++q) { u[q] = list[key[q] & 4095]; g[q] = gs[key[q] & 4095]; }
        if (vec) {
#pragma unroll
            for (int q = 0; q < BATCH; ++q) load4(X + (int64_t)u[q] * f.ldx, c4, f.k, true, x[q]);
        } else {
#pragma unroll
            for (int q = 0; q < BATCH; ++q) load4(X + (int64_t)u[q] * f.ldx, c4, f.k, false, x[q]);
        }
#pragma unroll
        for (int q = 0; q < BATCH; ++q)
            if (in && q0 + q < end) {
                const int at = (int)(key[q] >> 12) - local0;
                if (at != cur) {
                    if (cur >= 0) flush();
                    cur = at;
                    sum = *(const float4 *)(row_of(at) + c4);
                    sum_b = 0.f;
                }
                sum.x = fmaf(g[q], x[q][0], sum.x); sum.y = fmaf(g[q], x[q][1], sum.y);
                sum.z = fmaf(g[q], x[q][2], sum.z); sum.w = fmaf(g[q], x[q][3], sum.w);
                sum_b += g[q];
            }
    }
    if (in && cur >= 0) flush();
    __syncthreads();
    const int used = (to - from + part - 1) / part;   // groups that had places
    for (int g = 0; g < used; ++g) {
        const int item = aside_item[g];
        for (int c = tid; c < KP; c += 256) rows[item * KP + c] += aside[g * KP + c];
        if (tid == 0) row_b[item] += aside[GROUPS * KP + g];
    }
    __syncthreads();
}

// four columns of a row of dV
template <typename T>
__device__ __forceinline__ void store4(const Finish &f, int64_t i, int c, float4 v)
{
    if (!f.dV || i >= f.n_items || c >= f.k) return;
    T o[4] = {(T)(f.scale * v.x), (T)(f.scale * v.y), (T)(f.scale * v.z), (T)(f.scale * v.w)};
    T *to = (T *)f.dV + i * f.ld_dv + c;
    if (f.vec_dv) {
        __builtin_memcpy(__builtin_assume_aligned(to, 4 * sizeof(T)), o, 4 * sizeof(T));
    } else {
        for (int j = 0; j < 4; ++j)
            if (c + j < f.k) to[j] = o[j];
    }
}

template <typename T, int KP>
__device__ __forceinline__ void store_rows(const Finish &f, const float *rows, const float *row_b, int64_t i0)
{
    for (int i = threadIdx.x; i < 64 * KP / 4; i += 256) {
        const int r = i / (KP / 4), c = (i - r * (KP / 4)) * 4;
        store4<T>(f, i0 + r, c, *(const float4 *)(rows + r * KP + c));
    }
    if (f.db)
        for (int r = threadIdx.x; r < 64; r += 256)
            if (i0 + r < f.n_items) f.db[i0 + r] = f.scale * row_b[r];
}

// memory of the sums set aside (one row and one number a group), or a byte for each place of the lists
constexpr int aside_floats(int KP)
{
    const int sums = 256 / group_threads(KP) * (KP + 1), bytes = list_length(KP) / 4;
    return sums > bytes ? sums : bytes;
}

// T rows of a stage, in tiles of 32.  For the gradient two stages, each of which also holds 64 rows of sums at the end, fill 512 KP bytes
// of LDS; the statistics take half of that, for two workgroups a compute unit also at KP = 256.
constexpr int stage_tiles(int NS, bool grad) { return (NS == 1 ? 2 : 1) * (grad ? 2 : 1); }

// whether a compute unit holds two workgroups of walk_kernel by its registers
constexpr bool paired(int KP, int NS, int mode) { return KP * NS <= 256 && (mode == WALK_STATS || KP <= 128); }

// S_LIES, T_LIES: read as bf16 rows in memory (V; X too for the statistics)
//
// Bound by the matrix instructions together with what does not fit beside them: 16 exponentials a lane and tile (a quarter of the rate of
// the rest), the conversion of P to two parts of 16 bits, with fp32 operands the scaling of P and of each tile's product (600 vector
// instructions a wave and tile of 224 columns beside 84 matrix ones), and the clock under their load (bf16 2048 x 1 000 000 x 128, sums of
// dX: 1350 us, the same instructions on rows of zeros 1010 us).  A tile is 32 rows as the 32 x 32 instructions have it: 16 x 16 ones would read LDS twice as
// often for the same products.  128 S rows a workgroup: their operand (KP / 16 registers of 4 a part) and the sums of 32 x KP a wave
// fill the registers, so that a compute unit holds two workgroups up to 256 columns in all parts and one beyond; LDS serves four waves
// with one stage.  Sizes and what they measured (matrix unit busy, of the SIMDs' cycles):
//   bf16 2048 x 1 000 000 x 128: lse 0.66 ms (45 %), sums of dX 1.38 ms (66 %), dV finished 1.66 ms (52 %), all under the profiler
//   fp32 2048 x 26 744 x 200: lse 71 us (62 %), sums of dX 185 us (42 %), dV and db finished 289 us (34 %)
// = 3.7 PFLOP with the recomputed scores and both parts of P in 3.3 - 3.5 ms for the bf16 step, where a large product of the library
// reaches 1206 TFLOP/s.  (P in one part took 2.6 ms, and lost the gradient of users who are sure of their item.)
template <int KP, int NS, int MODE, bool S_LIES, bool T_LIES>
__global__ __launch_bounds__(256, paired(KP, NS, MODE) ? 2 : 1) void walk_kernel(WalkParams p)
{
    typedef typename std::conditional<NS == 2, float, __bf16>::type T;
    typedef typename std::conditional<NS == 2, _Float16, __bf16>::type E;
    constexpr int STEPS = KP / 16;
    constexpr int PART = STEPS * 64;                  // 16-byte pieces of a part of a tile
    constexpr bool GRAD = MODE != WALK_STATS, PAIRED = paired(KP, NS, MODE);
    constexpr int ABREAST = NS == 2 && !PAIRED ? 2 : 1;      // blocks of 32 columns whose products alternate
    constexpr int SUB = stage_tiles(NS, GRAD);
    constexpr int STAGE = PART * NS * SUB;
    // two stages: one is read while the other arrives (two arrays, so that the compiler sees that they are apart)
    __shared__ uint4 stage0[STAGE], stage1[STAGE];
    // of the stage's T rows: t_term, t_factor, t_unit (a fetch brings 64)
    constexpr int ROWS = SUB * 32 < 64 ? 64 : SUB * 32;
    __shared__ __align__(16) float terms0[(NS + 1) * ROWS], terms1[(NS + 1) * ROWS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = lane >> 5;
    // workgroups go to the eight XCDs in turn: splits are dealt so that an XCD's L2 sees each part of T from one split only
    int s_block, split;
    {
        const int id = blockIdx.x, whole = p.splits / 8 * 8 * p.s_blocks;
        if (id < whole) {
            s_block = (id >> 3) % p.s_blocks;
            split = (id >> 3) / p.s_blocks * 8 + (id & 7);
        } else {
            s_block = (id - whole) % p.s_blocks;
            split = p.splits / 8 * 8 + (id - whole) / p.s_blocks;
        }
    }
    const int64_t s_tile = (int64_t)s_block * 4 + wave;
    const int64_t s_row = s_tile * 32 + (lane & 31);

    uint4 sf[NS][STEPS];
#pragma unroll
    for (int q = 0; q < NS; ++q)
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
            sf[q][s] = S_LIES ? ((const uint4 *)(p.s_rows + min(s_row, p.s_n - 1) * p.s_ld))[2 * s + h]
                            : p.s_frag[(s_tile * NS + q) * PART + piece_at(s, lane & 31, h)];
    // split: a score is scale log2(e) 2^-(e_s + e_t) of a product; the T row's part leaves 2^24 to the S row's, so that a product of a T row's
    // parts (below 2^38) times its own power of two stays below 2^127 whatever the row holds
    const float s_unit = NS == 2 ? fminf(p.c * (p.s_unit[s_row] * 16777216.f) * 16777216.f, 3.402823466e38f) : 1.f;
    const float s_term = p.s_term ? p.s_term[s_row] * (NS == 1 ? p.c : 1.f) : 0.f;

    constexpr bool ITEMS = MODE == WALK_ITEMS || MODE == WALK_ITEMS_BASE;
    v16f acc[GRAD ? KP / 32 : 1] = {};
    float m = -3.402823466e38f, sum = 0.f, b_sum = 0.f;
    const int first = split * p.tiles_per_split, last = min(first + p.tiles_per_split, p.t_tiles);
    // this lane's pieces of the first product's operand (even and odd steps), and its 8 bytes of the second's, which ds_read_tr turns
    // round: 16 lanes read four rows by 16 columns and get four rows of a column each (rows 0..7 and 8..15 of a step of 16)
    const int at1[2] = {piece_at(0, lane & 31, h), piece_at(1, lane & 31, h) - 64};
    const int row2 = 4 * h + (lane >> 2 & 3), step2 = lane >> 4 & 1, h2 = lane >> 1 & 1;
    const int at2 = piece_at(step2, row2, h2) * 16 + (lane & 1) * 8, at2_high = piece_at(step2, row2 + 8, h2) * 16 + (lane & 1) * 8;

    auto fetch_stage = [&](int t, uint4 *to, float *terms) {
        if (T_LIES) {
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub) {
                // steps s of a wave have the parity of the wave; behind the last row: one whose term is -inf
                const int r = lane >> 1;
                const int64_t row = min((int64_t)(t + sub) * 32 + (r ^ (wave & 1) * 4), p.t_n - 1);
                const uint4 *from = (const uint4 *)(p.t_rows + row * p.t_ld) + ((lane & 1) ^ (r >> 3 & 1));
#pragma unroll
                for (int s = 0; s < (STEPS + 3) / 4; ++s)
                    if (STEPS % 4 == 0 || s * 4 + wave < STEPS)
                        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from + (s * 4 + wave) * 2),
                                                         (__attribute__((address_space(3))) void *)(to + sub * PART + (s * 4 + wave) * 64), 16, 0, 0);
            }
        } else {
            fetch<STAGE>(p.t_frag + (int64_t)t * PART * NS, to);
        }
        constexpr int EACH = ROWS / 64;
        if (wave < EACH) fetch_row(p.t_term + (int64_t)t * 32 + wave * 64, terms + wave * 64);
        else if (ITEMS && wave < 2 * EACH) fetch_row(p.t_factor + (int64_t)t * 32 + (wave - EACH) * 64, terms + wave * 64);
        else if (NS == 2 && wave == 2) fetch_row(p.t_unit + (int64_t)t * 32, terms + 2 * ROWS);
    };
    // The scores of one tile: split (d t_unit) s_unit + term, otherwise the sums begin with the terms.
    auto scores = [&](const uint4 *l1, const float *tt) {
        v16f d = {};
        float4 t4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) t4[q] = *(const float4 *)(tt + 8 * q + 4 * h);
        if (NS == 1) {
#pragma unroll
            for (int q = 0; q < 4; ++q) { d[4 * q] = t4[q].x; d[4 * q + 1] = t4[q].y; d[4 * q + 2] = t4[q].z; d[4 * q + 3] = t4[q].w; }
        }
        // split: two sums in turn, so that no matrix instruction waits for the one before (a wave is alone on its SIMD)
        v16f other = {};
        constexpr bool TWO = NS == 2 && GRAD && !PAIRED;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const uint4 a = l1[s * 64 + at1[s & 1]];
            v16f &d0 = TWO && (s & 1) ? other : d, &d1 = TWO && !(s & 1) ? other : d;
            d0 = product<NS>(a, sf[0][s], d0);
            if (NS == 2) {
                d1 = product<NS>(a, sf[NS - 1][s], d1);
                d0 = product<NS>(l1[PART + s * 64 + at1[s & 1]], sf[0][s], d0);
            }
        }
        if (TWO) {
            d += other;
            // the scaling stays behind the products: moved between them it took 512 registers and spilled (224 columns: sums of dX 204 us, so 182)
            __builtin_amdgcn_sched_barrier(0);
        }
        if (NS == 2) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 u4 = *(const float4 *)(tt + 2 * ROWS + 8 * q + 4 * h);
                d[4 * q] = fmaf(d[4 * q] * u4.x, s_unit, t4[q].x); d[4 * q + 1] = fmaf(d[4 * q + 1] * u4.y, s_unit, t4[q].y);
                d[4 * q + 2] = fmaf(d[4 * q + 2] * u4.z, s_unit, t4[q].z); d[4 * q + 3] = fmaf(d[4 * q + 3] * u4.w, s_unit, t4[q].w);
            }
        }
        return d;
    };
    // A stage's tiles (those behind the last row have terms of -inf and add nothing: no branch divides the code, so that the
    // exponentials of one tile go beside the matrix instructions of the next tile's scores and of the last one's sums).
    auto compute = [&](const uint4 *lds, const float *terms) {
        if (MODE == WALK_STATS) {
#pragma unroll 2
            for (int sub = 0; sub < SUB; ++sub) {
                const v16f d = scores(lds + sub * PART * NS, terms + sub * 32);
                reads_ahead<STEPS * NS, STEPS * (2 * NS - 1)>();
                online(d, NS == 2 ? 1.f : p.c, m, sum);
            }
            return;
        }
        // probabilities of a tile (times G for the items' side), as the operand of the second product: two parts in either type, since a
        // gradient is the difference of this product and the named items' rows, and only what P keeps is left of a user who is nearly
        // sure of its item.  bf16: hi + lo is off by at most 2^-16 of P, and near 1 by 2^-8 of 1 - P (one part lost such rows whole).
        // fp32: 22 bits, or an absolute step of 2^-39 of the largest of a S row's 32 elements.  That power of two is the tile's and the row's
        // own, taken off where the tile's product is added to the sums in fp32, so that neither an unlikely item nor one beside a user of
        // large G loses bits
        struct Operand { uint4 part[2][2]; float back; };
        auto probabilities = [&](const v16f &d, int sub) {
            float P[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) P[r] = exp2_raw(NS == 2 ? d[r] + s_term : fmaf(d[r], p.c, s_term));
            if (ITEMS) {
                {   // products rounded by themselves: dV has the same bits with and without db beside it
#pragma clang fp contract(off)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4 tg = *(const float4 *)(terms + ROWS + sub * 32 + 8 * q + 4 * h);
                        P[4 * q] *= tg.x; P[4 * q + 1] *= tg.y; P[4 * q + 2] *= tg.z; P[4 * q + 3] *= tg.w;
                    }
                }
                if (MODE == WALK_ITEMS_BASE) {
                    float b = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) b += P[r];
                    b_sum += b;
                }
            }
            Operand o;
            o.back = 1.f;
            if (NS == 2) {
                // times the T rows' powers of two, 2^-e (their parts are scaled by the inverse; G brings the 2^24 that they leave out); then
                // the S row's 32 elements (16 here, 16 in lane + or - 32) by the power of two that brings the largest to [2^14, 2^15)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    constexpr float REST = ITEMS ? 1.f : 16777216.f;
                    const float4 u4 = *(const float4 *)(terms + 2 * ROWS + sub * 32 + 8 * q + 4 * h);
                    P[4 * q] *= u4.x * REST; P[4 * q + 1] *= u4.y * REST; P[4 * q + 2] *= u4.z * REST; P[4 * q + 3] *= u4.w * REST;
                }
                float top = fabsf(P[0]);
#pragma unroll
                for (int r = 1; r < 16; ++r) top = fmaxf(top, fabsf(P[r]));
                const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                const uint32_t field = max(max((uint32_t)both[0], (uint32_t)both[1]) >> 23, 15u);
                const float up = __uint_as_float((268u - field) << 23);
                o.back = __uint_as_float((field - 14u) << 23);
#pragma unroll
                for (int r = 0; r < 16; ++r) P[r] *= up;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                typename std::conditional<NS == 1, b8, h8>::type hi, lo;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    hi[j] = (E)P[8 * e + j];
                    lo[j] = (E)(P[8 * e + j] - (float)hi[j]);
                }
                o.part[0][e] = __builtin_bit_cast(uint4, hi);
                o.part[1][e] = __builtin_bit_cast(uint4, lo);
            }
            return o;
        };
        // their product with the tile's rows: hi hi, hi lo and, where the rows have two parts, lo hi
        auto add_product = [&](const uint4 *l1, const Operand &o) {
#pragma unroll
            for (int kb = 0; kb < KP / 32; kb += ABREAST) {
                v16f part[ABREAST] = {};
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint4 a[ABREAST][NS];
#pragma unroll
                    for (int j = 0; j < ABREAST; ++j)
#pragma unroll
                        for (int q = 0; q < NS; ++q)
                            if (kb + j < KP / 32) {
                                const char *l2 = (const char *)(l1 + q * PART) + (kb + j) * 2048 + e * 512;
                                a[j][q] = turned(l2 + at2, l2 + at2_high);
                            }
#pragma unroll
                    for (int q = 0; q < NS + 1; ++q)
#pragma unroll
                        for (int j = 0; j < ABREAST; ++j)
                            if (kb + j < KP / 32) {
                                v16f &to = NS == 2 ? part[j] : acc[kb + j];
                                to = product<NS>(a[j][q >> 1], o.part[q & 1][e], to);
                            }
                }
                if (NS == 2) {
#pragma unroll
                    for (int j = 0; j < ABREAST; ++j)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (kb + j < KP / 32) acc[kb + j][r] = fmaf(part[j][r], o.back, acc[kb + j][r]);
                }
            }
        };
        v16f next = scores(lds, terms);
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
            const v16f d = next;
            if (sub + 1 < SUB) next = scores(lds + (sub + 1) * PART * NS, terms + (sub + 1) * 32);
            add_product(lds + sub * PART * NS, probabilities(d, sub));
        }
    };
    auto arrived = [&]() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };

    if (first < last) fetch_stage(first, stage0, terms0);
    for (int t = first; t < last; t += 2 * SUB) {
        arrived();
        if (t + SUB < last) fetch_stage(t + SUB, stage1, terms1);
        compute(stage0, terms0);
        if (t + SUB >= last) break;
        arrived();
        if (t + 2 * SUB < last) fetch_stage(t + 2 * SUB, stage0, terms0);
        compute(stage1, terms1);
    }

    const int64_t at = (int64_t)split * p.s_padded + s_row;
    if (MODE == WALK_STATS) {
        // lane and lane + 32 hold the same S row
        const float m2 = __shfl_xor(m, 32), s2 = __shfl_xor(sum, 32), top = fmaxf(m, m2);
        sum = sum * exp2_raw(m - top) + s2 * exp2_raw(m2 - top);
        if (h == 0) { p.out_m[at] = top; p.out_s[at] = sum; }
        return;
    }
    // split: G, and with it the sum for db, is 2^24 times itself
    b_sum = (b_sum + __shfl_xor(b_sum, 32)) * (NS == 2 ? 1.f / 16777216.f : 1.f);
    if (MODE == WALK_USERS) {
        for (int kb = 0; kb < KP / 32; ++kb)
            for (int q = 0; q < 4; ++q)
                *(float4 *)(p.out_acc + at * KP + kb * 32 + 8 * q + 4 * h) =
                    make_float4(acc[kb][4 * q], acc[kb][4 * q + 1], acc[kb][4 * q + 2], acc[kb][4 * q + 3]);
        return;
    }
    // dV: the places of the users walked are added here, to 64 rows a time (waves 0 and 1, then 2 and 3) whose sums lie in the first stage's
    // memory; one split finishes the rows, more leave parts of the gradient for join_kernel
    __shared__ float row_b[64], aside[aside_floats(KP)];
    __shared__ int counts[4], aside_item[32];
    static_assert(MODE == WALK_STATS || STAGE * 16 >= 64 * KP * 4, "a stage holds 64 rows of sums");
    static_assert(MODE == WALK_STATS || STAGE * 16 >= list_length(KP) * 12, "a stage holds a list and its order");
    float *rows = (float *)stage0;
    uint32_t *list = (uint32_t *)stage1;
    const int64_t i0 = (int64_t)s_block * S_ROWS;
    const Finish &f = p.f;
    __syncthreads();
    const int64_t from_place = first * 32ll * f.m, to_place = min(last * 32ll * f.m, f.n_places);
    const bool any = from_place < to_place && (!f.named || f.named[i0 >> 6] || f.named[(i0 >> 6) + 1]);
    auto lay = [&](int half) {                        // the sums of 64 items
        __syncthreads();
        if ((wave >> 1) == half) {
            const int r = (wave & 1) * 32 + (lane & 31);
            for (int kb = 0; kb < KP / 32; ++kb)
                for (int q = 0; q < 4; ++q)
                    *(float4 *)(rows + r * KP + kb * 32 + 8 * q + 4 * h) =
                        make_float4(-acc[kb][4 * q], -acc[kb][4 * q + 1], -acc[kb][4 * q + 2], -acc[kb][4 * q + 3]);
            if (h == 0) row_b[r] = -b_sum;
        }
        __syncthreads();
    };
    auto leave = [&](int half) {
        if (p.out_acc) {
            const int64_t to_row = (int64_t)split * p.s_padded + i0 + half * 64;
            for (int i = threadIdx.x; i < 64 * KP / 4; i += 256) ((float4 *)(p.out_acc + to_row * KP))[i] = ((const float4 *)rows)[i];
            if (p.out_b && threadIdx.x < 64) p.out_b[to_row + threadIdx.x] = row_b[threadIdx.x];
        } else {
            store_rows<T, KP>(f, rows, row_b, i0 + half * 64);
        }
    };
    if (!any) {                                       // nothing to add: no register is put aside for it
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
            lay(half);
            leave(half);
        }
        return;
    }
    // the places of all 128 items are found at once; where the lists do not hold them, those of 64 at a time in as many rounds as it takes
    bool find = true, at_once = true, more = false, fresh = true;
    int64_t step = -1;
    int total = 0, lower = 0;                         // of the sorted order: where the second half's items begin
#pragma unroll 1
    for (int half = 0; half < 2;) {
        if (fresh) {
            lay(half);
            fresh = false;
        }
        if (find) {
            total = find_places<KP>(f, list, counts, (uint8_t *)aside, at_once ? i0 : i0 + half * 64, at_once ? 128 : 64, from_place, to_place, step, more);
            if (at_once && more) {
                at_once = false;
                step = -1;
                __syncthreads();
                continue;
            }
            find = false;
            lower = 0;
            for (int hi = total; at_once && lower < hi;) {
                const int mid = (lower + hi) / 2;
                if (list[2 * list_length(KP) + mid] >> 12 < 64) lower = mid + 1;
                else hi = mid;
            }
        }
        const int from = at_once && half ? lower : 0, to = at_once && !half ? lower : total;
        if (from < to) add_places<T, KP>(f, rows, row_b, list, aside, aside_item, at_once ? half * 64 : 0, from, to);
        if (!at_once && more) {
            find = true;
            continue;
        }
        leave(half);
        ++half;
        fresh = true;
        find = !at_once;
        step = -1;
    }
}

// The statistics for few users, straight from V as it lies in memory: a wave takes 16 items at a time, its lanes 16 rows by four
// pieces of 16 bytes, which are the A operands of the 16 x 16 instructions (fp32: 16x16x4, a piece feeds four of them; bf16: 16x16x32).
// The order of the factors is the same in X's operand, so it does not matter.  V is read once for 16 UT users, the next tile's rows
// are on their way while one is computed: HBM-bound (fp32, one user x 1 000 000 x 128: 512 MB in 100 us, 5.1 TB/s; a sum over as much by
// the library 3.95 TB/s).  The first form, the walk after V had been put in its
// order, took 1650 us for this call.
struct DirectParams {
    const void *X, *V;
    const float *ibase;
    int64_t ldx, ldv, n, n_items, s_padded;
    int k;
    float c;
    float *out_m, *out_s;              // [workgroups][s_padded]
};

typedef float v4f __attribute__((ext_vector_type(4)));

template <typename T, bool VEC>
__device__ __forceinline__ uint4 piece(const T *row, int c, int k)
{
    constexpr int N = 16 / sizeof(T);
    if (VEC) return c < k ? *(const uint4 *)(row + c) : make_uint4(0, 0, 0, 0);
    T v[N];
    for (int j = 0; j < N; ++j) v[j] = c + j < k ? row[c + j] : (T)0.f;
    uint4 o;
    __builtin_memcpy(&o, v, 16);
    return o;
}

// workgroups of direct_kernel a compute unit holds by its registers: the tile, the next one and UT users' operand, and what else there is
constexpr int direct_resident(int KP, int UT, int size)
{
    const int r = (UT + 2) * KP * size / 16 + (size == 4 ? 36 : 60);
    return r <= 132 ? 4 : r <= 168 ? 3 : r <= 256 ? 2 : 1;
}

template <typename T, int KP, int UT, bool VEC>
__global__ __launch_bounds__(256, direct_resident(KP, UT, sizeof(T))) void direct_kernel(DirectParams p)
{
    constexpr int N = 16 / sizeof(T), STEPS = KP / (4 * N);
    __shared__ float lm[4][UT * 16], ls[4][UT * 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int64_t u0 = (int64_t)blockIdx.y * UT * 16;
    const T *X = (const T *)p.X, *V = (const T *)p.V;
    uint4 b[UT][STEPS];
#pragma unroll
    for (int t = 0; t < UT; ++t)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) b[t][s] = piece<T, VEC>(X + min(u0 + t * 16 + r, p.n - 1) * p.ldx, (s * 4 + g) * N, p.k);
    float m[UT], sum[UT];
    for (int t = 0; t < UT; ++t) { m[t] = -3.402823466e38f; sum[t] = 0.f; }
    const int64_t tiles = (p.n_items + 15) / 16, stride = (int64_t)gridDim.x * 4;
    int64_t i = (int64_t)blockIdx.x * 4 + wave;
    uint4 a[STEPS];
    float base[4];
    auto load = [&](int64_t tile, uint4 *to, float *bases) {
        const T *row = V + min(tile * 16 + r, p.n_items - 1) * p.ldv;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) to[s] = piece<T, VEC>(row, (s * 4 + g) * N, p.k);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t item = tile * 16 + 4 * g + e;
            bases[e] = item < p.n_items ? (p.ibase ? p.ibase[item] * p.c : 0.f) : -INFINITY;
        }
    };
    if (i < tiles) load(i, a, base);
    for (; i < tiles; i += stride) {
        uint4 next[STEPS];
        float next_base[4];
        if (i + stride < tiles) load(i + stride, next, next_base);
#pragma unroll
        for (int t = 0; t < UT; ++t) {
            v4f d = {};
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                if (sizeof(T) == 4) {
                    const v4f x = __builtin_bit_cast(v4f, a[s]), y = __builtin_bit_cast(v4f, b[t][s]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) d = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], d, 0, 0, 0);
                } else {
                    d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a[s]), __builtin_bit_cast(b8, b[t][s]), d, 0, 0, 0);
                }
            }
            float z[4], top = m[t];
#pragma unroll
            for (int e = 0; e < 4; ++e) { z[e] = fmaf(d[e], p.c, base[e]); top = fmaxf(top, z[e]); }
            float add = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) add += exp2_raw(z[e] - top);
            sum[t] = fmaf(sum[t], exp2_raw(m[t] - top), add);
            m[t] = top;
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) a[s] = next[s];
        for (int e = 0; e < 4; ++e) base[e] = next_base[e];
    }
#pragma unroll
    for (int t = 0; t < UT; ++t) {
        for (int o = 16; o < 64; o <<= 1) {
            const float m2 = __shfl_xor(m[t], o), s2 = __shfl_xor(sum[t], o), top = fmaxf(m[t], m2);
            sum[t] = sum[t] * exp2_raw(m[t] - top) + s2 * exp2_raw(m2 - top);
            m[t] = top;
        }
        if (g == 0) { lm[wave][t * 16 + r] = m[t]; ls[wave][t * 16 + r] = sum[t]; }
    }
    __syncthreads();
    if (threadIdx.x < UT * 16) {
        const int q = threadIdx.x;
        const float top = fmaxf(fmaxf(lm[0][q], lm[1][q]), fmaxf(lm[2][q], lm[3][q]));
        const float all = (ls[0][q] * exp2_raw(lm[0][q] - top) + ls[1][q] * exp2_raw(lm[1][q] - top)) +
                          (ls[2][q] * exp2_raw(lm[2][q] - top) + ls[3][q] * exp2_raw(lm[3][q] - top));
        p.out_m[blockIdx.x * p.s_padded + u0 + q] = top;
        p.out_s[blockIdx.x * p.s_padded + u0 + q] = all;
    }
}

// The same statistics from 4-bit operands: a lane of the instruction holds one block of 32 of a row and its scale, as it lies in
// memory.  A wave keeps UT tiles of 32 users (B operand) and walks item tiles of 32, the next one's codes on their way; the bases are
// the initial value of the sums.  Bound by the exponentials (v_exp_f32 at a quarter of the rate of the rest) and the maxima and sums
// beside them: 2048 x 125 000 x 128 in 63 us, 256 M exponentials at 26 us of issue, the vector unit busy in 88 % of the cycles.  Four user
// tiles a wave: one item tile's loads and scales serve 128 users (the first form had one and took 145 us).
struct MxWalkParams {
    const uint8_t *xc, *xs, *vc, *vs;
    const float *base;                 // ibase or null
    int64_t n, n_items, s_padded;
    int kb, t_tiles, tiles_per_split;
    float c;
    float *out_m, *out_s;
};

template <int STEPS, int UT>
__global__ __launch_bounds__(256, STEPS <= 2 ? 3 : 2) void walk_mx_kernel(MxWalkParams p)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
    const int64_t s0 = (int64_t)blockIdx.x * 32 * UT;
    v8i x[UT][STEPS];
    int sx[UT][STEPS];
    auto block_of = [&](const uint8_t *codes, const uint8_t *scales, int64_t row, int s, uint4 *c, int *scale) {
        const int b = 2 * s + h;
        *c = make_uint4(0, 0, 0, 0);
        *scale = 127;
        if (b < p.kb) {
            *c = *(const uint4 *)(codes + (row * p.kb + b) * 16);
            *scale = scales[row * p.kb + b];
        }
    };
#pragma unroll
    for (int t = 0; t < UT; ++t)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            uint4 c;
            block_of(p.xc, p.xs, min(s0 + t * 32 + r, p.n - 1), s, &c, &sx[t][s]);
            x[t][s] = v8i{(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0};
        }
    float m[UT], sum[UT];
#pragma unroll
    for (int t = 0; t < UT; ++t) { m[t] = -3.402823466e38f; sum[t] = 0.f; }
    const int split = blockIdx.y * 4 + wave;          // each wave walks items of its own
    const int first = split * p.tiles_per_split, last = min(first + p.tiles_per_split, p.t_tiles);
    const bool base_vec = p.base && ((uintptr_t)p.base & 15) == 0;
    uint4 a[STEPS];
    int sa[STEPS];
    float4 base[4];
    auto load = [&](int t, uint4 *to, int *scale, float4 *bases) {
        const int64_t item = min((int64_t)t * 32 + r, p.n_items - 1);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) block_of(p.vc, p.vs, item, s, &to[s], &scale[s]);
        if (base_vec && (t + 1) * 32ll <= p.n_items) {
#pragma unroll
            for (int q = 0; q < 4; ++q) bases[q] = *(const float4 *)(p.base + (int64_t)t * 32 + 8 * q + 4 * h);
        } else {
            float b[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int64_t i = (int64_t)t * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
                b[e] = i < p.n_items ? (p.base ? p.base[i] : 0.f) : -INFINITY;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) bases[q] = make_float4(b[4 * q], b[4 * q + 1], b[4 * q + 2], b[4 * q + 3]);
        }
    };
    if (first < last) load(first, a, sa, base);
    for (int t = first; t < last; ++t) {
        uint4 a2[STEPS];
        int sa2[STEPS];
        float4 base2[4];
        if (t + 1 < last) load(t + 1, a2, sa2, base2);
        v8i w[STEPS];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) w[s] = v8i{(int)a[s].x, (int)a[s].y, (int)a[s].z, (int)a[s].w, 0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < UT; ++u) {
            v16f d;
#pragma unroll
            for (int q = 0; q < 4; ++q) { d[4 * q] = base[q].x; d[4 * q + 1] = base[q].y; d[4 * q + 2] = base[q].z; d[4 * q + 3] = base[q].w; }
#pragma unroll
            for (int s = 0; s < STEPS; ++s) d = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[s], x[u][s], d, 4, 4, 0, sa[s], 0, sx[u][s]);
            online(d, p.c, m[u], sum[u]);
        }
#pragma unroll
        for (int s = 0; s < STEPS; ++s) { a[s] = a2[s]; sa[s] = sa2[s]; }
#pragma unroll
        for (int q = 0; q < 4; ++q) base[q] = base2[q];
    }
#pragma unroll
    for (int u = 0; u < UT; ++u) {
        const float top0 = m[u] , m2 = __shfl_xor(top0, 32), s2 = __shfl_xor(sum[u], 32), top = fmaxf(top0, m2);
        const float all = sum[u] * exp2_raw(top0 - top) + s2 * exp2_raw(m2 - top);
        const int64_t at = (int64_t)split * p.s_padded + s0 + u * 32 + r;
        if (h == 0) { p.out_m[at] = top; p.out_s[at] = all; }
    }
}

// ---------------------------------------------------------------------------- joins

// What the last kernel of the forward pass reads: the splits' maxima and sums, and the model for the scores of the named items.
struct Targets {
    const float *m, *s;
    int64_t s_padded;
    int splits, k, kb;
    const void *X, *V;                 // fp32, bf16, or the codes
    const uint8_t *xs, *vs;
    int64_t ldx, ldv, n_items;
    const float *ibase;
    float scale;
    const int32_t *ids;
    int64_t places, ld_ids, ld_logp;
    float *lse, *logp;
};

// e times the two scales' powers of two at once (one alone may leave fp32); NaN where a scale stands for it
__device__ __forceinline__ float mx_scaled(float e, int a, int b)
{
    return a == 255 || b == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(e, a + b - 254);
}

// lane l of 16: its share of <x, v>
template <typename T>
__device__ __forceinline__ float dot_share(const Targets &t, int64_t u, int64_t id, int l)
{
    const T *x = (const T *)t.X + u * t.ldx, *v = (const T *)t.V + id * t.ldv;
    float d = 0.f;
#pragma unroll 4
    for (int c = l; c < t.k; c += 16) d = fmaf(as_f32(x[c]), as_f32(v[c]), d);
    return d;
}

// ... of a 4-bit model: 8 columns a lane and step.  Sums of products of the grid are exact, the scales powers of two.
struct Mx {};
template <>
__device__ __forceinline__ float dot_share<Mx>(const Targets &t, int64_t u, int64_t id, int l)
{
    const uint32_t *x = (const uint32_t *)t.X + u * t.kb * 4, *v = (const uint32_t *)t.V + id * t.kb * 4;
    float d = 0.f;
#pragma unroll 2
    for (int c = l; c < t.kb * 4; c += 16) {
        const uint32_t a = x[c], b = v[c];
        const v2f a0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 1.0f, 0), b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 0);
        const v2f a1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 1.0f, 1), b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 1);
        const v2f a2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 1.0f, 2), b2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 2);
        const v2f a3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(a, 1.0f, 3), b3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(b, 1.0f, 3);
        const float e = a0[0] * b0[0] + a0[1] * b0[1] + a1[0] * b1[0] + a1[1] * b1[1] + a2[0] * b2[0] + a2[1] * b2[1] + a3[0] * b3[0] + a3[1] * b3[1];
        d += mx_scaled(e, t.xs[u * t.kb + (c >> 2)], t.vs[id * t.kb + (c >> 2)]);
    }
    return d;
}

// A workgroup a user: lse from the splits, then logp of the named items, 16 lanes a place (the score as one fp32 sum over the
// factors).  Bound by the latency of its gathers (2048 users x 20 places, 200 columns: 9 us).
template <typename T>
__global__ __launch_bounds__(256) void targets_kernel(Targets t)
{
    __shared__ float lm[4], ls[4];
    const int64_t u = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = threadIdx.x & 15;
    float top = -3.402823466e38f, sum = 0.f;
    for (int q = threadIdx.x; q < t.splits; q += 256) {
        const float a = t.m[q * t.s_padded + u], both = fmaxf(top, a);
        sum = sum * exp2f(top - both) + t.s[q * t.s_padded + u] * exp2f(a - both);
        top = both;
    }
    for (int o = 32; o; o >>= 1) {
        const float a = __shfl_xor(top, o), r = __shfl_xor(sum, o), both = fmaxf(top, a);
        sum = sum * exp2f(top - both) + r * exp2f(a - both);
        top = both;
    }
    if (lane == 0) { lm[wave] = top; ls[wave] = sum; }
    __syncthreads();
    top = fmaxf(fmaxf(lm[0], lm[1]), fmaxf(lm[2], lm[3]));
    sum = (ls[0] * exp2f(lm[0] - top) + ls[1] * exp2f(lm[1] - top)) + (ls[2] * exp2f(lm[2] - top) + ls[3] * exp2f(lm[3] - top));
    const float lse = (float)(((double)top + (double)log2f(sum)) * LN2);
    if (threadIdx.x == 0 && t.lse) t.lse[u] = lse;
    for (int64_t j = threadIdx.x >> 4; j < t.places; j += 16) {
        const int32_t id = t.ids[u * t.ld_ids + j];
        float out = 0.f;
        if (id >= t.n_items) {
            out = __uint_as_float(0x7fc00000u);
        } else if (id >= 0) {
            float d = dot_share<T>(t, u, id, l);
            for (int o = 8; o; o >>= 1) d += __shfl_xor(d, o);
            const float z = t.scale * (d + (t.ibase ? t.ibase[id] : 0.f));
            out = lse == -INFINITY ? -INFINITY : z - lse;
        }
        if (l == 0) t.logp[u * t.ld_logp + j] = out;
    }
}

// dX = scale (sum over the places of g v - G acc): four columns a thread, so that a user's row of V is read in long pieces.  Bound by the
// splits' sums and the gathers of V (2048 x 200, 20 places, 16 splits: 16 us, 46 MB).
struct JoinDx {
    const float *acc, *G;
    const void *V;
    const int32_t *ids;
    const float *dlogp;
    void *dX;
    int64_t s_padded, ldv, n_items, m, ld_ids, ld_dlogp, n, ld_dx;
    int splits, KP, k, vec_v;
    float scale;
    int64_t blocks;                    // workgroups it takes (none without dX)
};

template <typename T>
__device__ __forceinline__ void join_dx(const JoinDx &p, int64_t block)
{
    const int64_t at = block * 256 + threadIdx.x;
    const int64_t u = at / (p.KP / 4);
    const int c = (int)(at - u * (p.KP / 4)) * 4;
    if (u >= p.n || c >= p.k) return;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int q = 0; q < p.splits; ++q) {
        const float4 v = *(const float4 *)(p.acc + ((int64_t)q * p.s_padded + u) * p.KP + c);
        a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
    const float g0 = -p.G[u];
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    if (g0 != 0.f) { r[0] = g0 * a.x; r[1] = g0 * a.y; r[2] = g0 * a.z; r[3] = g0 * a.w; }      // (NaN != 0)
#pragma unroll 4
    for (int64_t j = 0; j < p.m; ++j) {
        const int32_t id = p.ids[u * p.ld_ids + j];
        if (id < 0 || id >= p.n_items) continue;
        const float g = p.dlogp[u * p.ld_dlogp + j];
        float v[4];
        load4((const T *)p.V + (int64_t)id * p.ldv, c, p.k, p.vec_v, v);
        for (int e = 0; e < 4; ++e) r[e] = fmaf(g, v[e], r[e]);
    }
    T *out = (T *)p.dX + u * p.ld_dx;
    for (int e = 0; e < 4; ++e)
        if (c + e < p.k) out[c + e] = (T)(p.scale * r[e]);
}

template <typename T>
__global__ __launch_bounds__(256) void join_dx_kernel(JoinDx p) { join_dx<T>(p, blockIdx.x); }

// dV and db where the walk was split (few items, many users): the sum of the splits' parts, four columns a thread.  The first x.blocks
// workgroups do dX: one launch for both, since each is a few microseconds.  Latency-bound.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(JoinDx x, const float *acc, const float *acc_b, int splits, int64_t s_padded, int KP, Finish f)
{
    if (blockIdx.x < x.blocks) {
        join_dx<T>(x, blockIdx.x);
        return;
    }
    const int64_t at = (blockIdx.x - x.blocks) * 256ll + threadIdx.x, i = at / (KP / 4);
    const int c = (int)(at - i * (KP / 4)) * 4;
    if (i >= f.n_items) return;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int q = 0; q < splits; ++q) {
        const float4 v = *(const float4 *)(acc + ((int64_t)q * s_padded + i) * KP + c);
        a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
    store4<T>(f, i, c, a);
    if (c == 0 && f.db) {
        float b = 0.f;
        for (int q = 0; q < splits; ++q) b += acc_b[(int64_t)q * s_padded + i];
        f.db[i] = f.scale * b;
    }
}

// ---------------------------------------------------------------------------- launches

namespace {

// the walks may read both matrices as they lie: bf16, no column missing to a multiple of 32, rows at 16-byte borders
bool rows_lie(const ifr_catalogue &c)
{
    return c.dtype == IFR_BF16 && c.k % 32 == 0 && c.ldx % 8 == 0 && c.ldv % 8 == 0 && (((uintptr_t)c.X | (uintptr_t)c.V) & 15) == 0;
}

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

// Splits of the T axis: the count with the shortest plan, in stages: rounds of resident workgroups times (a split's stages + what a
// workgroup costs besides, about four), plus what joining costs where there is more than one.  2048 users x 26 744 items leave 16
// workgroups without a split of dX and take 16 splits; dV's 209 workgroups take none, since five (two rounds and a join) cost more.
struct Split { int count, per; };

Split split_plan(int64_t s_blocks, int64_t t_tiles, int unit, int64_t resident, double join, double places = 0.0)
{
    const int64_t stages = (t_tiles + unit - 1) / unit;
    int64_t best = 1;
    double best_cost = 0;
    for (int64_t c = 1; c <= stages && c <= 4096; c = c < 16 ? c + 1 : c + c / 8) {
        const int64_t per = (stages + c - 1) / c;
        const double cost = (double)((s_blocks * c + resident - 1) / resident) * ((double)per + 4.0 + places / (double)(s_blocks * c)) + (c > 1 ? join * (double)c : 0.0);
        if (c == 1 || cost < best_cost) { best = c; best_cost = cost; }
    }
    Split s;
    s.per = (int)((stages + best - 1) / best) * unit;
    s.count = (int)((t_tiles + s.per - 1) / s.per);
    return s;
}

struct Side {                          // one matrix as the walks read it
    int64_t rows, tiles, padded;       // tiles of 32 rows; padded: rows up to whole S blocks
    bool lies;                         // bf16 rows of whole, aligned pieces: read as they lie
    float *units;
    uint4 *frag;
};

Side side(Pieces &w, const ifr_catalogue &c, bool users, bool lies)
{
    Side s;
    const int KP = pad_factors(c.k), NS = c.dtype == IFR_F32 ? 2 : 1;
    s.rows = users ? c.n : c.n_items;
    s.padded = up(s.rows, S_ROWS);
    s.tiles = s.padded / 32;
    s.lies = lies;
    s.units = w.take<float>(NS == 2 ? s.padded + 32 : 0);      // a fetch brings 64, also where a stage holds 32 rows
    s.frag = w.take<uint4>(s.lies ? 0 : s.tiles * NS * (KP / 16) * 64);
    return s;
}

template <typename T>
void launch_prepare(const PrepParams &p, int64_t x_tiles, hipStream_t s)
{
    constexpr int NS = sizeof(T) == 4 ? 2 : 1;
    hipLaunchKernelGGL((prepare_kernel<T, NS>), dim3((uint32_t)(p.v_blocks + x_tiles)), dim3(256), 32 * (p.KP + 1) * sizeof(float), s, p);
}

#define IFR_FOR_FACTORS(KP, CALL)                                                                                     \
    switch (KP) {                                                                                                     \
    case 32: CALL(32); break;                                                                                         \
    case 64: CALL(64); break;                                                                                         \
    case 96: CALL(96); break;                                                                                         \
    case 128: CALL(128); break;                                                                                       \
    case 160: CALL(160); break;                                                                                       \
    case 192: CALL(192); break;                                                                                       \
    case 224: CALL(224); break;                                                                                       \
    default: CALL(256); break;                                                                                        \
    }

template <int NS, int MODE>
void launch_walk(const WalkParams &p, int KP, hipStream_t s)
{
    const dim3 grid((uint32_t)(p.s_blocks * p.splits));
    const bool lies = !(MODE >= WALK_ITEMS ? p.s_frag : p.t_frag);
#define IFR_WALK(K)                                                                                                   \
    if (NS == 1 && lies) hipLaunchKernelGGL((walk_kernel<K, NS, MODE, NS == 1 && MODE != WALK_USERS, NS == 1 && MODE < WALK_ITEMS>), grid, dim3(256), 0, s, p); \
    else hipLaunchKernelGGL((walk_kernel<K, NS, MODE, false, false>), grid, dim3(256), 0, s, p)
    IFR_FOR_FACTORS(KP, IFR_WALK)
#undef IFR_WALK
}

int resident_blocks(int KP, int NS, int mode) { return mode == WALK_STATS || paired(KP, NS, mode) ? 512 : 256; }

// Users one pass over V serves (their operand stays in registers: at most 128 of them), and up to how many users the direct kernel is taken.
int direct_tiles(int KP, int64_t n) { return n <= 16 ? 1 : n <= 32 || KP > 128 ? 2 : 4; }

struct ForwardPlan {
    bool direct;
    Side x, v;
    float *term, *out_m, *out_s;
    Split split;
    int64_t s_padded, t_padded;
    int mx_users;                      // user tiles of a wave, 4-bit model
};

// The direct kernel is taken for what one pass over V serves.  Beyond, the walk is as fast where V needs no other order (bf16 1 000 000 x
// 128, 70 users: 66 us, 113 us in two passes) and faster where it does (fp32, 70 users: 374 us by the walk, 460 us in two passes).
int64_t direct_users(const ifr_catalogue &c) { return 16 * (pad_factors(c.k) > 128 ? 2 : 4); }

ForwardPlan forward_plan(Pieces &w, const ifr_catalogue &c, bool lies)
{
    ForwardPlan p = {};
    const int KP = pad_factors(c.k), NS = c.dtype == IFR_F32 ? 2 : 1;
    p.s_padded = up(c.n, S_ROWS);
    p.t_padded = up(c.n_items, S_ROWS);
    p.direct = c.dtype != IFR_MXFP4 && c.n <= direct_users(c);
    if (p.direct) {
        const int64_t want = (c.n_items + 63) / 64;
        const int64_t most = 256 * direct_resident(KP, direct_tiles(KP, c.n), c.dtype == IFR_F32 ? 4 : 2);      // one round of them
        p.split.count = (int)(want < most ? want : most);
        p.out_m = w.take<float>(p.split.count * p.s_padded);
        p.out_s = w.take<float>(p.split.count * p.s_padded);
        return p;
    }
    if (c.dtype != IFR_MXFP4) {
        p.x = side(w, c, true, lies);
        p.v = side(w, c, false, lies);
    }
    if (c.dtype == IFR_MXFP4) {                       // waves walk alone: 16 a compute unit, none with fewer than two tiles
        p.mx_users = c.n > 64 ? 4 : c.n > 32 ? 2 : 1;
        const int64_t s_tiles = (c.n + 32 * p.mx_users - 1) / (32 * p.mx_users), tiles = p.t_padded / 32;
        int64_t waves = (4096 + s_tiles - 1) / s_tiles;
        waves = waves < tiles / 2 ? waves : (tiles / 2 > 0 ? tiles / 2 : 1);
        p.split.per = (int)((tiles + waves - 1) / waves);
        p.split.count = (int)up((tiles + p.split.per - 1) / p.split.per, 4);
    } else {
        p.split = split_plan(p.s_padded / S_ROWS, p.t_padded / 32, stage_tiles(NS, false), resident_blocks(KP, NS, WALK_STATS), 0.0);
    }
    p.term = w.take<float>(c.dtype == IFR_MXFP4 ? 0 : p.t_padded + 32);         // a fetch brings 64, also where a stage holds 32 rows
    p.out_m = w.take<float>(p.split.count * p.s_padded);
    p.out_s = w.take<float>(p.split.count * p.s_padded);
    return p;
}

struct BackwardPlan {
    Side x, v;
    float *item_term, *user_term, *G, *G_scaled, *acc_x, *acc_v, *acc_b;
    int32_t *places;
    uint8_t *named;
    int64_t places_padded;
    Deal deal;                         // places dealt into buckets, or places null
    Split split_x, split_v;
};

// Places are dealt into buckets where the workgroups' looking through all of them takes longer than the dealing: with 524 288 places and
// 100 000 items dV takes 838 us dealt and 1164 us as they are, with 81 920 and 26 744 items 333 and 335 us.
bool deals(const ifr_catalogue &c, int64_t m, bool items) { return items && c.n * m >= DEAL_FROM && c.n * m < (int64_t)1 << 31 && c.n_items >= 16 * S_ROWS; }

BackwardPlan backward_plan(Pieces &w, const ifr_catalogue &c, int64_t m, bool dx, bool dv, bool db, bool lies)
{
    BackwardPlan p = {};
    const int KP = pad_factors(c.k), NS = c.dtype == IFR_F32 ? 2 : 1;
    const bool items = dv || db;
    p.x = side(w, c, true, false);
    p.v = side(w, c, false, lies);
    p.item_term = w.take<float>(p.v.padded);
    p.user_term = w.take<float>(p.x.padded);
    p.G = w.take<float>(p.x.padded);
    p.G_scaled = w.take<float>(NS == 2 ? p.x.padded : 0);
    p.places_padded = items ? up(c.n * m, CHUNK) : 0;
    p.places = w.take<int32_t>(p.places_padded);
    // flags save the search where most groups of 64 items are not named; where the places are as many as the groups, none is saved
    p.named = w.take<uint8_t>(p.places_padded && c.n_items > 64 * c.n * m ? up(p.v.padded / 64, 4) : 0);
    const int resident = resident_blocks(KP, NS, WALK_USERS);
    p.split_x = split_plan(p.x.padded / S_ROWS, p.v.tiles, stage_tiles(NS, true), resident, 0.05);
    // a hundred places take about as long as a stage, and so do the parts of a hundred blocks, written and read again
    const int64_t v_blocks = p.v.padded / S_ROWS;
    p.split_v = split_plan(v_blocks, p.x.tiles, stage_tiles(NS, true), resident, 0.1 + 0.01 * (double)v_blocks, items ? 0.01 * (double)(c.n * m) : 0.0);
    if (p.split_v.count == 1 && deals(c, m, items)) {
        Deal &d = p.deal;
        d.chunks = p.places_padded / CHUNK;
        d.n_items = c.n_items;
        d.bucket_items = up(up(c.n_items, S_ROWS) / S_ROWS, BUCKETS) / BUCKETS * S_ROWS;
        d.counts = w.take<uint32_t>(BUCKETS * d.chunks);
        d.bounds = w.take<uint32_t>(BUCKETS + 1);
        d.to = w.take<int32_t>(p.places_padded);
        d.place_of = w.take<uint32_t>(p.places_padded);
        d.places = p.places;
    }
    const bool parts = items && p.split_v.count > 1;
    p.acc_x = w.take<float>(dx ? p.split_x.count * p.x.padded * KP : 0);
    p.acc_v = w.take<float>(parts ? p.split_v.count * p.v.padded * KP : 0);
    p.acc_b = w.take<float>(db && parts ? p.split_v.count * p.v.padded : 0);
    return p;
}

}  // namespace

// The size does not depend on the matrices' addresses and strides: the larger of the two plans.
size_t logprob_workspace(const ifr_catalogue &c)
{
    Pieces a{nullptr}, b{nullptr};
    forward_plan(a, c, false);
    forward_plan(b, c, true);
    return a.used > b.used ? a.used : b.used;
}

size_t logprob_backward_workspace(const ifr_catalogue &c, int64_t m, bool want_dx, bool want_dv, bool want_db)
{
    Pieces a{nullptr}, b{nullptr};
    backward_plan(a, c, m, want_dx, want_dv, want_db, false);
    backward_plan(b, c, m, want_dx, want_dv, want_db, true);
    return a.used > b.used ? a.used : b.used;
}

static PrepParams prepare_sides(const ifr_catalogue &c, const Side &x, const Side &v, float *item_term)
{
    PrepParams p = {};
    p.V = c.V; p.X = c.X; p.ldv = c.ldv; p.ldx = c.ldx; p.n_items = c.n_items; p.n = c.n;
    p.v_blocks = v.lies ? (v.padded + 255) / 256 : v.tiles; p.v_padded = v.padded;
    p.k = c.k; p.KP = pad_factors(c.k);
    p.v_unit = v.units; p.x_unit = x.units; p.v_frag = v.frag; p.x_frag = x.frag;
    p.ibase = c.ibase; p.item_term = item_term;
    p.base_unit = c.dtype == IFR_F32 ? (float)(c.scale / LN2) : 1.f;
    p.lse_unit = c.dtype == IFR_F32 ? -LOG2E : (float)(-1.0 / c.scale);
    return p;
}

static void walk_sides(WalkParams &w, const ifr_catalogue &c, const Side &x, const Side &v, bool users_stay)
{
    const Side &s = users_stay ? x : v, &t = users_stay ? v : x;
    w.s_frag = s.frag; w.t_frag = t.frag; w.s_unit = s.units; w.t_unit = t.units; w.s_n = s.rows; w.t_n = t.rows;
    w.s_rows = (const __bf16 *)(users_stay ? c.X : c.V); w.t_rows = (const __bf16 *)(users_stay ? c.V : c.X);
    w.s_ld = users_stay ? c.ldx : c.ldv; w.t_ld = users_stay ? c.ldv : c.ldx;
    w.t_tiles = (int)((t.rows + 31) / 32); w.s_blocks = (int)(s.padded / S_ROWS); w.s_padded = s.padded;
}

template <typename T>
static void forward_typed(const ifr_catalogue &c, const ForwardPlan &p, hipStream_t s)
{
    constexpr int NS = sizeof(T) == 4 ? 2 : 1;
    launch_prepare<T>(prepare_sides(c, p.x, p.v, p.term), p.x.lies ? 0 : p.x.tiles, s);
    WalkParams w = {};
    walk_sides(w, c, p.x, p.v, true);
    w.t_term = p.term;
    w.c = (float)(c.scale / LN2); w.tiles_per_split = p.split.per; w.splits = p.split.count;
    w.out_m = p.out_m; w.out_s = p.out_s;
    launch_walk<NS, WALK_STATS>(w, pad_factors(c.k), s);
}

template <int STEPS>
static void launch_mx_users(const MxWalkParams &w, int users, dim3 grid, hipStream_t s)
{
    if (users == 1) hipLaunchKernelGGL((walk_mx_kernel<STEPS, 1>), grid, dim3(256), 0, s, w);
    else if (users == 2) hipLaunchKernelGGL((walk_mx_kernel<STEPS, 2>), grid, dim3(256), 0, s, w);
    else hipLaunchKernelGGL((walk_mx_kernel<STEPS, 4>), grid, dim3(256), 0, s, w);
}

static void launch_mx_walk(const ifr_catalogue &c, const ForwardPlan &p, hipStream_t s)
{
    const int kb = (c.k + 31) / 32;
    const MxWalkParams w = {(const uint8_t *)c.X, c.x_scales, (const uint8_t *)c.V, c.v_scales, c.ibase, c.n, c.n_items, p.s_padded, kb, (int)((c.n_items + 31) / 32),
                            p.split.per, (float)(c.scale / LN2), p.out_m, p.out_s};
    const dim3 grid((uint32_t)((c.n + 32 * p.mx_users - 1) / (32 * p.mx_users)), (uint32_t)(p.split.count / 4));
    if (kb <= 2) launch_mx_users<1>(w, p.mx_users, grid, s);
    else if (kb <= 4) launch_mx_users<2>(w, p.mx_users, grid, s);
    else if (kb <= 6) launch_mx_users<3>(w, p.mx_users, grid, s);
    else launch_mx_users<4>(w, p.mx_users, grid, s);
}

template <typename T, int KP, bool VEC>
static void launch_direct_tiles(const DirectParams &d, int tiles, int grid, hipStream_t s)
{
    const dim3 g((uint32_t)grid, (uint32_t)((d.n + tiles * 16 - 1) / (tiles * 16)));
    if (tiles == 1) hipLaunchKernelGGL((direct_kernel<T, KP, 1, VEC>), g, dim3(256), 0, s, d);
    else if (tiles == 2) hipLaunchKernelGGL((direct_kernel<T, KP, 2, VEC>), g, dim3(256), 0, s, d);
    else hipLaunchKernelGGL((direct_kernel<T, KP, (KP > 128 ? 2 : 4), VEC>), g, dim3(256), 0, s, d);
}

template <typename T>
static void launch_direct(const ifr_catalogue &c, const ForwardPlan &p, hipStream_t s)
{
    const int KP = pad_factors(c.k), tiles = direct_tiles(KP, c.n), N = 16 / sizeof(T);
    const bool vec = c.k % N == 0 && c.ldx % N == 0 && c.ldv % N == 0 && (((uintptr_t)c.X | (uintptr_t)c.V) & 15) == 0;
    const DirectParams d = {c.X, c.V, c.ibase, c.ldx, c.ldv, c.n, c.n_items, p.s_padded, c.k, (float)(c.scale / LN2), p.out_m, p.out_s};
#define IFR_DIRECT(K) vec ? launch_direct_tiles<T, K, true>(d, tiles, p.split.count, s) : launch_direct_tiles<T, K, false>(d, tiles, p.split.count, s)
    IFR_FOR_FACTORS(KP, IFR_DIRECT)
#undef IFR_DIRECT
}

int launch_logprob(const ifr_catalogue &c, const int32_t *ids, int64_t m, int64_t ld_ids, float *logp, int64_t ld_logp, float *lse,
                   void *ws, hipStream_t s)
{
    Pieces w{(char *)ws};
    const ForwardPlan p = forward_plan(w, c, rows_lie(c));
    const int kb = (c.k + 31) / 32;
    if (p.direct) {
        if (c.dtype == IFR_F32) launch_direct<float>(c, p, s);
        else launch_direct<__bf16>(c, p, s);
    } else {
        if (c.dtype == IFR_MXFP4) launch_mx_walk(c, p, s);
        else if (c.dtype == IFR_F32) forward_typed<float>(c, p, s);
        else forward_typed<__bf16>(c, p, s);
    }
    Targets t = {p.out_m, p.out_s, p.s_padded, p.split.count, c.k, kb, c.X, c.V, c.x_scales, c.v_scales, c.ldx, c.ldv, c.n_items, c.ibase, (float)c.scale,
                 ids, m, ld_ids, ld_logp, lse, logp};
    const dim3 grid((uint32_t)c.n);
    if (c.dtype == IFR_MXFP4) hipLaunchKernelGGL((targets_kernel<Mx>), grid, dim3(256), 0, s, t);
    else if (c.dtype == IFR_F32) hipLaunchKernelGGL((targets_kernel<float>), grid, dim3(256), 0, s, t);
    else hipLaunchKernelGGL((targets_kernel<__bf16>), grid, dim3(256), 0, s, t);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <typename T>
static void backward_typed(const ifr_catalogue &c, const int32_t *ids, int64_t m, int64_t ld_ids, const LogprobGrad &g, const BackwardPlan &p, hipStream_t s)
{
    constexpr int NS = sizeof(T) == 4 ? 2 : 1;
    const int KP = pad_factors(c.k);
    const float sc = (float)c.scale;
    const T *X = (const T *)c.X, *V = (const T *)c.V;
    auto fours = [&](const void *rows, int64_t ld) { return c.k % 4 == 0 && ld % 4 == 0 && ((uintptr_t)rows & (4 * sizeof(T) - 1)) == 0; };
    const bool items = g.dV || g.dibase;
    if (p.named) {
        const int64_t words = up(p.v.padded / 64, 4) / 4, want = (words + 255) / 256;
        hipLaunchKernelGGL(clear_kernel, dim3((uint32_t)(want < MAX_GRID ? want : MAX_GRID)), dim3(256), 0, s, (uint32_t *)p.named, words);
    }
    PrepParams pp = prepare_sides(c, p.x, p.v, p.item_term);
    pp.lse = g.lse; pp.dlogp = g.dlogp; pp.ids = ids; pp.m = m; pp.ld_ids = ld_ids; pp.ld_dlogp = g.ld_dlogp; pp.places_padded = p.places_padded;
    pp.user_term = p.user_term; pp.G = p.G; pp.G_scaled = p.G_scaled; pp.places = p.places; pp.named = p.named;
    launch_prepare<T>(pp, p.x.tiles, s);
    const bool dealt = p.deal.chunks > 0;
    if (dealt) {
        hipLaunchKernelGGL(deal_kernel<false>, dim3((uint32_t)p.deal.chunks), dim3(256), 0, s, p.deal);
        hipLaunchKernelGGL(deal_sums_kernel, dim3(1), dim3(1024), 0, s, p.deal);
        hipLaunchKernelGGL(deal_kernel<true>, dim3((uint32_t)p.deal.chunks), dim3(256), 0, s, p.deal);
    }
    WalkParams w = {};
    w.c = (float)(c.scale / LN2);
    JoinDx x = {};
    if (g.dX) {
        walk_sides(w, c, p.x, p.v, true);
        w.s_term = p.user_term; w.t_term = p.item_term; w.tiles_per_split = p.split_x.per; w.splits = p.split_x.count; w.out_acc = p.acc_x;
        launch_walk<NS, WALK_USERS>(w, KP, s);
        x = {p.acc_x, p.G, V, ids, g.dlogp, g.dX, p.x.padded, c.ldv, c.n_items, m, ld_ids, g.ld_dlogp, c.n, g.ld_dx, p.split_x.count, KP, c.k, fours(V, c.ldv), sc,
             (c.n * (KP / 4) + 255) / 256};
    }
    const bool parts = items && p.split_v.count > 1;
    if (items) {
        walk_sides(w, c, p.x, p.v, false);
        w.s_term = p.item_term; w.t_term = p.user_term; w.t_factor = NS == 2 ? p.G_scaled : p.G;
        w.tiles_per_split = p.split_v.per; w.splits = p.split_v.count;
        w.out_acc = parts ? p.acc_v : nullptr; w.out_b = p.acc_b;
        w.f = {dealt ? p.deal.to : p.places, p.named, X, g.dlogp, g.dV, g.dibase, dealt ? p.deal.place_of : nullptr, p.deal.bounds, p.deal.bucket_items, c.n * m, m, c.ldx, g.ld_dlogp, g.ld_dv, c.n_items, c.k, sc, fours(X, c.ldx), fours(g.dV, g.ld_dv)};
        if (NS == 2 || g.dibase) launch_walk<NS, WALK_ITEMS_BASE>(w, KP, s);
        else launch_walk<1, WALK_ITEMS>(w, KP, s);
    }
    if (g.dX && !parts) hipLaunchKernelGGL((join_dx_kernel<T>), dim3((uint32_t)x.blocks), dim3(256), 0, s, x);
    if (parts) {
        const dim3 grid((uint32_t)(x.blocks + (c.n_items * (KP / 4) + 255) / 256));
        hipLaunchKernelGGL((join_kernel<T>), grid, dim3(256), 0, s, x, p.acc_v, p.acc_b, p.split_v.count, p.v.padded, KP, w.f);
    }
}

int launch_logprob_backward(const ifr_catalogue &c, const int32_t *ids, int64_t m, int64_t ld_ids, const LogprobGrad &g, void *ws,
                            hipStream_t s)
{
    Pieces w{(char *)ws};
    const BackwardPlan p = backward_plan(w, c, m, g.dX != nullptr, g.dV != nullptr, g.dibase != nullptr, rows_lie(c));
    if (c.dtype == IFR_F32) backward_typed<float>(c, ids, m, ld_ids, g, p, s);
    else backward_typed<__bf16>(c, ids, m, ld_ids, g, p, s);
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

}  // namespace ifr
