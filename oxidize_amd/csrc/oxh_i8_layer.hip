/* oxh_i8_layer.hip — what stands around the int8 products of a layer: the norm that makes their tokens, products with bias,
 * activation and residual, the gated product and the feed-forward block (oxh_i8_rmsnorm, oxh_i8_matmul_ex, oxh_i8_linear_ex,
 * oxh_i8_gated, oxh_i8_ffn). */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oxhip.h"
#include "oxh_internal.h"
#include "oxh_device.inc"
#include "i8_tiles.inc"
#include "i8_products.inc"
#include "i8_host.inc"

/* Bytes that the L2s are told not to keep: results of a launch, which nobody reads before the next one. */
typedef uint32_t Stored8 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t Stored16 __attribute__((ext_vector_type(4), aligned(2)));
template <typename W, typename V> __device__ __forceinline__ void store_past(void *to, const V &v)
{
    static_assert(sizeof(V) % sizeof(W) == 0, "whole stores");
    struct All { W w[sizeof(V) / sizeof(W)]; };
    const All all = __builtin_bit_cast(All, v);
#pragma unroll
    for (uint32_t i = 0; i < sizeof(V) / sizeof(W); i++) __builtin_nontemporal_store(all.w[i], (W *)to + i);
}

/* ─── norm ────────────────────────────────────────────────────────────── */

struct I8Norm {
    const void *x, *add;
    void *sum, *y;
    size_t x_stride, add_stride, sum_stride, y_stride;
    const float *weight;
    int8_t *q;
    size_t q_stride;
    float *scale;
    double eps;
    uint32_t cols;
};

/* Values c .. c + 7 of a row, those behind the last one 0. */
template <typename T> __device__ __forceinline__ void norm_load8(const T *from, uint32_t c, uint32_t cols, float (&v)[8])
{
    if (c + 8u <= cols) {
        const Run<T, 8> r = *reinterpret_cast<const Run<T, 8> *>(from + c);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32(r.v[i]);
    } else
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) v[i] = c + i < cols ? to_f32(from[c + i]) : 0.0f;
}

template <typename T> __device__ __forceinline__ void norm_store8(T *to, uint32_t c, uint32_t cols, const float (&v)[8])
{
    if (c + 8u <= cols) {
        Run<T, 8> r;
#pragma unroll
        for (int i = 0; i < 8; i++) r.v[i] = from_f32<T>(v[i]);
        store_past<Stored16>(to + c, r);
    } else
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++)
            if (c + i < cols) to[c + i] = from_f32<T>(v[i]);
}

/* the sum over the wave's lanes, in every lane, by exchanges within rows of sixteen and four scalar reads */
__device__ __forceinline__ double wave_sum(double v)
{
    auto with = [&](auto exchange) {
        const uint2 bits = __builtin_bit_cast(uint2, v);
        v += __builtin_bit_cast(double, make_uint2((uint32_t)exchange((int)bits.x), (uint32_t)exchange((int)bits.y)));
    };
    with([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, false); });       /* lane ^ 1 */
    with([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, false); });       /* lane ^ 2 */
    with([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x141, 0xF, 0xF, false); });      /* mirrored in 8 */
    with([](int x) { return __builtin_amdgcn_update_dpp(0, x, 0x140, 0xF, 0xF, false); });      /* mirrored in 16 */
    auto row = [&](int lane) {
        const uint2 bits = __builtin_bit_cast(uint2, v);
        return __builtin_bit_cast(double, make_uint2((uint32_t)__builtin_amdgcn_readlane((int)bits.x, lane), (uint32_t)__builtin_amdgcn_readlane((int)bits.y, lane)));
    };
    return (row(0) + row(16)) + (row(32) + row(48));
}

/* A row by a workgroup, eight values to a thread and step: s = x + add in 32 bits, the sum of its squares (each exact) and the norm in 64; y is
 * rounded once.  The first HELD steps' values stay in registers; what is longer is
 * read three times.  sum and y go only to places that the same thread has read for the last time: they may be x or add.  Bound by memory: 4096 rows
 * of 4096 bf16 with add and sum in 26 us, 4.5 TB/s read and written (30 with ordinary stores), of 14336 in 92, 4.5 TB/s (114); one row of
 * 4096 in 3.3, a trip to memory and two barriers. */
template <typename T, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void k_i8_rmsnorm(const I8Norm p)
{
    constexpr uint32_t STEP = 8u * THREADS, WAVES = THREADS / 64;
    __shared__ double s_sum[(HELD + 1) * WAVES];
    __shared__ uint32_t s_top[THREADS / 64];
    const size_t row = blockIdx.x;
    const T *x = (const T *)p.x + row * p.x_stride, *add = p.add ? (const T *)p.add + row * p.add_stride : nullptr;
    const uint32_t cols = p.cols, c0 = 8u * threadIdx.x, wave = threadIdx.x >> 6;
    auto weights = [&](uint32_t c, float (&v)[8]) {
        if (p.weight) norm_load8(p.weight, c, cols, v);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 1.0f;
    };
    auto load = [&](uint32_t c, float (&v)[8]) {
        norm_load8(x, c, cols, v);
        if (add) {
            float a[8];
            norm_load8(add, c, cols, a);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] += a[i];
        }
    };
    auto square = [](const float (&v)[8], double &squares) {
#pragma unroll
        for (int i = 0; i < 8; i++) squares = __builtin_fma((double)v[i], (double)v[i], squares);
    };
    float s[HELD][8], w[HELD][8];
#pragma unroll
    for (int i = 0; i < HELD; i++) load(c0 + STEP * i, s[i]);
#pragma unroll
    for (int i = 0; i < HELD; i++) weights(c0 + STEP * i, w[i]);
    /* 512 neighbouring values' squares by a wave, and those sums in the order of the columns: the same for any THREADS and HELD that hold a row */
    double sums[HELD + 1];
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        sums[i] = 0.0;
        square(s[i], sums[i]);
        if (p.sum) norm_store8((T *)p.sum + row * p.sum_stride, c0 + STEP * i, cols, s[i]);
    }
    const bool longer = cols > STEP * HELD;
    sums[HELD] = 0.0;
    for (uint32_t c = c0 + STEP * HELD; c < cols; c += STEP) {
        float v[8];
        load(c, v);
        square(v, sums[HELD]);
    }
#pragma unroll
    for (int i = 0; i < HELD; i++) sums[i] = wave_sum(sums[i]);
    if (longer) sums[HELD] = wave_sum(sums[HELD]);
    double squares = 0.0;
    if (THREADS > 64) {
        if ((threadIdx.x & 63u) == 0u)
#pragma unroll
            for (int i = 0; i <= HELD; i++) s_sum[WAVES * i + wave] = sums[i];
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < HELD * WAVES; i++) squares += s_sum[i];
        if (longer)
#pragma unroll
            for (uint32_t i = HELD * WAVES; i < (HELD + 1) * WAVES; i++) squares += s_sum[i];
    } else
#pragma unroll
        for (int i = 0; i <= HELD; i++) squares += sums[i];
    const double r = 1.0 / sqrt(squares / (double)cols + p.eps);
    /* what stands for places behind the last column is 0 or, where r is no number, as little one as the row itself */
    auto normed = [&](float (&v)[8], const float (&g)[8]) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)((double)v[i] * r * (double)g[i]);
    };
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        normed(s[i], w[i]);
        top = max(top, i8_top8(s[i]));
    }
    for (uint32_t c = c0 + STEP * HELD; c < cols; c += STEP) {
        float v[8], g[8];
        load(c, v);
        weights(c, g);
        normed(v, g);
        top = max(top, i8_top8(v));
    }
    top = wave_top(top);
    if (THREADS > 64) {
        if ((threadIdx.x & 63u) == 0u) s_top[wave] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < THREADS / 64; i++) top = max(top, s_top[i]);
    }
    float inv;
    const float scale = i8_scale(top, inv);
    if (threadIdx.x == 0u) p.scale[row] = scale;
    const uint32_t end = (cols + 15u) & ~15u;
    auto store = [&](uint32_t c, const float (&y)[8]) {
        if (c >= end) return;
        store_past<Stored8>(p.q + row * p.q_stride + c, inv != 0.0f ? i8_codes8(y, scale, inv) : make_uint2(0u, 0u));
        if (p.y) norm_store8((T *)p.y + row * p.y_stride, c, cols, y);
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) store(c0 + STEP * i, s[i]);
    for (uint32_t c = c0 + STEP * HELD; c < end; c += STEP) {
        float v[8], g[8];
        load(c, v);
        weights(c, g);
        if (p.sum) norm_store8((T *)p.sum + row * p.sum_stride, c, cols, v);
        normed(v, g);
        store(c, v);
    }
}

/* ─── products with an epilogue ───────────────────────────────────────── */

/* 1 / (1 + 2^t), by the instructions for both (a unit in the last place each; results below 2^-126 are 0) */
__device__ __forceinline__ float i8_logistic(float t) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(t)); }

/* v P(X <= v) of a normal X.  P(X > z) = 2^(-z^2 / (2 ln 2)) R(z) falls as fast as its first factor; R = erfcx(z / sqrt(2)) / 2 has no scale of its own and is a
 * polynomial of degree 8 in 1 / (1 + 0.3 z) without a constant term, fitted to least relative error (2.4 * 2^-24) over 0 <= z <= 13.5, where the first
 * factor leaves the f32 numbers.  v v times the constant is rounded three times ahead of 2^x, which counts as v^2: in units of 2^-24 the whole is
 * within 20 + 1.2 v^2 below 0 and within 20 above (2^21 values each: 9.0 off in -1 .. 0, 14 in -4 .. -2, 46 in -8 .. -6, 127 in -13 .. -10; 8.7 above). */
__device__ __forceinline__ float i8_gelu(float v)
{
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, fabsf(v), 1.0f));
    float r = 0.03593168780207634f;
    r = __builtin_fmaf(r, t, -0.1582757830619812f);
    r = __builtin_fmaf(r, t, 0.2082061916589737f);
    r = __builtin_fmaf(r, t, -0.05539347976446152f);
    r = __builtin_fmaf(r, t, 0.12946900725364685f);
    r = __builtin_fmaf(r, t, 0.09963755309581757f);
    r = __builtin_fmaf(r, t, 0.12079835683107376f);
    r = __builtin_fmaf(r, t, 0.11962639540433884f);
    const float above = __builtin_amdgcn_exp2f(v * v * -0.72134752f) * (r * t);
    return v * (v > 0.0f ? 1.0f - above : above);
}

/* In 32 bits; a NaN stays one.  SILU's exponent is rounded once: -1 / ln 2 is the sum of two f32 numbers (within 6 + 1.01 |v| units of 2^-24; 8 off in
 * -8 .. -4, 47 in -80 .. -30).  The tanh form's, -2u / ln 2, is rounded three times and has two rounded constants (6 + 3.4 |2u|; 16 off in -4 .. -2, 155 in -10 ..
 * -8, where it is below 2^-68). */
template <uint32_t ACT> __device__ __forceinline__ float i8_activate(float v)
{
    if (ACT == OXH_ACT_RELU) return v < 0.0f ? 0.0f : v;
    if (ACT == OXH_ACT_SILU) return v * i8_logistic(__builtin_fmaf(v, -1.44269502f, v * -1.92596299e-8f));
    if (ACT == OXH_ACT_GELU) return i8_gelu(v);
    return v * i8_logistic(v * __builtin_fmaf(v * v, -0.10294324f, -2.30220820f));      /* (1 + tanh(u)) / 2 = 1 / (1 + exp(-2u)) */
}

/* Of many values at a time: what an activation waits for, an exponential and a reciprocal, is under way for all of them, where a branch on its kind for each
 * value would end every one's chain first (4096 tokens over 14336 x 4096, bias and GELU: 269 us; like this 262). */
template <uint32_t N> __device__ __forceinline__ void i8_activate_all(uint32_t act, float (&v)[N][4])
{
    auto all = [&](auto kind) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) v[i][k] = i8_activate<kind.value>(v[i][k]);
    };
    if (act == OXH_ACT_RELU) all(I8Num<OXH_ACT_RELU>{});
    else if (act == OXH_ACT_SILU) all(I8Num<OXH_ACT_SILU>{});
    else if (act == OXH_ACT_GELU) all(I8Num<OXH_ACT_GELU>{});
    else if (act == OXH_ACT_GELU_TANH) all(I8Num<OXH_ACT_GELU_TANH>{});
}

/* sum * q_scale * w_scale + bias */
template <uint32_t N, uint32_t M> __device__ __forceinline__ void i8_scaled(const v4i (&sums)[N][M], const I8RowFactors (&f)[N][M], uint32_t m, float st, bool bias, float (&v)[N][4])
{
#pragma unroll
    for (uint32_t i = 0; i < N; i++)
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) v[i][k] = (float)sums[i][m][k] * st * f[i][m].s[k];
    if (bias)
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) v[i][k] += f[i][m].b[k];
}

/* A lane's results, rows r + 16 i .. + 3 of token t, to memory, whole lines at a time.  A wave holds four rows of each of sixteen tokens: a store of those as
 * they are writes 32 (16-bit results) or 64 neighbouring bytes of a token's row.  So lanes change places first, without LDS: of two fragments of
 * 16-bit results the lanes of odd rows of sixteen give their share of the first for their neighbours' of the second, and have 16 bytes each of one,
 * 64 of a token; then of two such the lanes of the upper eight tokens give the first for the lower eight's second, and a store writes 128
 * bytes of each of eight tokens.  The L2s are told to keep none of it: a launch's results would push the operands of its other tiles out.  (4096 tokens over
 * 14336 x 4096, bf16, bias and GELU: 259 us without all that, 235 with the first change, 234 with both, 217 with the stores past the L2s; gate and up 413,
 * 387, 385 and 366.)  Every lane takes part, whether its token is there or not.
 *
 * i8_put_pieces: pieces of 16 bytes that a lane has of its token: `PIECES` of them, SPAN rows apart from `row` on, HAS rows of W's size each. */
template <typename W, uint32_t PIECES>
__device__ __forceinline__ void i8_put_pieces(W *out, size_t stride, uint32_t row, uint32_t rows, uint32_t t, uint32_t n_vec, const uint4 (&piece)[PIECES], bool past)
{
    constexpr uint32_t HAS = 16u / sizeof(W), SPAN = 4u * HAS;
    auto store = [&](uint32_t token, uint32_t at, const uint4 &what) {
        if (token >= n_vec) return;
        W *to = out + (size_t)token * stride + at;
        const Run<W, HAS> all = __builtin_bit_cast(Run<W, HAS>, what);
        if (at + HAS <= rows) {
            if (past) store_past<Stored16>(to, what);
            else *reinterpret_cast<Run<W, HAS> *>(to) = all;
        } else
#pragma unroll
            for (uint32_t k = 0; k < HAS - 1u; k++)
                if (at + k < rows) to[k] = all.v[k];
    };
    if constexpr (PIECES % 2u == 0u) {
        const uint32_t upper = (threadIdx.x >> 3) & 1u;
        row += SPAN * upper;
#pragma unroll
        for (uint32_t i = 0; i < PIECES; i += 2u) {
            const uint4 x = piece[i], y = piece[i + 1u];
            auto low = [](uint32_t a, uint32_t b) { return (uint32_t)__builtin_amdgcn_update_dpp((int)a, (int)b, 0x128, 0xF, 0xC, false); };     /* a, in the upper eight lanes the lower's b */
            auto high = [](uint32_t a, uint32_t b) { return (uint32_t)__builtin_amdgcn_update_dpp((int)b, (int)a, 0x128, 0xF, 0x3, false); };    /* b, in the lower eight the upper's a */
            store(t - 8u * upper, row + SPAN * i, make_uint4(low(x.x, y.x), low(x.y, y.y), low(x.z, y.z), low(x.w, y.w)));
            store(t + 8u - 8u * upper, row + SPAN * i, make_uint4(high(x.x, y.x), high(x.y, y.y), high(x.z, y.z), high(x.w, y.w)));
        }
    } else
#pragma unroll
        for (uint32_t i = 0; i < PIECES; i++) store(t, row + SPAN * i, piece[i]);
}

template <uint32_t N>
__device__ __forceinline__ void i8_put_f32(float *out, size_t stride, uint32_t r, uint32_t rows, uint32_t t, uint32_t n_vec, const float (&v)[N][4], bool past)
{
    uint4 piece[N];
#pragma unroll
    for (uint32_t i = 0; i < N; i++) piece[i] = __builtin_bit_cast(uint4, (v4f){ v[i][0], v[i][1], v[i][2], v[i][3] });
    i8_put_pieces((uint32_t *)out, stride, r, rows, t, n_vec, piece, past);
}

template <uint32_t N> __device__ __forceinline__ void i8_put_all(const I8Product &p, uint32_t r, uint32_t t, const float (&v)[N][4])
{
    const uint32_t rows = (uint32_t)p.w.rows;
    if (p.out_type == OXH_F32) {
        i8_put_f32((float *)p.out, p.out_stride, r, rows, t, p.n_vec, v, true);
        return;
    }
    /* the two 16-bit types differ in their rounding only */
    uint2 four[N];
    auto round = [&](auto zero) {
        typedef decltype(zero) T;
        typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
            four[i] = __builtin_bit_cast(uint2, (T4){ from_f32<T>(v[i][0]), from_f32<T>(v[i][1]), from_f32<T>(v[i][2]), from_f32<T>(v[i][3]) });
    };
    if (p.out_type == OXH_F16) round((_Float16)0);
    else round((__bf16)0.0f);
    uint16_t *out = (uint16_t *)p.out;
    if constexpr (N % 2u == 0u) {
        uint4 piece[N / 2u];
#pragma unroll
        for (uint32_t i = 0; i < N; i += 2u) {
            const auto lo = __builtin_amdgcn_permlane16_swap(four[i].x, four[i + 1u].x, false, false), hi = __builtin_amdgcn_permlane16_swap(four[i].y, four[i + 1u].y, false, false);
            piece[i / 2u] = make_uint4(lo[0], hi[0], lo[1], hi[1]);
        }
        const uint32_t kq = (threadIdx.x >> 4) & 3u;
        i8_put_pieces(out, p.out_stride, r - 4u * kq + 16u * (kq & 1u) + 8u * (kq >> 1), rows, t, p.n_vec, piece, true);
    } else {
        static_assert(N == 1u, "fragments in pairs, or one");
        if (t >= p.n_vec || r >= rows) return;
        uint16_t *to = out + (size_t)t * p.out_stride + r;
        const Run<uint16_t, 4> all = __builtin_bit_cast(Run<uint16_t, 4>, four[0]);
        if (r + 4u <= rows) *reinterpret_cast<Run<uint16_t, 4> *>(to) = all;
        else
#pragma unroll
            for (uint32_t k = 0; k < 3u; k++)
                if (r + k < rows) to[k] = all.v[k];
    }
}

/* Partial sums the same way: rows of rows_pad of a token and matrix, as k_i8_join reads them.  Up to 8 MB of them stay in the L2s for it (us kept and past
 * them: 2000 x 9000, gate and up under 60, 3.8 MB: 13.7 and 14.3; 1168 x 14272 under 310, 7.2: 19.8, 20.4; 2000 x 14000 under 260, 10.4: 24.7, 24.2; 4096 x
 * 14336 under 333, 21.8: 39.4, 36.1, and 39.1 kept in half lines; under 1000, 32.8: 81.8, 78.8). */
template <typename P, uint32_t N, uint32_t M> __device__ __forceinline__ void i8_part(const P &p, uint32_t split, uint32_t r, uint32_t t, const v4i (&sums)[N][M])
{
#pragma unroll
    for (uint32_t m = 0; m < M; m++) {
        float v[N][4];
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) v[i][k] = __int_as_float(sums[i][m][k]);
        float *out = (float *)p.parts + ((size_t)split * p.n_vec * M + m) * p.rows_pad;
        i8_put_f32(out, (size_t)M * p.rows_pad, r, p.rows_pad, t, p.n_vec, v, (size_t)p.splits * p.n_vec * M * p.rows_pad > ((size_t)2 << 20));
    }
}

/* products whose columns are shared out, without what is made of their sums */
struct I8Sums : I8Product {
    static constexpr bool TOGETHER = true, SUMS = true;
    explicit I8Sums(const I8Product &p) : I8Product(p) {}
};
template <uint32_t N> __device__ __forceinline__ void i8_row_factors(const I8Sums &, uint32_t, I8RowFactors (&)[N][1]) {}

/* Scales (or biases, if there are any) of matrix m's rows r + 16 i .. + 3, 16 bytes a load where all four exist; behind the last row the last
 * one again. */
template <uint32_t N, uint32_t M>
__device__ __forceinline__ void i8_rows4(const float *from, uint32_t r, uint32_t rows, uint32_t m, float (I8RowFactors::*to)[4], I8RowFactors (&f)[N][M])
{
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
        const uint32_t at = r + 16u * i;
        if (!from)
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) (f[i][m].*to)[k] = 0.0f;
        else if (at + 4u <= rows) {
            const Run<float, 4> v = *reinterpret_cast<const Run<float, 4> *>(from + at);
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) (f[i][m].*to)[k] = v.v[k];
        } else
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) (f[i][m].*to)[k] = from[min(at + k, rows - 1u)];
    }
}

struct I8ProductEx : I8Product {
    static constexpr uint32_t RULE = I8_EX;
    static constexpr bool TOGETHER = true;
    const void *residual;
    size_t residual_stride;
    uint32_t act;
};

template <uint32_t N> __device__ __forceinline__ void i8_row_factors(const I8ProductEx &p, uint32_t r, I8RowFactors (&f)[N][1])
{
    i8_rows4(p.w.d_scale, r, (uint32_t)p.w.rows, 0u, &I8RowFactors::s, f);
    i8_rows4(p.bias, r, (uint32_t)p.w.rows, 0u, &I8RowFactors::b, f);
}

/* four neighbouring values of the residual, as i8_store4 stores them */
template <typename T> __device__ __forceinline__ v4f residual4(const T *from, uint32_t left)
{
    if (left >= 4u) {
        const Run<T, 4> r = *reinterpret_cast<const Run<T, 4> *>(from);
        return v4f{ to_f32(r.v[0]), to_f32(r.v[1]), to_f32(r.v[2]), to_f32(r.v[3]) };
    }
    return v4f{ to_f32(from[0]), left > 1u ? to_f32(from[1]) : 0.0f, left > 2u ? to_f32(from[2]) : 0.0f, 0.0f };
}
template <typename T, uint32_t N> __device__ __forceinline__ void residual_all(const T *from, uint32_t left, float (&v)[N][4])
{
    v4f more[N];
#pragma unroll
    for (uint32_t i = 0; i < N; i++) more[i] = 16u * i < left ? residual4(from + 16u * i, left - 16u * i) : v4f{ 0.0f, 0.0f, 0.0f, 0.0f };
#pragma unroll
    for (uint32_t i = 0; i < N; i++)
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) v[i][k] += more[i][k];
}

/* the residual of one fragment's rows; 0 where there is none, or no such row or token */
__device__ __forceinline__ v4f i8_beside(const I8ProductEx &p, uint32_t r, uint32_t t)
{
    const uint32_t rows = (uint32_t)p.w.rows;
    if (!p.residual || r >= rows || t >= p.n_vec) return v4f{ 0.0f, 0.0f, 0.0f, 0.0f };
    const size_t at = (size_t)t * p.residual_stride + r;
    if (p.out_type == OXH_F32) return residual4((const float *)p.residual + at, rows - r);
    if (p.out_type == OXH_F16) return residual4((const _Float16 *)p.residual + at, rows - r);
    return residual4((const __bf16 *)p.residual + at, rows - r);
}

__device__ __forceinline__ void i8_results(const I8ProductEx &p, uint32_t r, uint32_t t, const v4i (&sums)[1], const I8RowFactors (&f)[1], float st, v4f beside)
{
    float v[1][4];
    i8_scaled(reinterpret_cast<const v4i(&)[1][1]>(sums), reinterpret_cast<const I8RowFactors(&)[1][1]>(f), 0u, st, p.bias != nullptr, v);
    i8_activate_all(p.act, v);
    if (p.residual)
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) v[0][k] += beside[k];
    i8_put_all(p, r, t, v);
}

template <uint32_t N>
__device__ __forceinline__ void i8_results(const I8ProductEx &p, uint32_t r, uint32_t t, const v4i (&sums)[N][1], const I8RowFactors (&f)[N][1], float st)
{
    float v[N][4];
    i8_scaled(sums, f, 0u, st, p.bias != nullptr, v);
    i8_activate_all(p.act, v);
    if (p.residual && r < (uint32_t)p.w.rows) {
        const size_t at = (size_t)min(t, p.n_vec - 1u) * p.residual_stride + r;
        const uint32_t left = (uint32_t)p.w.rows - r;
        if (p.out_type == OXH_F32) residual_all((const float *)p.residual + at, left, v);
        else if (p.out_type == OXH_F16) residual_all((const _Float16 *)p.residual + at, left, v);
        else residual_all((const __bf16 *)p.residual + at, left, v);
    }
    i8_put_all(p, r, t, v);
}

/* ─── gated products ──────────────────────────────────────────────────── */

/* w and bias are the gate's */
struct I8GatedProduct : I8Product {
    static constexpr uint32_t MATRICES = 2, RULE = I8_GATED;
    static constexpr bool TOGETHER = true;
    const int8_t *up;
    const float *up_scale, *up_bias;
    uint32_t act;
};

__device__ __forceinline__ const int8_t *i8_codes_of(const I8GatedProduct &p, uint32_t m) { return m ? p.up : p.w.d_w; }

template <uint32_t N> __device__ __forceinline__ void i8_row_factors(const I8GatedProduct &p, uint32_t r, I8RowFactors (&f)[N][2])
{
    const uint32_t rows = (uint32_t)p.w.rows;
    i8_rows4(p.w.d_scale, r, rows, 0u, &I8RowFactors::s, f);
    i8_rows4(p.up_scale, r, rows, 1u, &I8RowFactors::s, f);
    i8_rows4(p.bias, r, rows, 0u, &I8RowFactors::b, f);
    i8_rows4(p.up_bias, r, rows, 1u, &I8RowFactors::b, f);
}

struct I8GatedSums : I8GatedProduct {
    static constexpr bool SUMS = true;
    explicit I8GatedSums(const I8GatedProduct &p) : I8GatedProduct(p) {}
};

template <uint32_t N>
__device__ __forceinline__ void i8_results(const I8GatedProduct &p, uint32_t r, uint32_t t, const v4i (&sums)[N][2], const I8RowFactors (&f)[N][2], float st)
{
    float v[N][4], up[N][4];
    i8_scaled(sums, f, 0u, st, p.bias != nullptr, v);
    i8_activate_all(p.act, v);
    i8_scaled(sums, f, 1u, st, p.up_bias != nullptr, up);
#pragma unroll
    for (uint32_t i = 0; i < N; i++)
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) v[i][k] *= up[i][k];
    i8_put_all(p, r, t, v);
}

/* of one fragment's rows, as the kernels for few tokens and the joined parts have them */
template <typename P, uint32_t M> __device__ __forceinline__ void i8_row_factors(const P &p, uint32_t r, I8RowFactors (&f)[M])
{
    i8_row_factors<1u>(p, r, reinterpret_cast<I8RowFactors(&)[1][M]>(f));
}
__device__ __forceinline__ void i8_results(const I8GatedProduct &p, uint32_t r, uint32_t t, const v4i (&sums)[2], const I8RowFactors (&f)[2], float st, I8Nothing)
{
    i8_results<1u>(p, r, t, reinterpret_cast<const v4i(&)[1][2]>(sums), reinterpret_cast<const I8RowFactors(&)[1][2]>(f), st);
}

/* ─── host side ───────────────────────────────────────────────────────── */

static int check_again(const char *who, const char *name, const void *d, uint32_t type, size_t stride, size_t cols)
{
    return d ? check_floats(who, name, type, d, stride, cols) : OXH_OK;
}

extern "C" int oxh_i8_rmsnorm(const OxhI8Norm *norm, uint32_t x_type, const void *d_x, size_t x_stride, size_t n_vec, size_t cols, int8_t *d_q,
                              size_t q_stride, float *d_scale, void *stream)
{
    static const char who[] = "oxh_i8_rmsnorm";
    int rc;
    if (!norm) return I8_ARG("%s: NULL norm", who);
    if (!(norm->eps >= 0.0f)) return I8_ARG("%s: eps must be >= 0", who);
    if (n_vec == 0) return OXH_OK;
    if ((rc = check_cols(who, cols)) || (rc = check_floats(who, "d_x", x_type, d_x, x_stride, cols)) ||
        (rc = check_rows(who, "d_q", d_q, q_stride, cols)) || (rc = check_again(who, "d_add", norm->d_add, x_type, norm->add_stride, cols)) ||
        (rc = check_again(who, "d_sum", norm->d_sum, x_type, norm->sum_stride, cols)) ||
        (rc = check_again(who, "d_y", norm->d_y, x_type, norm->y_stride, cols)) ||
        (rc = check_again(who, "d_weight", norm->d_weight, OXH_F32, cols, cols)))
        return rc;
    if (!d_scale) return I8_ARG("%s: NULL pointer (d_scale)", who);
    if (norm->d_sum && norm->d_sum == norm->d_y) return I8_ARG("%s: d_sum and d_y are the same memory", who);
    const void *const outs[2] = { norm->d_sum, norm->d_y }, *const ins[2] = { d_x, norm->d_add };
    const size_t out_strides[2] = { norm->sum_stride, norm->y_stride }, in_strides[2] = { x_stride, norm->add_stride };
    for (int o = 0; o < 2; o++)
        for (int i = 0; i < 2; i++)
            if (outs[o] && outs[o] == ins[i] && out_strides[o] != in_strides[i])
                return I8_ARG("%s: an output in place of an input must have its stride", who);
    if (n_vec > OXH_I8_MAX_ROWS) return I8_ARG("%s: at most %zu rows per call", who, OXH_I8_MAX_ROWS);
    if ((rc = ready())) return rc;
    const I8Norm p = { d_x, norm->d_add, norm->d_sum, norm->d_y, x_stride, norm->add_stride, norm->sum_stride, norm->y_stride, norm->d_weight,
                       d_q, q_stride, d_scale, (double)norm->eps, (uint32_t)cols };
    const dim3 grid((uint32_t)n_vec);
    const hipStream_t st = stream_of(stream);
#define OXH_NORM_K(T, THREADS, HELD) hipLaunchKernelGGL((k_i8_rmsnorm<T, THREADS, HELD>), grid, dim3(THREADS), 0, st, p)
    /* Threads to a row: as few as hold its values in a step or two, so that they are read once (us of 4096 bf16 rows with 256 threads and two
     * steps, 512 and one, 512 and two, 1024 and two: of 4096 values 26.0, 28.7, 35.9, 77; one row 3.8, 3.5, 4.5, 5.8; 4096 f32 rows 38.1, 36.4; 2048 bf16 rows of
     * 8192 with 512 and two, 1024 and one: 27.5, 37.8; 4096 of 14336 with 1024 and two, 512 and two, which reads some twice more: 92, 96). */
#define OXH_NORM(T)                                                                                                              \
    do {                                                                                                                         \
        if (cols <= 512u) OXH_NORM_K(T, 64, 1);                                                                                  \
        else if (cols <= 1024u) OXH_NORM_K(T, 128, 1);                                                                           \
        else if (cols <= 2048u) OXH_NORM_K(T, 256, 1);                                                                           \
        else if (cols <= 4096u && sizeof(T) == 2 && n_vec >= 1024u) OXH_NORM_K(T, 256, 2);                                       \
        else if (cols <= 4096u) OXH_NORM_K(T, 512, 1);                                                                           \
        else if (cols <= 8192u) OXH_NORM_K(T, 512, 2);                                                                           \
        else OXH_NORM_K(T, 1024, 2);                                                                                             \
    } while (0)
    if (x_type == OXH_F32) OXH_NORM(float);
    else if (x_type == OXH_F16) OXH_NORM(_Float16);
    else OXH_NORM(__bf16);
#undef OXH_NORM
#undef OXH_NORM_K
    return launched(who);
}

static int check_activation(const char *who, uint32_t act)
{
    return act <= OXH_ACT_GELU_TANH ? OXH_OK : I8_ARG("%s: the activation is not an OXH_ACT_", who);
}

static int check_epilogue(const char *who, const OxhI8Epilogue *e, uint32_t out_type, const void *d_out, size_t out_stride, size_t rows)
{
    int rc;
    if (!e) return OXH_OK;
    if ((rc = check_activation(who, e->act)) || (rc = check_again(who, "d_bias", e->d_bias, OXH_F32, rows, rows)) ||
        (rc = check_again(who, "d_residual", e->d_residual, out_type, e->residual_stride, rows)))
        return rc;
    if (e->d_residual && e->d_residual == d_out && e->residual_stride != out_stride)
        return I8_ARG("%s: results in place of the residual must have its stride", who);
    return OXH_OK;
}

static I8ProductEx product_ex(const I8Product &p, const OxhI8Epilogue *e)
{
    I8ProductEx x = { p, nullptr, 0, OXH_ACT_NONE };
    if (e) {
        x.bias = e->d_bias;
        x.residual = e->d_residual;
        x.residual_stride = e->residual_stride;
        x.act = e->act;
    }
    return x;
}

/* sizes that every product here has to keep to */
static int check_sizes(const char *who, size_t n_vec, size_t rows)
{
    if (n_vec > OXH_I8_MAX_ROWS) return I8_ARG("%s: at most %zu tokens per call", who, OXH_I8_MAX_ROWS);
    if (n_vec * rows > OXH_I8_MAX_RESULTS) return I8_ARG("%s: at most %zu results per call", who, OXH_I8_MAX_RESULTS);
    return OXH_OK;
}

static int check_tokens(const char *who, const int8_t *d_q, size_t q_stride, const float *d_q_scale, size_t cols)
{
    const int rc = check_rows(who, "d_q", d_q, q_stride, cols);
    if (rc) return rc;
    return d_q_scale ? OXH_OK : I8_ARG("%s: NULL pointer (d_q_scale)", who);
}

static int check_optional_workspace(const char *who, const void *d_workspace, size_t bytes)
{
    if (d_workspace && bytes && ((uintptr_t)d_workspace & 15u)) return I8_ARG("%s: workspace must be 16-byte aligned", who);
    return OXH_OK;
}

extern "C" int oxh_i8_matmul_ex(const OxhI8Matrix *w, const int8_t *d_q, size_t q_stride, const float *d_q_scale, size_t n_vec,
                                const OxhI8Epilogue *e, uint32_t out_type, void *d_out, size_t out_stride, void *d_workspace,
                                size_t workspace_bytes, void *stream)
{
    static const char who[] = "oxh_i8_matmul_ex";
    int rc;
    if ((rc = check_matrix(who, w))) return rc;
    if (n_vec == 0 || w->rows == 0) return OXH_OK;
    if ((rc = check_tokens(who, d_q, q_stride, d_q_scale, w->cols)) || (rc = check_floats(who, "d_out", out_type, d_out, out_stride, w->rows)) ||
        (rc = check_epilogue(who, e, out_type, d_out, out_stride, w->rows)) || (rc = check_sizes(who, n_vec, w->rows)) ||
        (rc = check_optional_workspace(who, d_workspace, workspace_bytes)) || (rc = ready()))
        return rc;
    I8ProductEx p = product_ex(i8_product(w, d_q, q_stride, d_q_scale, n_vec, nullptr, out_type, d_out, out_stride), e);
    return product_launch<I8ProductEx, I8Sums>(p, i8_choice(w->rows, w->cols, n_vec, d_workspace ? workspace_bytes : 0, i8_cus(), I8_EX), d_workspace,
                                               stream_of(stream), who);
}

extern "C" int oxh_i8_linear_ex(const OxhI8Matrix *w, uint32_t x_type, const void *d_x, size_t x_stride, size_t n_vec, const OxhI8Epilogue *e,
                                uint32_t out_type, void *d_out, size_t out_stride, void *d_workspace, size_t workspace_bytes, void *stream)
{
    static const char who[] = "oxh_i8_linear_ex";
    int rc;
    if ((rc = check_matrix(who, w))) return rc;
    if (n_vec == 0 || w->rows == 0) return OXH_OK;
    if ((rc = check_floats(who, "d_x", x_type, d_x, x_stride, w->cols)) || (rc = check_floats(who, "d_out", out_type, d_out, out_stride, w->rows)) ||
        (rc = check_epilogue(who, e, out_type, d_out, out_stride, w->rows)) || (rc = check_sizes(who, n_vec, w->rows)))
        return rc;
    if (d_out == d_x) return I8_ARG("%s: results in place of the tokens", who);      /* workgroups that quantise for themselves read all of them */
    if ((rc = check_linear_workspace(who, w, n_vec, d_workspace, workspace_bytes)) || (rc = ready()) ||
        (rc = check_linear_workspace(who, w, n_vec, d_workspace, workspace_bytes)))    /* once more: the way depends on the device */
        return rc;
    I8ProductEx p = product_ex(i8_product(w, nullptr, 0, nullptr, n_vec, nullptr, out_type, d_out, out_stride), e);
    return linear_launch<I8ProductEx, I8Sums>(p, x_type, d_x, x_stride, d_workspace, workspace_bytes, stream_of(stream), who);
}

static OxhI8Matrix gate_of(const OxhI8Gated *g) { return { g->d_w_gate, g->stride, g->d_s_gate, g->rows, g->cols }; }

static int check_gated(const char *who, const OxhI8Gated *g)
{
    int rc;
    if (!g) return I8_ARG("%s: NULL matrices", who);
    if ((rc = check_cols(who, g->cols)) || (rc = check_rows(who, "d_w_gate", g->d_w_gate, g->stride, g->cols)) ||
        (rc = check_rows(who, "d_w_up", g->d_w_up, g->stride, g->cols)))
        return rc;
    if (!g->d_s_gate || !g->d_s_up) return I8_ARG("%s: NULL pointer (the matrices' scales)", who);
    if ((rc = check_again(who, "d_b_gate", g->d_b_gate, OXH_F32, g->rows, g->rows)) ||
        (rc = check_again(who, "d_b_up", g->d_b_up, OXH_F32, g->rows, g->rows)))
        return rc;
    if (g->rows > OXH_I8_MAX_ROWS) return I8_ARG("%s: at most %zu rows", who, OXH_I8_MAX_ROWS);
    return check_activation(who, g->act);
}

static int gated_launch(const OxhI8Gated *g, const int8_t *q, size_t q_stride, const float *q_scale, size_t n, uint32_t out_type, void *out,
                        size_t out_stride, void *ws, size_t ws_bytes, hipStream_t st, const char *who)
{
    const OxhI8Matrix gate = gate_of(g);
    I8GatedProduct p = { i8_product(&gate, q, q_stride, q_scale, n, g->d_b_gate, out_type, out, out_stride), g->d_w_up, g->d_s_up, g->d_b_up, g->act };
    return product_launch<I8GatedProduct, I8GatedSums>(p, i8_choice(g->rows, g->cols, n, ws_bytes, i8_cus(), I8_GATED), ws, st, who);
}

/* as product_parts() */
static size_t gated_parts(size_t rows, size_t cols, size_t n)
{
    const size_t cus = i8_cus(), in_all = i8_rows_in_all(rows, 2u);
    return most_parts(in_all, cols, n, [&](size_t m) {
        const I8Choice c = i8_choice(rows, cols, m, SIZE_MAX, cus, I8_GATED);
        return c.team ? (size_t)0 : parts_bytes(in_all, m, c.way.splits);
    });
}

extern "C" size_t oxh_i8_gated_workspace(const OxhI8Gated *g, size_t n_vec)
{
    return g && workable(g->rows, g->cols, n_vec) ? gated_parts(g->rows, g->cols, n_vec) : 0;
}

extern "C" int oxh_i8_gated(const OxhI8Gated *g, const int8_t *d_q, size_t q_stride, const float *d_q_scale, size_t n_vec, uint32_t out_type,
                            void *d_out, size_t out_stride, void *d_workspace, size_t workspace_bytes, void *stream)
{
    static const char who[] = "oxh_i8_gated";
    int rc;
    if ((rc = check_gated(who, g))) return rc;
    if (n_vec == 0 || g->rows == 0) return OXH_OK;
    if ((rc = check_tokens(who, d_q, q_stride, d_q_scale, g->cols)) || (rc = check_floats(who, "d_out", out_type, d_out, out_stride, g->rows)) ||
        (rc = check_sizes(who, n_vec, g->rows)) || (rc = check_optional_workspace(who, d_workspace, workspace_bytes)) || (rc = ready()))
        return rc;
    return gated_launch(g, d_q, q_stride, d_q_scale, n_vec, out_type, d_out, out_stride, d_workspace, d_workspace ? workspace_bytes : 0,
                        stream_of(stream), who);
}

/* The block's workspace: h in f32, rows of up64(ffn); behind it the gated product's partial sums, and when those are done the codes
 * and sums of the down projection. */
static size_t ffn_h_bytes(size_t ffn, size_t n) { return up256(n * up64(ffn) * 4u); }

extern "C" size_t oxh_i8_ffn_workspace(const OxhI8Gated *g, const OxhI8Matrix *down, size_t n_vec)
{
    if (!g || !down || !workable(g->rows, g->cols, n_vec) || !workable(down->rows, down->cols, n_vec)) return 0;
    const size_t first = gated_parts(g->rows, g->cols, n_vec), second = linear_bytes(down->rows, down->cols, n_vec);
    return ffn_h_bytes(g->rows, n_vec) + (first > second ? first : second);
}

/* h and the codes have to fit, partial sums are used where they do */
static int check_ffn_workspace(const char *who, const OxhI8Gated *g, const OxhI8Matrix *down, size_t n_vec, const void *d_workspace, size_t bytes)
{
    const LinearParts l = linear_parts(down->rows, down->cols, n_vec);
    if (!d_workspace || bytes < ffn_h_bytes(g->rows, n_vec) + (l.fused ? 0 : l.parts)) return I8_ARG("%s: workspace too small (see oxh_i8_ffn_workspace)", who);
    if ((uintptr_t)d_workspace & 255u) return I8_ARG("%s: workspace must be 256-byte aligned", who);
    return OXH_OK;
}

extern "C" int oxh_i8_ffn(const OxhI8Gated *g, const OxhI8Matrix *down, const int8_t *d_q, size_t q_stride, const float *d_q_scale, size_t n_vec,
                          const OxhI8Epilogue *e, uint32_t out_type, void *d_out, size_t out_stride, void *d_workspace, size_t workspace_bytes,
                          void *stream)
{
    static const char who[] = "oxh_i8_ffn";
    int rc;
    if ((rc = check_gated(who, g)) || (rc = check_matrix(who, down))) return rc;
    if (g->rows == 0 || down->cols != g->rows) return I8_ARG("%s: the down matrix must have as many columns as the gate has rows", who);
    if (n_vec == 0 || down->rows == 0) return OXH_OK;
    if ((rc = check_tokens(who, d_q, q_stride, d_q_scale, g->cols)) || (rc = check_floats(who, "d_out", out_type, d_out, out_stride, down->rows)) ||
        (rc = check_epilogue(who, e, out_type, d_out, out_stride, down->rows)) || (rc = check_sizes(who, n_vec, g->rows)) ||
        (rc = check_sizes(who, n_vec, down->rows)) || (rc = check_ffn_workspace(who, g, down, n_vec, d_workspace, workspace_bytes)) || (rc = ready()) ||
        (rc = check_ffn_workspace(who, g, down, n_vec, d_workspace, workspace_bytes)))
        return rc;
    const hipStream_t st = stream_of(stream);
    const size_t h_bytes = ffn_h_bytes(g->rows, n_vec), h_stride = up64(g->rows);
    uint8_t *rest = (uint8_t *)d_workspace + h_bytes;
    if ((rc = gated_launch(g, d_q, q_stride, d_q_scale, n_vec, OXH_F32, d_workspace, h_stride, rest, workspace_bytes - h_bytes, st, who))) return rc;
    I8ProductEx p = product_ex(i8_product(down, nullptr, 0, nullptr, n_vec, nullptr, out_type, d_out, out_stride), e);
    return linear_launch<I8ProductEx, I8Sums>(p, OXH_F32, d_workspace, h_stride, rest, workspace_bytes - h_bytes, st, who);
}

extern "C" int oxh_internal_i8_layer_init(void)
{
    hipError_t e;
    if ((e = product_init<I8ProductEx>()) != hipSuccess) return (int)e;
    if ((e = product_init<I8Sums>()) != hipSuccess) return (int)e;
    if ((e = product_init<I8GatedProduct>()) != hipSuccess) return (int)e;
    return (int)product_init<I8GatedSums>();
}

/* ─── which kernels run, for tests ────────────────────────────────────── */

extern "C" int oxh_debug_i8_layer_kernel(size_t rows, size_t cols, size_t n_vec, size_t n_cu, size_t ws_bytes, int gated, uint32_t out[4])
{
    static const char who[] = "oxh_debug_i8_layer_kernel";
    if (!out || !rows || !n_vec || !n_cu) return I8_ARG("%s: NULL or empty", who);
    const int rc = check_cols(who, cols);
    if (rc) return rc;
    const uint32_t rule = gated ? I8_GATED : I8_EX;
    i8_describe(i8_choice(rows, cols, n_vec, ws_bytes, n_cu, rule), rows, cols, n_vec, n_cu, rule, out);
    return OXH_OK;
}
