/* oxh_i8.hip — int8 rows with one scale per row: the quantiser, the product of tokens with a matrix, and the experts'
 * products of a mixture-of-experts layer (oxh_i8_*, oxh_moe_ffn_i8). */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oxhip.h"
#include "oxh_internal.h"
#include "oxh_device.inc"
#include "i8_tiles.inc"

#pragma clang fp contract(off)

typedef float v4f __attribute__((ext_vector_type(4)));

/* ─── floats ──────────────────────────────────────────────────────────── */

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }      /* to nearest, ties to even */

/* N neighbouring values that are aligned to their elements only */
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Run { T v[N]; };

__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

/* ─── rows of floats to codes ─────────────────────────────────────────── */

/* The integer nearest to v / s, ties to even.  v * inv is within 2^-15 of the quotient, so its rounding is off by one at
 * most, next to a half; the remainder v - t * s has no more bits than an f32 holds (it is a multiple of half a unit of
 * s's last place and no larger than half of s and a bit), the fused operation gives it exactly, and which side of the half it lies
 * on says whether the rounding was right. */
__device__ __forceinline__ float i8_settle(float v, float t, float s)
{
    const float r = __builtin_fmaf(-t, s, v), twice = r + r;
    const bool odd = ((int)t & 1) != 0;
    if (twice > s || (twice == s && odd)) return t + 1.0f;
    if (twice < -s || (twice == -s && odd)) return t - 1.0f;
    return t;
}

/* The codes of eight values as bytes.  Only where a product lies within 2^-14 of a half (eight values in a thousand) is the
 * remainder looked at: five instructions a value instead of a dozen. */
__device__ __forceinline__ uint2 i8_codes8(const float (&v)[8], float s, float inv)
{
    float t[8], far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float x = v[i] * inv;
        t[i] = rintf(x);
        far = fmaxf(far, fabsf(x - t[i]));
    }
    if (far > 0.5f - 0x1p-14f) {
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = i8_settle(v[i], t[i], s);
    }
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; i++) b[i] = (uint32_t)(int)t[i];
    auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
    };
    return make_uint2(four(b[0], b[1], b[2], b[3]), four(b[4], b[5], b[6], b[7]));
}

/* Values c .. c + 7 of a row of cols, those behind the last one 0; up: NULL, or the row of SwiGLU's other factor. */
template <typename T, bool GLU>
__device__ __forceinline__ void i8_values8(const T *__restrict__ x, const T *__restrict__ up, uint32_t c, uint32_t cols, float (&v)[8])
{
    if (c + 8u <= cols) {
        const Run<T, 8> r = *reinterpret_cast<const Run<T, 8> *>(x + c);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32(r.v[i]);
        if (GLU) {
            const Run<T, 8> u = *reinterpret_cast<const Run<T, 8> *>(up + c);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = silu(v[i]) * to_f32(u.v[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] = c + i < cols ? to_f32(x[c + i]) : 0.0f;
            if (GLU) v[i] = c + i < cols ? silu(v[i]) * to_f32(up[c + i]) : 0.0f;
        }
    }
}

__device__ __forceinline__ uint32_t i8_top8(const float (&v)[8])
{
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return top;
}

/* the largest of sixteen neighbouring lanes' values, and of the wave's; every lane receives it, all lanes take part */
__device__ __forceinline__ uint32_t row_top(uint32_t top)
{
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));       /* lane ^ 1 */
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));       /* lane ^ 2 */
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x141, 0xF, 0xF, false));      /* mirrored in 8 */
    return max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x140, 0xF, 0xF, false));     /* mirrored in 16 */
}
__device__ __forceinline__ uint32_t wave_top(uint32_t top)
{
    const int row = (int)row_top(top);
    return max(max((uint32_t)__builtin_amdgcn_readlane(row, 0), (uint32_t)__builtin_amdgcn_readlane(row, 16)),
               max((uint32_t)__builtin_amdgcn_readlane(row, 32), (uint32_t)__builtin_amdgcn_readlane(row, 48)));
}

/* scale and 1 / scale of a row whose largest magnitude has the bits `top` (those of an infinity or a NaN are the
 * largest); a row without codes gets inv 0 */
__device__ __forceinline__ float i8_scale(uint32_t top, float &inv)
{
    inv = 0.0f;
    if (top >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    const float s = __uint_as_float(top) / 127.0f;
    if (s < 1.17549435e-38f) return 0.0f;
    inv = 1.0f / s;
    return s;
}

/* A row by a workgroup, eight values to a thread and step: once for the largest magnitude, once for the codes.  The first
 * HELD steps' values stay in registers; what is longer is read (and, GLU, computed) a second time.  Bound by memory: 4096 x 14336 bf16
 * in 35 us, 5.1 TB/s read and written, of silu(x) * up in 66, 4.5 TB/s; one row of 4096 in 2.2 us, a trip to memory and two barriers. */
template <typename T, bool GLU, int THREADS, int HELD>
__device__ __forceinline__ void i8_quantize_row(const T *__restrict__ xr, const T *__restrict__ ur, uint32_t cols, int8_t *__restrict__ qr,
                                                float *__restrict__ scale)
{
    constexpr uint32_t STEP = 8u * THREADS;
    __shared__ uint32_t s_top[THREADS / 64];
    const uint32_t c0 = 8u * threadIdx.x;
    float v[HELD][8];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < HELD; i++) i8_values8<T, GLU>(xr, ur, c0 + STEP * i, cols, v[i]);
#pragma unroll
    for (int i = 0; i < HELD; i++) top = max(top, i8_top8(v[i]));
    for (uint32_t c = c0 + STEP * HELD; c < cols; c += STEP) {
        float t[8];
        i8_values8<T, GLU>(xr, ur, c, cols, t);
        top = max(top, i8_top8(t));
    }
    top = wave_top(top);
    if (THREADS > 64) {
        if ((threadIdx.x & 63u) == 0u) s_top[threadIdx.x >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < THREADS / 64; i++) top = max(top, s_top[i]);
    }
    float inv;
    const float s = i8_scale(top, inv);
    if (threadIdx.x == 0u) *scale = s;
    const uint32_t end = (cols + 15u) & ~15u;
    auto store = [&](uint32_t c, const float (&t)[8]) {
        if (c < end) *reinterpret_cast<uint2 *>(qr + c) = inv != 0.0f ? i8_codes8(t, s, inv) : make_uint2(0u, 0u);
    };
#pragma unroll
    for (int i = 0; i < HELD; i++) store(c0 + STEP * i, v[i]);
    for (uint32_t c = c0 + STEP * HELD; c < end; c += STEP) {
        float t[8];
        i8_values8<T, GLU>(xr, ur, c, cols, t);
        store(c, t);
    }
}

template <typename T, bool GLU, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void
k_i8_quantize(const T *__restrict__ x, size_t x_stride, uint32_t cols, const T *__restrict__ up, int8_t *__restrict__ q,
              size_t q_stride, float *__restrict__ scale)
{
    const size_t row = blockIdx.x;
    i8_quantize_row<T, GLU, THREADS, HELD>(x + row * x_stride, GLU ? up + row * x_stride : nullptr, cols, q + row * q_stride, scale + row);
}

/* ─── products ────────────────────────────────────────────────────────── */

/* The sixteen codes at columns k.. of a row, those from cols on as 0 (k a multiple of 16). */
__device__ __forceinline__ v4i i8_piece(const int8_t *row, uint32_t k, uint32_t cols)
{
    v4i v = { 0, 0, 0, 0 };
    if (k < cols) {
        v = *reinterpret_cast<const v4i *>(row + k);
        if (cols - k < 16u)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t left = cols - k > 4u * i ? cols - k - 4u * i : 0u;
                if (left < 4u) v[i] &= (int)((1u << (8u * left)) - 1u);
            }
    }
    return v;
}

/* what a wave's lanes wrote to LDS before, its other lanes read after (LDS serves a wave in order) */
__device__ __forceinline__ void i8_wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

/* Four neighbouring results of a token, aligned to their elements only; the last rows of a matrix one by one. */
template <typename T> __device__ __forceinline__ void i8_store4(T *out, const float (&v)[4], uint32_t rows_left)
{
    if (rows_left >= 4u) {
        Run<T, 4> r;
#pragma unroll
        for (int i = 0; i < 4; i++) r.v[i] = from_f32<T>(v[i]);
        *reinterpret_cast<Run<T, 4> *>(out) = r;
    } else
#pragma unroll
        for (uint32_t i = 0; i < 3u; i++)
            if (i < rows_left) out[i] = from_f32<T>(v[i]);
}

/* Workgroup b of n takes place i8_place() of the tiles' order: the workgroups of an XCD (every eighth one) take a run of it. */
__device__ __forceinline__ uint32_t i8_place(uint32_t b, uint32_t n)
{
    const uint32_t per = n / 8u, more = n % 8u, x = b % 8u;
    return x * per + min(x, more) + b / 8u;
}

/* The tile at place i: an order that goes through the token tiles with up to eight row tiles at each, so that what an XCD's
 * 32 CUs read at a time is 8 + 4 operand tiles through its L2, where one row tile under 32 token tiles is 33 (8192 x
 * 8192 x 8192: 473 us, 435 in this order; 406 with what i8_tile has learnt since, 2700 TOPS). */
__device__ __forceinline__ void i8_tile_at(uint32_t i, uint32_t row_tiles, uint32_t tok_tiles, uint32_t &row, uint32_t &tok)
{
    const uint32_t group = i / (8u * tok_tiles), in = i - group * 8u * tok_tiles, high = min(8u, row_tiles - 8u * group);
    row = 8u * group + in % high;
    tok = in / high;
}

/* What the product's kernels take: the matrix, quantised tokens, and where the results go. */
struct I8Product {
    OxhI8Matrix w;
    const int8_t *q;
    size_t q_stride;
    const float *q_scale, *bias;
    void *out;
    size_t out_stride;
    int *parts;                     /* partial sums [split][token][rows_pad] of a product whose columns are shared out */
    uint32_t n_vec, splits, row_tiles, tok_tiles, whole, rows_pad, out_type;
};

/* four rows' results of a token from their sums, in out_type */
__device__ __forceinline__ void i8_results(const I8Product &p, uint32_t r, uint32_t t, const v4i &sums, const float (&sw)[4],
                                           const float (&b)[4], float st)
{
    const uint32_t rows = (uint32_t)p.w.rows;
    float v[4];
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++) {
        v[k] = (float)sums[k] * st * sw[k];
        if (p.bias) v[k] += b[k];
    }
    const size_t at = (size_t)t * p.out_stride + r;
    if (p.out_type == OXH_F32) i8_store4((float *)p.out + at, v, rows - r);
    else if (p.out_type == OXH_F16) i8_store4((_Float16 *)p.out + at, v, rows - r);
    else i8_store4((__bf16 *)p.out + at, v, rows - r);
}

__device__ __forceinline__ void i8_row_factors(const I8Product &p, uint32_t r, float (&sw)[4], float (&b)[4])
{
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++) {
        const uint32_t rk = min(r + k, (uint32_t)p.w.rows - 1u);
        sw[k] = p.w.d_scale[rk];
        b[k] = p.bias ? p.bias[rk] : 0.0f;
    }
}

/* The tile at rows r0.., tokens t0.., over part `split` of the columns: results, or partial sums. */
template <typename G> __device__ __forceinline__ void i8_product_tile(const I8Product &p, uint32_t r0, uint32_t t0, uint32_t split)
{
    const uint32_t rows = (uint32_t)p.w.rows, cols = (uint32_t)p.w.cols;
    const uint32_t ws = (uint32_t)p.w.stride, qs = (uint32_t)p.q_stride;
    const uint32_t stages = (cols + 127u) / 128u, first = split * stages / p.splits, end = (split + 1u) * stages / p.splits;
    const uint32_t k0 = 128u * first, kn = min(cols, 128u * end) - k0;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, wr = wave / G::WT, wt = wave % G::WT;
    const uint32_t row = r0 + wr * G::RF * 16u + 4u * (lane >> 4), tok = t0 + wt * G::TF * 16u + (lane & 15u);
    /* a wave's factors are asked for before the product, so that no result waits for one; the largest tile has no registers
     * for that and asks for all of them at its end */
    constexpr bool EARLY = G::RF * G::TF <= 16u;
    float sw[G::RF][4], b[G::RF][4], st[G::TF];
    auto factors = [&]() {
        if (p.parts) return;
#pragma unroll
        for (uint32_t i = 0; i < G::RF; i++) i8_row_factors(p, row + 16u * i, sw[i], b[i]);
#pragma unroll
        for (uint32_t j = 0; j < G::TF; j++) st[j] = p.q_scale[min(tok + 16u * j, p.n_vec - 1u)];
    };
    if (EARLY) factors();
    v4i acc[G::RF][G::TF];
    const int8_t *w = p.w.d_w + (size_t)r0 * p.w.stride + k0;
    i8_tile<G>([&](uint32_t) { return w; }, [&](uint32_t r) { return min(r, rows - 1u - r0) * ws; },
               p.q + (size_t)t0 * p.q_stride + k0, [&](uint32_t t) { return min(t, p.n_vec - 1u - t0) * qs; }, kn, acc);
    if (!EARLY) factors();
#pragma unroll
    for (uint32_t j = 0; j < G::TF; j++) {
        const uint32_t t = tok + 16u * j;
        if (t >= p.n_vec) break;
#pragma unroll
        for (uint32_t i = 0; i < G::RF; i++) {
            const uint32_t r = row + 16u * i;
            if (r >= rows) break;
            if (p.parts) *reinterpret_cast<v4i *>(p.parts + ((size_t)split * p.n_vec + t) * p.rows_pad + r) = acc[i][j];
            else i8_results(p, r, t, acc[i][j], sw[i], b[i], st[j]);
        }
    }
}

template <typename G>
__global__ __launch_bounds__(G::WAVES * 64, 2) void k_i8_tiles(const I8Product p)
{
    const uint32_t tiles = p.row_tiles * p.tok_tiles, split = blockIdx.x / tiles;
    uint32_t row, tok;
    i8_tile_at(i8_place(blockIdx.x - split * tiles, tiles), p.row_tiles, p.tok_tiles, row, tok);
    i8_product_tile<G>(p, row * G::ROWS, tok * G::TOK, split);
}

/* A last round that would leave half of the CUs idle and more is done in tiles of half the rows: places from p.whole on, two
 * workgroups to each. */
template <typename G, typename H>
__global__ __launch_bounds__(G::WAVES * 64, 2) void k_i8_tiles_tail(const I8Product p)
{
    static_assert(G::TOK == H::TOK && G::ROWS == 2u * H::ROWS && G::WAVES == H::WAVES && G::LDS_BYTES == H::LDS_BYTES, "the same launch");
    uint32_t row, tok;
    if (blockIdx.x < p.whole) {
        i8_tile_at(i8_place(blockIdx.x, p.whole), p.row_tiles, p.tok_tiles, row, tok);
        i8_product_tile<G>(p, row * G::ROWS, tok * G::TOK, 0u);
    } else {
        const uint32_t h = i8_place(blockIdx.x - p.whole, gridDim.x - p.whole);
        i8_tile_at(p.whole + h / 2u, p.row_tiles, p.tok_tiles, row, tok);
        const uint32_t r0 = row * G::ROWS + (h & 1u) * H::ROWS;
        if (r0 < (uint32_t)p.w.rows) i8_product_tile<H>(p, r0, tok * H::TOK, 0u);
    }
}

/* The sums of a product whose columns were shared out: integers, the same in any order.  Four rows to a thread, four parts under
 * way at a time (333 x 4096 in five parts: 9 us one after the other, 7.7 like this). */
__global__ __launch_bounds__(256) void k_i8_join(const I8Product p)
{
    const uint32_t r = (blockIdx.x * 256u + threadIdx.x) * 4u, t = blockIdx.y;
    if (r >= (uint32_t)p.w.rows) return;
    const size_t part = (size_t)p.n_vec * p.rows_pad;
    const int *from = p.parts + (size_t)t * p.rows_pad + r;
    float sw[4], b[4];
    i8_row_factors(p, r, sw, b);
    const float st = p.q_scale[t];
    v4i sums = { 0, 0, 0, 0 };
    for (uint32_t s0 = 0; s0 < p.splits; s0 += 4u) {
        v4i v[4];
#pragma unroll
        for (uint32_t s = 0; s < 4u; s++) v[s] = *reinterpret_cast<const v4i *>(from + part * min(s0 + s, p.splits - 1u));
#pragma unroll
        for (uint32_t s = 0; s < 4u; s++)
            if (s0 + s < p.splits) sums += v[s];
    }
    i8_results(p, r, t, sums, sw, b, st);
}

/* ─── few tokens ──────────────────────────────────────────────────────── */

/* Up to sixteen tokens: the matrix is streamed once and everything else has to stay out of its way.  `team` waves of a
 * workgroup of sixteen share the columns of a group of 16 rows, at most ST stages of 128 columns a wave.  A wave requests all
 * that it multiplies at once: weights eight rows of 128 bytes an instruction, turned into operands through 2 KiB of LDS of its own
 * (loaded in the operand's order, sixteen rows of 64 bytes an instruction, one wave per CU takes 9.0 us for 16.8 MB where it
 * takes 5.5 this way); tokens straight from L2, which all workgroups read.  The waves' sums are joined in LDS, where
 * each leaves its own at the start of its 2 KiB.  Bound by HBM; few rows by the latency of one trip to it. */
#define FEW_TOKENS 16u
#define FEW_WAVES 16u
#define FEW_TURN_BYTES (FEW_WAVES * 2048u)

/* This wave's weights: stages first .. of the group's rows at `rows` (this lane's, lane / 8 and lane / 8 + 8); stages that are not
 * there are the last one again. */
template <int ST>
__device__ __forceinline__ void few_weights(v4i (&w)[ST][2], const int8_t *const (&rows)[2], uint32_t first, uint32_t stages, uint32_t last_piece)
{
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (uint32_t i = 0; i < ST; i++)
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++)
            w[i][h] = *reinterpret_cast<const v4i *>(rows[h] + 16u * min(8u * min(first + i, stages - 1u) + (lane & 7u), last_piece));
}

/* acc += a stage's weights, through `turn`, times tokens b(0), b(1).  Piece c of row r lies at slot c ^ ((r >> 1) & 7) of its
 * 128 bytes, as in i8_tiles.inc. */
template <typename B> __device__ __forceinline__ void few_stage(v4i &acc, const v4i (&w)[2], uint8_t *turn, B b)
{
    const uint32_t lane = threadIdx.x & 63u, r16 = lane & 15u, kq = lane >> 4, swz = (r16 >> 1) & 7u;
    const uint32_t wr = 128u * (lane >> 3) + 16u * ((lane & 7u) ^ ((lane >> 4) & 7u));
    *reinterpret_cast<v4i *>(turn + wr) = w[0];
    *reinterpret_cast<v4i *>(turn + 1024u + (wr ^ 64u)) = w[1];
    i8_wave_sync();
    const v4i a0 = *reinterpret_cast<const v4i *>(turn + 128u * r16 + 16u * (kq ^ swz));
    const v4i a1 = *reinterpret_cast<const v4i *>(turn + 128u * r16 + 16u * ((4u + kq) ^ swz));
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, b(0u), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, b(1u), acc, 0, 0, 0);
    i8_wave_sync();
}

/* The sums of a group of rows and up to sixteen tokens over `mine` stages from `first` on, left in this wave's `turn`.
 * q_row: this lane's token, lane % 16. */
template <int ST>
__device__ __forceinline__ void few_sums(const int8_t *const (&rows)[2], const int8_t *q_row, uint32_t cols, uint32_t first, uint32_t mine,
                                         uint8_t *turn)
{
    const uint32_t lane = threadIdx.x & 63u, kq = lane >> 4, stages = (cols + 127u) / 128u, last_piece = (cols - 1u) / 16u;
    v4i w[ST][2], q[2][2];
    auto tokens = [&](uint32_t i) {
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++)
            q[i & 1u][h] = *reinterpret_cast<const v4i *>(q_row + 16u * min(8u * min(first + i, stages - 1u) + 4u * h + kq, last_piece));
    };
    tokens(0u);
    few_weights<ST>(w, rows, first, stages, last_piece);
    v4i acc = { 0, 0, 0, 0 };
#pragma unroll
    for (uint32_t i = 0; i < ST; i++) {
        if (i + 1u < ST) tokens(i + 1u);
        if (i < mine) {
            if (128u * (first + i + 1u) > cols) {           /* the tokens' columns behind the last one count as 0 */
#pragma unroll
                for (uint32_t h = 0; h < 2u; h++)
#pragma unroll
                    for (uint32_t d = 0; d < 4u; d++) {
                        const uint32_t at = 128u * (first + i) + 64u * h + 16u * kq + 4u * d, left = cols > at ? cols - at : 0u;
                        if (left < 4u) q[i & 1u][h][d] &= (int)((1u << (8u * left)) - 1u);
                    }
            }
            few_stage(acc, w[i], turn, [&](uint32_t h) { return q[i & 1u][h]; });
        }
    }
    *reinterpret_cast<v4i *>(turn + 16u * lane) = acc;
}

/* Part `part` of `parts` of a row's stages. */
__device__ __forceinline__ void few_part(uint32_t stages, uint32_t part, uint32_t parts, uint32_t &first, uint32_t &mine)
{
    first = part * stages / parts;
    mine = (part + 1u) * stages / parts - first;
}

/* The joined sums of the `count` waves from `wave` on. */
__device__ __forceinline__ v4i few_join(const uint8_t *turns, uint32_t wave, uint32_t count)
{
    v4i sums = { 0, 0, 0, 0 };
    for (uint32_t k = 0; k < count; k += 4u) {                      /* four reads under way at a time */
        v4i v[4];
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++)
            v[i] = *reinterpret_cast<const v4i *>(turns + 2048u * (wave + min(k + i, count - 1u)) + 16u * (threadIdx.x & 63u));
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++)
            if (k + i < count) sums += v[i];
    }
    return sums;
}

/* quantised tokens */
template <int ST>
__global__ __launch_bounds__(1024, ST <= 4 ? 8 : 4) void k_i8_few(const I8Product p, uint32_t team, uint32_t groups)
{
    __shared__ __attribute__((aligned(16))) uint8_t turns[FEW_TURN_BYTES];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t rows = (uint32_t)p.w.rows, cols = (uint32_t)p.w.cols, teams = FEW_WAVES / team, r16 = lane & 15u;
    const uint32_t r0 = 16u * min(blockIdx.x * teams + wave / team, groups - 1u);
    uint32_t first, mine;
    few_part((cols + 127u) / 128u, wave % team, team, first, mine);
    const int8_t *w[2];
#pragma unroll
    for (uint32_t h = 0; h < 2u; h++) w[h] = p.w.d_w + (size_t)min(r0 + 8u * h + (lane >> 3), rows - 1u) * p.w.stride;
    /* what the results of this wave's rows need, if it is one that joins */
    const uint32_t g = blockIdx.x * teams + wave, r = 16u * g + 4u * (lane >> 4);
    float sw[4], b[4];
    float st;
    auto factors = [&]() {
        i8_row_factors(p, min(r, rows - 1u), sw, b);
        st = p.q_scale[min(r16, p.n_vec - 1u)];
    };
    /* asked for early where a trip to memory is what the launch takes; late where the registers are wanted for weights */
    if (ST <= 2) factors();
    few_sums<ST>(w, p.q + (size_t)min(r16, p.n_vec - 1u) * p.q_stride, cols, first, mine, turns + 2048u * wave);
    if (ST > 2) factors();
    __syncthreads();
    if (wave < teams && g < groups && r < rows && r16 < p.n_vec) i8_results(p, r, r16, few_join(turns, wave * team, team), sw, b, st);
}

/* 17 to 64 tokens, TF fragments of sixteen: the same, but a stage's tokens come as the weights do, eight rows of 128 bytes an
 * instruction, and are turned the same way, the next stage's requested as soon as these are in LDS. */
template <int TF>
__global__ __launch_bounds__(1024) void k_i8_few_wide(const I8Product p, uint32_t team, uint32_t groups)
{
    constexpr uint32_t ST = 2;                      /* few_team() gives these tokens no more */
    constexpr uint32_t TURN = TF > 2 ? TF * 1024u : 2048u;
    __shared__ __attribute__((aligned(16))) uint8_t turns[FEW_WAVES * TURN];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t rows = (uint32_t)p.w.rows, cols = (uint32_t)p.w.cols, teams = FEW_WAVES / team, r16 = lane & 15u, kq = lane >> 4;
    const uint32_t r0 = 16u * min(blockIdx.x * teams + wave / team, groups - 1u);
    const uint32_t stages = (cols + 127u) / 128u, last_piece = (cols - 1u) / 16u;
    uint32_t first, mine;
    few_part(stages, wave % team, team, first, mine);
    uint8_t *const turn = turns + TURN * wave;
    const int8_t *wrow[2];
#pragma unroll
    for (uint32_t h = 0; h < 2u; h++) wrow[h] = p.w.d_w + (size_t)min(r0 + 8u * h + (lane >> 3), rows - 1u) * p.w.stride;
    v4i w[ST][2], q[TF][2];
    few_weights<ST>(w, wrow, first, stages, last_piece);
    auto tokens = [&](uint32_t i) {
        const uint32_t at = 16u * min(8u * min(first + i, stages - 1u) + (lane & 7u), last_piece);
#pragma unroll
        for (uint32_t j = 0; j < TF; j++)
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++)
                q[j][h] = *reinterpret_cast<const v4i *>(p.q + (size_t)min(16u * j + 8u * h + (lane >> 3), p.n_vec - 1u) * p.q_stride + at);
    };
    tokens(0u);
    const uint32_t swz = (r16 >> 1) & 7u, wr = 128u * (lane >> 3) + 16u * ((lane & 7u) ^ ((lane >> 4) & 7u));
    const uint32_t rd[2] = { 128u * r16 + 16u * (kq ^ swz), 128u * r16 + 16u * ((4u + kq) ^ swz) };
    auto turned = [&](const v4i (&from)[2], v4i (&to)[2]) {
        *reinterpret_cast<v4i *>(turn + wr) = from[0];
        *reinterpret_cast<v4i *>(turn + 1024u + (wr ^ 64u)) = from[1];
        i8_wave_sync();
        to[0] = *reinterpret_cast<const v4i *>(turn + rd[0]);
        to[1] = *reinterpret_cast<const v4i *>(turn + rd[1]);
        i8_wave_sync();
    };
    v4i acc[TF];
#pragma unroll
    for (uint32_t j = 0; j < TF; j++) acc[j] = v4i{ 0, 0, 0, 0 };
#pragma unroll
    for (uint32_t i = 0; i < ST; i++) {
        if (i < mine) {
            if (128u * (first + i + 1u) > cols) {           /* the weights' columns behind the last one count as 0 */
#pragma unroll
                for (uint32_t d = 0; d < 4u; d++) {
                    const uint32_t at = 128u * (first + i) + 16u * (lane & 7u) + 4u * d, left = cols > at ? cols - at : 0u;
                    const int mask = left < 4u ? (int)((1u << (8u * left)) - 1u) : -1;
                    w[i][0][d] &= mask;
                    w[i][1][d] &= mask;
                }
            }
            v4i a[2], b[TF][2];
            turned(w[i], a);
#pragma unroll
            for (uint32_t j = 0; j < TF; j++) turned(q[j], b[j]);
            if (i + 1u < ST) tokens(i + 1u);
#pragma unroll
            for (uint32_t j = 0; j < TF; j++) {
                acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[0], b[j][0], acc[j], 0, 0, 0);
                acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[1], b[j][1], acc[j], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < TF; j++) *reinterpret_cast<v4i *>(turn + 1024u * j + 16u * lane) = acc[j];
    __syncthreads();
    /* a wave joins a fragment of a team's, or several */
    for (uint32_t x = wave; x < teams * TF; x += FEW_WAVES) {
        const uint32_t mate = x / TF, j = x % TF, g = blockIdx.x * teams + mate, r = 16u * g + 4u * kq, t = 16u * j + r16;
        if (g >= groups || r >= rows || t >= p.n_vec) continue;
        float sw[4], b[4];
        i8_row_factors(p, r, sw, b);
        const float st = p.q_scale[t];
        v4i sums = { 0, 0, 0, 0 };
        for (uint32_t k = 0; k < team; k++) sums += *reinterpret_cast<const v4i *>(turns + TURN * (mate * team + k) + 1024u * j + 16u * lane);
        i8_results(p, r, t, sums, sw, b, st);
    }
}

/* Float tokens, which every workgroup quantises for itself (k_i8_quantize's codes): their values are requested before the weights
 * and wait in registers; the codes lie in LDS in the order the MFMA takes them, [16-column piece][token]. */
#define FEW_HELD 4u                                    /* times eight values of a token that a lane holds */
#define FEW_HEAD_BYTES (FEW_TURN_BYTES + 128u)         /* and the scales, a maximum per wave */

/* Codes of a row that `per` neighbouring waves hold, wave - w0 the first of them, this one from value 8 * (64 * w0 + lane) on, 512 * per apart;
 * piece after piece n pieces apart, up to `end` codes.  Returns the scale; `store`: whether there is a row. */
template <uint32_t HELD>
__device__ __forceinline__ float few_codes(const float (&v)[HELD][8], uint32_t per, uint32_t w0, uint32_t wave, uint32_t *s_top, bool store,
                                           uint8_t *codes, uint32_t n, uint32_t end)
{
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < HELD; i++) top = max(top, i8_top8(v[i]));
    top = wave_top(top);
    if (lane == 0u) s_top[wave] = top;
    __syncthreads();
    top = row_top((lane & 15u) < per ? s_top[min(wave - w0 + (lane & 15u), FEW_WAVES - 1u)] : top);
    float inv;
    const float s = i8_scale(top, inv);
    if (store) {
#pragma unroll
        for (uint32_t i = 0; i < HELD; i++) {
            const uint32_t c = 8u * (64u * w0 + lane) + 512u * per * i;
            if (c < end)
                *reinterpret_cast<uint2 *>(codes + 16u * n * (c / 16u) + (c & 8u)) = inv != 0.0f ? i8_codes8(v[i], s, inv) : make_uint2(0u, 0u);
        }
    }
    return s;
}

template <typename XT, int ST>
__global__ __launch_bounds__(1024) void
k_i8_few_float(const I8Product p, const XT *__restrict__ x, size_t x_stride, uint32_t team, uint32_t groups)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t few_shared[];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    float *const s_scale = reinterpret_cast<float *>(few_shared + FEW_TURN_BYTES);
    uint32_t *const s_top = reinterpret_cast<uint32_t *>(few_shared + FEW_TURN_BYTES + 64u);
    uint8_t *const codes = few_shared + FEW_HEAD_BYTES;
    const uint32_t r16 = lane & 15u, kq = lane >> 4;
    const uint32_t rows = (uint32_t)p.w.rows, cols = (uint32_t)p.w.cols, n = p.n_vec, teams = FEW_WAVES / team;
    const uint32_t stages = (cols + 127u) / 128u, pieces = 8u * stages;
    uint32_t first, mine;
    few_part(stages, wave % team, team, first, mine);

    /* tokens: waves per * t .. of token t */
    const uint32_t per = n == 1u ? 16u : n == 2u ? 8u : n <= 4u ? 4u : n <= 8u ? 2u : 1u;
    const uint32_t t = wave / per, w0 = wave % per, c0 = 8u * (64u * w0 + lane), step = 512u * per;
    float v[FEW_HELD][8];
    const XT *xr = x + (size_t)min(t, n - 1u) * x_stride;
#pragma unroll
    for (uint32_t i = 0; i < FEW_HELD; i++) i8_values8<XT, false>(xr, nullptr, c0 + step * i, t < n ? cols : 0u, v[i]);
    const uint32_t r0 = 16u * min(blockIdx.x * teams + wave / team, groups - 1u);
    const int8_t *wrow[2];
#pragma unroll
    for (uint32_t h = 0; h < 2u; h++) wrow[h] = p.w.d_w + (size_t)min(r0 + 8u * h + (lane >> 3), rows - 1u) * p.w.stride;
    const uint32_t g = blockIdx.x * teams + wave, r = 16u * g + 4u * kq;
    float sw[4], b[4];
    if (ST <= 2) i8_row_factors(p, min(r, rows - 1u), sw, b);
    v4i w[ST][2];
    few_weights<ST>(w, wrow, first, stages, (cols - 1u) / 16u);

    const float s = few_codes(v, per, w0, wave, s_top, t < n, codes + 16u * t, n, 16u * pieces);
    if (t < n && w0 == 0u && lane == 0u) s_scale[t] = s;
    __syncthreads();

    const uint8_t *mine_codes = codes + 16u * (kq * n + min(r16, n - 1u));
    v4i acc = { 0, 0, 0, 0 };
#pragma unroll
    for (uint32_t i = 0; i < ST; i++)
        if (i < mine)
            few_stage(acc, w[i], few_shared + 2048u * wave,
                      [&](uint32_t h) { return *reinterpret_cast<const v4i *>(mine_codes + 16u * n * (8u * (first + i) + 4u * h)); });
    *reinterpret_cast<v4i *>(few_shared + 2048u * wave + 16u * lane) = acc;
    if (ST > 2) i8_row_factors(p, min(r, rows - 1u), sw, b);
    __syncthreads();
    if (wave < teams && g < groups && r < rows && r16 < n) i8_results(p, r, r16, few_join(few_shared, wave * team, team), sw, b, s_scale[r16]);
}

/* ─── experts ─────────────────────────────────────────────────────────── */

/* Up to a number of pairs of an expert: n of them from sorted pair `first` on; n 0: nothing.  The expert's tiles are `count` from
 * entry `base` on; all: tiles there are. */
struct I8ExpertTile {
    uint32_t expert, first, n, all, base, count, unused[2];
};

/* The first launch of a layer: a workgroup per token to quantise it, and one that cuts the experts' runs of the sorted pairs into tiles
 * of `tok`; entries behind the last tile say so. */
template <typename T, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void
k_i8_experts_begin(const T *__restrict__ x, size_t x_stride, uint32_t cols, int8_t *__restrict__ q, size_t q_stride,
                   float *__restrict__ scale, const uint32_t *__restrict__ offsets, uint32_t n_expert, uint32_t pairs, uint32_t tok,
                   I8ExpertTile *__restrict__ tiles, uint32_t n_tiles)
{
    __shared__ uint32_t s_first[OXH_SELECT_MAX_EXPERTS + 1], s_tile[OXH_SELECT_MAX_EXPERTS + 1];
    if (blockIdx.x != 0u) {
        const size_t row = blockIdx.x - 1u;
        i8_quantize_row<T, false, THREADS, HELD>(x + row * x_stride, nullptr, cols, q + row * q_stride, scale + row);
        return;
    }
    for (uint32_t e = threadIdx.x; e <= n_expert; e += THREADS) s_first[e] = min(offsets[e], pairs);
    __syncthreads();
    if (threadIdx.x < 64u) {                        /* eight experts to a lane: where their tiles start */
        uint32_t own[8], sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) {
            const uint32_t e = 8u * threadIdx.x + i;
            const uint32_t n = e < n_expert && s_first[e + 1u] > s_first[e] ? s_first[e + 1u] - s_first[e] : 0u;
            own[i] = (n + tok - 1u) / tok;
            sum += own[i];
        }
        uint32_t upto = sum;
#pragma unroll
        for (uint32_t d = 1; d < 64u; d <<= 1) {
            const uint32_t v = __shfl_up(upto, d);
            if (threadIdx.x >= d) upto += v;
        }
        uint32_t at = upto - sum;
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) {
            if (8u * threadIdx.x + i <= n_expert) s_tile[8u * threadIdx.x + i] = at;
            at += own[i];
        }
        if (threadIdx.x == 63u && n_expert == OXH_SELECT_MAX_EXPERTS) s_tile[n_expert] = at;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n_tiles; i += THREADS) {
        I8ExpertTile t = { 0u, 0u, 0u, s_tile[n_expert], 0u, 0u, { 0u, 0u } };
        if (i < s_tile[n_expert]) {
            uint32_t lo = 0, hi = n_expert;         /* the last expert whose tiles start at i or before */
            while (hi - lo > 1u) {
                const uint32_t mid = (lo + hi) / 2u;
                if (s_tile[mid] <= i) lo = mid;
                else hi = mid;
            }
            t.expert = lo;
            t.first = s_first[lo] + tok * (i - s_tile[lo]);
            t.n = min(tok, s_first[lo + 1u] - t.first);
            t.base = s_tile[lo];
            t.count = min(s_tile[lo + 1u], n_tiles) - t.base;       /* offsets out of order can ask for more tiles than any routing has */
        }
        tiles[i] = t;
    }
}

/* What the experts' products read and write: gate and up (UP) over tokens through perm into h, or down over the pairs' codes
 * into y. */
struct I8Experts {
    const int8_t *w[2];
    const float *s[2];
    size_t stride;
    const int8_t *q;
    size_t q_stride;
    const float *q_scale;
    const uint32_t *perm;
    const I8ExpertTile *tiles;
    float *out;
    size_t out_stride;
    uint32_t rows, cols, n_tok, n_tiles, row_tiles;
};

/* the row of codes of a tile's pair j */
template <bool UP> __device__ __forceinline__ uint32_t i8_pair_row(const I8Experts &p, const I8ExpertTile &t, uint32_t j)
{
    const uint32_t pair = t.first + min(j, t.n - 1u);
    return UP ? min(p.perm[pair], p.n_tok - 1u) : pair;
}

/* The scales of four rows of the expert (UP: of gate's and of up's). */
template <bool UP> __device__ __forceinline__ void i8_pair_scales(const I8Experts &p, const I8ExpertTile &t, uint32_t r, float (&s0)[4], float (&s1)[4])
{
    const size_t row0 = (size_t)t.expert * p.rows;
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++) {
        const uint32_t rk = min(r + k, p.rows - 1u);
        s0[k] = p.s[0][row0 + rk];
        s1[k] = UP ? p.s[1][row0 + rk] : 0.0f;
    }
}

/* Four rows' results of a pair from its sums.  The quantiser's silu, so that h has the codes that oxh_i8_quantize gives of gate and up: an
 * exponential of the instruction's kind, 2^(g * -1.4427), takes 2000 tokens over 8 of 128 experts 6 us less (245 and 251), but its rounded
 * argument alone is 0.8 |g| units of 2^-24 off in the result (64 at -80), where this stays within 7. */
template <bool UP>
__device__ __forceinline__ Run<float, 4> i8_pair_values(const v4i &first, const v4i &second, const float (&s0)[4], const float (&s1)[4], float st)
{
    Run<float, 4> r;
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++) {
        r.v[k] = (float)first[k] * st * s0[k];
        if (UP) r.v[k] = silu(r.v[k]) * ((float)second[k] * st * s1[k]);
    }
    return r;
}

/* A tile's results to memory, for products of few columns, which are half stores.  A wave holds four rows of each of sixteen tokens,
 * 64 bytes of an output row at a time; stored like that a launch writes 2.8 TB/s (131 MB beside the products of 768 columns: 47 us
 * more; a fill of them takes 22).  So the workgroup's results are gathered in its LDS, token by token, and written 16 bytes
 * to a lane along the rows (30 us).  Long products (i8_product_tile) are 3 % faster without the two barriers this takes.
 *
 * PER: a wave's fragments of 16 rows; value(i, j): its four results of fragment i, tokens j, as T.  out: the tile's first
 * token and row; rows, toks: how many of them there are.  T's of four bytes may be ints as well. */
template <typename G, typename T, uint32_t PER, typename Value>
__device__ __forceinline__ void i8_store_tile(Value value, T *out, size_t out_stride, uint32_t rows, uint32_t toks)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t i8_lds[];
    constexpr uint32_t ROWS = 16u * PER * G::WR, ROW_BYTES = ROWS * sizeof(T), PITCH = ROW_BYTES + 16u, THREADS = 64u * G::WAVES;
    constexpr uint32_t JC = G::TF * 16u * G::WT * PITCH <= G::LDS_BYTES ? G::TF : G::TF / 2u;       /* of a wave's tokens at a time */
    static_assert(JC * 16u * G::WT * PITCH <= G::LDS_BYTES, "half of the tokens fit");
    constexpr uint32_t CHUNKS = ROW_BYTES / 16u, STEP = 16u / sizeof(T);
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, wr = wave / G::WT, wt = wave % G::WT;
#pragma unroll
    for (uint32_t j0 = 0; j0 < G::TF; j0 += JC) {
        __syncthreads();                            /* operands, or the tokens before, are read */
#pragma unroll
        for (uint32_t j = j0; j < j0 + JC; j++)
#pragma unroll
            for (uint32_t i = 0; i < PER; i++) {
                const Run<T, 4> r = value(i, j);
                uint8_t *to = i8_lds + (16u * (wt * JC + j - j0) + (lane & 15u)) * PITCH + (16u * (wr * PER + i) + 4u * (lane >> 4)) * sizeof(T);
                typedef T T4 __attribute__((ext_vector_type(4)));
                *reinterpret_cast<T4 *>(to) = T4{ r.v[0], r.v[1], r.v[2], r.v[3] };
            }
        __syncthreads();
#pragma unroll 4
        for (uint32_t f = threadIdx.x; f < 16u * G::WT * JC * CHUNKS; f += THREADS) {
            const uint32_t at = f / CHUNKS, c = f % CHUNKS, tok = 16u * (at / (16u * JC) * G::TF + j0) + at % (16u * JC), r = c * STEP;
            if (tok >= toks || r >= rows) continue;
            const Run<T, STEP> v = *reinterpret_cast<const Run<T, STEP> *>(i8_lds + at * PITCH + 16u * c);
            T *to = out + (size_t)tok * out_stride + r;
            if (r + STEP <= rows) *reinterpret_cast<Run<T, STEP> *>(to) = v;
            else
#pragma unroll
                for (uint32_t k = 0; k < STEP - 1u; k++)
                    if (r + k < rows) to[k] = v.v[k];
        }
    }
}

/* A tile of an expert's rows and pairs.  UP: the tile's fragments of 16 rows are gate's and up's by turns, so that a wave holds
 * both factors of a result. */
template <typename G, bool UP> __device__ __forceinline__ void i8_experts_tile(const I8Experts &p, const I8ExpertTile &t, uint32_t row_tile)
{
    constexpr uint32_t OUT_ROWS = UP ? G::ROWS / 2u : G::ROWS;
    const uint32_t r0 = row_tile * OUT_ROWS, stride = (uint32_t)p.stride, qs = (uint32_t)p.q_stride;
    const size_t at = ((size_t)t.expert * p.rows + r0) * p.stride;
    const int8_t *w0 = p.w[0] + at, *w1 = p.w[1] + at, *q = UP ? p.q : p.q + (size_t)t.first * p.q_stride;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, wr = wave / G::WT, wt = wave % G::WT;
    constexpr uint32_t PER = UP ? G::RF / 2u : G::RF;               /* results' fragments of a wave */
    const uint32_t row = r0 + wr * PER * 16u + 4u * (lane >> 4), tok = wt * G::TF * 16u + (lane & 15u);
    float s0[PER][4], s1[PER][4], st[G::TF];
#pragma unroll
    for (uint32_t i = 0; i < PER; i++) i8_pair_scales<UP>(p, t, row + 16u * i, s0[i], s1[i]);
#pragma unroll
    for (uint32_t j = 0; j < G::TF; j++) st[j] = p.q_scale[i8_pair_row<UP>(p, t, tok + 16u * j)];
    v4i acc[G::RF][G::TF];
    i8_tile<G>([&](uint32_t o) { return UP && ((o >> 1) & 1u) ? w1 : w0; },
               [&](uint32_t r) { return min(UP ? 16u * (r >> 5) + (r & 15u) : r, p.rows - 1u - r0) * stride; }, q,
               [&](uint32_t j) { return (UP ? i8_pair_row<UP>(p, t, j) : min(j, t.n - 1u)) * qs; }, p.cols, acc);
    i8_store_tile<G, float, PER>(
        [&](uint32_t i, uint32_t j) {
            return i8_pair_values<UP>(acc[UP ? 2u * i : i][j], acc[UP ? 2u * i + 1u : i][j], s0[i], s1[i], st[j]);
        },
        p.out + (size_t)t.first * p.out_stride + r0, p.out_stride, p.rows - r0, t.n);
}

/* G: as many pairs as a table entry can have; H, Q: fewer, for the last ones of an expert's.  2000 tokens, 8 of 128 experts of 2048 x 768:
 * gate and up in 113 us (403 MB of weights, which take 65 alone, and 100 Gop, which take 37, with the empty places of the tiles 47), down in 79 (201 MB, and 131 of
 * results). */
template <typename G, typename H, typename Q, bool UP>
__global__ __launch_bounds__(G::WAVES * 64, 2) void k_i8_experts(const I8Experts p)
{
    /* those that there are, dealt to the XCDs evenly; the tiles of an expert that share weights next to each other */
    const uint32_t all = min(p.tiles[0].all, p.n_tiles) * p.row_tiles;
    if (blockIdx.x >= all) return;
    const uint32_t i = i8_place(blockIdx.x, all);
    const I8ExpertTile any = p.tiles[i / p.row_tiles];
    const uint32_t in = i - any.base * p.row_tiles, row_tile = in / any.count;
    const I8ExpertTile t = p.tiles[any.base + in % any.count];
    if (Q::TOK < H::TOK && t.n <= Q::TOK) i8_experts_tile<Q, UP>(p, t, row_tile);
    else if (t.n <= H::TOK) i8_experts_tile<H, UP>(p, t, row_tile);
    else i8_experts_tile<G, UP>(p, t, row_tile);
}

/* Up to sixteen pairs of an expert, as k_i8_few: `team` waves share a group of 16 rows; UP: half of them take gate, half up.  Bound by
 * memory: 8 experts of 4096 x 14336, 16 tokens of two: gate and up in 155 us, 6.1 TB/s, down in 98, 4.8 TB/s. */
template <int ST, bool UP>
__global__ __launch_bounds__(1024, ST <= 4 ? 8 : 4) void k_i8_experts_few(const I8Experts p, uint32_t team, uint32_t groups)
{
    __shared__ __attribute__((aligned(16))) uint8_t turns[FEW_TURN_BYTES];
    const I8ExpertTile t = p.tiles[blockIdx.y];
    if (t.n == 0u) return;
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t teams = FEW_WAVES / team, parts = UP ? team / 2u : team, r16 = lane & 15u;
    const uint32_t r0 = 16u * min(blockIdx.x * teams + wave / team, groups - 1u), which = wave % team / parts;
    uint32_t first, mine;
    few_part((p.cols + 127u) / 128u, wave % parts, parts, first, mine);
    const int8_t *w[2];
#pragma unroll
    for (uint32_t h = 0; h < 2u; h++)
        w[h] = p.w[which] + ((size_t)t.expert * p.rows + min(r0 + 8u * h + (lane >> 3), p.rows - 1u)) * p.stride;
    const uint32_t g = blockIdx.x * teams + wave, r = 16u * g + 4u * (lane >> 4), q_row = i8_pair_row<UP>(p, t, r16);
    float s0[4], s1[4], st;
    auto factors = [&]() {
        i8_pair_scales<UP>(p, t, min(r, p.rows - 1u), s0, s1);
        st = p.q_scale[q_row];
    };
    if (ST <= 2) factors();
    few_sums<ST>(w, p.q + (size_t)q_row * p.q_stride, p.cols, first, mine, turns + 2048u * wave);
    if (ST > 2) factors();
    __syncthreads();
    if (wave < teams && g < groups && r16 < t.n && r < p.rows) {
        const v4i a = few_join(turns, wave * team, parts);
        const Run<float, 4> v = i8_pair_values<UP>(a, UP ? few_join(turns, wave * team + parts, parts) : a, s0, s1, st);
        i8_store4(p.out + (size_t)(t.first + r16) * p.out_stride + r, v.v, p.rows - r);
    }
}

/* ─── the experts of a few tokens, pair by pair ───────────────────────── */

/* A decode step has a handful of pairs, hardly two of one expert, and what it takes is launches: here there are two.  Nothing is sorted or
 * tabled; a pair's expert is read from its id, and each launch quantises what it multiplies by itself, as k_i8_few_float does.  The sums are
 * integers and the float steps those of the other kernels: the same results, bit by bit.  One token, 8 experts of 2048 x 768: 9.4 and
 * 6.5 us for 25 and 13 MB, a chain of id, weights and tokens, quantisation and joins behind the memory's 4.1 and 2. */
struct I8Pairs {
    I8Experts e;
    const int32_t *ids;
    const float *weights;
    uint32_t k, n_expert;
};
__device__ __forceinline__ uint32_t i8_pair_expert(const I8Pairs &p, uint32_t pair) { return min((uint32_t)p.ids[pair], p.n_expert - 1u); }

/* h of pair blockIdx.y: `team` waves to a group of 16 rows, half of them gate, half up (k_i8_experts_few) */
template <typename XT, int ST>
__global__ __launch_bounds__(1024, ST <= 4 ? 8 : 4) void
k_i8_pair_up(const I8Pairs p, const XT *__restrict__ x, size_t x_stride, uint32_t team, uint32_t groups)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t few_shared[];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint32_t *const s_top = reinterpret_cast<uint32_t *>(few_shared + FEW_TURN_BYTES + 64u);
    uint8_t *const codes = few_shared + FEW_HEAD_BYTES, *const turn = few_shared + 2048u * wave;
    const uint32_t rows = p.e.rows, cols = p.e.cols, stages = (cols + 127u) / 128u, kq = lane >> 4;
    const uint32_t teams = FEW_WAVES / team, parts = team / 2u, which = wave % team / parts;
    float v[1][8];                                  /* 8192 columns a workgroup, as many as eight waves take of an expert's rows */
    i8_values8<XT, false>(x + (size_t)(blockIdx.y / p.k) * x_stride, nullptr, 8u * (64u * wave + lane), cols, v[0]);
    const I8ExpertTile t = { i8_pair_expert(p, blockIdx.y), blockIdx.y, 1u, 0u, 0u, 0u, { 0u, 0u } };
    const uint32_t r0 = 16u * min(blockIdx.x * teams + wave / team, groups - 1u);
    uint32_t first, mine;
    few_part(stages, wave % parts, parts, first, mine);
    const int8_t *wrow[2];
#pragma unroll
    for (uint32_t h = 0; h < 2u; h++)
        wrow[h] = p.e.w[which] + ((size_t)t.expert * rows + min(r0 + 8u * h + (lane >> 3), rows - 1u)) * p.e.stride;
    v4i w[ST][2];
    few_weights<ST>(w, wrow, first, stages, (cols - 1u) / 16u);
    const uint32_t g = blockIdx.x * teams + wave, r = 16u * g + 4u * kq;
    float s0[4], s1[4];
    if (ST <= 2) i8_pair_scales<true>(p.e, t, min(r, rows - 1u), s0, s1);
    const float st = few_codes(v, FEW_WAVES, wave, wave, s_top, true, codes, 1u, 128u * stages);
    __syncthreads();
    v4i acc = { 0, 0, 0, 0 };
#pragma unroll
    for (uint32_t i = 0; i < ST; i++)
        if (i < mine)
            few_stage(acc, w[i], turn, [&](uint32_t h) { return *reinterpret_cast<const v4i *>(codes + 16u * (8u * (first + i) + 4u * h + kq)); });
    *reinterpret_cast<v4i *>(turn + 16u * lane) = acc;
    if (ST > 2) i8_pair_scales<true>(p.e, t, min(r, rows - 1u), s0, s1);
    __syncthreads();
    if (wave < teams && g < groups && r < rows && (lane & 15u) == 0u) {
        const Run<float, 4> hv = i8_pair_values<true>(few_join(few_shared, wave * team, parts), few_join(few_shared, wave * team + parts, parts), s0, s1, st);
        i8_store4(p.e.out + (size_t)blockIdx.y * p.e.out_stride + r, hv.v, rows - r);
    }
}

/* Results of token blockIdx.y, 16 rows of them: `per` waves to each of its pairs. */
#define FEW_PAIRS_BYTES (FEW_HEAD_BYTES + 64u * OXH_SELECT_MAX_TOPK)       /* and a term per pair and row */
template <typename T, int ST>
__global__ __launch_bounds__(1024, ST <= 4 ? 8 : 4) void
k_i8_pair_down(const I8Pairs p, const float *__restrict__ h, size_t h_stride, T *__restrict__ out, size_t out_stride, uint32_t per)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t few_shared[];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    float *const s_scale = reinterpret_cast<float *>(few_shared + FEW_TURN_BYTES), *const s_term = reinterpret_cast<float *>(few_shared + FEW_HEAD_BYTES);
    uint32_t *const s_top = reinterpret_cast<uint32_t *>(few_shared + FEW_TURN_BYTES + 64u);
    const uint32_t rows = p.e.rows, cols = p.e.cols, stages = (cols + 127u) / 128u, kq = lane >> 4, r0 = 16u * blockIdx.x;
    const uint32_t j = min(wave / per, p.k - 1u), w0 = wave % per, pair = blockIdx.y * p.k + j;
    const bool live = wave < per * p.k;
    constexpr int HELD = ST <= 4 ? 1 : 2;           /* 512 columns a wave */
    uint8_t *const codes = few_shared + FEW_PAIRS_BYTES + 128u * stages * j, *const turn = few_shared + 2048u * wave;
    float v[HELD][8];
#pragma unroll
    for (uint32_t i = 0; i < HELD; i++)
        i8_values8<float, false>(h + (size_t)pair * h_stride, nullptr, 8u * (64u * w0 + lane) + 512u * per * i, cols, v[i]);
    uint32_t first, mine;
    few_part(stages, w0, per, first, mine);
    const int8_t *wrow[2];
    const size_t row0 = (size_t)i8_pair_expert(p, pair) * rows;
#pragma unroll
    for (uint32_t i = 0; i < 2u; i++) wrow[i] = p.e.w[0] + (row0 + min(r0 + 8u * i + (lane >> 3), rows - 1u)) * p.e.stride;
    v4i w[ST][2];
    few_weights<ST>(w, wrow, first, stages, (cols - 1u) / 16u);
    /* a thread per pair and row for the terms */
    const uint32_t tj = min(threadIdx.x / 16u, p.k - 1u), tr = threadIdx.x % 16u, t_pair = blockIdx.y * p.k + tj;
    const float sw = p.e.s[0][(size_t)i8_pair_expert(p, t_pair) * rows + min(r0 + tr, rows - 1u)], weight = p.weights[t_pair];
    const float st = few_codes(v, per, w0, wave, s_top, live, codes, 1u, 128u * stages);
    if (live && w0 == 0u && lane == 0u) s_scale[j] = st;
    __syncthreads();
    v4i acc = { 0, 0, 0, 0 };
#pragma unroll
    for (uint32_t i = 0; i < ST; i++)
        if (i < mine)
            few_stage(acc, w[i], turn, [&](uint32_t q) { return *reinterpret_cast<const v4i *>(codes + 16u * (8u * (first + i) + 4u * q + kq)); });
    if ((lane & 15u) == 0u) *reinterpret_cast<v4i *>(turn + 16u * kq) = acc;
    __syncthreads();
    if (threadIdx.x < 16u * p.k) {
        int sum = 0;
#pragma unroll 4
        for (uint32_t i = 0; i < per; i++) sum += *reinterpret_cast<const int *>(few_shared + 2048u * (tj * per + i) + 4u * tr);
        s_term[threadIdx.x] = weight * ((float)sum * s_scale[tj] * sw);
    }
    __syncthreads();
    if (threadIdx.x < 16u && r0 + threadIdx.x < rows) {
        float total = 0.0f;
        for (uint32_t i = 0; i < p.k; i++) total += s_term[16u * i + threadIdx.x];
        out[blockIdx.y * out_stride + r0 + threadIdx.x] = from_f32<T>(total);
    }
}

/* out[t] = sum over t's pairs, in their order, of weight * y.  Four columns to a thread, eight of the token's pairs under way at a
 * time.  Bound by memory: 2000 tokens, 8 x 2048 each, in 21.6 us, 6.4 TB/s. */
template <typename T>
__global__ __launch_bounds__(256) void
k_i8_combine(const float *__restrict__ y, size_t y_stride, const float *__restrict__ weights, const uint32_t *__restrict__ slot_pos,
             uint32_t k, uint32_t pairs, uint32_t cols, T *__restrict__ out, size_t out_stride)
{
    const size_t t = blockIdx.y;
    const uint32_t c = 4u * (blockIdx.x * 256u + threadIdx.x);
    if (c >= cols) return;
    float acc[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
    for (uint32_t j0 = 0; j0 < k; j0 += 8u) {
        v4f v[8];
        float w[8];
#pragma unroll
        for (uint32_t j = 0; j < 8u; j++) {                         /* past the end: the last pair again */
            const size_t pair = t * k + min(j0 + j, k - 1u);
            w[j] = weights[pair];
            v[j] = *reinterpret_cast<const v4f *>(y + (size_t)min(slot_pos[pair], pairs - 1u) * y_stride + c);
        }
#pragma unroll
        for (uint32_t j = 0; j < 8u; j++)
            if (j0 + j < k)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[i] += w[j] * v[j][i];
    }
    i8_store4(out + t * out_stride + c, acc, cols - c);
}

/* ─── host side ───────────────────────────────────────────────────────── */

#define I8_ARG(...) oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: " __VA_ARGS__)

static size_t up16(size_t v) { return (v + 15u) & ~(size_t)15u; }
static size_t up64(size_t v) { return (v + 63u) & ~(size_t)63u; }
static size_t up256(size_t v) { return (v + 255u) & ~(size_t)255u; }
static size_t elem_bytes(uint32_t type) { return type == OXH_F32 ? 4u : 2u; }
static bool known_type(uint32_t type) { return type == OXH_F32 || type == OXH_F16 || type == OXH_BF16; }

static int ready(void) { return oxh_internal_device() < 0 ? oxh_init(0) : OXH_OK; }
static hipStream_t stream_of(void *s) { return (hipStream_t)(s ? s : oxh_internal_stream()); }
static int launched(const char *who)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? OXH_OK : oxh_internal_errorf(OXH_ERR_HIP, "HIP error in %s: %s", who, hipGetErrorString(e));
}

/* OXH_I8_MAX_ROWS: a workgroup of 1024 threads each is a grid of 2^31 threads.  OXH_I8_MAX_RESULTS: 2^30 threads in tiles of 256 x 256, and
 * they do not fit this memory in f32.  OXH_MOE_I8_MAX_VALUES: tiles of 128 x 64 below 2^32 threads, and 128 GiB of h or y. */

/* a tile's rows lie within 32 bits of its first one */
#define I8_MAX_STRIDE ((size_t)1 << 23)

static int check_rows(const char *who, const char *name, const void *d, size_t stride, size_t cols)
{
    if (!d) return I8_ARG("%s: NULL pointer (%s)", who, name);
    if ((uintptr_t)d & 15u) return I8_ARG("%s: %s must be 16-byte aligned", who, name);
    if (stride % 16u) return I8_ARG("%s: the stride of %s must be a multiple of 16", who, name);
    if (stride < cols) return I8_ARG("%s: the stride of %s is less than cols", who, name);
    if (stride > I8_MAX_STRIDE) return I8_ARG("%s: the stride of %s is more than %zu bytes", who, name, I8_MAX_STRIDE);
    return OXH_OK;
}

static int check_cols(const char *who, size_t cols)
{
    if (cols == 0) return I8_ARG("%s: cols is 0", who);
    if (cols > OXH_I8_MAX_COLS)
        return oxh_internal_errorf(OXH_ERR_TOO_WIDE, "%s: %zu columns: the int32 sums hold %u", who, cols, OXH_I8_MAX_COLS);
    return OXH_OK;
}

static int check_floats(const char *who, const char *name, uint32_t type, const void *d, size_t stride, size_t cols)
{
    if (!known_type(type)) return I8_ARG("%s: the type of %s is not OXH_F32, OXH_F16 or OXH_BF16", who, name);
    if (!d) return I8_ARG("%s: NULL pointer (%s)", who, name);
    if ((uintptr_t)d % elem_bytes(type)) return I8_ARG("%s: %s is not aligned to its elements", who, name);
    if (stride < cols) return I8_ARG("%s: the stride of %s is less than its columns", who, name);
    return OXH_OK;
}

/* Threads to a row: as many as hold its values with one step or two, so that it is read once; for many rows of middling length a workgroup of 256
 * with four steps, of which a CU holds more (4096 rows, us with 64 threads and two steps, 256 and one, 256 and four, 1024 and two: of 1024
 * values 5.3, 6.1, 8.9, 20; of 2048 10, 7.8, 10, 20; of 4096 18, 13.7, 13.6, 22; of 8192 35, 26, 22, 26; of 14336 71, 52, 40, 36.  512 rows
 * of 8192: 18, 7.3, 6.0, 5.4). */
static int quantize_launch(uint32_t type, const void *x, size_t x_stride, size_t n, size_t cols, const void *up, int8_t *q,
                           size_t q_stride, float *scale, hipStream_t st, const char *who)
{
    const dim3 grid((uint32_t)n);
#define OXH_QUANT_K(T, GLU, THREADS, HELD)                                                                                       \
    hipLaunchKernelGGL((k_i8_quantize<T, GLU, THREADS, HELD>), grid, dim3(THREADS), 0, st, (const T *)x, x_stride, (uint32_t)cols, \
                       (const T *)up, q, q_stride, scale)
#define OXH_QUANT_S(T, GLU)                                                                                                      \
    do {                                                                                                                         \
        if (cols <= 512u) OXH_QUANT_K(T, GLU, 64, 1);                                                                            \
        else if (cols <= 1024u) OXH_QUANT_K(T, GLU, 64, 2);                                                                      \
        else if (cols <= 2048u) OXH_QUANT_K(T, GLU, 256, 1);                                                                     \
        else if (cols <= 8192u && n >= 1024u) OXH_QUANT_K(T, GLU, 256, 4);                                                       \
        else OXH_QUANT_K(T, GLU, 1024, 2);                                                                                       \
    } while (0)
#define OXH_QUANT(T)                                                                                                             \
    do {                                                                                                                         \
        if (up) OXH_QUANT_S(T, true);                                                                                            \
        else OXH_QUANT_S(T, false);                                                                                              \
    } while (0)
    if (type == OXH_F32) OXH_QUANT(float);
    else if (type == OXH_F16) OXH_QUANT(_Float16);
    else OXH_QUANT(__bf16);
#undef OXH_QUANT
#undef OXH_QUANT_S
#undef OXH_QUANT_K
    return launched(who);
}

extern "C" int oxh_i8_quantize(uint32_t x_type, const void *d_x, size_t x_stride, size_t n_vec, size_t cols, const void *d_up,
                               int8_t *d_q, size_t q_stride, float *d_scale, void *stream)
{
    static const char who[] = "oxh_i8_quantize";
    int rc;
    if (n_vec == 0) return OXH_OK;
    if ((rc = check_cols(who, cols)) || (rc = check_floats(who, "d_x", x_type, d_x, x_stride, cols)) ||
        (rc = check_rows(who, "d_q", d_q, q_stride, cols)))
        return rc;
    if (d_up && (rc = check_floats(who, "d_up", x_type, d_up, x_stride, cols))) return rc;
    if (!d_scale) return I8_ARG("%s: NULL pointer (d_scale)", who);
    if (n_vec > OXH_I8_MAX_ROWS) return I8_ARG("%s: at most %zu rows per call", who, OXH_I8_MAX_ROWS);
    if ((rc = ready())) return rc;
    return quantize_launch(x_type, d_x, x_stride, n_vec, cols, d_up, d_q, q_stride, d_scale, stream_of(stream), who);
}

static int check_matrix(const char *who, const OxhI8Matrix *w)
{
    int rc;
    if (!w) return I8_ARG("%s: NULL matrix", who);
    if ((rc = check_cols(who, w->cols)) || (rc = check_rows(who, "the matrix", w->d_w, w->stride, w->cols))) return rc;
    if (!w->d_scale) return I8_ARG("%s: NULL pointer (the matrix's scales)", who);
    if (w->rows > OXH_I8_MAX_ROWS) return I8_ARG("%s: at most %zu rows", who, OXH_I8_MAX_ROWS);
    return OXH_OK;
}

typedef I8Geom<8, 4, 2, 4, 5> I8Large;        /* 256 x 256, a workgroup per CU */
typedef I8Geom<4, 4, 2, 4, 5> I8Half;         /* 128 x 256, one */
typedef I8Geom<4, 3, 2, 4, 5> I8Wide;         /* 128 x 192, one */
typedef I8Geom<2, 4, 4, 2, 5> I8Mid;          /* 128 x 128, two */
/* 64 x 64, two, with a ring of nine: where there is hardly a tile per CU, loads have to be under way for four stages (4096 x 4096 under 96
 * to 256 tokens: 10.1 to 11.4 us, with five blocks and four tiles to a CU 12.7 to 16.5) */
typedef I8Geom<2, 2, 2, 2, 9> I8Small;
typedef I8Geom<2, 2, 2, 2, 5> I8Many;         /* 64 x 64, four: many tiles of few columns (151936 x 896 under 64 tokens: 42.8 us, 45.5 in I8Small) */

typedef I8Geom<2, 4, 4, 2, 5> I8Mid128;     /* 128 rows x 128, 64, 32 pairs */
typedef I8Geom<2, 2, 4, 2, 5> I8Mid64;
typedef I8Geom<2, 1, 4, 2, 5> I8Mid32;
typedef I8Geom<2, 2, 2, 2, 5> I8Small64;    /* 64 rows x 64, 32 pairs */
typedef I8Geom<2, 1, 2, 2, 5> I8Small32;

/* How a product runs: on which tile, its columns in how many parts. */
enum { I8_LARGE = 0, I8_HALF, I8_WIDE, I8_MID, I8_SMALL, I8_MANY, I8_TILES };
struct I8Way {
    int tile;
    uint32_t splits;
};

static size_t parts_bytes(size_t rows, size_t n, uint32_t splits) { return splits > 1 ? (size_t)splits * n * ((rows + 3u) & ~(size_t)3u) * 4u : 0; }
#define I8_MAX_PARTS_BYTES ((size_t)64 << 20)

/* The tiles: how many a CU holds at a time, and the microseconds that a stage of 128 columns takes a CU that works on so many of them, in a
 * launch that is done at once and round after round.  These, and the other times of product_us(), are fitted to 5000 launches
 * (256 to 151936 rows, 512 to 16000 columns, 17 to 4096 tokens, every tile, 1 to 8 parts) over three to six matrices in turn, which the
 * last cache holds wholly or in part: the way they choose takes 0.9 % more than the best of its launches on the average, 14 % at the worst
 * (6416 x 512 under 1400 tokens, 20.2 us against 17.7).  They serve matrices that come from memory as well, though a launch of 65 to 500 tokens takes up to
 * half as long again: over 800 MB of matrices in turn 0.8 % and 15 % (76 sizes, 2048 x 2048 to 28672 x 4096 and 6000 x 16000, 17 to 2048 tokens;
 * 6000 x 16000 under 333, 67.2 us against 58.4), over three of the same 0.9 % and 17 %; where they choose nine to twelve parts
 * (60 sizes, 64 to 9000 rows) 0.6 % and 5 %, over three 2.2 % and 15 %.  128 x 192 is there for token counts that leave tiles of 128 and 256 half empty (4096 x 14336 under
 * 333: 34.8 us in four parts, 37.0 the best without it; from memory 38.8 and 41.5). */
struct I8Pace {
    uint32_t rows, tok, held;
    double alone[4], rounds;
};
static const I8Pace i8_pace[I8_TILES] = {
    { 256, 256, 1, { 1.28 }, 1.41 },
    { 128, 256, 1, { 0.89 }, 0.72 },
    { 128, 192, 1, { 0.74 }, 0.71 },
    { 128, 128, 2, { 0.55, 0.94 }, 0.86 },
    { 64, 64, 2, { 0.20, 0.39 }, 0.46 },
    { 64, 64, 4, { 0.27, 0.46, 0.55, 0.92 }, 0.90 },
};

static size_t tile_count(const I8Pace &t, size_t rows, size_t n)
{
    return ((rows + t.rows - 1) / t.rows) * ((n + t.tok - 1) / t.tok);
}
#define I8_MAX_TILES ((size_t)1 << 23)      /* of 512 threads: a grid of 2^32 */

/* What a product takes: rounds of what the CUs hold at a time, the last one with as many tiles to a CU as are left, and a tile's results, which
 * take a CU's time where no other tile is multiplied meanwhile; results and partial sums in memory, and the second launch that
 * those take. */
static double product_us(int tile, uint32_t splits, size_t rows, size_t stages, size_t n, size_t cus)
{
    const I8Pace &t = i8_pace[tile];
    const size_t tiles = tile_count(t, rows, n) * splits;
    const size_t k = (stages + splits - 1) / splits, rounds = tiles / (cus * t.held), rest = tiles - rounds * cus * t.held;
    const double end = 0.61 + (t.held == 1 ? 1.2 * t.rows * t.tok / 65536.0 : 0.0);
    double us = 3.0 + (double)rounds * ((double)k * t.rounds + end);
    if (rest) {
        const bool halves = tile == I8_LARGE && splits == 1 && rest <= cus / 2;
        const I8Pace &last = halves ? i8_pace[I8_HALF] : t;
        us += (double)k * (rounds && t.held == 1 ? last.rounds : last.alone[(rest + cus - 1) / cus - 1]) + end;
    }
    us += (double)n * (double)rows * 4.0 / 3.1e6;
    if (splits > 1) us += 3.6 + (double)splits * (double)n * (double)rows * 8.0 / 5.2e6;
    return us;
}

static I8Way i8_way(size_t rows, size_t cols, size_t n, size_t ws_bytes, size_t cus)
{
    const size_t stages = (cols + 127u) / 128u;
    I8Way best = { I8_SMALL, 1 };
    double least = 1e30;
    for (uint32_t splits = 1; splits <= 12 && splits <= stages; splits++) {
        const size_t need = parts_bytes(rows, n, splits);
        if (splits > 1 && (need > ws_bytes || need > I8_MAX_PARTS_BYTES || n > 65535u)) break;
        for (int tile = 0; tile < I8_TILES; tile++) {
            if (tile > I8_LARGE && tile_count(i8_pace[tile], rows, n) * splits >= I8_MAX_TILES) continue;
            const double us = product_us(tile, splits, rows, stages, n, cus);
            if (us < least) {
                least = us;
                best = { tile, splits };
            }
        }
    }
    return best;
}

/* The kernel of a product over quantised tokens: `tile` in `splits` parts, or with `team` the few tokens'. */
struct I8Choice {
    uint32_t team;
    I8Way way;
};

/* compute units; a count to plan a workspace with when there is no device yet */
static size_t i8_cus(void) { return oxh_internal_n_cu() > 0 ? (size_t)oxh_internal_n_cu() : 256u; }

/* the large tiles whose last round is done in half tiles: places behind the whole ones, or 0 */
static uint32_t i8_tail(uint32_t tiles, uint32_t splits, size_t cus)
{
    const uint32_t rest = tiles % (uint32_t)cus;
    return splits == 1u && rest <= cus / 2u ? rest : 0u;
}

template <typename G> static void tiles_launch(I8Product &p, hipStream_t st)
{
    p.row_tiles = (uint32_t)((p.w.rows + G::ROWS - 1u) / G::ROWS);
    p.tok_tiles = (p.n_vec + G::TOK - 1u) / G::TOK;
    const uint32_t tiles = p.row_tiles * p.tok_tiles;
    if constexpr (G::ROWS == I8Large::ROWS && G::TOK == I8Large::TOK) {
        const uint32_t rest = i8_tail(tiles, p.splits, i8_cus());
        if (rest) {
            p.whole = tiles - rest;
            hipLaunchKernelGGL((k_i8_tiles_tail<G, I8Half>), dim3(p.whole + 2u * rest), dim3(G::WAVES * 64u), G::LDS_BYTES, st, p);
            return;
        }
    }
    hipLaunchKernelGGL(k_i8_tiles<G>, dim3(tiles * p.splits), dim3(G::WAVES * 64u), G::LDS_BYTES, st, p);
}

/* The kernels for few tokens: how many waves share a group of 16 rows (0: they cannot take the product).  Four stages a wave leave room
 * for two workgroups on a CU, and where the groups are few, all of a CU's sixteen waves are wanted. */
#define FEW_WIDE_TOKENS 64u
#define FEW_MAX_STAGES 8u
static uint32_t few_waves(size_t rows, size_t cols, size_t cus)
{
    const size_t groups = (rows + 15u) / 16u, stages = (cols + 127u) / 128u;
    uint32_t team = 1;
    while (team < FEW_WAVES && (stages > 4u * team || groups * team < cus * FEW_WAVES)) team *= 2u;
    return stages > FEW_MAX_STAGES * team ? 0u : team;
}

/* Whether they should.  They reach a matrix sooner than the tiles, which need the first two stages of a tile before they multiply, but
 * tokens read once per group of rows cost more than they do in tiles.  So they take, with matrices that come from memory and the
 * tiles' time behind theirs:
 *  - what is a workgroup per CU and two stages a wave, up to 64 tokens (4096 x 4096 under one: 6.7 us, 8.2; sixteen: 7.4, 9.0; 64:
 *    9.3, 12.8; 500 x 3001 under sixteen: 5.5, 7.6);
 *  - up to eight of what is a workgroup per CU and four stages (2048 x 7000: 8.1, 8.5; sixteen: 9.4, 8.6), or more on most of the
 *    CUs (4096 x 14336: 15.0, 15.2; but 571 x 11128 under one: 9.3, 8.0);
 *  - up to eight of what is more, if it is one and a half and a wave has two stages (14336 x 4096: 14.6, 15.5; 151936 x 896 under one:
 *    27.3, 29.7; but 6000 x 16000 under one: 23.2, 22.8; 14631 x 629: 6.4, 5.4). */
static uint32_t few_team(size_t rows, size_t cols, size_t n, size_t cus)
{
    const size_t groups = (rows + 15u) / 16u, stages = (cols + 127u) / 128u, all = cus * FEW_WAVES;
    const uint32_t team = few_waves(rows, cols, cus);
    size_t most = 0;
    if (groups * team > all) most = 2u * groups * team >= 3u * all && stages >= 2u * team ? 8u : 0u;
    else if (stages <= 2u * team) most = FEW_WIDE_TOKENS;
    else if (stages <= 4u * team || 4u * groups * team >= 3u * all) most = 8u;
    return n <= most ? team : 0u;
}

/* the kernels' instance for waves of up to so many stages */
static uint32_t few_held(uint32_t stages) { return stages <= 2u ? 2u : stages <= 4u ? 4u : FEW_MAX_STAGES; }

struct FewGrid {
    uint32_t groups, wgs, held;     /* held: few_held() of a wave's stages */
};
static FewGrid few_grid(size_t rows, size_t cols, uint32_t team)
{
    FewGrid g;
    g.groups = (uint32_t)((rows + 15u) / 16u);
    g.wgs = (g.groups + FEW_WAVES / team - 1u) / (FEW_WAVES / team);
    g.held = few_held(((uint32_t)((cols + 127u) / 128u) + team - 1u) / team);
    return g;
}

static void few_launch(const I8Product &p, uint32_t team, hipStream_t st)
{
    const FewGrid g = few_grid(p.w.rows, p.w.cols, team);
    const dim3 grid(g.wgs), block(64u * FEW_WAVES);
    if (p.n_vec > 48u) hipLaunchKernelGGL(k_i8_few_wide<4>, grid, block, 0, st, p, team, g.groups);
    else if (p.n_vec > 32u) hipLaunchKernelGGL(k_i8_few_wide<3>, grid, block, 0, st, p, team, g.groups);
    else if (p.n_vec > 16u) hipLaunchKernelGGL(k_i8_few_wide<2>, grid, block, 0, st, p, team, g.groups);
    else if (g.held == 2u) hipLaunchKernelGGL(k_i8_few<2>, grid, block, 0, st, p, team, g.groups);
    else if (g.held == 4u) hipLaunchKernelGGL(k_i8_few<4>, grid, block, 0, st, p, team, g.groups);
    else hipLaunchKernelGGL(k_i8_few<8>, grid, block, 0, st, p, team, g.groups);
}

static size_t few_float_lds(size_t cols, size_t n) { return FEW_HEAD_BYTES + n * ((cols + 127u) & ~(size_t)127u); }
template <typename XT> static void few_float_launch(const I8Product &p, const XT *x, size_t x_stride, uint32_t team, hipStream_t st)
{
    const FewGrid g = few_grid(p.w.rows, p.w.cols, team);
    const dim3 grid(g.wgs), block(64u * FEW_WAVES);
    const size_t lds = few_float_lds(p.w.cols, p.n_vec);
    if (g.held == 2u) hipLaunchKernelGGL((k_i8_few_float<XT, 2>), grid, block, lds, st, p, x, x_stride, team, g.groups);
    else if (g.held == 4u) hipLaunchKernelGGL((k_i8_few_float<XT, 4>), grid, block, lds, st, p, x, x_stride, team, g.groups);
    else hipLaunchKernelGGL((k_i8_few_float<XT, 8>), grid, block, lds, st, p, x, x_stride, team, g.groups);
}

static I8Choice i8_choice(size_t rows, size_t cols, size_t n, size_t ws_bytes, size_t cus)
{
    I8Choice c = { few_team(rows, cols, n, cus), { 0, 1u } };
    if (!c.team) c.way = i8_way(rows, cols, n, ws_bytes, cus);
    return c;
}

static int matmul_launch(const OxhI8Matrix *w, const int8_t *q, size_t q_stride, const float *q_scale, size_t n, const float *bias,
                         uint32_t out_type, void *out, size_t out_stride, void *ws, size_t ws_bytes, hipStream_t st, const char *who)
{
    I8Product p = { *w, q, q_stride, q_scale, bias, out, out_stride, nullptr, (uint32_t)n, 1u, 0u, 0u, 0u,
                    (uint32_t)((w->rows + 3u) & ~(size_t)3u), out_type };
    const I8Choice choice = i8_choice(w->rows, w->cols, n, ws_bytes, i8_cus());
    if (choice.team) {
        few_launch(p, choice.team, st);
        return launched(who);
    }
    const I8Way way = choice.way;
    p.splits = way.splits;
    if (way.splits > 1) p.parts = (int *)ws;
    if (way.tile == I8_LARGE) tiles_launch<I8Large>(p, st);
    else if (way.tile == I8_HALF) tiles_launch<I8Half>(p, st);
    else if (way.tile == I8_WIDE) tiles_launch<I8Wide>(p, st);
    else if (way.tile == I8_MID) tiles_launch<I8Mid>(p, st);
    else if (way.tile == I8_SMALL) tiles_launch<I8Small>(p, st);
    else tiles_launch<I8Many>(p, st);
    if (way.splits > 1) hipLaunchKernelGGL(k_i8_join, dim3((p.rows_pad / 4u + 255u) / 256u, p.n_vec), dim3(256), 0, st, p);
    return launched(who);
}

template <typename K> static hipError_t whole_lds(K kernel)
{
    return hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
}

extern "C" int oxh_internal_i8_init(void)
{
    hipError_t e;
    if ((e = whole_lds(k_i8_tiles<I8Large>)) != hipSuccess) return (int)e;
    if ((e = whole_lds(k_i8_tiles_tail<I8Large, I8Half>)) != hipSuccess) return (int)e;
    if ((e = whole_lds(k_i8_tiles<I8Half>)) != hipSuccess) return (int)e;
    if ((e = whole_lds(k_i8_tiles<I8Wide>)) != hipSuccess) return (int)e;
    if ((e = whole_lds(k_i8_tiles<I8Mid>)) != hipSuccess) return (int)e;
    if ((e = whole_lds(k_i8_tiles<I8Small>)) != hipSuccess) return (int)e;
    if ((e = whole_lds(k_i8_experts<I8Mid128, I8Mid64, I8Mid32, true>)) != hipSuccess) return (int)e;
    if ((e = whole_lds(k_i8_experts<I8Mid128, I8Mid64, I8Mid32, false>)) != hipSuccess) return (int)e;
    return (int)hipSuccess;
}

extern "C" size_t oxh_i8_matmul_workspace(const OxhI8Matrix *w, size_t n_vec)
{
    if (!w || n_vec == 0 || w->rows == 0 || w->cols == 0 || w->cols > OXH_I8_MAX_COLS || w->rows > OXH_I8_MAX_ROWS || n_vec > OXH_I8_MAX_ROWS)
        return 0;
    if (few_team(w->rows, w->cols, n_vec, i8_cus())) return 0;
    return parts_bytes(w->rows, n_vec, i8_way(w->rows, w->cols, n_vec, SIZE_MAX, i8_cus()).splits);
}

extern "C" int oxh_i8_matmul(const OxhI8Matrix *w, const int8_t *d_q, size_t q_stride, const float *d_q_scale, size_t n_vec,
                             const float *d_bias, uint32_t out_type, void *d_out, size_t out_stride, void *d_workspace,
                             size_t workspace_bytes, void *stream)
{
    static const char who[] = "oxh_i8_matmul";
    int rc;
    if ((rc = check_matrix(who, w))) return rc;
    if (n_vec == 0 || w->rows == 0) return OXH_OK;
    if ((rc = check_rows(who, "d_q", d_q, q_stride, w->cols)) || (rc = check_floats(who, "d_out", out_type, d_out, out_stride, w->rows)))
        return rc;
    if (!d_q_scale) return I8_ARG("%s: NULL pointer (d_q_scale)", who);
    if (n_vec > OXH_I8_MAX_ROWS) return I8_ARG("%s: at most %zu tokens per call", who, OXH_I8_MAX_ROWS);
    if (n_vec * w->rows > OXH_I8_MAX_RESULTS) return I8_ARG("%s: at most %zu results per call", who, OXH_I8_MAX_RESULTS);
    if (d_workspace && workspace_bytes && ((uintptr_t)d_workspace & 15u)) return I8_ARG("%s: workspace must be 16-byte aligned", who);
    if ((rc = ready())) return rc;
    return matmul_launch(w, d_q, q_stride, d_q_scale, n_vec, d_bias, out_type, d_out, out_stride, d_workspace,
                         d_workspace ? workspace_bytes : 0, stream_of(stream), who);
}

/* Whether a product quantises its tokens in the launch itself: every workgroup does it again, so for few values (a second
 * launch costs about 3 us, the values of one token of 4096 about 1) and while there is no more than a workgroup per CU
 * (14336 x 4096 under one token, 448 workgroups: 16.5 us fused, 15.2 in two). */
static bool linear_fused(size_t rows, size_t cols, size_t n, size_t cus)
{
    const size_t per = n == 1 ? 16 : n == 2 ? 8 : n <= 4 ? 4 : n <= 8 ? 2 : 1;      /* waves a token, as in the kernel */
    const uint32_t team = few_waves(rows, cols, cus);
    return team && n <= FEW_TOKENS && n * cols <= 16384u && cols <= 512u * per * FEW_HELD && few_grid(rows, cols, team).wgs <= cus;
}

/* the workspace otherwise: codes and scales of the tokens, the partial sums of the product */
struct LinearParts {
    size_t q_stride, q, scale, parts, parts_bytes, total;
};
static LinearParts linear_parts(size_t rows, size_t cols, size_t n)
{
    LinearParts p;
    p.q_stride = up64(cols);
    p.q = 0;
    p.scale = p.q_stride * n;
    p.parts = p.scale + up16(4u * n);
    p.parts_bytes = few_team(rows, cols, n, i8_cus()) ? 0 : parts_bytes(rows, n, i8_way(rows, cols, n, SIZE_MAX, i8_cus()).splits);
    p.total = linear_fused(rows, cols, n, i8_cus()) ? 0 : p.parts + p.parts_bytes;
    return p;
}

extern "C" size_t oxh_i8_linear_workspace(const OxhI8Matrix *w, size_t n_vec)
{
    if (!w || n_vec == 0 || w->rows == 0 || w->cols == 0 || w->cols > OXH_I8_MAX_COLS || w->rows > OXH_I8_MAX_ROWS || n_vec > OXH_I8_MAX_ROWS)
        return 0;
    return linear_parts(w->rows, w->cols, n_vec).total;
}

/* codes and scales have to fit; partial sums are used where they do, so a buffer for more tokens serves fewer as well */
static int check_linear_workspace(const char *who, const OxhI8Matrix *w, size_t n_vec, const void *d_workspace, size_t bytes)
{
    const LinearParts l = linear_parts(w->rows, w->cols, n_vec);
    if (l.total && (!d_workspace || bytes < l.parts)) return I8_ARG("%s: workspace too small (see oxh_i8_linear_workspace)", who);
    if (l.total && ((uintptr_t)d_workspace & 15u)) return I8_ARG("%s: workspace must be 16-byte aligned", who);
    return OXH_OK;
}

extern "C" int oxh_i8_linear(const OxhI8Matrix *w, uint32_t x_type, const void *d_x, size_t x_stride, size_t n_vec,
                             const float *d_bias, uint32_t out_type, void *d_out, size_t out_stride, void *d_workspace,
                             size_t workspace_bytes, void *stream)
{
    static const char who[] = "oxh_i8_linear";
    int rc;
    if ((rc = check_matrix(who, w))) return rc;
    if (n_vec == 0 || w->rows == 0) return OXH_OK;
    if ((rc = check_floats(who, "d_x", x_type, d_x, x_stride, w->cols)) ||
        (rc = check_floats(who, "d_out", out_type, d_out, out_stride, w->rows)))
        return rc;
    if (n_vec > OXH_I8_MAX_ROWS) return I8_ARG("%s: at most %zu tokens per call", who, OXH_I8_MAX_ROWS);
    if (n_vec * w->rows > OXH_I8_MAX_RESULTS) return I8_ARG("%s: at most %zu results per call", who, OXH_I8_MAX_RESULTS);
    if ((rc = check_linear_workspace(who, w, n_vec, d_workspace, workspace_bytes)) || (rc = ready()) ||
        (rc = check_linear_workspace(who, w, n_vec, d_workspace, workspace_bytes)))    /* once more: the way depends on the device */
        return rc;
    const LinearParts l = linear_parts(w->rows, w->cols, n_vec);
    hipStream_t st = stream_of(stream);
    if (l.total == 0) {
        I8Product p = { *w, nullptr, 0, nullptr, d_bias, d_out, out_stride, nullptr, (uint32_t)n_vec, 1u, 0u, 0u, 0u, 0u, out_type };
        const uint32_t team = few_waves(w->rows, w->cols, i8_cus());
        if (x_type == OXH_F32) few_float_launch(p, (const float *)d_x, x_stride, team, st);
        else if (x_type == OXH_F16) few_float_launch(p, (const _Float16 *)d_x, x_stride, team, st);
        else few_float_launch(p, (const __bf16 *)d_x, x_stride, team, st);
        return launched(who);
    }
    int8_t *q = (int8_t *)d_workspace;
    float *scale = (float *)((uint8_t *)d_workspace + l.scale);
    if ((rc = quantize_launch(x_type, d_x, x_stride, n_vec, w->cols, nullptr, q, l.q_stride, scale, st, who))) return rc;
    return matmul_launch(w, q, l.q_stride, scale, n_vec, d_bias, out_type, d_out, out_stride, (uint8_t *)d_workspace + l.parts,
                         workspace_bytes - l.parts, st, who);
}

/* ─── experts ─────────────────────────────────────────────────────────── */

/* Pairs of a table entry: by how many an expert gets on average (6: 64 experts of 2048 x 1408 take 120 us in tiles of 64, 127 in the few
 * tokens' way; 9: 122 and 137; 4: 118 and 121, and 8 of 4096 x 14336 277 and 269.  62: 128 of 2048 x 768 take 190 us in tiles of 128, 202 of 64; 25:
 * 16 of 568 x 6448 take 86 and 75). */
static uint32_t experts_tok(size_t pairs, size_t n_expert)
{
    const size_t avg = pairs / n_expert;
    return avg <= 4 ? FEW_TOKENS : avg <= 44 ? 64u : 128u;
}

/* The most tiles any routing can need: an expert's runs make at most one tile that is not full. */
static size_t experts_tiles(size_t pairs, size_t n_expert, uint32_t tok)
{
    const size_t most = pairs / tok + n_expert;
    return most < pairs ? most : pairs;
}

struct MoeI8Parts {
    size_t q_stride, h_stride, y_stride, qh_stride;    /* bytes, floats, floats, bytes */
    size_t tiles, q, q_scale, h, qh, qh_scale, y, total;
    uint32_t tok, n_tiles;
};

static int moe_parts(const char *who, const OxhMoeI8 *m, size_t n_tok, MoeI8Parts *p)
{
    int rc;
    if (!m) return I8_ARG("%s: NULL layer", who);
    if (m->n_expert == 0 || m->n_expert > OXH_SELECT_MAX_EXPERTS) return I8_ARG("%s: n_expert must be 1..%u", who, OXH_SELECT_MAX_EXPERTS);
    if (m->top_k == 0 || m->top_k > OXH_SELECT_MAX_TOPK || m->top_k > m->n_expert)
        return I8_ARG("%s: top_k must be 1..%u and at most n_expert", who, OXH_SELECT_MAX_TOPK);
    if ((rc = check_cols(who, m->hidden)) || (rc = check_cols(who, m->ffn))) return rc;
    if (n_tok == 0 || n_tok > OXH_SELECT_MAX_TOKENS) return I8_ARG("%s: n_tok must be 1..%u", who, OXH_SELECT_MAX_TOKENS);
    const size_t pairs = n_tok * m->top_k;
    p->q_stride = up64(m->hidden);
    p->qh_stride = up64(m->ffn);
    p->h_stride = up64(m->ffn);
    p->y_stride = up64(m->hidden);
    if (pairs * (m->hidden > m->ffn ? m->hidden : m->ffn) > OXH_MOE_I8_MAX_VALUES)
        return I8_ARG("%s: n_tok * top_k * max(hidden, ffn) is more than %zu", who, OXH_MOE_I8_MAX_VALUES);
    if (n_tok * p->q_stride > 0xFFFFFFFFull) return I8_ARG("%s: the tokens' codes exceed 4 GiB", who);
    p->tok = experts_tok(pairs, m->n_expert);
    p->n_tiles = (uint32_t)experts_tiles(pairs, m->n_expert, p->tok);
    size_t at = 0;
#define OXH_PART(FIELD, BYTES) p->FIELD = at; at = up256(at + (BYTES))
    OXH_PART(tiles, experts_tiles(pairs, m->n_expert, FEW_TOKENS) * sizeof(I8ExpertTile));   /* more tokens never need less */
    OXH_PART(q, n_tok * p->q_stride);
    OXH_PART(q_scale, n_tok * 4u);
    OXH_PART(h, pairs * p->h_stride * 4u);
    OXH_PART(qh, pairs * p->qh_stride);
    OXH_PART(qh_scale, pairs * 4u);
    OXH_PART(y, pairs * p->y_stride * 4u);
#undef OXH_PART
    p->total = at;
    return OXH_OK;
}

template <typename G, typename H, typename Q, bool UP> static void experts_launch(I8Experts &e, hipStream_t st)
{
    const uint32_t out_rows = UP ? G::ROWS / 2u : G::ROWS;
    e.row_tiles = (e.rows + out_rows - 1u) / out_rows;
    hipLaunchKernelGGL((k_i8_experts<G, H, Q, UP>), dim3(e.row_tiles * e.n_tiles), dim3(G::WAVES * 64u), G::LDS_BYTES, st, e);
}

/* How a product of the experts runs under a table whose entries have up to `tok` pairs: on the kernel for few pairs, `team` waves to a group of
 * rows as few_team(), half of them gate where it is up's, or (held 0) on tiles. */
struct ExpertsWay {
    uint32_t team, held;
};
static ExpertsWay experts_way(bool up, size_t rows, size_t cols, uint32_t tok, size_t n_tiles, size_t cus)
{
    const uint32_t groups = (uint32_t)((rows + 15u) / 16u), stages = (uint32_t)((cols + 127u) / 128u), halves = up ? 2u : 1u;
    if (tok != FEW_TOKENS || stages > FEW_MAX_STAGES * FEW_WAVES / halves) return { 0u, 0u };
    uint32_t team = halves;
    while (team < FEW_WAVES && (stages * halves > 4u * team || (size_t)groups * n_tiles * team < cus * FEW_WAVES)) team *= 2u;
    const uint32_t parts = team / halves;
    return { team, few_held((stages + parts - 1u) / parts) };
}
template <bool UP> static void experts_few_launch(I8Experts &e, ExpertsWay way, hipStream_t st)
{
    const uint32_t groups = (e.rows + 15u) / 16u, teams = FEW_WAVES / way.team;
    const dim3 grid((groups + teams - 1u) / teams, e.n_tiles), block(64u * FEW_WAVES);
    if (way.held == 2u) hipLaunchKernelGGL((k_i8_experts_few<2, UP>), grid, block, 0, st, e, way.team, groups);
    else if (way.held == 4u) hipLaunchKernelGGL((k_i8_experts_few<4, UP>), grid, block, 0, st, e, way.team, groups);
    else hipLaunchKernelGGL((k_i8_experts_few<8, UP>), grid, block, 0, st, e, way.team, groups);
}

/* Whether a layer goes pair by pair, in two launches instead of five.  It saves 5 to 7 us and pays in two ways: every workgroup quantises again,
 * which shows once the weights take longer than that (7168 x 2048, 8 pairs of 44 MB: 82.2 us, 81.9 sorted; 128 experts of 2048 x 768, 8 pairs
 * of 4.7 MB: 15.6 and 21.0, 32 of them: 31.0 and 38.7; 64 of 2048 x 1408, 18 of 8.7 MB: 41.8 and 40.7); and pairs of one expert read its weights
 * each for itself (8 experts of 1024 x 2048, 32 pairs: 28.7 and 23.2).  A wave's columns of an expert's rows are loaded at once, and the
 * codes have to fit. */
#define PAIRS_MAX_BYTES ((size_t)160 << 20)
struct PairsPlan {
    uint32_t team, per;             /* waves to 16 rows of h; to a pair of the results */
    uint32_t up_held, down_held;    /* the kernels' instances; down has no <2> */
    size_t up_lds, down_lds;
    bool taken;
};
static PairsPlan pairs_plan(const OxhMoeI8 *m, size_t n_tok, size_t cus)
{
    PairsPlan l = { 2u, FEW_WAVES / (uint32_t)m->top_k, 0, 0, 0, 0, false };
    const size_t up_stages = (m->hidden + 127u) / 128u, down_stages = (m->ffn + 127u) / 128u, groups = (m->ffn + 15u) / 16u, pairs = n_tok * m->top_k;
    while (l.team < FEW_WAVES && (up_stages * 2u > 4u * l.team || groups * pairs * l.team < cus * FEW_WAVES)) l.team *= 2u;
    l.up_held = few_held(((uint32_t)up_stages + l.team / 2u - 1u) / (l.team / 2u));
    l.down_held = ((uint32_t)down_stages + l.per - 1u) / l.per <= 4u ? 4u : FEW_MAX_STAGES;
    l.up_lds = FEW_HEAD_BYTES + 128u * up_stages;
    l.down_lds = FEW_PAIRS_BYTES + 128u * down_stages * m->top_k;
    l.taken = pairs <= 2u * m->n_expert && pairs * 3u * m->hidden * m->ffn <= PAIRS_MAX_BYTES && pairs <= 65535u &&
              up_stages <= FEW_MAX_STAGES * FEW_WAVES / 2u && down_stages <= FEW_MAX_STAGES * l.per && l.up_lds <= 65536u && l.down_lds <= 65536u;
    return l;
}

template <typename T> static void pair_up_launch(const I8Pairs &p, const PairsPlan &l, uint32_t pairs, const void *x, size_t x_stride, hipStream_t st)
{
    const uint32_t groups = (p.e.rows + 15u) / 16u, teams = FEW_WAVES / l.team;
    const dim3 grid((groups + teams - 1u) / teams, pairs), block(64u * FEW_WAVES);
    if (l.up_held == 2u) hipLaunchKernelGGL((k_i8_pair_up<T, 2>), grid, block, l.up_lds, st, p, (const T *)x, x_stride, l.team, groups);
    else if (l.up_held == 4u) hipLaunchKernelGGL((k_i8_pair_up<T, 4>), grid, block, l.up_lds, st, p, (const T *)x, x_stride, l.team, groups);
    else hipLaunchKernelGGL((k_i8_pair_up<T, 8>), grid, block, l.up_lds, st, p, (const T *)x, x_stride, l.team, groups);
}

template <typename T> static void pair_down_launch(const I8Pairs &p, const PairsPlan &l, uint32_t n_tok, const float *h, size_t h_stride, void *out, size_t out_stride, hipStream_t st)
{
    const dim3 grid((p.e.rows + 15u) / 16u, n_tok), block(64u * FEW_WAVES);
    if (l.down_held == 4u) hipLaunchKernelGGL((k_i8_pair_down<T, 4>), grid, block, l.down_lds, st, p, h, h_stride, (T *)out, out_stride, l.per);
    else hipLaunchKernelGGL((k_i8_pair_down<T, 8>), grid, block, l.down_lds, st, p, h, h_stride, (T *)out, out_stride, l.per);
}

template <bool UP> static void experts_run(I8Experts &e, uint32_t tok, hipStream_t st)
{
    const ExpertsWay way = experts_way(UP, e.rows, e.cols, tok, e.n_tiles, i8_cus());
    if (way.held) experts_few_launch<UP>(e, way, st);
    else if (tok <= 64u) experts_launch<I8Small64, I8Small32, I8Small32, UP>(e, st);
    else experts_launch<I8Mid128, I8Mid64, I8Mid32, UP>(e, st);
}

template <typename T>
static void experts_begin(const void *x, size_t x_stride, size_t n_tok, size_t cols, int8_t *q, size_t q_stride, float *scale,
                          const uint32_t *offsets, size_t n_expert, size_t pairs, uint32_t tok, I8ExpertTile *tiles, uint32_t n_tiles,
                          hipStream_t st)
{
    const dim3 grid((uint32_t)n_tok + 1u);
#define OXH_BEGIN(THREADS, HELD)                                                                                                 \
    hipLaunchKernelGGL((k_i8_experts_begin<T, THREADS, HELD>), grid, dim3(THREADS), 0, st, (const T *)x, x_stride, (uint32_t)cols, q, \
                       q_stride, scale, offsets, (uint32_t)n_expert, (uint32_t)pairs, tok, tiles, n_tiles)
    if (cols <= 2048u) OXH_BEGIN(256, 1);           /* as quantize_launch(); the table wants 256 threads */
    else if (cols <= 8192u && n_tok >= 1024u) OXH_BEGIN(256, 4);
    else OXH_BEGIN(1024, 2);
#undef OXH_BEGIN
}

extern "C" int oxh_moe_i8_workspace_bytes(const OxhMoeI8 *m, size_t n_tok, size_t *bytes)
{
    MoeI8Parts p;
    const int rc = moe_parts("oxh_moe_i8_workspace_bytes", m, n_tok, &p);
    if (rc) return rc;
    if (bytes) *bytes = p.total;
    return OXH_OK;
}

extern "C" int oxh_moe_ffn_i8(const OxhMoeI8 *m, const OxhRouting *routing, uint32_t x_type, const void *d_x, size_t x_stride,
                              size_t n_tok, uint32_t out_type, void *d_out, size_t out_stride, void *d_workspace,
                              size_t workspace_bytes, void *stream)
{
    static const char who[] = "oxh_moe_ffn_i8";
    int rc;
    MoeI8Parts p;
    if ((rc = moe_parts(who, m, n_tok, &p))) return rc;
    if ((rc = check_rows(who, "d_w_gate", m->d_w_gate, m->gate_up_stride, m->hidden)) ||
        (rc = check_rows(who, "d_w_up", m->d_w_up, m->gate_up_stride, m->hidden)) ||
        (rc = check_rows(who, "d_w_down", m->d_w_down, m->down_stride, m->ffn)) ||
        (rc = check_floats(who, "d_x", x_type, d_x, x_stride, m->hidden)) ||
        (rc = check_floats(who, "d_out", out_type, d_out, out_stride, m->hidden)))
        return rc;
    if (!m->d_s_gate || !m->d_s_up || !m->d_s_down || !routing || !routing->d_weights || !routing->d_offsets || !routing->d_perm ||
        !routing->d_slot_pos || !d_workspace)
        return I8_ARG("%s: NULL pointer", who);
    if (workspace_bytes < p.total) return I8_ARG("%s: workspace too small (see oxh_moe_i8_workspace_bytes)", who);
    if ((uintptr_t)d_workspace & 255u) return I8_ARG("%s: workspace must be 256-byte aligned", who);
    if ((rc = ready())) return rc;
    hipStream_t st = stream_of(stream);
    uint8_t *ws = (uint8_t *)d_workspace;
    int8_t *q = (int8_t *)(ws + p.q), *qh = (int8_t *)(ws + p.qh);
    float *q_scale = (float *)(ws + p.q_scale), *qh_scale = (float *)(ws + p.qh_scale), *h = (float *)(ws + p.h), *y = (float *)(ws + p.y);
    const size_t pairs = n_tok * m->top_k;
    const PairsPlan few = pairs_plan(m, n_tok, i8_cus());
    if (few.taken && routing->d_ids) {
        I8Pairs a = { { { m->d_w_gate, m->d_w_up }, { m->d_s_gate, m->d_s_up }, m->gate_up_stride, nullptr, 0, nullptr, nullptr, nullptr, h, p.h_stride,
                        (uint32_t)m->ffn, (uint32_t)m->hidden, (uint32_t)n_tok, 0u, 0u }, routing->d_ids, routing->d_weights, (uint32_t)m->top_k, (uint32_t)m->n_expert };
        if (x_type == OXH_F32) pair_up_launch<float>(a, few, (uint32_t)pairs, d_x, x_stride, st);
        else if (x_type == OXH_F16) pair_up_launch<_Float16>(a, few, (uint32_t)pairs, d_x, x_stride, st);
        else pair_up_launch<__bf16>(a, few, (uint32_t)pairs, d_x, x_stride, st);
        if ((rc = launched(who))) return rc;
        a.e = { { m->d_w_down, m->d_w_down }, { m->d_s_down, m->d_s_down }, m->down_stride, nullptr, 0, nullptr, nullptr, nullptr, nullptr, 0,
                (uint32_t)m->hidden, (uint32_t)m->ffn, (uint32_t)n_tok, 0u, 0u };
        if (out_type == OXH_F32) pair_down_launch<float>(a, few, (uint32_t)n_tok, h, p.h_stride, d_out, out_stride, st);
        else if (out_type == OXH_F16) pair_down_launch<_Float16>(a, few, (uint32_t)n_tok, h, p.h_stride, d_out, out_stride, st);
        else pair_down_launch<__bf16>(a, few, (uint32_t)n_tok, h, p.h_stride, d_out, out_stride, st);
        return launched(who);
    }
    I8ExpertTile *tiles = (I8ExpertTile *)(ws + p.tiles);
    if (x_type == OXH_F32) experts_begin<float>(d_x, x_stride, n_tok, m->hidden, q, p.q_stride, q_scale, routing->d_offsets, m->n_expert, pairs, p.tok, tiles, p.n_tiles, st);
    else if (x_type == OXH_F16) experts_begin<_Float16>(d_x, x_stride, n_tok, m->hidden, q, p.q_stride, q_scale, routing->d_offsets, m->n_expert, pairs, p.tok, tiles, p.n_tiles, st);
    else experts_begin<__bf16>(d_x, x_stride, n_tok, m->hidden, q, p.q_stride, q_scale, routing->d_offsets, m->n_expert, pairs, p.tok, tiles, p.n_tiles, st);
    if ((rc = launched(who))) return rc;
    I8Experts up = { { m->d_w_gate, m->d_w_up }, { m->d_s_gate, m->d_s_up }, m->gate_up_stride, q, p.q_stride, q_scale, routing->d_perm, tiles,
                     h, p.h_stride, (uint32_t)m->ffn, (uint32_t)m->hidden, (uint32_t)n_tok, p.n_tiles, 0u };
    experts_run<true>(up, p.tok, st);
    if ((rc = launched(who))) return rc;
    if ((rc = quantize_launch(OXH_F32, h, p.h_stride, pairs, m->ffn, nullptr, qh, p.qh_stride, qh_scale, st, who))) return rc;
    I8Experts down = { { m->d_w_down, m->d_w_down }, { m->d_s_down, m->d_s_down }, m->down_stride, qh, p.qh_stride, qh_scale, routing->d_perm,
                       tiles, y, p.y_stride, (uint32_t)m->hidden, (uint32_t)m->ffn, (uint32_t)n_tok, p.n_tiles, 0u };
    experts_run<false>(down, p.tok, st);
    if ((rc = launched(who))) return rc;
#define OXH_COMBINE(T)                                                                                                           \
    hipLaunchKernelGGL(k_i8_combine<T>, dim3((uint32_t)((m->hidden + 1023u) / 1024u), (uint32_t)n_tok), dim3(256), 0, st, y, p.y_stride, \
                       routing->d_weights, routing->d_slot_pos, (uint32_t)m->top_k, (uint32_t)pairs, (uint32_t)m->hidden,        \
                       (T *)d_out, out_stride)
    if (out_type == OXH_F32) OXH_COMBINE(float);
    else if (out_type == OXH_F16) OXH_COMBINE(_Float16);
    else OXH_COMBINE(__bf16);
#undef OXH_COMBINE
    return launched(who);
}

/* ─── which kernels run, for tests ────────────────────────────────────── */

extern "C" int oxh_debug_i8_kernel(size_t rows, size_t cols, size_t n_vec, size_t n_cu, size_t ws_bytes, int floats, uint32_t out[4])
{
    static const char who[] = "oxh_debug_i8_kernel";
    if (!out || !rows || !n_vec || !n_cu) return I8_ARG("%s: NULL or empty", who);
    const int rc = check_cols(who, cols);
    if (rc) return rc;
    if (floats && linear_fused(rows, cols, n_vec, n_cu)) {
        out[0] = 3u;
        out[1] = few_waves(rows, cols, n_cu);
        out[2] = few_grid(rows, cols, out[1]).held;
        out[3] = (uint32_t)n_vec;
        return OXH_OK;
    }
    const I8Choice c = i8_choice(rows, cols, n_vec, ws_bytes, n_cu);
    if (c.team) {
        out[0] = n_vec > FEW_TOKENS ? 2u : 1u;
        out[1] = c.team;
        out[2] = few_grid(rows, cols, c.team).held;
        out[3] = (uint32_t)((n_vec + 15u) / 16u);
        return OXH_OK;
    }
    out[0] = 0u;
    out[1] = (uint32_t)c.way.tile;
    out[2] = c.way.splits;
    out[3] = c.way.tile == I8_LARGE ? i8_tail((uint32_t)tile_count(i8_pace[I8_LARGE], rows, n_vec), c.way.splits, n_cu) : 0u;
    return OXH_OK;
}

extern "C" int oxh_debug_moe_i8_kernels(const OxhMoeI8 *m, size_t n_tok, int ids, size_t n_cu, uint32_t out[4])
{
    static const char who[] = "oxh_debug_moe_i8_kernels";
    MoeI8Parts p;
    if (!out || !n_cu) return I8_ARG("%s: NULL or empty", who);
    const int rc = moe_parts(who, m, n_tok, &p);
    if (rc) return rc;
    const PairsPlan few = pairs_plan(m, n_tok, n_cu);
    out[0] = few.taken && ids;
    out[1] = out[0] ? 1u : p.tok;
    out[2] = out[0] ? few.up_held : experts_way(true, m->ffn, m->hidden, p.tok, p.n_tiles, n_cu).held;
    out[3] = out[0] ? few.down_held : experts_way(false, m->hidden, m->ffn, p.tok, p.n_tiles, n_cu).held;
    return OXH_OK;
}
