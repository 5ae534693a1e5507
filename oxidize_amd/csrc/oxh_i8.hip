/* oxh_i8.hip — int8 rows with one scale per row: the quantiser, the product of tokens with a matrix, and the experts'
 * products of a mixture-of-experts layer (oxh_i8_*, oxh_moe_ffn_i8). */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oxhip.h"
#include "oxh_internal.h"
#include "oxh_device.inc"
#include "i8_tiles.inc"
#include "i8_products.inc"
#include "i8_host.inc"

template <typename T, bool GLU, int THREADS, int HELD>
__global__ __launch_bounds__(THREADS) void
k_i8_quantize(const T *__restrict__ x, size_t x_stride, uint32_t cols, const T *__restrict__ up, int8_t *__restrict__ q,
              size_t q_stride, float *__restrict__ scale)
{
    const size_t row = blockIdx.x;
    i8_quantize_row<T, GLU, THREADS, HELD>(x + row * x_stride, GLU ? up + row * x_stride : nullptr, cols, q + row * q_stride, scale + row);
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

/* Threads to a row: as many as hold its values with one step or two, so that it is read once; for many rows of middling length a workgroup of 256
 * with four steps, of which a CU holds more (4096 rows, us with 64 threads and two steps, 256 and one, 256 and four, 1024 and two: of 1024
 * values 5.3, 6.1, 8.9, 20; of 2048 10, 7.8, 10, 20; of 4096 18, 13.7, 13.6, 22; of 8192 35, 26, 22, 26; of 14336 71, 52, 40, 36.  512 rows
 * of 8192: 18, 7.3, 6.0, 5.4). */
extern "C" int oxh_internal_i8_quantize(uint32_t type, const void *x, size_t x_stride, size_t n, size_t cols, const void *up, int8_t *q,
                                        size_t q_stride, float *scale, void *stream, const char *who)
{
    const hipStream_t st = (hipStream_t)stream;
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
    return oxh_internal_i8_quantize(x_type, d_x, x_stride, n_vec, cols, d_up, d_q, q_stride, d_scale, stream_of(stream), who);
}

extern "C" int oxh_internal_i8_init(void)
{
    hipError_t e;
    if ((e = product_init<I8Product>()) != hipSuccess) return (int)e;
    if ((e = whole_lds(k_i8_experts<I8Mid128, I8Mid64, I8Mid32, true>)) != hipSuccess) return (int)e;
    if ((e = whole_lds(k_i8_experts<I8Mid128, I8Mid64, I8Mid32, false>)) != hipSuccess) return (int)e;
    return (int)hipSuccess;
}

extern "C" size_t oxh_i8_matmul_workspace(const OxhI8Matrix *w, size_t n_vec)
{
    return w && workable(w->rows, w->cols, n_vec) ? product_parts(w->rows, w->cols, n_vec) : 0;
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
    I8Product p = i8_product(w, d_q, q_stride, d_q_scale, n_vec, d_bias, out_type, d_out, out_stride);
    return product_launch(p, i8_choice(w->rows, w->cols, n_vec, d_workspace ? workspace_bytes : 0, i8_cus(), I8_PLAIN), d_workspace, stream_of(stream), who);
}

extern "C" size_t oxh_i8_linear_workspace(const OxhI8Matrix *w, size_t n_vec)
{
    return w && workable(w->rows, w->cols, n_vec) ? linear_bytes(w->rows, w->cols, n_vec) : 0;
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
    I8Product p = i8_product(w, nullptr, 0, nullptr, n_vec, d_bias, out_type, d_out, out_stride);
    return linear_launch(p, x_type, d_x, x_stride, d_workspace, workspace_bytes, stream_of(stream), who);
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
    if (cols <= 2048u) OXH_BEGIN(256, 1);           /* as oxh_internal_i8_quantize(); the table wants 256 threads */
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
    if ((rc = oxh_internal_i8_quantize(OXH_F32, h, p.h_stride, pairs, m->ffn, nullptr, qh, p.qh_stride, qh_scale, st, who))) return rc;
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
    i8_describe(i8_choice(rows, cols, n_vec, ws_bytes, n_cu, I8_PLAIN), rows, cols, n_vec, n_cu, I8_PLAIN, out);
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
