/* oxh_select.hip — routing for models with many experts: softmax or sigmoid scores, a bias on the choice, expert groups,
 * up to 512 experts and 16 choices, and the pairs sorted by expert (oxh_moe_select).
 *
 * A wave per token, lane l the experts l, l + 64, ...  Scores are 64-bit: two keys next to each other at the border
 * of the choice are told apart as the definition tells them, which 32 bits do not always do (among 256 sigmoids the
 * eighth and ninth lie within 1e-7 of each other in about one token of 40 000).
 *
 * Sorting needs no sort: a workgroup takes at most 64 tokens, and a token chooses an expert at most once, so the
 * tokens of an expert are a 64-bit mask in LDS; its count is the mask's population and a pair's rank the population
 * below its token.  Bound by the instructions of 64-bit exponentials and of the rounds of the choice (about 5000 cycles a token, four
 * waves to a SIMD): 4096 tokens, 8 of 256 sigmoids in groups, in 12 us and the positions in 5.5.  For a few tokens one workgroup does all of it in one launch.  Above, every workgroup leaves its
 * counts (a byte each) and a second launch adds up those of the workgroups before it. */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oxhip.h"
#include "oxh_internal.h"
#include "oxh_device.inc"

#pragma clang fp contract(off)

#define SEL_TOKENS 64u              /* a workgroup's tokens, at most: bits of a mask */
#define SEL_WAVES 16u

/* 1 / 13! .. 1 / 0!, an argument of the kernel so that they are scalar operands, not registers that every wave fills one by one */
#define EXP_TERMS 14
struct ExpSeries {
    double c[EXP_TERMS];
};

struct SelectArgs {
    ExpSeries exp;
    const void *logits;
    size_t stride;
    const float *bias;
    int32_t *ids;
    float *weights;
    uint32_t *counts, *offsets, *perm, *slot_pos;
    uint8_t *hist;                  /* [workgroup][hist_stride] counts; NULL for a launch of one workgroup */
    uint32_t n_tok, tok_per_wg, rows, rows_per_wg, n_expert, k, n_group, top_group, group_best, score, renorm, hist_stride;
    float scale;
};

/* The order of 64-bit keys as the order of integers; the least key there is, -inf, maps to more than the two below. */
__device__ __forceinline__ uint64_t sortable(double key)
{
    const uint64_t b = (uint64_t)__double_as_longlong(key);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
#define KEY_MASKED 1ull             /* chosen after all others */
#define KEY_NONE 0ull               /* never chosen */

/* e^x for x <= 709: x = k ln 2 + r, the series of e^r to its thirteenth power (|r| <= 0.347: what is left out is 4e-18 of it).  Half of
 * the instructions of the library's, which also looks after what cannot come here. */
__device__ __forceinline__ double exp64(double x, const ExpSeries &s)
{
    x = fmax(x, -750.0);
    const double k = rint(x * 1.4426950408889634074);
    double r = __builtin_fma(-k, 0x1.62e42fee00000p-1, x);          /* ln 2 in two parts, the first of 32 bits: k times it is exact */
    r = __builtin_fma(-k, 0x1.a39ef35793c76p-33, r);
    double e = s.c[0];
#pragma unroll
    for (int i = 1; i < EXP_TERMS; i++) e = __builtin_fma(e, r, s.c[i]);
    return __builtin_ldexp(e, (int)k);
}

/* v's neighbour in a step of a reduction over 16 lanes (lane ^ 1, lane ^ 2, mirrored in 8, mirrored in 16): no trip through LDS */
template <int STEP> __device__ __forceinline__ uint32_t dpp_step(uint32_t v)
{
    constexpr int ctrl = STEP == 0 ? 0xB1 : STEP == 1 ? 0x4E : STEP == 2 ? 0x141 : 0x140;
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF, 0xF, false);
}
template <int STEP> __device__ __forceinline__ double dpp_step(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)(((uint64_t)dpp_step<STEP>((uint32_t)(b >> 32)) << 32) | dpp_step<STEP>((uint32_t)b)));
}

__device__ __forceinline__ double lane_double(double v, int lane)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}

__device__ __forceinline__ double wave_sum64(double v)
{
    v += dpp_step<0>(v);
    v += dpp_step<1>(v);
    v += dpp_step<2>(v);
    v += dpp_step<3>(v);
    return (lane_double(v, 0) + lane_double(v, 16)) + (lane_double(v, 32) + lane_double(v, 48));
}

__device__ __forceinline__ uint32_t wave_max32(uint32_t v)
{
    v = max(v, dpp_step<0>(v));
    v = max(v, dpp_step<1>(v));
    v = max(v, dpp_step<2>(v));
    v = max(v, dpp_step<3>(v));
    return max(max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16)),
               max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48)));
}

/* The lane that holds the largest 64-bit key: by its upper half, by the lower one only where that does not tell, and of equal keys the one
 * of the lowest expert, `at` (expert e is lane e % 64's). */
__device__ __forceinline__ int wave_argmax64(uint64_t key, uint32_t at)
{
    const uint32_t hi = (uint32_t)(key >> 32), top = wave_max32(hi);
    unsigned long long who = __ballot(hi == top);
    if (who & (who - 1ull)) {
        const uint32_t lo = hi == top ? (uint32_t)key : 0u, low = wave_max32(lo);
        const bool equal = hi == top && lo == low;
        who = __ballot(equal);
        if (who & (who - 1ull)) return (int)(~wave_max32(equal ? ~at : 0u) & 63u);
    }
    return __builtin_ctzll(who);
}

/* what a wave's lanes wrote to LDS before, its other lanes read after */
__device__ __forceinline__ void sel_wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename T> __device__ __forceinline__ float sel_load(const void *p, size_t i);
template <> __device__ __forceinline__ float sel_load<float>(const void *p, size_t i) { return ((const float *)p)[i]; }
template <> __device__ __forceinline__ float sel_load<_Float16>(const void *p, size_t i) { return (float)((const _Float16 *)p)[i]; }
template <> __device__ __forceinline__ float sel_load<__bf16>(const void *p, size_t i)
{
    return __uint_as_float((uint32_t)((const uint16_t *)p)[i] << 16);
}

/* exclusive prefix of the experts' totals (in s_total) into s_base; one wave */
__device__ __forceinline__ void sel_scan(const uint32_t *s_total, uint32_t *s_base, uint32_t n_expert, uint32_t lane)
{
    uint32_t own[8], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8u; i++) {
        own[i] = 8u * lane + i < n_expert ? s_total[8u * lane + i] : 0u;
        sum += own[i];
    }
    uint32_t upto = sum;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t v = __shfl_up(upto, d);
        if (lane >= d) upto += v;
    }
    uint32_t at = upto - sum;
#pragma unroll
    for (uint32_t i = 0; i < 8u; i++) {
        s_base[8u * lane + i] = at;
        at += own[i];
    }
}

template <typename T, int NPL>
__global__ __launch_bounds__(1024) void k_moe_select(const SelectArgs a)
{
    __shared__ unsigned long long s_mask[OXH_SELECT_MAX_EXPERTS];
    __shared__ double s_key[SEL_WAVES][NPL * 64];
    __shared__ double s_score[SEL_WAVES][NPL * 64];
    __shared__ uint16_t s_id[SEL_TOKENS * OXH_SELECT_MAX_TOPK];
    __shared__ uint32_t s_total[OXH_SELECT_MAX_EXPERTS], s_base[OXH_SELECT_MAX_EXPERTS];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t t0 = blockIdx.x * a.tok_per_wg, here = min(a.tok_per_wg, a.n_tok - t0), E = a.n_expert;
    for (uint32_t e = tid; e < OXH_SELECT_MAX_EXPERTS; e += blockDim.x) s_mask[e] = 0ull;
    __syncthreads();
    for (uint32_t tt = wave; tt < here; tt += SEL_WAVES) {
        const size_t row = (size_t)(t0 + tt) * a.stride;
        const double ninf = -__builtin_inf();
        const bool softmax = a.score == OXH_SCORE_SOFTMAX;
        uint64_t key[NPL];
        uint32_t at[NPL];
        float x[NPL], bias[NPL], top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < NPL; i++) x[i] = sel_load<T>(a.logits, row + min(lane + 64u * i, E - 1u));
#pragma unroll
        for (int i = 0; i < NPL; i++) bias[i] = a.bias ? a.bias[min(lane + 64u * i, E - 1u)] : 0.0f;
#pragma unroll
        for (int i = 0; i < NPL; i++) {
            /* a NaN is masked as -inf is */
            x[i] = lane + 64u * i < E && x[i] == x[i] ? fminf(x[i], 3.402823466e38f) : -__builtin_inff();
            top = fmaxf(top, x[i]);
            s_score[wave][lane + 64u * i] = (double)x[i];
        }
        /* A lane's experts one after the other, in a loop that stays a loop: a wave comes here once, and what it does not have to
         * fetch of the program it does not wait for.  e^(x - top), or 1 / (1 + e^-x) with the sum within range (below e^-708 it is 0) */
        top = softmax ? wave_max(top) : 0.0f;
        double z = 0.0;
#pragma unroll 1
        for (uint32_t e = lane; e < NPL * 64u; e += 64u) {
            const double v = s_score[wave][e];
            const double d = exp64(softmax ? v - (double)top : fmin(-v, 708.0), a.exp);
            double r = __builtin_amdgcn_rcp(1.0 + d);
            r = __builtin_fma(__builtin_fma(-(1.0 + d), r, 1.0), r, r);
            r = __builtin_fma(__builtin_fma(-(1.0 + d), r, 1.0), r, r);
            r = softmax ? d : r;
            r = v < (softmax ? -3.5e38 : -708.0) ? 0.0 : r;
            z += r;
            s_score[wave][e] = r;
        }
        double factor = 1.0;
        if (softmax) {
            z = wave_sum64(z);
            factor = z > 0.0 ? 1.0 / z : 0.0;
        }
#pragma unroll
        for (int i = 0; i < NPL; i++) {
            const uint32_t e = lane + 64u * i;
            const double p = s_score[wave][e] * factor, kv = p + (double)bias[i];
            const bool live = x[i] > -__builtin_inff() && kv > ninf;        /* a NaN is not */
            key[i] = e < E ? live ? sortable(kv) : KEY_MASKED : KEY_NONE;
            at[i] = e;
            s_score[wave][e] = live ? p : 0.0;
            if (a.n_group > 1u) s_key[wave][e] = live ? kv : ninf;
        }
        sel_wave_sync();
        if (a.n_group > 1u) {
            /* `share` neighbouring lanes look through a group, every one at each share-th of its keys, and put their best two
             * together */
            const uint32_t size = E / a.n_group, share = 1u << (31u - (uint32_t)__builtin_clz(64u / a.n_group));
            const uint32_t mine = lane / share, from = lane % share;
            double b1 = ninf, b2 = ninf;
            if (mine < a.n_group)
#pragma unroll 2
                for (uint32_t j = from; j < size; j += share) {
                    const double v = s_key[wave][mine * size + j];
                    b2 = fmax(b2, fmin(b1, v));
                    b1 = fmax(b1, v);
                }
#pragma unroll 1
            for (uint32_t d = 1; d < share; d <<= 1) {
                const double o1 = __shfl_xor(b1, (int)d), o2 = __shfl_xor(b2, (int)d);
                b2 = fmax(fmin(b1, o1), fmax(b2, o2));
                b1 = fmax(b1, o1);
            }
            /* a masked expert does not count */
            const uint64_t rank = sortable(a.group_best == 2u && b2 > ninf ? b1 + b2 : b1);
            uint32_t before = 0;
#pragma unroll 1
            for (uint32_t g = 0; g < a.n_group; g++) {
                const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)rank, (int)(g * share));
                const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(rank >> 32), (int)(g * share));
                const uint64_t other = ((uint64_t)hi << 32) | lo;
                before += other > rank || (other == rank && g < mine) ? 1u : 0u;
            }
            /* bit g * share: whether group g is kept */
            const unsigned long long kept = __ballot(mine < a.n_group && before < a.top_group);
#pragma unroll
            for (int i = 0; i < NPL; i++) {
                const uint32_t e = lane + 64u * i;
                if (e < E && !((kept >> (e / size * share)) & 1ull)) key[i] = KEY_NONE;
            }
        }
        /* a lane's keys in descending order, equal ones in the experts', of which only the first one is looked at */
#pragma unroll
        for (int n = NPL - 1; n > 0; n--)
#pragma unroll
            for (int i = 0; i < n; i++) {
                const bool swap = key[i + 1] > key[i];
                const uint64_t high = swap ? key[i + 1] : key[i], low = swap ? key[i] : key[i + 1];
                const uint32_t first = swap ? at[i + 1] : at[i], second = swap ? at[i] : at[i + 1];
                key[i] = high;
                key[i + 1] = low;
                at[i] = first;
                at[i + 1] = second;
            }
        uint32_t my_id = 0;
#pragma unroll 1
        for (uint32_t j = 0; j < a.k; j++) {
            const int owner = wave_argmax64(key[0], at[0]);
            const uint32_t id = (uint32_t)__builtin_amdgcn_readlane((int)at[0], owner);
            my_id = lane == j ? id : my_id;
            if ((int)lane == owner) {
#pragma unroll
                for (int i = 0; i + 1 < NPL; i++) {
                    key[i] = key[i + 1];
                    at[i] = at[i + 1];
                }
                key[NPL - 1] = KEY_NONE;
            }
        }
        const double my_p = lane < a.k ? s_score[wave][my_id] : 0.0;
        const double sum = wave_sum64(my_p);
        double w = my_p;
        if (a.renorm) w = sum > 0.0 ? my_p / sum : 0.0;
        if (lane < a.k) {
            const size_t pair = (size_t)(t0 + tt) * a.k + lane;
            a.ids[pair] = (int32_t)my_id;
            a.weights[pair] = (float)(w * (double)a.scale);
            s_id[tt * a.k + lane] = (uint16_t)my_id;
            atomicOr(&s_mask[my_id], 1ull << tt);
        }
        sel_wave_sync();
    }
    __syncthreads();
    if (a.hist) {
        for (uint32_t e = tid; e < a.hist_stride; e += blockDim.x)
            a.hist[(size_t)blockIdx.x * a.hist_stride + e] = e < E ? (uint8_t)__popcll(s_mask[e]) : (uint8_t)0;
        return;
    }
    for (uint32_t e = tid; e < E; e += blockDim.x) s_total[e] = (uint32_t)__popcll(s_mask[e]);
    __syncthreads();
    if (wave == 0u) sel_scan(s_total, s_base, E, lane);
    __syncthreads();
    for (uint32_t e = tid; e < E; e += blockDim.x) {
        a.counts[e] = s_total[e];
        a.offsets[e] = s_base[e];
    }
    if (tid == 0u) a.offsets[E] = a.n_tok * a.k;
    for (uint32_t i = tid; i < here * a.k; i += blockDim.x) {
        const uint32_t tt = i / a.k, e = s_id[i];
        const uint32_t pos = s_base[e] + (uint32_t)__popcll(s_mask[e] & ((1ull << tt) - 1ull));
        a.perm[pos] = t0 + tt;
        a.slot_pos[i] = pos;
    }
}

#define PLACE_THREADS 1024u
#define PLACE_COPIES 8u
#define PLACE_WORDS (OXH_SELECT_MAX_EXPERTS / 2u)

/* The positions of the pairs of many workgroups' tokens: the counts of all workgroups give the experts' runs, those of
 * the workgroups before this one where its own pairs start in them.  Sixteen counts to a load, rows dealt to the threads;
 * they are added up two to a word (an expert has at most one pair of a token, 65535 in all).  Up to 256 rows of counts have a workgroup
 * each; more are taken several by one, for each looks through all of them (65535 tokens over 128 experts, both launches: 71 us, 87.9 with a
 * workgroup to each of 1024 rows). */
__global__ __launch_bounds__(PLACE_THREADS) void k_moe_place(const SelectArgs a)
{
    __shared__ unsigned long long s_mask[OXH_SELECT_MAX_EXPERTS];
    /* eight copies of the sums, in other banks, for neighbouring slices: a wave's lanes hardly meet in one word (2000 tokens over 64
     * experts, both launches: 9.8 us, 11.3 with one copy) */
    __shared__ uint32_t s_all[PLACE_COPIES][PLACE_WORDS + 8u], s_bef[PLACE_COPIES][PLACE_WORDS + 8u];
    __shared__ uint32_t s_total[OXH_SELECT_MAX_EXPERTS], s_base[OXH_SELECT_MAX_EXPERTS];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, E = a.n_expert;
    const uint32_t row0 = blockIdx.x * a.rows_per_wg, rows = min(a.rows_per_wg, a.rows - row0);
    static_assert(SEL_TOKENS * OXH_SELECT_MAX_TOPK <= PLACE_THREADS, "a row's choices are one a thread at most");
    uint32_t id;
    const uint32_t tt = tid / a.k;                      /* the row's token whose choice this thread has */
    auto choices = [&](uint32_t row) {
        const uint32_t t0 = row * a.tok_per_wg, n_pairs = min(a.tok_per_wg, a.n_tok - t0) * a.k;
        id = (uint32_t)a.ids[(size_t)t0 * a.k + min(tid, n_pairs - 1u)];
    };
    auto marks = [&](uint32_t n_pairs) {
        if (tid < n_pairs) atomicOr(&s_mask[id], 1ull << tt);
    };
    /* the loads first: this workgroup's first choices, the first rows of counts */
    choices(row0);
    const uint32_t chunks = a.hist_stride / 16u, slices = PLACE_THREADS / chunks, c = tid % chunks, first = tid / chunks;
    uint32_t all[8] = { 0u }, bef[8] = { 0u };         /* experts 4i, 4i + 2 and 4i + 1, 4i + 3 of the chunk */
    auto counts = [&](uint32_t b) { return *reinterpret_cast<const u32x4 *>(a.hist + (size_t)min(b, a.rows - 1u) * a.hist_stride + 16u * c); };
    auto add = [&](const u32x4 &v, uint32_t b) {
        const uint32_t there = b < a.rows ? 0x00FF00FFu : 0u, before = b < row0 ? 0x00FF00FFu : 0u;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            all[2 * i] += v[i] & there;
            all[2 * i + 1] += (v[i] >> 8) & there;
            bef[2 * i] += v[i] & before;
            bef[2 * i + 1] += (v[i] >> 8) & before;
        }
    };
    if (tid < slices * chunks) {
        if (a.rows <= slices) add(counts(first), first);
        else
            for (uint32_t b = first; b < a.rows; b += 4u * slices) {       /* four loads under way at a time */
                u32x4 v[4];
#pragma unroll
                for (uint32_t j = 0; j < 4u; j++) v[j] = counts(b + j * slices);
#pragma unroll
                for (uint32_t j = 0; j < 4u; j++) add(v[j], b + j * slices);
            }
    }
    for (uint32_t e = tid; e < OXH_SELECT_MAX_EXPERTS; e += PLACE_THREADS) s_mask[e] = 0ull;
    for (uint32_t i = tid; i < PLACE_COPIES * (PLACE_WORDS + 8u); i += PLACE_THREADS) s_all[0][i] = s_bef[0][i] = 0u;
    __syncthreads();
    marks(min(a.tok_per_wg, a.n_tok - row0 * a.tok_per_wg) * a.k);
    if (tid < slices * chunks)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (all[i]) atomicAdd(&s_all[first % PLACE_COPIES][8u * c + i], all[i]);
            if (bef[i]) atomicAdd(&s_bef[first % PLACE_COPIES][8u * c + i], bef[i]);
        }
    __syncthreads();
    if (tid < 2u * PLACE_WORDS) {
        uint32_t *const word = (tid < PLACE_WORDS ? s_all[0] : s_bef[0]) + tid % PLACE_WORDS;
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < PLACE_COPIES; i++) sum += word[i * (PLACE_WORDS + 8u)];
        *word = sum;
    }
    __syncthreads();
    /* expert 4q + r of the words: word 2q + (r & 1), half r >> 1 */
    auto half = [](const uint32_t *w, uint32_t e) { return (w[2u * (e / 4u) + (e & 1u)] >> (8u * (e & 2u))) & 0xFFFFu; };
    for (uint32_t e = tid; e < E; e += PLACE_THREADS) s_total[e] = half(s_all[0], e);
    __syncthreads();
    if (wave == 0u) sel_scan(s_total, s_base, E, lane);
    __syncthreads();
    if (blockIdx.x == 0u) {
        for (uint32_t e = tid; e < E; e += PLACE_THREADS) {
            a.counts[e] = s_total[e];
            a.offsets[e] = s_base[e];
        }
        if (tid == 0u) a.offsets[E] = a.n_tok * a.k;
    }
    for (uint32_t row = row0; row < row0 + rows; row++) {
        const uint32_t t0 = row * a.tok_per_wg, n_pairs = min(a.tok_per_wg, a.n_tok - t0) * a.k;
        if (row > row0) {                               /* the row before is done: its pairs lie before this one's */
            choices(row);
            __syncthreads();
            for (uint32_t e = tid; e < E; e += PLACE_THREADS) {
                s_base[e] += (uint32_t)__popcll(s_mask[e]);
                s_mask[e] = 0ull;
            }
            __syncthreads();
            marks(n_pairs);
            __syncthreads();
        }
        if (tid < n_pairs) {
            const uint32_t pos = s_base[id] + half(s_bef[0], id) + (uint32_t)__popcll(s_mask[id] & ((1ull << tt) - 1ull));
            a.perm[pos] = t0 + tt;
            a.slot_pos[(size_t)t0 * a.k + tid] = pos;
        }
    }
}

/* ─── host side ───────────────────────────────────────────────────────── */

/* One workgroup and one launch for as many tokens as it has waves; few experts take less of a wave's time (256 experts, 16 tokens: 10.5 us,
 * in two launches 10.3; 64 tokens: 29.3 and 10.6; 64 experts, 24 tokens: 6.3 and 8.0). */
static bool sel_single(const OxhMoeRouter *r, size_t n_tok) { return n_tok <= (r->n_expert <= 64u ? 2u : 1u) * SEL_WAVES; }

/* A workgroup's tokens otherwise: one wave to a SIMD while there are CUs left (256 experts, 65 tokens: 10.3 us in workgroups of four, 13.5 of
 * sixteen), then more, for the second launch looks through the counts of all workgroups: no more than 256 of them up to 8192 tokens. */
static uint32_t sel_tok_per_wg(size_t n_tok)
{
    if (n_tok <= 1024u) return 4u;
    if (n_tok <= 2048u) return 8u;
    return n_tok <= 4096u ? 16u : n_tok <= 8192u ? 32u : SEL_TOKENS;
}

static uint32_t sel_hist_stride(size_t n_expert) { return ((uint32_t)n_expert + 15u) & ~15u; }

static int sel_check(const OxhMoeRouter *r, size_t n_tok, const char *who)
{
    if (!r) return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: NULL router", who);
    if (r->score != OXH_SCORE_SOFTMAX && r->score != OXH_SCORE_SIGMOID)
        return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: score %u is not one of OXH_SCORE_*", who, r->score);
    if (r->n_expert == 0 || r->n_expert > OXH_SELECT_MAX_EXPERTS)
        return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: n_expert must be 1..%u", who, OXH_SELECT_MAX_EXPERTS);
    size_t open = r->n_expert;
    if (r->n_group > 1) {
        if (r->n_group > OXH_SELECT_MAX_GROUPS || r->n_expert % r->n_group)
            return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: n_group must be at most %u and divide n_expert", who,
                                       OXH_SELECT_MAX_GROUPS);
        if (r->top_group == 0 || r->top_group > r->n_group)
            return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: top_group must be 1..n_group", who);
        if (r->group_best != 1 && r->group_best != 2)
            return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: group_best must be 1 or 2", who);
        open = r->n_expert / r->n_group * r->top_group;
    }
    if (r->top_k == 0 || r->top_k > OXH_SELECT_MAX_TOPK || r->top_k > open)
        return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: top_k must be 1..%u and at most the experts of the kept groups (%zu)",
                                   who, OXH_SELECT_MAX_TOPK, open);
    if (n_tok > OXH_SELECT_MAX_TOKENS)
        return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: at most %u tokens per call", who, OXH_SELECT_MAX_TOKENS);
    return OXH_OK;
}

static size_t sel_workspace(const OxhMoeRouter *r, size_t n_tok)
{
    const uint32_t per = sel_tok_per_wg(n_tok);
    const size_t wgs = (n_tok + per - 1u) / per;
    /* where a workgroup takes more tokens there are fewer of them: never less than for fewer tokens */
    return sel_single(r, n_tok) ? 0 : (n_tok > 1024u && wgs < 256u ? 256u : wgs) * sel_hist_stride(r->n_expert);
}

extern "C" int oxh_moe_select_workspace(const OxhMoeRouter *r, size_t n_tok, size_t *bytes)
{
    const int rc = sel_check(r, n_tok, "oxh_moe_select_workspace");
    if (rc) return rc;
    if (bytes) *bytes = sel_workspace(r, n_tok);
    return OXH_OK;
}

template <typename T> static void sel_launch(const SelectArgs &a, uint32_t wgs, hipStream_t st)
{
    const dim3 grid(wgs), block(64u * SEL_WAVES);
    if (a.n_expert <= 64u) hipLaunchKernelGGL((k_moe_select<T, 1>), grid, block, 0, st, a);
    else if (a.n_expert <= 128u) hipLaunchKernelGGL((k_moe_select<T, 2>), grid, block, 0, st, a);
    else if (a.n_expert <= 256u) hipLaunchKernelGGL((k_moe_select<T, 4>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((k_moe_select<T, 8>), grid, block, 0, st, a);
}

extern "C" int oxh_moe_select(const OxhMoeRouter *r, uint32_t logits_type, const void *d_logits, size_t logits_stride,
                              size_t n_tok, const OxhRouting *out, void *d_workspace, size_t workspace_bytes, void *stream)
{
    static const char who[] = "oxh_moe_select";
    int rc = sel_check(r, n_tok, who);
    if (rc) return rc;
    if (logits_type != OXH_F32 && logits_type != OXH_F16 && logits_type != OXH_BF16)
        return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: logits_type %u is not OXH_F32, OXH_F16 or OXH_BF16", who, logits_type);
    if (n_tok == 0) return OXH_OK;
    if (!d_logits || !out || !out->d_ids || !out->d_weights || !out->d_counts || !out->d_offsets || !out->d_perm || !out->d_slot_pos)
        return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: NULL pointer", who);
    if ((uintptr_t)d_logits % (logits_type == OXH_F32 ? 4u : 2u))
        return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: d_logits is not aligned to its elements", who);
    if (logits_stride < r->n_expert) return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: logits_stride < n_expert", who);
    const size_t need = sel_workspace(r, n_tok);
    if (need && (!d_workspace || workspace_bytes < need))
        return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: workspace too small (see oxh_moe_select_workspace)", who);
    if (need && ((uintptr_t)d_workspace & 15u))
        return oxh_internal_errorf(OXH_ERR_ARG, "invalid argument: %s: workspace must be 16-byte aligned", who);
    if (oxh_internal_device() < 0 && (rc = oxh_init(0))) return rc;
    SelectArgs a = {};
    double term = 1.0;                              /* n!, exact */
    for (int n = 0; n < EXP_TERMS; n++) {
        a.exp.c[EXP_TERMS - 1 - n] = 1.0 / term;
        term *= n + 1;
    }
    a.logits = d_logits;
    a.stride = logits_stride;
    a.bias = r->d_bias;
    a.ids = out->d_ids;
    a.weights = out->d_weights;
    a.counts = out->d_counts;
    a.offsets = out->d_offsets;
    a.perm = out->d_perm;
    a.slot_pos = out->d_slot_pos;
    a.hist = need ? (uint8_t *)d_workspace : nullptr;
    a.n_tok = (uint32_t)n_tok;
    a.tok_per_wg = need ? sel_tok_per_wg(n_tok) : SEL_TOKENS;
    a.n_expert = (uint32_t)r->n_expert;
    a.k = (uint32_t)r->top_k;
    a.n_group = r->n_group > 1 ? (uint32_t)r->n_group : 1u;
    a.top_group = (uint32_t)r->top_group;
    a.group_best = r->group_best;
    a.score = r->score;
    a.renorm = r->renorm ? 1u : 0u;
    a.hist_stride = sel_hist_stride(r->n_expert);
    a.scale = r->scale;
    const uint32_t wgs = (a.n_tok + a.tok_per_wg - 1u) / a.tok_per_wg;
    a.rows = wgs;
    a.rows_per_wg = (wgs + 255u) / 256u;
    hipStream_t st = (hipStream_t)(stream ? stream : oxh_internal_stream());
    if (logits_type == OXH_F32) sel_launch<float>(a, wgs, st);
    else if (logits_type == OXH_F16) sel_launch<_Float16>(a, wgs, st);
    else sel_launch<__bf16>(a, wgs, st);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && need) {
        hipLaunchKernelGGL(k_moe_place, dim3((wgs + a.rows_per_wg - 1u) / a.rows_per_wg), dim3(PLACE_THREADS), 0, st, a);
        e = hipGetLastError();
    }
    if (e != hipSuccess) return oxh_internal_errorf(OXH_ERR_HIP, "HIP error in %s: %s", who, hipGetErrorString(e));
    return OXH_OK;
}
