/* oxh_i8.hip — int8 rows with one scale per row: the quantiser, the product of tokens with a matrix, and the experts'
 * products of a mixture-of-experts layer (oxh_i8_*, oxh_moe_ffn_i8). */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "oxhip.h"
#include "oxh_internal.h"
#include "oxh_device.inc"

#pragma clang fp contract(off)

typedef int v4i __attribute__((ext_vector_type(4)));

/* ─── floats ──────────────────────────────────────────────────────────── */

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }      /* to nearest, ties to even */

/* N neighbouring values that are aligned to their elements only */
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Run { T v[N]; };

/* ─── rows of floats to codes ─────────────────────────────────────────── */

/* The integer nearest to v / s, ties to even.  v * inv is within 2^-15 of the quotient, so its rounding is off by one at
 * most, next to a half; the remainder v - t * s has no more bits than an f32 holds (it is a multiple of half a unit of
 * s's last place and no larger than half of s and a bit), the fused operation gives it exactly, and which side of the half it lies
 * on says whether the rounding was right. */
__device__ __forceinline__ int i8_code(float v, float s, float inv)
{
    float t = rintf(v * inv);
    const float r = __builtin_fmaf(-t, s, v), twice = r + r;
    const bool odd = ((int)t & 1) != 0;
    if (twice > s || (twice == s && odd)) t += 1.0f;
    else if (twice < -s || (twice == -s && odd)) t -= 1.0f;
    return (int)t;
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

__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

/* A workgroup per row, eight values to a thread and step: once for the largest magnitude, once for the codes. */
template <typename T, bool GLU>
__global__ __launch_bounds__(256) void
k_i8_quantize(const T *__restrict__ x, size_t x_stride, uint32_t cols, const T *__restrict__ up, int8_t *__restrict__ q,
              size_t q_stride, float *__restrict__ scale)
{
    __shared__ uint32_t s_top[4];
    const size_t row = blockIdx.x;
    const T *xr = x + row * x_stride, *ur = GLU ? up + row * x_stride : nullptr;
    auto value = [&](uint32_t c) {
        const float v = to_f32(xr[c]);
        return GLU ? silu(v) * to_f32(ur[c]) : v;
    };
    uint32_t top = 0;
    for (uint32_t c = threadIdx.x; c < cols; c += 256u) top = max(top, __float_as_uint(value(c)) & 0x7FFFFFFFu);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if ((threadIdx.x & 63u) == 0u) s_top[threadIdx.x >> 6] = top;
    __syncthreads();
    top = max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]));
    float inv;
    const float s = i8_scale(top, inv);
    if (threadIdx.x == 0u) scale[row] = s;
    for (uint32_t c = threadIdx.x; c < ((cols + 15u) & ~15u); c += 256u)
        q[row * q_stride + c] = (int8_t)(inv != 0.0f && c < cols ? i8_code(value(c), s, inv) : 0);
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

/* 16 rows x 16 tokens of a wave: lane l supplies sixteen columns of row l % 16 and of token l % 16, and receives the sums
 * of token l % 16 and rows 4 * (l / 16) .. +3.  Zeroing one operand behind the last column is enough. */
__device__ __forceinline__ v4i i8_wave_sums(const int8_t *w_row, const int8_t *q_row, uint32_t cols, uint32_t lane)
{
    v4i acc = { 0, 0, 0, 0 };
    for (uint32_t k0 = 0; k0 < cols; k0 += 64u) {
        const uint32_t k = k0 + 16u * (lane >> 4);
        const v4i a = i8_piece(w_row, k, cols), b = i8_piece(q_row, k, cols);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, acc, 0, 0, 0);
    }
    return acc;
}

template <typename T>
__global__ __launch_bounds__(256) void
k_i8_matmul(const OxhI8Matrix w, const int8_t *__restrict__ q, size_t q_stride, const float *__restrict__ q_scale, uint32_t n_vec,
            const float *__restrict__ bias, T *__restrict__ out, size_t out_stride)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, rows = (uint32_t)w.rows;
    const uint32_t r0 = blockIdx.x * 64u + 16u * wave, t = blockIdx.y * 16u + (lane & 15u);
    if (r0 >= rows) return;
    const v4i acc = i8_wave_sums(w.d_w + (size_t)min(r0 + (lane & 15u), rows - 1u) * w.stride,
                                 q + (size_t)min(t, n_vec - 1u) * q_stride, (uint32_t)w.cols, lane);
    if (t >= n_vec) return;
    const float st = q_scale[t];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t r = r0 + 4u * (lane >> 4) + i;
        if (r >= rows) break;
        float v = (float)acc[i] * st * w.d_scale[r];
        if (bias) v += bias[r];
        out[(size_t)t * out_stride + r] = from_f32<T>(v);
    }
}

/* An expert's run of the sorted pairs, as far as it lies among them. */
__device__ __forceinline__ uint32_t i8_run(const uint32_t *offsets, uint32_t e, uint32_t pairs, uint32_t &first)
{
    first = min(offsets[e], pairs);
    const uint32_t end = min(offsets[e + 1u], pairs);
    return end > first ? end - first : 0u;
}

/* h = silu(gate) * up of an expert's pairs; the pairs' tokens through perm */
__global__ __launch_bounds__(256) void
k_i8_experts_up(const OxhMoeI8 m, const OxhRouting rt, const int8_t *__restrict__ q, size_t q_stride,
                const float *__restrict__ q_scale, uint32_t n_tok, uint32_t pairs, float *__restrict__ h, size_t h_stride)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, e = blockIdx.y, ffn = (uint32_t)m.ffn;
    const uint32_t r0 = blockIdx.x * 64u + 16u * wave;
    if (r0 >= ffn) return;
    uint32_t first;
    const uint32_t n = i8_run(rt.d_offsets, e, pairs, first);
    const size_t row = (size_t)e * ffn + min(r0 + (lane & 15u), ffn - 1u);
    for (uint32_t j0 = 0; j0 < n; j0 += 16u) {
        const uint32_t j = first + min(j0 + (lane & 15u), n - 1u), tok = min(rt.d_perm[j], n_tok - 1u);
        const int8_t *qr = q + (size_t)tok * q_stride;
        const v4i g = i8_wave_sums(m.d_w_gate + row * m.gate_up_stride, qr, (uint32_t)m.hidden, lane);
        const v4i u = i8_wave_sums(m.d_w_up + row * m.gate_up_stride, qr, (uint32_t)m.hidden, lane);
        if (j0 + (lane & 15u) >= n) continue;
        const float st = q_scale[tok];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t r = r0 + 4u * (lane >> 4) + i;
            if (r >= ffn) break;
            const float gv = (float)g[i] * st * m.d_s_gate[(size_t)e * ffn + r], uv = (float)u[i] * st * m.d_s_up[(size_t)e * ffn + r];
            h[(size_t)j * h_stride + r] = silu(gv) * uv;
        }
    }
}

__global__ __launch_bounds__(256) void
k_i8_experts_down(const OxhMoeI8 m, const OxhRouting rt, const int8_t *__restrict__ q, size_t q_stride,
                  const float *__restrict__ q_scale, uint32_t pairs, float *__restrict__ y, size_t y_stride)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, e = blockIdx.y, rows = (uint32_t)m.hidden;
    const uint32_t r0 = blockIdx.x * 64u + 16u * wave;
    if (r0 >= rows) return;
    uint32_t first;
    const uint32_t n = i8_run(rt.d_offsets, e, pairs, first);
    const size_t row = (size_t)e * rows + min(r0 + (lane & 15u), rows - 1u);
    for (uint32_t j0 = 0; j0 < n; j0 += 16u) {
        const uint32_t j = first + min(j0 + (lane & 15u), n - 1u);
        const v4i s = i8_wave_sums(m.d_w_down + row * m.down_stride, q + (size_t)j * q_stride, (uint32_t)m.ffn, lane);
        if (j0 + (lane & 15u) >= n) continue;
        const float st = q_scale[j];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t r = r0 + 4u * (lane >> 4) + i;
            if (r >= rows) break;
            y[(size_t)j * y_stride + r] = (float)s[i] * st * m.d_s_down[(size_t)e * rows + r];
        }
    }
}

/* out[t] = sum over t's pairs, in their order, of weight * y */
template <typename T>
__global__ __launch_bounds__(256) void
k_i8_combine(const float *__restrict__ y, size_t y_stride, const float *__restrict__ weights, const uint32_t *__restrict__ slot_pos,
             uint32_t k, uint32_t pairs, uint32_t cols, T *__restrict__ out, size_t out_stride)
{
    const size_t t = blockIdx.y;
    const uint32_t c = blockIdx.x * 256u + threadIdx.x;
    if (c >= cols) return;
    float acc = 0.0f;
    for (uint32_t j = 0; j < k; j++) acc += weights[t * k + j] * y[(size_t)min(slot_pos[t * k + j], pairs - 1u) * y_stride + c];
    out[t * out_stride + c] = from_f32<T>(acc);
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

/* rows or tokens: the launches count them in 32 bits, in grids of up to 2^31 threads a dimension */
#define I8_MAX_ROWS ((size_t)1 << 23)

static int check_rows(const char *who, const char *name, const void *d, size_t stride, size_t cols)
{
    if (!d) return I8_ARG("%s: NULL pointer (%s)", who, name);
    if ((uintptr_t)d & 15u) return I8_ARG("%s: %s must be 16-byte aligned", who, name);
    if (stride % 16u) return I8_ARG("%s: the stride of %s must be a multiple of 16", who, name);
    if (stride < cols) return I8_ARG("%s: the stride of %s is less than cols", who, name);
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

static int quantize_launch(uint32_t type, const void *x, size_t x_stride, size_t n, size_t cols, const void *up, int8_t *q,
                           size_t q_stride, float *scale, hipStream_t st, const char *who)
{
    const dim3 grid((uint32_t)n), block(256);
#define OXH_QUANT(T)                                                                                                             \
    do {                                                                                                                         \
        if (up) hipLaunchKernelGGL((k_i8_quantize<T, true>), grid, block, 0, st, (const T *)x, x_stride, (uint32_t)cols,         \
                                   (const T *)up, q, q_stride, scale);                                                           \
        else hipLaunchKernelGGL((k_i8_quantize<T, false>), grid, block, 0, st, (const T *)x, x_stride, (uint32_t)cols,           \
                                (const T *)nullptr, q, q_stride, scale);                                                         \
    } while (0)
    if (type == OXH_F32) OXH_QUANT(float);
    else if (type == OXH_F16) OXH_QUANT(_Float16);
    else OXH_QUANT(__bf16);
#undef OXH_QUANT
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
    if (n_vec > I8_MAX_ROWS) return I8_ARG("%s: at most %zu rows per call", who, I8_MAX_ROWS);
    if ((rc = ready())) return rc;
    return quantize_launch(x_type, d_x, x_stride, n_vec, cols, d_up, d_q, q_stride, d_scale, stream_of(stream), who);
}

static int check_matrix(const char *who, const OxhI8Matrix *w)
{
    int rc;
    if (!w) return I8_ARG("%s: NULL matrix", who);
    if ((rc = check_cols(who, w->cols)) || (rc = check_rows(who, "the matrix", w->d_w, w->stride, w->cols))) return rc;
    if (!w->d_scale) return I8_ARG("%s: NULL pointer (the matrix's scales)", who);
    if (w->rows > I8_MAX_ROWS) return I8_ARG("%s: at most %zu rows", who, I8_MAX_ROWS);
    return OXH_OK;
}

static int matmul_launch(const OxhI8Matrix *w, const int8_t *q, size_t q_stride, const float *q_scale, size_t n, const float *bias,
                         uint32_t out_type, void *out, size_t out_stride, hipStream_t st, const char *who)
{
    for (size_t t0 = 0; t0 < n; t0 += 65535u * 16u) {
        const size_t here = n - t0 < 65535u * 16u ? n - t0 : 65535u * 16u;
        const dim3 grid((uint32_t)((w->rows + 63u) / 64u), (uint32_t)((here + 15u) / 16u)), block(256);
#define OXH_MM(T)                                                                                                                \
    hipLaunchKernelGGL(k_i8_matmul<T>, grid, block, 0, st, *w, q + t0 * q_stride, q_stride, q_scale + t0, (uint32_t)here, bias,  \
                       (T *)out + t0 * out_stride, out_stride)
        if (out_type == OXH_F32) OXH_MM(float);
        else if (out_type == OXH_F16) OXH_MM(_Float16);
        else OXH_MM(__bf16);
#undef OXH_MM
    }
    return launched(who);
}

extern "C" size_t oxh_i8_matmul_workspace(const OxhI8Matrix *w, size_t n_vec)
{
    (void)w;
    (void)n_vec;
    return 0;
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
    if (n_vec > I8_MAX_ROWS) return I8_ARG("%s: at most %zu tokens per call", who, I8_MAX_ROWS);
    if (d_workspace && workspace_bytes && ((uintptr_t)d_workspace & 15u)) return I8_ARG("%s: workspace must be 16-byte aligned", who);
    if ((rc = ready())) return rc;
    return matmul_launch(w, d_q, q_stride, d_q_scale, n_vec, d_bias, out_type, d_out, out_stride, stream_of(stream), who);
}

/* the codes and scales of the tokens */
struct LinearParts {
    size_t q_stride, q, scale, total;
};
static LinearParts linear_parts(size_t cols, size_t n)
{
    LinearParts p;
    p.q_stride = up64(cols);
    p.q = 0;
    p.scale = p.q_stride * n;
    p.total = p.scale + up16(4u * n);
    return p;
}

extern "C" size_t oxh_i8_linear_workspace(const OxhI8Matrix *w, size_t n_vec)
{
    return w && w->cols && w->cols <= OXH_I8_MAX_COLS && n_vec <= I8_MAX_ROWS ? linear_parts(w->cols, n_vec).total : 0;
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
    if (n_vec > I8_MAX_ROWS) return I8_ARG("%s: at most %zu tokens per call", who, I8_MAX_ROWS);
    const LinearParts p = linear_parts(w->cols, n_vec);
    if (!d_workspace || workspace_bytes < p.total) return I8_ARG("%s: workspace too small (see oxh_i8_linear_workspace)", who);
    if ((uintptr_t)d_workspace & 15u) return I8_ARG("%s: workspace must be 16-byte aligned", who);
    if ((rc = ready())) return rc;
    int8_t *q = (int8_t *)d_workspace;
    float *scale = (float *)((uint8_t *)d_workspace + p.scale);
    if ((rc = quantize_launch(x_type, d_x, x_stride, n_vec, w->cols, nullptr, q, p.q_stride, scale, stream_of(stream), who))) return rc;
    return matmul_launch(w, q, p.q_stride, scale, n_vec, d_bias, out_type, d_out, out_stride, stream_of(stream), who);
}

/* ─── experts ─────────────────────────────────────────────────────────── */

struct MoeI8Parts {
    size_t q_stride, h_stride, y_stride, qh_stride;    /* bytes, floats, floats, bytes */
    size_t q, q_scale, h, qh, qh_scale, y, total;
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
    size_t at = 0;
#define OXH_PART(FIELD, BYTES) p->FIELD = at; at = up256(at + (BYTES))
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
    if ((rc = quantize_launch(x_type, d_x, x_stride, n_tok, m->hidden, nullptr, q, p.q_stride, q_scale, st, who))) return rc;
    hipLaunchKernelGGL(k_i8_experts_up, dim3((uint32_t)((m->ffn + 63u) / 64u), (uint32_t)m->n_expert), dim3(256), 0, st, *m, *routing,
                       q, p.q_stride, q_scale, (uint32_t)n_tok, (uint32_t)pairs, h, p.h_stride);
    if ((rc = launched(who))) return rc;
    if ((rc = quantize_launch(OXH_F32, h, p.h_stride, pairs, m->ffn, nullptr, qh, p.qh_stride, qh_scale, st, who))) return rc;
    hipLaunchKernelGGL(k_i8_experts_down, dim3((uint32_t)((m->hidden + 63u) / 64u), (uint32_t)m->n_expert), dim3(256), 0, st, *m,
                       *routing, qh, p.qh_stride, qh_scale, (uint32_t)pairs, y, p.y_stride);
    if ((rc = launched(who))) return rc;
#define OXH_COMBINE(T)                                                                                                           \
    hipLaunchKernelGGL(k_i8_combine<T>, dim3((uint32_t)((m->hidden + 255u) / 256u), (uint32_t)n_tok), dim3(256), 0, st, y, p.y_stride, \
                       routing->d_weights, routing->d_slot_pos, (uint32_t)m->top_k, (uint32_t)pairs, (uint32_t)m->hidden,        \
                       (T *)d_out, out_stride)
    if (out_type == OXH_F32) OXH_COMBINE(float);
    else if (out_type == OXH_F16) OXH_COMBINE(_Float16);
    else OXH_COMBINE(__bf16);
#undef OXH_COMBINE
    return launched(who);
}
