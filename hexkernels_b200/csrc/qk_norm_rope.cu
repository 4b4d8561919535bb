// qk_norm_rope.cu -- new tokens on their way into the attention layer: RMS
// norm of every query and key head, rotation by the token's position, queries
// to a dense array, keys and values to their slots of the paged cache, in one
// pass over the projection's output.
//
//   y = x * rsqrt(mean(x^2) + eps) * gain      (per head; norm = 0: y = x)
//   (a, b) -> (a c - b s, a s + b c)           for each pair of y's first
//                                              rot_dim columns, c and s from
//                                              row position of the tables
//
// Everything between the load and the one rounding at the store is fp32.
// HBM-bound: each row is read once and written once, 4 bytes a value.
#include "ew_launch.cuh"
#include "paged.cuh"

namespace hx {
namespace {

constexpr int kMaxD = 256;

struct NormRope {
    const void *q, *k, *v, *q_gain, *k_gain;
    int64_t q_stride, k_stride, v_stride;
    const float *cos_t, *sin_t;
    const int *positions, *slots;
    void *q_out, *k_pages, *v_pages;
    float *scores;
    int tokens, heads, kv_heads, dim, rot, halves, norm, table_len;
    int num_pages, page_size;
    float eps;
    int *err_word;
};

// Where a token of this position and slot goes; false for one that is skipped
// (padding, or an index out of range, which is flagged).
__device__ __forceinline__ bool token_place(const NormRope &a, int pos, int slot, int64_t &page,
                                            int &off) {
    page = 0;
    off = 0;
    if (a.slots) {
        if (slot < 0) return false;
        page = slot / a.page_size;
        off = slot % a.page_size;
        if (page >= a.num_pages) {
            flag_index(a.err_word);
            return false;
        }
    }
    if (a.rot > 0 && (pos < 0 || pos >= a.table_len)) {
        flag_index(a.err_word);
        return false;
    }
    return true;
}

// Rows of a token: its query heads, its key heads, its value heads.
template <typename T>
__device__ __forceinline__ const T *row_source(const NormRope &a, int t, int r) {
    if (r < a.heads) return (const T *)a.q + (int64_t)t * a.q_stride + (int64_t)r * a.dim;
    r -= a.heads;
    if (r < a.kv_heads) return (const T *)a.k + (int64_t)t * a.k_stride + (int64_t)r * a.dim;
    return (const T *)a.v + (int64_t)t * a.v_stride + (int64_t)(r - a.kv_heads) * a.dim;
}
template <typename T>
__device__ __forceinline__ T *row_target(const NormRope &a, int t, int r, int64_t page, int off) {
    if (r < a.heads) return (T *)a.q_out + ((int64_t)t * a.heads + r) * a.dim;
    r -= a.heads;
    T *pages = r < a.kv_heads ? (T *)a.k_pages : (T *)a.v_pages;
    if (r >= a.kv_heads) r -= a.kv_heads;
    return pages + ((page * a.kv_heads + r) * a.page_size + off) * a.dim;
}

// Four values as 32-bit floats, and back.
template <typename T>
__device__ __forceinline__ void widen(uint2 w, float (&x)[4]) {
    const float2 a = unpack2<T>(w.x), b = unpack2<T>(w.y);
    x[0] = a.x;
    x[1] = a.y;
    x[2] = b.x;
    x[3] = b.y;
}
template <typename T>
__device__ __forceinline__ uint2 narrow(const float (&x)[4]) {
    return make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
}

// Head sizes that are multiples of 8, 8-byte aligned rows: LPR lanes a row (8
// values a lane), 256 / LPR rows at a time, every thread in the same columns
// of all its rows, so that a token's cosines and sines and the gains are read
// once.  A lane's 8 values are two pieces of 4 chosen so that a pair never
// leaves the lane: columns 4c.. and rot/2 + 4c.. when halves turn together,
// 8c.. and 8c + 4.. otherwise; in both the lane's four pairs are 4c .. 4c + 3.
// `ysplit` blocks share a token when tokens are few.
template <typename T, int LPR>
__global__ void __launch_bounds__(256, 4) norm_rope_kernel(const NormRope a, int ysplit) {
    constexpr int kRows = 256 / LPR, U = 4;
    const int c = threadIdx.x % LPR, slot = threadIdx.x / LPR;
    const int per_token = a.heads + a.kv_heads * (a.v ? 2 : 1);
    const bool in_row = c * 8 < a.dim, turns = c * 8 < a.rot;
    const int o0 = turns && a.halves ? 4 * c : 8 * c;
    const int o1 = turns && a.halves ? a.rot / 2 + 4 * c : 8 * c + 4;
    // the gains of this lane's columns, as they are stored
    uint2 gq0, gq1, gk0, gk1;
    const uint2 ones = make_uint2(pack2<T>(1.0f, 1.0f), pack2<T>(1.0f, 1.0f));
    auto gain_of = [&](const void *g, uint2 &x, uint2 &y) {
        x = y = ones;
        if (g && a.norm && in_row) {
            x = *reinterpret_cast<const uint2 *>((const T *)g + o0);
            y = *reinterpret_cast<const uint2 *>((const T *)g + o1);
        }
    };
    gain_of(a.q_gain, gq0, gq1);
    gain_of(a.k_gain, gk0, gk1);
    const float inv_dim = 1.0f / (float)a.dim;
    const int64_t items = (int64_t)a.tokens * ysplit;
    const int step = kRows * ysplit;
    // a token's position and slot, fetched while the token before it is worked on
    auto fetch = [&](int64_t item, int &pos, int &at) {
        const int t = (int)(item / ysplit);
        pos = a.rot > 0 ? a.positions[t] : 0;
        at = a.slots ? a.slots[t] : 0;
    };
    int pos_next = 0, slot_next = 0;
    if ((int64_t)blockIdx.x < items) fetch(blockIdx.x, pos_next, slot_next);
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int t = (int)(item / ysplit), pos = pos_next, at = slot_next;
        if (item + gridDim.x < items) fetch(item + gridDim.x, pos_next, slot_next);
        int64_t page;
        int off;
        if (!token_place(a, pos, at, page, off)) continue;
        float4 cs = make_float4(1.0f, 1.0f, 1.0f, 1.0f), sn = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (turns) {
            cs = *reinterpret_cast<const float4 *>(a.cos_t + (int64_t)pos * (a.rot / 2) + 4 * c);
            sn = *reinterpret_cast<const float4 *>(a.sin_t + (int64_t)pos * (a.rot / 2) + 4 * c);
        }
        const float cv[4] = {cs.x, cs.y, cs.z, cs.w}, sv[4] = {sn.x, sn.y, sn.z, sn.w};
        // (rows of one warp may end at different passes; all lanes stay for the shuffles)
        for (int r0 = (int)(item % ysplit) * kRows; r0 < per_token; r0 += U * step) {
            uint2 w0[U], w1[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int r = r0 + u * step + slot;
                w0[u] = w1[u] = make_uint2(0, 0);
                if (r < per_token && in_row) {
                    const T *src = row_source<T>(a, t, r);
                    w0[u] = *reinterpret_cast<const uint2 *>(src + o0);
                    w1[u] = *reinterpret_cast<const uint2 *>(src + o1);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int r = r0 + u * step + slot;
                if (r0 + u * step >= per_token) break;
                float x[4], y[4];
                widen<T>(w0[u], x);
                widen<T>(w1[u], y);
                float inv = 1.0f;
                if (a.norm) {
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; i++) sum += x[i] * x[i] + y[i] * y[i];
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    inv = rsqrtf(sum * inv_dim + a.eps);
                }
                if (r >= per_token || !in_row) continue;
                T *dst = row_target<T>(a, t, r, page, off);
                if (r < a.heads + a.kv_heads) {
                    const bool is_q = r < a.heads;
                    float g0[4], g1[4];
                    widen<T>(is_q ? gq0 : gk0, g0);
                    widen<T>(is_q ? gq1 : gk1, g1);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        x[i] *= inv * g0[i];
                        y[i] *= inv * g1[i];
                    }
                    if (a.halves) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float p = x[i], q = y[i];
                            x[i] = p * cv[i] - q * sv[i];
                            y[i] = p * sv[i] + q * cv[i];
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; i += 2) {
                            const float p = x[i], q = x[i + 1], e = y[i], f = y[i + 1];
                            x[i] = p * cv[i / 2] - q * sv[i / 2];
                            x[i + 1] = p * sv[i / 2] + q * cv[i / 2];
                            y[i] = e * cv[2 + i / 2] - f * sv[2 + i / 2];
                            y[i + 1] = e * sv[2 + i / 2] + f * cv[2 + i / 2];
                        }
                    }
                    w0[u] = narrow<T>(x);
                    w1[u] = narrow<T>(y);
                    if (a.scores && !is_q && c == 0)
                        a.scores[(page * a.kv_heads + (r - a.heads)) * a.page_size + off] = 0.0f;
                }
                *reinterpret_cast<uint2 *>(dst + o0) = w0[u];
                *reinterpret_cast<uint2 *>(dst + o1) = w1[u];
            }
        }
    }
}

// Any head size up to 256, any alignment: one warp per row, the row in shared
// memory for its partner columns.
template <typename T>
__global__ void __launch_bounds__(256) norm_rope_any_kernel(const NormRope a) {
    __shared__ float rows[8][kMaxD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_token = a.heads + a.kv_heads * (a.v ? 2 : 1);
    const int64_t n = (int64_t)a.tokens * per_token;
    float *x = rows[warp];
    for (int64_t w = (int64_t)blockIdx.x * 8 + warp; w < n; w += (int64_t)gridDim.x * 8) {
        const int t = (int)(w / per_token), r = (int)(w % per_token);
        const int pos = a.rot > 0 ? a.positions[t] : 0;
        int off;
        int64_t page;
        if (!token_place(a, pos, a.slots ? a.slots[t] : 0, page, off)) continue;
        const T *src = row_source<T>(a, t, r);
        T *dst = row_target<T>(a, t, r, page, off);
        if (r >= a.heads + a.kv_heads) {
            for (int i = lane; i < a.dim; i += 32) dst[i] = src[i];
            continue;
        }
        const T *gain = (const T *)(r < a.heads ? a.q_gain : a.k_gain);
        float sum = 0.0f;
        for (int i = lane; i < a.dim; i += 32) {
            x[i] = to_f32(src[i]);
            sum += x[i] * x[i];
        }
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (a.norm) {
            const float inv = rsqrtf(sum / (float)a.dim + a.eps);
            for (int i = lane; i < a.dim; i += 32)
                x[i] = x[i] * inv * (gain ? to_f32(gain[i]) : 1.0f);
        }
        __syncwarp();
        const int half = a.rot / 2;
        for (int i = lane; i < a.dim; i += 32) {
            float y = x[i];
            if (i < a.rot) {
                const int p = a.halves ? (i < half ? i : i - half) : i >> 1;
                const bool first = a.halves ? i < half : (i & 1) == 0;
                const float other = a.halves ? x[first ? i + half : i - half] : x[i ^ 1];
                const float c = a.cos_t[(int64_t)pos * half + p];
                const float s = a.sin_t[(int64_t)pos * half + p];
                y = first ? y * c - other * s : other * s + y * c;
            }
            dst[i] = from_f32<T>(y);
        }
        if (a.scores && r >= a.heads && lane == 0)
            a.scores[(page * a.kv_heads + (r - a.heads)) * a.page_size + off] = 0.0f;
        __syncwarp();
    }
}

// Whether the tensors and strides allow the 8- and 16-byte accesses above.
bool wide_rows(const NormRope &a) {
    const uintptr_t p8 = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out |
                         (uintptr_t)a.k_pages | (uintptr_t)a.v_pages | (uintptr_t)a.q_gain |
                         (uintptr_t)a.k_gain;
    const uintptr_t p16 = (uintptr_t)a.cos_t | (uintptr_t)a.sin_t;
    const int64_t strides = (a.heads ? a.q_stride : 0) | (a.kv_heads ? a.k_stride : 0) |
                            (a.v ? a.v_stride : 0);
    return a.dim % 8 == 0 && a.rot % 8 == 0 && strides % 4 == 0 && p8 % 8 == 0 &&
           (a.rot == 0 || p16 % 16 == 0);
}

template <typename T, int LPR>
void launch_wide(Dev *d, const NormRope &a) {
    constexpr auto kern = norm_rope_kernel<T, LPR>;
    const int rows = a.heads + a.kv_heads * (a.v ? 2 : 1);
    const int passes = (rows + 256 / LPR - 1) / (256 / LPR);
    // few tokens: a block per pass, so that a token's rows go out at once
    const int ysplit = a.tokens < 4 * d->sms ? passes : 1;
    kern<<<resident_blocks<kern>(d, (int64_t)a.tokens * ysplit * 256), 256, 0, d->stream>>>(a, ysplit);
}
template <typename T>
void launch_rows(Dev *d, const NormRope &a) {
    if (!wide_rows(a)) {
        constexpr auto kern = norm_rope_any_kernel<T>;
        const int64_t rows = (int64_t)a.tokens * (a.heads + a.kv_heads * (a.v ? 2 : 1));
        kern<<<resident_blocks<kern>(d, rows * 32), 256, 0, d->stream>>>(a);
    } else if (a.dim <= 64) {
        launch_wide<T, 8>(d, a);
    } else if (a.dim <= 128) {
        launch_wide<T, 16>(d, a);
    } else {
        launch_wide<T, 32>(d, a);
    }
}

}  // namespace
}  // namespace hx

using namespace hx;

HX_EXPORT int hexcuda_qk_norm_rope(int dev, int dtype, const void *q, int64_t q_stride,
                                   const void *k, int64_t k_stride, const void *v,
                                   int64_t v_stride, const void *q_gain, const void *k_gain,
                                   const float *cos_t, const float *sin_t,
                                   const int32_t *positions, const int32_t *slots, void *q_out,
                                   void *k_pages, void *v_pages, float *scores, int tokens,
                                   int heads, int kv_heads, int head_dim, int rot_dim, int halves,
                                   int norm, int table_len, int num_pages, int page_size,
                                   float eps) {
    const char *name = "qk_norm_rope";
    if (dtype != HEXCUDA_F16 && dtype != HEXCUDA_BF16)
        return fail(HEXCUDA_ERR_ARG, "%s: dtype %d", name, dtype);
    if (tokens < 0 || heads < 0 || kv_heads < 0 || head_dim < 1 || head_dim > kMaxD)
        return fail(HEXCUDA_ERR_ARG, "%s: tokens %d heads %d kv_heads %d head_dim %d (1 to %d)",
                    name, tokens, heads, kv_heads, head_dim, kMaxD);
    if (rot_dim < 0 || rot_dim > head_dim || rot_dim % 2 != 0 || (rot_dim > 0 && table_len < 1))
        return fail(HEXCUDA_ERR_ARG, "%s: rot_dim %d of head_dim %d, table_len %d", name, rot_dim,
                    head_dim, table_len);
    if (norm && !(eps >= 0.0f)) return fail(HEXCUDA_ERR_ARG, "%s: eps %g", name, (double)eps);
    if (tokens == 0 || heads + (int64_t)kv_heads == 0) return HEXCUDA_OK;
    if ((heads > 0 && (!q || !q_out)) || (rot_dim > 0 && (!cos_t || !sin_t || !positions)) ||
        (kv_heads > 0 && (!k || !k_pages || !slots || !v != !v_pages)))
        return fail(HEXCUDA_ERR_ARG, "%s: null pointer", name);
    if ((heads > 0 && q_stride < (int64_t)heads * head_dim) ||
        (kv_heads > 0 && (k_stride < (int64_t)kv_heads * head_dim ||
                          (v && v_stride < (int64_t)kv_heads * head_dim))))
        return fail(HEXCUDA_ERR_ARG, "%s: a row stride is shorter than its heads", name);
    if (kv_heads > 0 &&
        (num_pages < 1 || page_size < 1 || (int64_t)num_pages * page_size > 0x7fffffff))
        return fail(HEXCUDA_ERR_ARG, "%s: num_pages %d page_size %d", name, num_pages, page_size);
    if ((int64_t)heads + 2 * (int64_t)kv_heads > (1 << 20))
        return fail(HEXCUDA_ERR_ARG, "%s: heads %d kv_heads %d", name, heads, kv_heads);
    Dev *d = get_dev(dev);
    if (!d) return HEXCUDA_ERR_NODEV;
    NormRope a;
    a.q = q;
    a.k = k;
    a.v = kv_heads > 0 ? v : nullptr;
    a.q_gain = q_gain;
    a.k_gain = k_gain;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.positions = positions;
    a.slots = slots;
    a.q_out = q_out;
    a.k_pages = k_pages;
    a.v_pages = v_pages;
    a.scores = kv_heads > 0 ? scores : nullptr;
    a.tokens = tokens;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.dim = head_dim;
    a.rot = rot_dim;
    a.halves = halves;
    a.norm = norm;
    a.table_len = table_len;
    a.num_pages = num_pages;
    a.page_size = page_size;
    a.eps = eps;
    a.err_word = d->err_word;
    launch_begin(d);
    if (dtype == HEXCUDA_F16)
        launch_rows<__half>(d, a);
    else
        launch_rows<__nv_bfloat16>(d, a);
    return launch_end(d, name);
}
