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

// Position and slot of a token; false for a token that is skipped (padding,
// or an index out of range, which is flagged).
__device__ __forceinline__ bool token_place(const NormRope &a, int t, int &pos, int64_t &page,
                                            int &off) {
    pos = a.rot > 0 ? a.positions[t] : 0;
    page = 0;
    off = 0;
    if (a.slots) {
        const int slot = a.slots[t];
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
        int pos, off;
        int64_t page;
        if (!token_place(a, t, pos, page, off)) continue;
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
    const int64_t rows = (int64_t)tokens * (heads + kv_heads * (a.v ? 2 : 1));
    if (dtype == HEXCUDA_F16) {
        constexpr auto kern = norm_rope_any_kernel<__half>;
        kern<<<resident_blocks<kern>(d, rows * 32), 256, 0, d->stream>>>(a);
    } else {
        constexpr auto kern = norm_rope_any_kernel<__nv_bfloat16>;
        kern<<<resident_blocks<kern>(d, rows * 32), 256, 0, d->stream>>>(a);
    }
    return launch_end(d, name);
}
