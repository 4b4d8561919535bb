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
// HBM-bound: each row is read once and written once, 4 bytes a value.  Measured
// with 32 + 2 x 8 heads of 128: 16384 tokens 78 to 83 us from box to box for 411 MB, 5.0
// to 5.3 TB/s (a copy 6.5); one token 5 us on the device.
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
    int page_shift;         // log2 of page_size, or -1
    float eps;
    int *err_word;
};

// Where a token of this position and slot goes; false for one that is skipped
// (padding, or an index out of range, which is flagged).
__device__ __forceinline__ bool token_place(const NormRope &a, int pos, int slot, int64_t &page,
                                            int &off) {
    page = 0;
    off = 0;
    if (a.slots && slot < 0) return false;
    if (a.kv_heads > 0) {       // (without a cache any other slot marks a token that counts)
        page = a.page_shift >= 0 ? slot >> a.page_shift : slot / a.page_size;
        off = slot - (int)page * a.page_size;
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

// Packed pairs of 32-bit floats (one instruction for two).
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
template <typename T>
__device__ __forceinline__ void widen(const uint4 &w, uint64_t (&x)[4]) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = unpack2<T>(v[i]);
        x[i] = pair(f.x, f.y);
    }
}
template <typename T>
__device__ __forceinline__ uint4 narrow(const uint64_t (&x)[4]) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = unpair(x[i]);
        v[i] = pack2<T>(f.x, f.y);
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// Head sizes and rot_dim that are multiples of 16, 16-byte aligned rows: a block
// takes up to U passes of 128 / LPR rows of a token, LPR lanes a row (16 values a
// lane), all loads in flight together; blocks are short and many, so that those
// which load and those which compute overlap.  A lane's 16 values are two pieces
// of 8, chosen so that a pair never leaves the lane: columns 8c.. and rot/2 +
// 8c.. when halves turn together, 16c.. and 16c + 8.. otherwise; in both the
// lane's eight pairs are 8c .. 8c + 7.  What bounds it besides HBM is the number
// of instructions, a third of them the same for every warp of a token (its slot
// and pointers): hence the small block, 16 values a lane and 32-bit strides.
constexpr int U = 3;

constexpr int kWideThreads = 128;

template <typename T, int LPR, bool HALVES>
__global__ void __launch_bounds__(kWideThreads, 8) norm_rope_kernel(const NormRope a, int passes) {
    constexpr int kRows = kWideThreads / LPR;
    const int c = threadIdx.x % LPR, t = blockIdx.x;
    const int r0 = blockIdx.y * passes * kRows + threadIdx.x / LPR;
    const int k_end = a.heads + a.kv_heads, r_end = k_end + (a.v ? a.kv_heads : 0);
    const int pos = a.rot > 0 ? a.positions[t] : 0, slot = a.slots ? a.slots[t] : 0;
    const bool in_row = c * 16 < a.dim, turns = c * 16 < a.rot;
    const int o0 = turns && HALVES ? 8 * c : 16 * c;
    const int o1 = turns && HALVES ? a.rot / 2 + 8 * c : 16 * c + 8;
    // (strides and head offsets are below 2^31 here)
    const T *qs = (const T *)a.q + (int64_t)t * (int)a.q_stride;
    const T *ks = (const T *)a.k + (int64_t)t * (int)a.k_stride;
    const T *vs = (const T *)a.v + (int64_t)t * (int)a.v_stride;
    uint4 wx[U], wy[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int r = r0 + u * kRows;
        wx[u] = wy[u] = make_uint4(0, 0, 0, 0);
        if (u < passes && r < r_end && in_row && slot >= 0) {
            const T *p = (r < a.heads ? qs : r < k_end ? ks : vs) +
                         (r - (r < a.heads ? 0 : r < k_end ? a.heads : k_end)) * a.dim;
            wx[u] = *reinterpret_cast<const uint4 *>(p + o0);
            wy[u] = *reinterpret_cast<const uint4 *>(p + o1);
        }
    }
    int64_t page;
    int off;
    if (!token_place(a, pos, slot, page, off)) return;
    // (read where the lane's columns turn: a sine of 0 would not leave the others
    // alone, since 0 times an infinity is not 0)
    uint64_t cs[4] = {0, 0, 0, 0}, sn[4] = {0, 0, 0, 0};
    if (turns) {
        const int64_t o = (int64_t)pos * (a.rot / 2) + 8 * c;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float4 f = reinterpret_cast<const float4 *>(a.cos_t + o)[i];
            const float4 g = reinterpret_cast<const float4 *>(a.sin_t + o)[i];
            cs[2 * i] = pair(f.x, f.y);
            cs[2 * i + 1] = pair(f.z, f.w);
            sn[2 * i] = pair(g.x, g.y);
            sn[2 * i + 1] = pair(g.z, g.w);
        }
    }
    const int64_t kv_at = page * (int64_t)(a.kv_heads * a.page_size * a.dim) + off * a.dim;
    T *qd = (T *)a.q_out + (int64_t)t * (a.heads * a.dim);
    T *kd = (T *)a.k_pages + kv_at, *vd = (T *)a.v_pages + kv_at;
    const float inv_dim = 1.0f / (float)a.dim;
    const uint64_t minus = pair(-1.0f, -1.0f);
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (u >= passes) break;
        const int r = r0 + u * kRows;
        uint64_t x[4], y[4];
        widen<T>(wx[u], x);
        widen<T>(wy[u], y);
        float inv = 1.0f;
        if (a.norm) {
            uint64_t s2 = mul2(x[0], x[0]);
#pragma unroll
            for (int i = 1; i < 4; i++) s2 = fma2(x[i], x[i], s2);
#pragma unroll
            for (int i = 0; i < 4; i++) s2 = fma2(y[i], y[i], s2);
            const float2 s = unpair(s2);
            float sum = s.x + s.y;
            // (all lanes take part, also those past the row or the token)
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            inv = rsqrtf(fmaf(sum, inv_dim, a.eps));
        }
        if (r >= r_end || !in_row) continue;
        const bool is_q = r < a.heads;
        T *p = (is_q ? qd : r < k_end ? kd : vd) +
               (r - (is_q ? 0 : r < k_end ? a.heads : k_end)) * (is_q ? a.dim : a.page_size * a.dim);
        if (r < k_end) {
            const T *gain = (const T *)(is_q ? a.q_gain : a.k_gain);
            const uint64_t iv = pair(inv, inv);
            if (a.norm && gain) {
                uint64_t g[4], h[4];
                widen<T>(*reinterpret_cast<const uint4 *>(gain + o0), g);
                widen<T>(*reinterpret_cast<const uint4 *>(gain + o1), h);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[i] = mul2(x[i], mul2(iv, g[i]));
                    y[i] = mul2(y[i], mul2(iv, h[i]));
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    x[i] = mul2(x[i], iv);
                    y[i] = mul2(y[i], iv);
                }
            }
            if (!turns) {
                // (y as it is)
            } else if (HALVES) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint64_t f = x[i];
                    x[i] = fma2(f, cs[i], mul2(mul2(y[i], sn[i]), minus));
                    y[i] = fma2(f, sn[i], mul2(y[i], cs[i]));
                }
            } else {
                auto turn = [](uint64_t &v, float co, float si) {
                    const float2 f = unpair(v);
                    v = pair(f.x * co - f.y * si, f.x * si + f.y * co);
                };
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 c0 = unpair(cs[i / 2]), s0 = unpair(sn[i / 2]);
                    const float2 c1 = unpair(cs[2 + i / 2]), s1 = unpair(sn[2 + i / 2]);
                    turn(x[i], i & 1 ? c0.y : c0.x, i & 1 ? s0.y : s0.x);
                    turn(y[i], i & 1 ? c1.y : c1.x, i & 1 ? s1.y : s1.x);
                }
            }
            wx[u] = narrow<T>(x);
            wy[u] = narrow<T>(y);
            if (a.scores && !is_q && c == 0)
                a.scores[(page * a.kv_heads + (r - a.heads)) * a.page_size + off] = 0.0f;
        }
        *reinterpret_cast<uint4 *>(p + o0) = wx[u];
        *reinterpret_cast<uint4 *>(p + o1) = wy[u];
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

// Whether the tensors and strides allow the 16-byte accesses above.
bool wide_rows(const NormRope &a) {
    const uintptr_t p = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out |
                        (uintptr_t)a.k_pages | (uintptr_t)a.v_pages | (uintptr_t)a.q_gain |
                        (uintptr_t)a.k_gain | (uintptr_t)a.cos_t | (uintptr_t)a.sin_t;
    const int64_t strides = (a.heads ? a.q_stride : 0) | (a.kv_heads ? a.k_stride : 0) |
                            (a.v ? a.v_stride : 0);
    // (strides and offsets between heads are 32-bit there)
    if (((int64_t)a.heads + a.kv_heads * (int64_t)a.page_size) * a.dim > 0x7fffffff ||
        a.q_stride > 0x7fffffff || a.k_stride > 0x7fffffff || a.v_stride > 0x7fffffff)
        return false;
    return a.dim % 16 == 0 && a.rot % 16 == 0 && strides % 8 == 0 && p % 16 == 0;
}

template <typename T, int LPR, bool HALVES>
void launch_wide(Dev *d, const NormRope &a) {
    const int rows = a.heads + a.kv_heads * (a.v ? 2 : 1);
    constexpr int kRows = kWideThreads / LPR;
    const int all = (rows + kRows - 1) / kRows;
    // few tokens: a block per pass, so that a token's rows go out at once (16 and 64
    // tokens 8.2 us, with U passes a block 10.2; 4096 tokens 34.9 and 28.7, from 253
    // to 1200 the same; L2 flushed)
    const int passes = a.tokens < 4 * d->sms ? 1 : all < U ? all : U;
    const dim3 grid((unsigned)a.tokens, (unsigned)((all + passes - 1) / passes));
    norm_rope_kernel<T, LPR, HALVES><<<grid, kWideThreads, 0, d->stream>>>(a, passes);
}
template <typename T, int LPR>
void launch_halves(Dev *d, const NormRope &a) {
    if (a.halves)
        launch_wide<T, LPR, true>(d, a);
    else
        launch_wide<T, LPR, false>(d, a);
}
template <typename T>
void launch_norm_rope(Dev *d, const NormRope &a) {
    if (!wide_rows(a)) {
        constexpr auto kern = norm_rope_any_kernel<T>;
        const int64_t rows = (int64_t)a.tokens * (a.heads + a.kv_heads * (a.v ? 2 : 1));
        kern<<<resident_blocks<kern>(d, rows * 32), 256, 0, d->stream>>>(a);
    } else if (a.dim <= 64) {
        launch_halves<T, 4>(d, a);
    } else if (a.dim <= 128) {
        launch_halves<T, 8>(d, a);
    } else {
        launch_halves<T, 16>(d, a);
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
    if ((int64_t)heads + 2 * (int64_t)kv_heads > (1 << 16))
        return fail(HEXCUDA_ERR_ARG, "%s: heads %d kv_heads %d", name, heads, kv_heads);
    Dev *d = get_dev(dev);
    if (!d) return HEXCUDA_ERR_NODEV;
    const int64_t row = (int64_t)heads * head_dim, kv_row = (int64_t)kv_heads * head_dim;
    const int64_t last = tokens - 1;
    if ((overlap16(q_out, tokens * row, q, last * q_stride + row) &&
         !(q_out == q && (tokens == 1 || q_stride == row))) ||
        (kv_row > 0 && (overlap16(q_out, tokens * row, k, last * k_stride + kv_row) ||
                        overlap16(q_out, tokens * row, v, last * v_stride + kv_row))))
        return fail(HEXCUDA_ERR_ARG, "%s: q_out overlaps an input and is not q in its layout", name);
    if (overlap16(k_pages, num_pages * kv_row * page_size, v_pages, num_pages * kv_row * page_size))
        return fail(HEXCUDA_ERR_ARG, "%s: k_pages and v_pages overlap", name);
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
    a.page_shift = -1;
    for (int i = 0; i < 31; i++)
        if (page_size == 1 << i) a.page_shift = i;
    a.eps = eps;
    a.err_word = d->err_word;
    launch_begin(d);
    if (dtype == HEXCUDA_F16)
        launch_norm_rope<__half>(d, a);
    else
        launch_norm_rope<__nv_bfloat16>(d, a);
    return launch_end(d, name);
}
