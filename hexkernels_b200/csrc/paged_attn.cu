// paged_attn.cu -- attention of new tokens over a paged key / value cache,
// the entry point and the CUDA-core path.
//
//   out[r, h] = sum_j softmax_j(scale * q[r, h] . K[j]) V[j],
//   lse[r, h] = log sum_j exp(scale * q[r, h] . K[j])
//
// over the cached tokens j that the row sees (paged.cuh), K and V of query
// head h's key head h / (heads / kv_heads).  A row that sees nothing gets
// zeros and minus infinity.
#include <math.h>

#include "paged.cuh"

namespace hx {

int check_paged(const char *name, int dtype, const void *table, const void *kv_lens,
                const void *q_offs, int batch, int total_q, int max_q, int heads, int kv_heads,
                int head_dim, int num_pages, int page_size, int max_pages, float scale) {
    if (dtype != HEXCUDA_F16 && dtype != HEXCUDA_BF16)
        return fail(HEXCUDA_ERR_ARG, "%s: dtype %d", name, dtype);
    if (batch < 0 || total_q < 0 || max_q < 0)
        return fail(HEXCUDA_ERR_ARG, "%s: batch %d total_q %d max_q %d", name, batch, total_q,
                    max_q);
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads > 65535 || head_dim < 1 ||
        head_dim > 256)
        return fail(HEXCUDA_ERR_ARG,
                    "%s: heads %d kv_heads %d (a divisor) head_dim %d (1 to 256)", name, heads,
                    kv_heads, head_dim);
    if (num_pages < 1 || page_size < 1 || max_pages < 1 ||
        (int64_t)num_pages * page_size > 0x7fffffff || (int64_t)max_pages * page_size > 0x7fffffff)
        return fail(HEXCUDA_ERR_ARG, "%s: num_pages %d page_size %d max_pages %d", name, num_pages,
                    page_size, max_pages);
    if (!(scale > 0.0f) || isinf(scale))
        return fail(HEXCUDA_ERR_ARG, "%s: scale %g is not positive and finite", name,
                    (double)scale);
    if (batch > 0 && total_q > 0 && (!table || !kv_lens || !q_offs))
        return fail(HEXCUDA_ERR_ARG, "%s: null pointer", name);
    return HEXCUDA_OK;
}

namespace {

constexpr int kMaxD = 256;

// Any head size, page size and alignment: one warp per query row and head.
// Lane t scores key t of a run of 32, the warp reduces the run's maximum and
// sum with shuffles, and lane t accumulates output columns t, t + 32, ...
template <typename T>
__global__ void __launch_bounds__(128) paged_attn_any_kernel(
    const T *__restrict__ q, const T *__restrict__ kp, const T *__restrict__ vp,
    T *__restrict__ out, float *__restrict__ lse, const PagedSeqs s, int heads, int kv_heads,
    int dim, float scale) {
    __shared__ float sq[4][kMaxD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int b = blockIdx.y; b < s.batch; b += gridDim.y) {
      int first;
      const int q_len = seq_q_len(s, b, first), kv_len = seq_kv_len(s, b);
      const int64_t rows = (int64_t)q_len * heads;
      for (int64_t i = (int64_t)blockIdx.x * 4 + warp; i < rows; i += (int64_t)gridDim.x * 4) {
        const int64_t w = (int64_t)first * heads + i;
        const int h = (int)(i % heads);
        const int seen = seen_by(s, kv_len, q_len, (int)(i / heads));
        const int kvh = h / (heads / kv_heads);
        __syncwarp();
        for (int d = lane; d < dim; d += 32) sq[warp][d] = to_f32(q[w * dim + d]);
        __syncwarp();
        float acc[kMaxD / 32];
#pragma unroll
        for (int u = 0; u < kMaxD / 32; u++) acc[u] = 0.0f;
        float m = -INFINITY, l = 0.0f;
        for (int j0 = 0; j0 < seen; j0 += 32) {
            const int j = j0 + lane;
            int64_t row = -1;
            float x = -INFINITY;
            if (j < seen) {
                const int page = seq_page(s, b, j / s.page_size);
                if (page >= 0) {
                    row = ((int64_t)page * kv_heads + kvh) * s.page_size + j % s.page_size;
                    float a = 0.0f;
                    for (int d = 0; d < dim; d++) a += sq[warp][d] * to_f32(kp[row * dim + d]);
                    x = a * scale;
                }
            }
            float top = x;
            for (int o = 16; o > 0; o >>= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float m_new = fmaxf(m, top);
            const float ref = m_new == -INFINITY ? 0.0f : m_new;
            const float corr = expf(m - ref);
            const float p = row >= 0 ? expf(x - ref) : 0.0f;
            float sum = p;
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l = l * corr + sum;
#pragma unroll
            for (int u = 0; u < kMaxD / 32; u++) acc[u] *= corr;
            const int n = min(32, seen - j0);
            for (int e = 0; e < n; e++) {
                const float pe = __shfl_sync(0xffffffffu, p, e);
                const int64_t re = __shfl_sync(0xffffffffu, row, e);
                if (re < 0) continue;
#pragma unroll
                for (int u = 0; u < kMaxD / 32; u++) {
                    const int d = lane + 32 * u;
                    if (d < dim) acc[u] += pe * to_f32(vp[re * dim + d]);
                }
            }
            m = m_new;
        }
#pragma unroll
        for (int u = 0; u < kMaxD / 32; u++) {
            const int d = lane + 32 * u;
            // (a sum that is not a number divides too: only an empty row gives zeros)
            if (d < dim) out[w * dim + d] = from_f32<T>(l == 0.0f ? 0.0f : acc[u] / l);
        }
        if (lse && lane == 0) lse[w] = l == 0.0f ? -INFINITY : m + logf(l);
      }
    }
}

}  // namespace
}  // namespace hx

using namespace hx;

HX_EXPORT int hexcuda_paged_attn_workspace(int dev, size_t *bytes) {
    Dev *d = get_dev(dev);
    if (!d) return HEXCUDA_ERR_NODEV;
    if (!bytes) return fail(HEXCUDA_ERR_ARG, "paged_attn_workspace: null pointer");
    *bytes = 256;
    return HEXCUDA_OK;
}

HX_EXPORT int hexcuda_paged_attn(int dev, int dtype, const void *q, const void *k_pages,
                                 const void *v_pages, const int32_t *block_table,
                                 const int32_t *kv_lens, const int32_t *q_offs, void *out,
                                 float *lse, void *workspace, size_t workspace_bytes, int batch,
                                 int total_q, int max_q, int heads, int kv_heads, int head_dim,
                                 int num_pages, int page_size, int max_pages, float scale,
                                 int causal) {
    if (int rc = check_paged("paged_attn", dtype, block_table, kv_lens, q_offs, batch, total_q,
                             max_q, heads, kv_heads, head_dim, num_pages, page_size, max_pages,
                             scale))
        return rc;
    if (batch == 0 || total_q == 0) return HEXCUDA_OK;
    if (!q || !k_pages || !v_pages || !out || !workspace)
        return fail(HEXCUDA_ERR_ARG, "paged_attn: null pointer");
    Dev *d = get_dev(dev);
    if (!d) return HEXCUDA_ERR_NODEV;
    size_t need = 0;
    if (int rc = hexcuda_paged_attn_workspace(dev, &need)) return rc;
    if (workspace_bytes < need || ((uintptr_t)workspace & 15u))
        return fail(HEXCUDA_ERR_ARG,
                    "paged_attn: workspace of %zu bytes, %zu needed, 16-byte aligned",
                    workspace_bytes, need);
    PagedSeqs s{block_table, kv_lens, q_offs, batch, total_q, num_pages, page_size,
                max_pages, causal, d->err_word};
    launch_begin(d);
    const int ny = batch < 1024 ? batch : 1024;
    const dim3 grid((unsigned)((d->sms * 16 + ny - 1) / ny), (unsigned)ny);
    if (dtype == HEXCUDA_F16)
        paged_attn_any_kernel<__half><<<grid, 128, 0, d->stream>>>(
            (const __half *)q, (const __half *)k_pages, (const __half *)v_pages, (__half *)out, lse,
            s, heads, kv_heads, head_dim, scale);
    else
        paged_attn_any_kernel<__nv_bfloat16><<<grid, 128, 0, d->stream>>>(
            (const __nv_bfloat16 *)q, (const __nv_bfloat16 *)k_pages,
            (const __nv_bfloat16 *)v_pages, (__nv_bfloat16 *)out, lse, s, heads, kv_heads, head_dim,
            scale);
    return launch_end(d, "paged_attn");
}
