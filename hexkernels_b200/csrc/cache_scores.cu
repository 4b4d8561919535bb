// cache_scores.cu -- the attention weight that each cached token collects:
//
//   scores[slot(j), kvh] += sum over the new tokens r that see j, and over
//                           the query heads h of kvh, of
//                           exp(scale * q[r, h] . K[j] - lse[r, h])
//
// with lse from paged_attn.  A key's weights are summed in fp32 by one CTA
// in a fixed order and added to the cache's score once, so the result does
// not depend on scheduling unless two sequences share the key's page (their
// two additions then come in either order).
#include <math.h>

#include "paged_tc.cuh"

namespace hx {
namespace {

// Any head size, page size and alignment: one thread per key.
template <typename T>
__global__ void __launch_bounds__(128) cache_scores_any_kernel(
    const T *__restrict__ q, const float *__restrict__ lse, const T *__restrict__ kp,
    float *scores, const PagedSeqs s, int heads, int kv_heads, int dim, float scale, int tiles) {
    const int64_t n = (int64_t)s.batch * kv_heads * tiles;
    const int group = heads / kv_heads;
    for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
        const int tile = (int)(w % tiles);
        const int kvh = (int)(w / tiles % kv_heads), b = (int)(w / tiles / kv_heads);
        const int kv_len = seq_kv_len(s, b);
        const int j = tile * 128 + threadIdx.x;
        if (j >= kv_len) continue;
        int first;
        const int q_len = seq_q_len(s, b, first);
        const int page = seq_page(s, b, j / s.page_size);
        if (page < 0) continue;
        const int64_t row = ((int64_t)page * kv_heads + kvh) * s.page_size + j % s.page_size;
        // the first new token that sees key j
        int t0 = 0;
        if (s.causal) t0 = max(0, j - (kv_len - q_len));
        float sum = 0.0f;
        for (int t = t0; t < q_len; t++)
            for (int g = 0; g < group; g++) {
                const int64_t r = (int64_t)(first + t) * heads + kvh * group + g;
                const float z = lse[r];
                if (z == -INFINITY) continue;
                float a = 0.0f;
                for (int d = 0; d < dim; d++)
                    a += to_f32(q[r * dim + d]) * to_f32(kp[row * dim + d]);
                sum += expf(a * scale - z);
            }
        if (t0 < q_len) atomicAdd(&scores[row], sum);
    }
}

}  // namespace
}  // namespace hx

using namespace hx;

HX_EXPORT int hexcuda_cache_scores(int dev, int dtype, const void *q, const float *lse,
                                   const void *k_pages, const int32_t *block_table,
                                   const int32_t *kv_lens, const int32_t *q_offs, float *scores,
                                   int batch, int total_q, int max_q, int heads, int kv_heads,
                                   int head_dim, int num_pages, int page_size, int max_pages,
                                   float scale, int causal) {
    if (int rc = check_paged("cache_scores", dtype, block_table, kv_lens, q_offs, batch, total_q,
                             max_q, heads, kv_heads, head_dim, num_pages, page_size, max_pages,
                             scale))
        return rc;
    if (batch == 0 || total_q == 0) return HEXCUDA_OK;
    if (!q || !lse || !k_pages || !scores)
        return fail(HEXCUDA_ERR_ARG, "cache_scores: null pointer");
    Dev *d = get_dev(dev);
    if (!d) return HEXCUDA_ERR_NODEV;
    PagedSeqs s{block_table, kv_lens, q_offs, batch, total_q, num_pages, page_size,
                max_pages, causal, d->err_word};
    if (paged_tc_fits(q, k_pages, nullptr, nullptr, heads, kv_heads, head_dim, num_pages, page_size)) {
        launch_begin(d);
        if (int rc = launch_scores_tc(d, s, dtype, q, lse, k_pages, scores, max_q, heads, kv_heads,
                                      head_dim, scale))
            return rc;
        return launch_end(d, "cache_scores");
    }
    launch_begin(d);
    const int tiles = (int)(((int64_t)max_pages * page_size + 127) / 128);
    const int64_t items = (int64_t)batch * kv_heads * tiles;
    const int grid = (int)(items < (int64_t)d->sms * 16 ? items : (int64_t)d->sms * 16);
    if (dtype == HEXCUDA_F16)
        cache_scores_any_kernel<__half><<<grid, 128, 0, d->stream>>>(
            (const __half *)q, lse, (const __half *)k_pages, scores, s, heads, kv_heads, head_dim,
            scale, tiles);
    else
        cache_scores_any_kernel<__nv_bfloat16><<<grid, 128, 0, d->stream>>>(
            (const __nv_bfloat16 *)q, lse, (const __nv_bfloat16 *)k_pages, scores, s, heads,
            kv_heads, head_dim, scale, tiles);
    return launch_end(d, "cache_scores");
}
