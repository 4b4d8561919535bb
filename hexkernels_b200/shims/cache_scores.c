/* candidate_kernel for cache_scores on the B200 (libhexcuda), on one device. */
#include "hexcuda.h"
#include "kernel_api/cache_scores.h"
void candidate_kernel(int dtype, const uint16_t *q, const float *lse, const uint16_t *k_pages,
                      const int32_t *block_table, const int32_t *kv_lens, const int32_t *q_offs,
                      float *scores, int batch, int total_q, int max_q, int heads, int kv_heads,
                      int head_dim, int num_pages, int page_size, int max_pages, float scale,
                      int causal) {
    hexcuda_host_cache_scores(dtype, q, lse, k_pages, block_table, kv_lens, q_offs,
        scores, batch, total_q, max_q, heads, kv_heads, head_dim, num_pages, page_size,
        max_pages, scale, causal);
}
