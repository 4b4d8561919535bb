/* candidate_kernel for cache_evict on the B200 (libhexcuda), on one device. */
#include "hexcuda.h"
#include "kernel_api/cache_evict.h"
void candidate_kernel(uint16_t *k_pages, uint16_t *v_pages, float *scores,
                      const int32_t *block_table, const int32_t *dst_table, const int32_t *kv_lens,
                      int32_t *new_lens, int32_t *kept, int batch, int kv_heads, int head_dim,
                      int num_pages, int page_size, int max_pages, int dst_max_pages, int budget,
                      int sink, int recent) {
    hexcuda_host_cache_evict(k_pages, v_pages, scores, block_table, dst_table, kv_lens,
        new_lens, kept, batch, kv_heads, head_dim, num_pages, page_size, max_pages,
        dst_max_pages, budget, sink, recent);
}
