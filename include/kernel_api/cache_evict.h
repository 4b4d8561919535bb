/* New task header: cut the sequences of a paged cache to the tokens of the highest collected weight
 * (arguments as in hexcuda.h, on host memory; 16-bit heads as bit patterns,
 * dtype 0 binary16 and 1 bfloat16).  The
 * counterpart of kernels/expert/kv_cache_update: rows leave the cache. */
#ifndef HEXCUDA_KAPI_CACHE_EVICT_H
#define HEXCUDA_KAPI_CACHE_EVICT_H
#include <stdint.h>
void candidate_kernel(uint16_t *k_pages, uint16_t *v_pages, float *scores,
                      const int32_t *block_table, const int32_t *dst_table, const int32_t *kv_lens,
                      int32_t *new_lens, int32_t *kept, int batch, int kv_heads, int head_dim,
                      int num_pages, int page_size, int max_pages, int dst_max_pages, int budget,
                      int sink, int recent);
#endif
