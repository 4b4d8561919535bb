/* New task header: attention weight that cached tokens collect
 * (arguments as in hexcuda.h, on host memory; 16-bit heads as bit patterns,
 * dtype 0 binary16 and 1 bfloat16).  Sums the columns of
 * the softmax matrix that paged_attn leaves out. */
#ifndef HEXCUDA_KAPI_CACHE_SCORES_H
#define HEXCUDA_KAPI_CACHE_SCORES_H
#include <stdint.h>
void candidate_kernel(int dtype, const uint16_t *q, const float *lse, const uint16_t *k_pages,
                      const int32_t *block_table, const int32_t *kv_lens, const int32_t *q_offs,
                      float *scores, int batch, int total_q, int max_q, int heads, int kv_heads,
                      int head_dim, int num_pages, int page_size, int max_pages, float scale,
                      int causal);
#endif
