/* New task header: attention of new tokens over a paged key / value cache
 * (arguments as in hexcuda.h, on host memory; 16-bit heads as bit patterns,
 * dtype 0 binary16 and 1 bfloat16).  Generalises
 * kernels/expert/fp16_flash_attention_tile/kernel_api.h:12-42 (one head, SK <=
 * 64) to shared key heads, ragged batches and a paged cache. */
#ifndef HEXCUDA_KAPI_PAGED_ATTN_H
#define HEXCUDA_KAPI_PAGED_ATTN_H
#include <stdint.h>
void candidate_kernel(int dtype, const uint16_t *q, const uint16_t *k_pages,
                      const uint16_t *v_pages, const int32_t *block_table, const int32_t *kv_lens,
                      const int32_t *q_offs, uint16_t *out, float *lse, int batch, int total_q,
                      int max_q, int heads, int kv_heads, int head_dim, int num_pages,
                      int page_size, int max_pages, float scale, int causal);
#endif
