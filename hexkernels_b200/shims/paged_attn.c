/* candidate_kernel for paged_attn on the B200 (libhexcuda), on one device. */
#include "hexcuda.h"
#include "kernel_api/paged_attn.h"
void candidate_kernel(int dtype, const uint16_t *q, const uint16_t *k_pages,
                      const uint16_t *v_pages, const int32_t *block_table, const int32_t *kv_lens,
                      const int32_t *q_offs, uint16_t *out, float *lse, int batch, int total_q,
                      int max_q, int heads, int kv_heads, int head_dim, int num_pages,
                      int page_size, int max_pages, float scale, int causal) {
    hexcuda_host_paged_attn(dtype, q, k_pages, v_pages, block_table, kv_lens, q_offs, out,
        lse, batch, total_q, max_q, heads, kv_heads, head_dim, num_pages, page_size,
        max_pages, scale, causal);
}
