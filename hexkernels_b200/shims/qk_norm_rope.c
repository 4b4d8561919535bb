/* candidate_kernel for qk_norm_rope on the B200 (libhexcuda), on one device. */
#include "hexcuda.h"
#include "kernel_api/qk_norm_rope.h"
void candidate_kernel(int dtype, const uint16_t *q, int64_t q_stride, const uint16_t *k,
                      int64_t k_stride, const uint16_t *v, int64_t v_stride,
                      const uint16_t *q_gain, const uint16_t *k_gain, const float *cos_t,
                      const float *sin_t, const int32_t *positions, const int32_t *slots,
                      uint16_t *q_out, uint16_t *k_pages, uint16_t *v_pages, float *scores,
                      int tokens, int heads, int kv_heads, int head_dim, int rot_dim, int halves,
                      int norm, int table_len, int num_pages, int page_size, float eps) {
    hexcuda_host_qk_norm_rope(dtype, q, q_stride, k, k_stride, v, v_stride, q_gain,
        k_gain, cos_t, sin_t, positions, slots, q_out, k_pages, v_pages, scores, tokens,
        heads, kv_heads, head_dim, rot_dim, halves, norm, table_len, num_pages, page_size,
        eps);
}
