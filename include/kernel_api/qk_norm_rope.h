/* New task header: RMS norm and rotation of new tokens' query and key heads, keys and values
 * to their slots of a paged cache
 * (arguments as in hexcuda.h, on host memory; 16-bit heads as bit patterns,
 * dtype 0 binary16 and 1 bfloat16).  One token of
 * kernels/expert/rope_pair_fp16 and kernels/expert/kv_cache_update for a
 * ragged batch of 16-bit heads. */
#ifndef HEXCUDA_KAPI_QK_NORM_ROPE_H
#define HEXCUDA_KAPI_QK_NORM_ROPE_H
#include <stdint.h>
void candidate_kernel(int dtype, const uint16_t *q, int64_t q_stride, const uint16_t *k,
                      int64_t k_stride, const uint16_t *v, int64_t v_stride,
                      const uint16_t *q_gain, const uint16_t *k_gain, const float *cos_t,
                      const float *sin_t, const int32_t *positions, const int32_t *slots,
                      uint16_t *q_out, uint16_t *k_pages, uint16_t *v_pages, float *scores,
                      int tokens, int heads, int kv_heads, int head_dim, int rot_dim, int halves,
                      int norm, int table_len, int num_pages, int page_size, float eps);
#endif
