// paged.cuh -- what the kernels of the paged key / value cache share: the
// cache's description, the 16-bit element types, and the checks of indices
// that live on the device (page numbers, lengths, row offsets).
//
// The cache: pages [num_pages][kv_heads][page_size][head_dim]; token j of
// sequence b lies in page table[b * max_pages + j / page_size] at offset
// j % page_size.  The new tokens of a call are rows q_offs[b] .. q_offs[b + 1]
// of q and the last ones of the sequence's kv_lens[b] cached tokens.
//
// The host cannot see those indices, so every kernel checks them before it
// uses them: what is out of range is skipped (clamped, for a length; taken for a
// page of zeros by the attention) and raises kErrIndex in the device's error word, which hexcuda_sync reports.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "hx_internal.h"

namespace hx {

struct PagedSeqs {
    const int *table, *kv_lens, *q_offs;
    int batch, total_q, num_pages, page_size, max_pages;
    int causal;
    int *err_word;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else if constexpr (std::is_same<T, __half>::value) return __half2float(x);
    else return __bfloat162float(x);
}
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
    if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}
// two values as one 32-bit word, the first in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value)
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
}

__device__ __forceinline__ void flag_index(int *err_word) { atomicOr(err_word, kErrIndex); }

// Cached tokens of sequence b, within what its row of the table can name.
__device__ __forceinline__ int seq_kv_len(const PagedSeqs &s, int b) {
    const int n = s.kv_lens[b];
    const long long cap = (long long)s.max_pages * s.page_size;
    if (n >= 0 && n <= cap) return n;
    flag_index(s.err_word);
    return n < 0 ? 0 : (int)cap;
}
// First row and number of the new tokens of sequence b; none when the offsets
// are not ascending or leave q.
__device__ __forceinline__ int seq_q_len(const PagedSeqs &s, int b, int &first) {
    first = s.q_offs[b];
    const int end = s.q_offs[b + 1];
    if (first >= 0 && end >= first && end <= s.total_q) return end - first;
    flag_index(s.err_word);
    first = 0;
    return 0;
}
// Page of a sequence's page number i (i * page_size < its cached tokens);
// -1, and the error word raised, when the table names none.
__device__ __forceinline__ int seq_page(const PagedSeqs &s, int b, int i) {
    const int p = s.table[(int64_t)b * s.max_pages + i];
    if (p >= 0 && p < s.num_pages) return p;
    flag_index(s.err_word);
    return -1;
}
// How many of the cached tokens new token t (of q_len) sees: all of them, or
// with the causal rule those up to its own place.
__device__ __forceinline__ int seen_by(const PagedSeqs &s, int kv_len, int q_len, int t) {
    if (!s.causal) return kv_len;
    const int n = kv_len - q_len + t + 1;
    return n < 0 ? 0 : n;
}

}  // namespace hx
