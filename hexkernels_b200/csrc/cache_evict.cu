// cache_evict.cu -- cut every sequence of a paged cache to at most `budget`
// tokens: its first `sink`, its last `recent`, and between them those with the
// highest collected weight (cache_scores), for each key head on its own.
// What stays keeps its order and moves to the front of the sequence's pages
// (or of other pages); which tokens stayed is written to `kept`.
//
// Two launches: the choice (one CTA per sequence and key head, a radix select
// on the scores' bits and a prefix sum in index order, so ties go to the
// lowest index), then the move of K, V and score rows.
#include <math.h>

#include "paged.cuh"

namespace hx {
namespace {

struct Evict {
    void *k_pages, *v_pages;
    float *scores;
    const int *table, *dst_table, *kv_lens;
    int *new_lens, *kept;
    int batch, kv_heads, dim, num_pages, page_size, max_pages, dst_max_pages;
    int budget, sink, recent;
    int *err_word;
};

__device__ __forceinline__ int evict_len(const Evict &a, int b) {
    const int n = a.kv_lens[b];
    const long long cap = (long long)a.max_pages * a.page_size;
    if (n >= 0 && n <= cap) return n;
    flag_index(a.err_word);
    return n < 0 ? 0 : (int)cap;
}
__device__ __forceinline__ int evict_page(const Evict &a, const int *table, int width, int b,
                                          int i) {
    const int p = table[(int64_t)b * width + i];
    if (p >= 0 && p < a.num_pages) return p;
    flag_index(a.err_word);
    return -1;
}

// Order of the scores as unsigned integers: not-a-number lowest, then minus
// infinity up to infinity, the two zeros equal.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (isnan(x)) return 0u;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;

__device__ __forceinline__ uint32_t score_key(const Evict &a, int b, int h, int j) {
    const int page = evict_page(a, a.table, a.max_pages, b, j / a.page_size);
    if (page < 0) return 0u;
    return order_key(
        a.scores[((int64_t)page * a.kv_heads + h) * a.page_size + j % a.page_size]);
}

// Exclusive prefix sum over the block of two packed counts (16 bits each fit
// 1024 threads); returns this thread's, and the block's total in `total`.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *warp_sums, uint32_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        uint32_t y = warp_sums[lane];
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        warp_sums[lane] = y;
    }
    __syncthreads();
    total = warp_sums[31];
    return x - v + (warp > 0 ? warp_sums[warp - 1] : 0u);
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const Evict a) {
    __shared__ int hist[256];
    __shared__ uint32_t warp_sums[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_left;
    const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads;
    const int n = evict_len(a, b);
    int *kept = a.kept + (int64_t)blockIdx.x * a.budget;
    const int m = min(n, a.budget);
    for (int j = m + threadIdx.x; j < a.budget; j += kSelThreads) kept[j] = -1;
    if (n <= a.budget) {
        for (int j = threadIdx.x; j < n; j += kSelThreads) kept[j] = j;
        return;
    }
    // the sinks and the recent ones stay whatever their weight
    const int lo = a.sink, hi = n - a.recent;
    const int want = a.budget - a.sink - a.recent;
    for (int j = threadIdx.x; j < a.sink; j += kSelThreads) kept[j] = j;
    for (int j = threadIdx.x; j < a.recent; j += kSelThreads)
        kept[a.budget - a.recent + j] = hi + j;
    if (want == 0) return;
    // the want-th highest key, byte by byte from the top
    uint32_t prefix = 0, mask = 0;
    int left = want;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (int j = lo + threadIdx.x; j < hi; j += kSelThreads) {
            const uint32_t key = score_key(a, b, h, j);
            if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int bin = 255, rest = left;
            while (bin > 0 && hist[bin] < rest) rest -= hist[bin--];
            s_prefix = prefix | (uint32_t)bin << shift;
            s_left = rest;
        }
        __syncthreads();
        prefix = s_prefix;
        left = s_left;
        mask |= 255u << shift;
        __syncthreads();
    }
    // in index order: every key above it, and the first `left` equal to it
    int above = 0, equal = 0;
    for (int j0 = lo; j0 < hi; j0 += kSelThreads) {
        const int j = j0 + threadIdx.x;
        uint32_t flags = 0;
        if (j < hi) {
            const uint32_t key = score_key(a, b, h, j);
            flags = key > prefix ? 1u : key == prefix ? 0x10000u : 0u;
        }
        uint32_t total;
        const uint32_t before = block_scan(flags, warp_sums, total);
        const int eq = equal + (int)(before >> 16);
        const int at = above + (int)(before & 0xffffu) + min(eq, left);
        if (flags == 1u || (flags != 0 && eq < left)) kept[a.sink + at] = j;
        above += (int)(total & 0xffffu);
        equal += (int)(total >> 16);
    }
}

// One CTA per sequence, key head, tensor (K, V, scores) and column slice.  Kept
// token i comes from place kept[i] >= i, so the rows are moved in ascending
// chunks: a chunk's rows are all read before any of them is written, and no
// later chunk reads what an earlier one wrote, also when the target pages are
// the source's.
template <typename W>
__global__ void __launch_bounds__(256) evict_move_kernel(const Evict a, int row_words, int slices) {
    const int parts = 2 * slices + 1;
    const int part = blockIdx.x % parts;
    const int bh = blockIdx.x / parts;
    const int b = bh / a.kv_heads, h = bh % a.kv_heads;
    const int n = min(evict_len(a, b), a.budget);
    const int *kept = a.kept + (int64_t)bh * a.budget;
    auto source = [&](int i) -> int64_t {
        const int j = kept[i];
        const int page = evict_page(a, a.table, a.max_pages, b, j / a.page_size);
        return page < 0 ? -1 : ((int64_t)page * a.kv_heads + h) * a.page_size + j % a.page_size;
    };
    auto target = [&](int i) -> int64_t {
        const int page = evict_page(a, a.dst_table, a.dst_max_pages, b, i / a.page_size);
        return page < 0 ? -1 : ((int64_t)page * a.kv_heads + h) * a.page_size + i % a.page_size;
    };
    if (part == 2 * slices) {
        if (h == 0 && threadIdx.x == 0) a.new_lens[b] = n;
        for (int i0 = 0; i0 < n; i0 += 256) {
            const int i = i0 + threadIdx.x;
            int64_t from = -1, to = -1;
            float x = 0.0f;
            if (i < n) {
                from = source(i);
                to = target(i);
                if (from >= 0) x = a.scores[from];
            }
            __syncthreads();
            if (from >= 0 && to >= 0 && from != to) a.scores[to] = x;
        }
        return;
    }
    W *pages = reinterpret_cast<W *>(part < slices ? a.k_pages : a.v_pages);
    const int words = row_words / slices, col0 = part % slices * words;
    const int64_t total = (int64_t)n * words;
    constexpr int U = 4;
    for (int64_t w0 = 0; w0 < total; w0 += 256 * U) {
        W x[U];
        int64_t at[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t w = w0 + u * 256 + threadIdx.x;
            at[u] = -1;
            if (w < total) {
                const int i = (int)(w / words), c = col0 + (int)(w % words);
                const int64_t from = source(i), to = target(i);
                if (from >= 0 && to >= 0 && from != to) {
                    x[u] = pages[from * row_words + c];
                    at[u] = to * row_words + c;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++)
            if (at[u] >= 0) pages[at[u]] = x[u];
    }
}

}  // namespace
}  // namespace hx

using namespace hx;

HX_EXPORT int hexcuda_cache_evict(int dev, void *k_pages, void *v_pages, float *scores,
                                  const int32_t *block_table, const int32_t *dst_table,
                                  const int32_t *kv_lens, int32_t *new_lens, int32_t *kept,
                                  int batch, int kv_heads, int head_dim, int num_pages,
                                  int page_size, int max_pages, int dst_max_pages, int budget,
                                  int sink, int recent) {
    const char *name = "cache_evict";
    if (batch < 0 || kv_heads < 1 || head_dim < 1 || head_dim > 256 || kv_heads > 65535)
        return fail(HEXCUDA_ERR_ARG, "%s: batch %d kv_heads %d head_dim %d (1 to 256)", name, batch,
                    kv_heads, head_dim);
    if (num_pages < 1 || page_size < 1 || max_pages < 1 ||
        (int64_t)num_pages * page_size > 0x7fffffff || (int64_t)max_pages * page_size > 0x7fffffff)
        return fail(HEXCUDA_ERR_ARG, "%s: num_pages %d page_size %d max_pages %d", name, num_pages,
                    page_size, max_pages);
    if (budget < 1 || sink < 0 || recent < 0 || (int64_t)sink + recent > budget)
        return fail(HEXCUDA_ERR_ARG, "%s: budget %d sink %d recent %d", name, budget, sink, recent);
    const int width = dst_table ? dst_max_pages : max_pages;
    if (width < 1 || (int64_t)width * page_size > 0x7fffffff ||
        (int64_t)width * page_size < (dst_table ? budget : 1))
        return fail(HEXCUDA_ERR_ARG, "%s: dst_max_pages %d of %d tokens hold no budget of %d", name,
                    width, page_size, budget);
    if (batch == 0) return HEXCUDA_OK;
    if (!k_pages || !v_pages || !scores || !block_table || !kv_lens || !new_lens || !kept)
        return fail(HEXCUDA_ERR_ARG, "%s: null pointer", name);
    if ((int64_t)batch * kv_heads > (1 << 24))
        return fail(HEXCUDA_ERR_ARG, "%s: batch %d kv_heads %d", name, batch, kv_heads);
    Dev *d = get_dev(dev);
    if (!d) return HEXCUDA_ERR_NODEV;
    Evict a{k_pages, v_pages, scores, block_table, dst_table ? dst_table : block_table, kv_lens,
            new_lens, kept, batch, kv_heads, head_dim, num_pages, page_size, max_pages, width,
            budget, sink, recent, d->err_word};
    launch_begin(d);
    const int bh = batch * kv_heads;
    evict_select_kernel<<<bh, kSelThreads, 0, d->stream>>>(a);
    const bool vec = head_dim % 8 == 0 && (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15u) == 0;
    if (vec) {
        const int slices = head_dim % 64 == 0 ? head_dim / 32 : 1;
        evict_move_kernel<uint4><<<bh * (2 * slices + 1), 256, 0, d->stream>>>(a, head_dim / 8,
                                                                               slices);
    } else {
        evict_move_kernel<uint16_t><<<bh * 3, 256, 0, d->stream>>>(a, head_dim, 1);
    }
    return launch_end(d, name, 2);
}
