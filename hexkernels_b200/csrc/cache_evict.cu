// cache_evict.cu -- cut every sequence of a paged cache to at most `budget`
// tokens: its first `sink`, its last `recent`, and between them those with the
// highest collected weight (cache_scores), for each key head on its own.
// What stays keeps its order and moves to the front of the sequence's pages
// (or of other pages); which tokens stayed is written to `kept`.
//
// Two launches: the choice (a radix select on the scores' bits, then the places
// in index order, so ties go to the lowest index), then the move of K, V and
// score rows.  Both are bound by what they read and write once, and for few
// sequences by latency.  Measured among other calls, to other pages, 8 key heads of 128
// to a quarter of their length: 1 x 4099: 20 us (choice 15, move 9, overlapping); 32 x
// 8192: 105 us (25 and 78, the move at 5.6 TB/s); 8 heads of 64, 1 x 131072 to 8192: 41
// us (30 and 12; the choice is three passes, each with barriers over the cluster).
// In place the move of few sequences takes longer, since a slice's chunks follow one
// another (128-wide heads, L2 flushed: 1 x 131072 97 us for 50, 32 x 8192 130 for 122).
// The choice's CTAs and shared memory go by the table's width: what it could name,
// not the lengths, which the host cannot see.
#include <math.h>

#include <algorithm>

#include "paged.cuh"
#include "tc_common.cuh"

namespace hx {
namespace {

struct Evict {
    void *k_pages, *v_pages;
    float *scores;
    const int *table, *dst_table, *kv_lens;
    int *new_lens, *kept;
    int batch, kv_heads, dim, num_pages, page_size, max_pages, dst_max_pages;
    int budget, sink, recent;
    int page_shift;         // log2 of page_size, or -1
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

constexpr int kBins = 2048;             // 11 bits of a key a pass (the last pass has 10)
constexpr int kSmemKeys = 49152;        // keys of a CTA that fit shared memory
constexpr int kMaxCluster = 8;

// shared memory of one CTA of the cluster that works on a (sequence, key head)
struct Select {
    alignas(16) int hist[2][kBins];
    int warp_sum[32], warp_eq[32];
    int counts[2];                      // keys above the threshold, equal to it
    int bin, left;
};

// Same variable in the shared memory of the cluster's CTA `rank`.
__device__ __forceinline__ int peer_int(const int *p, uint32_t rank) {
    int v;
    asm volatile("ld.shared::cluster.b32 %0, [%1];"
                 : "=r"(v)
                 : "r"(tc::mapa_shared(tc::smem_u32(p), rank))
                 : "memory");
    return v;
}
__device__ __forceinline__ int2 peer_pair(const int *p, uint32_t rank) {
    int2 v;
    asm volatile("ld.shared::cluster.v2.b32 {%0, %1}, [%2];"
                 : "=r"(v.x), "=r"(v.y)
                 : "r"(tc::mapa_shared(tc::smem_u32(p), rank))
                 : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    return n;
}

// The choice.  A cluster of CTAs works on one sequence and key head, each on a
// contiguous range of places whose keys it keeps in shared memory (SMEM; read
// again from the cache otherwise).  Three passes over 11, 11 and 10 bits find
// the want-th highest key: each CTA counts its keys that share the bits found
// so far by their next bits, every CTA adds up the cluster's counts (over
// distributed shared memory) and finds the bin where the count from the top
// reaches what is wanted.  Then the places are written in ascending order,
// each warp on a contiguous run, with ballots for the ranks in it.
template <bool SMEM, int kSelThreads>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const Evict a) {
    constexpr int kWarps = kSelThreads / 32, kPer = kBins / kSelThreads;
    tc::launch_dependents();
    __shared__ Select sh;
    extern __shared__ uint32_t keys[];
    const uint32_t ranks = cluster_size(), rank = tc::cluster_ctarank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int bh = blockIdx.x / ranks;
    const int b = bh / a.kv_heads, h = bh % a.kv_heads;
    const int n = evict_len(a, b);
    const int all = kSelThreads * (int)ranks, me = (int)rank * kSelThreads + (int)threadIdx.x;
    int *kept = a.kept + (int64_t)bh * a.budget;
    const int m = min(n, a.budget);
    for (int j = m + me; j < a.budget; j += all) kept[j] = -1;
    if (n <= a.budget) {            // (the whole cluster)
        for (int j = me; j < n; j += all) kept[j] = j;
        return;
    }
    // the sinks and the recent ones stay whatever their weight
    const int lo = a.sink, hi = n - a.recent;
    const int want = a.budget - a.sink - a.recent;
    for (int j = me; j < a.sink; j += all) kept[j] = j;
    for (int j = me; j < a.recent; j += all) kept[a.budget - a.recent + j] = hi + j;
    if (want == 0) return;
    // this CTA's places: [first, first + count), a multiple of 32 but for the last
    const int per = ((hi - lo + (int)ranks - 1) / (int)ranks + 31) & ~31;
    const int first = lo + (int)rank * per;
    const int count = max(0, min(per, hi - first));
    auto page_no = [&](int j) { return a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size; };
    auto read_key = [&](int i) -> uint32_t {
        const int j = first + i, pi = page_no(j);
        const int page = evict_page(a, a.table, a.max_pages, b, pi);
        if (page < 0) return 0u;
        return order_key(
            a.scores[((int64_t)page * a.kv_heads + h) * a.page_size + (j - pi * a.page_size)]);
    };
    auto key_at = [&](int i) { return SMEM ? keys[i] : read_key(i); };
    // one more key in the bin for each lane whose `in` is set; equal scores are
    // common, and lanes that agree on the bin add once
    auto count_in = [&](int *hist, bool in, int bin) {
        const uint32_t who = __ballot_sync(0xffffffffu, in);
        if (who == 0) return;
        const int leader = __ffs((int)who) - 1;
        const int bin0 = __shfl_sync(0xffffffffu, bin, leader);
        if (__ballot_sync(0xffffffffu, in && bin != bin0) == 0) {
            if (lane == leader) atomicAdd(&hist[bin0], __popc(who));
        } else if (in) {
            atomicAdd(&hist[bin], 1);
        }
    };
    for (int i = threadIdx.x; i < kBins; i += kSelThreads) sh.hist[0][i] = 0;
    __syncthreads();
    if (SMEM) {
        // sixteen keys a thread at a time: all their pages, then all their scores,
        // then the first pass's count while they are in registers
        constexpr int U = 16;
        for (int i0 = warp * 32; i0 < count; i0 += U * kSelThreads) {
            int page[U];
            float x[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = i0 + lane + u * kSelThreads;
                page[u] = 0;
                if (i < count) page[u] = a.table[(int64_t)b * a.max_pages + page_no(first + i)];
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = i0 + lane + u * kSelThreads, j = first + i;
                x[u] = 0.0f;
                if (i < count && page[u] >= 0 && page[u] < a.num_pages)
                    x[u] = a.scores[((int64_t)page[u] * a.kv_heads + h) * a.page_size +
                                    (j - page_no(j) * a.page_size)];
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = i0 + lane + u * kSelThreads;
                if (i - lane >= count) break;
                uint32_t key = order_key(x[u]);
                if (i < count) {
                    if (page[u] < 0 || page[u] >= a.num_pages) {
                        flag_index(a.err_word);
                        key = 0u;
                    }
                    keys[i] = key;
                }
                count_in(sh.hist[0], i < count, (int)(key >> 21));
            }
        }
    }
    uint32_t prefix = 0, mask = 0;
    int left = want;
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        int *hist = sh.hist[pass & 1];
        if (pass > 0) {
            for (int i = threadIdx.x; i < kBins; i += kSelThreads) hist[i] = 0;
            __syncthreads();
        }
        if (pass > 0 || !SMEM) {
#pragma unroll 4
            for (int i0 = warp * 32; i0 < count; i0 += kSelThreads) {
                const int i = i0 + lane;
                const uint32_t key = i < count ? key_at(i) : 0u;
                count_in(hist, i < count && (key & mask) == prefix,
                         (int)(key >> shift & ((1u << bits) - 1)));
            }
        }
        tc::cluster_sync_all();
        // thread t has the kPer bins from kBins - 1 - kPer * t down
        const int top = kBins - 1 - kPer * (int)threadIdx.x;
        int in_bin[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i += 2) {
            int2 v[kMaxCluster];
            if (ranks == 1) {
                v[0] = *reinterpret_cast<const int2 *>(&hist[top - i - 1]);
#pragma unroll
                for (int r = 1; r < kMaxCluster; r++) v[r] = int2{0, 0};
            } else {
#pragma unroll
                for (int r = 0; r < kMaxCluster; r++)
                    v[r] = r < (int)ranks ? peer_pair(&hist[top - i - 1], r) : int2{0, 0};
            }
            in_bin[i] = in_bin[i + 1] = 0;
#pragma unroll
            for (int r = 0; r < kMaxCluster; r++) {
                in_bin[i] += v[r].y;
                in_bin[i + 1] += v[r].x;
            }
        }
        int mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) mine += in_bin[i];
        int upto = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        if (lane == 31) sh.warp_sum[warp] = upto;
        __syncthreads();
        // (every warp scans the warps' sums for itself)
        int v = lane < kWarps ? sh.warp_sum[lane] : 0;
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += y;
        }
        const int before_warp = __shfl_sync(0xffffffffu, v, warp > 0 ? warp - 1 : 0);
        if (warp > 0) upto += before_warp;
        int before = upto - mine;
        if (before < left && left <= upto) {
            int bin = 0, rest = 0;
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                if (before < left && left <= before + in_bin[i]) {
                    bin = top - i;
                    rest = left - before;
                }
                before += in_bin[i];
            }
            sh.bin = bin;
            sh.left = rest;
        }
        __syncthreads();
        prefix |= (uint32_t)sh.bin << shift;
        left = sh.left;
        mask |= ((1u << bits) - 1) << shift;
        // (the next pass counts in the other histogram: peers may still read this one)
    }
    // ranks: keys above the threshold and equal to it in the places before a warp's run
    const int run = ((count + kWarps - 1) / kWarps + 31) / 32 * 32;     // whole ballots
    const int i_lo = min(count, warp * run), i_hi = min(count, i_lo + run);
    int above = 0, equal = 0;
#pragma unroll 4
    for (int i0 = i_lo; i0 < i_hi; i0 += 32) {
        const bool in = i0 + lane < i_hi;
        const uint32_t key = in ? key_at(i0 + lane) : 0u;
        above += __popc(__ballot_sync(0xffffffffu, in && key > prefix));
        equal += __popc(__ballot_sync(0xffffffffu, in && key == prefix));
    }
    if (lane == 0) {
        sh.warp_sum[warp] = above;
        sh.warp_eq[warp] = equal;
    }
    __syncthreads();
    if (warp == 0) {
        int x = lane < kWarps ? sh.warp_sum[lane] : 0, y = lane < kWarps ? sh.warp_eq[lane] : 0;
        const int x0 = x, y0 = y;
        for (int o = 1; o < 32; o <<= 1) {
            const int p = __shfl_up_sync(0xffffffffu, x, o), q = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) {
                x += p;
                y += q;
            }
        }
        sh.warp_sum[lane] = x - x0;
        sh.warp_eq[lane] = y - y0;
        if (lane == 31) {
            sh.counts[0] = x;
            sh.counts[1] = y;
        }
    }
    tc::cluster_sync_all();
    above = sh.warp_sum[warp];
    equal = sh.warp_eq[warp];
    for (uint32_t r = 0; r < rank; r++) {
        above += peer_int(&sh.counts[0], r);
        equal += peer_int(&sh.counts[1], r);
    }
    // every key above the threshold, and the first `left` equal to it
    const uint32_t below = (1u << lane) - 1;
#pragma unroll 4
    for (int i0 = i_lo; i0 < i_hi; i0 += 32) {
        const bool in = i0 + lane < i_hi;
        const uint32_t key = in ? key_at(i0 + lane) : 0u;
        const uint32_t gt = __ballot_sync(0xffffffffu, in && key > prefix);
        const uint32_t eq = __ballot_sync(0xffffffffu, in && key == prefix);
        const int e = equal + __popc(eq & below);
        const int at = above + __popc(gt & below) + min(e, left);
        if ((gt >> lane & 1) || ((eq >> lane & 1) && e < left))
            kept[a.sink + at] = first + i0 + lane;
        above += __popc(gt);
        equal += __popc(eq);
    }
    tc::cluster_sync_all();         // no CTA leaves while a peer may read its counts
}

// The move of K, V and score rows.  Kept token i comes from place kept[i] >= i.
// A CTA works on one sequence and key head in chunks of 256 kept tokens: each
// thread looks up the rows of one token (places, pages) for all, then the rows
// are copied, all loads of a chunk in flight together.
//
// In place (the target's first page is the source's): a CTA moves one column
// slice of K or V (or the scores), chunk after ascending chunk.  A chunk's rows
// are all read before any of them is written, and no later chunk reads what an
// earlier one wrote.  To other pages: each CTA takes chunks of its own.
constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 256;

template <typename W>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const Evict a, int row_words,
                                                                  int slices) {
    constexpr int U = 8;
    __shared__ int64_t from[2][kMoveRows], to[2][kMoveRows];
    tc::grid_dependency_wait();
    const int parts = 2 * slices + 1;
    const int part = blockIdx.x % parts;
    const int bh = blockIdx.x / parts;
    const int b = bh / a.kv_heads, h = bh % a.kv_heads;
    const int n = min(evict_len(a, b), a.budget);
    const int *kept = a.kept + (int64_t)bh * a.budget;
    const bool is_score = part == 2 * slices;
    if (is_score && h == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.new_lens[b] = n;
    if (n == 0) return;
    const bool in_place = a.table[(int64_t)b * a.max_pages] == a.dst_table[(int64_t)b * a.dst_max_pages];
    if (in_place && blockIdx.y != 0) return;
    // this thread's token of the chunk at i0: the rows of the cache it leaves and
    // goes to, -1 when there is nothing to move
    auto look_up = [&](int i0, int buf) {
        const int i = i0 + threadIdx.x;
        int64_t f = -1, t = -1;
        if (i < n) {
            const int j = kept[i], pj = j / a.page_size, pi = i / a.page_size;
            const int source = evict_page(a, a.table, a.max_pages, b, pj);
            const int target = evict_page(a, a.dst_table, a.dst_max_pages, b, pi);
            if (source >= 0 && target >= 0) {
                f = ((int64_t)source * a.kv_heads + h) * a.page_size + (j - pj * a.page_size);
                t = ((int64_t)target * a.kv_heads + h) * a.page_size + (i - pi * a.page_size);
                if (f == t) t = -1;
            }
        }
        from[buf][threadIdx.x] = f;
        to[buf][threadIdx.x] = t;
    };
    // in place: every chunk of one slice; else every `stride`-th chunk, whole rows
    const int pieces = is_score ? 1 : slices;
    const int words = is_score ? 1 : in_place ? row_words / slices : row_words;
    const int col0 = in_place && !is_score ? part % slices * words : 0;
    const int stride = in_place ? 1 : pieces * (int)gridDim.y;
    const int chunk0 = in_place ? 0 : (is_score ? 0 : part % slices * (int)gridDim.y) + (int)blockIdx.y;
    const int chunks = (n + kMoveRows - 1) / kMoveRows;
    if (chunk0 >= chunks) return;
    // threads of a row: the power of two from `words` on, so that no division is left
    int shift = 0;
    while ((1 << shift) < words) shift++;
    const int c = threadIdx.x & ((1 << shift) - 1), row0 = threadIdx.x >> shift;
    const int rows = kMoveThreads >> shift;
    W *pages = reinterpret_cast<W *>(part < slices ? a.k_pages : a.v_pages);
    int buf = 0;
    look_up(chunk0 * kMoveRows, buf);
    __syncthreads();
    for (int chunk = chunk0; chunk < chunks; chunk += stride, buf ^= 1) {
        if (is_score) {
            float x = 0.0f;
            const int64_t t = to[buf][threadIdx.x];
            if (t >= 0) x = a.scores[from[buf][threadIdx.x]];
            if (chunk + stride < chunks) look_up((chunk + stride) * kMoveRows, buf ^ 1);
            __syncthreads();
            if (t >= 0) a.scores[t] = x;
            continue;
        }
        // rows of a chunk that its threads can hold in registers at once
        for (int r0 = 0; r0 < kMoveRows; r0 += rows * U) {
            W x[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int r = r0 + u * rows + row0;
                if (r < kMoveRows && c < words && to[buf][r] >= 0)
                    x[u] = pages[from[buf][r] * row_words + col0 + c];
            }
            if (r0 == 0 && chunk + stride < chunks)
                look_up((chunk + stride) * kMoveRows, buf ^ 1);
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int r = r0 + u * rows + row0;
                if (r < kMoveRows && c < words && to[buf][r] >= 0)
                    pages[to[buf][r] * row_words + col0 + c] = x[u];
            }
        }
        __syncthreads();
    }
}

template <bool SMEM, int kThreads>
int launch_select(Dev *d, const Evict &a, int ranks, size_t smem) {
    static bool allowed[64] = {};
    auto kern = evict_select_kernel<SMEM, kThreads>;
    if (smem > 24576 && !allowed[d->ordinal & 63]) {
        if (int rc = check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                kSmemKeys * 4),
                           "cudaFuncSetAttribute(evict_select)"))
            return rc;
        allowed[d->ordinal & 63] = true;
    }
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)ranks;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.batch * a.kv_heads * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = d->stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return check(cudaLaunchKernelEx(&cfg, kern, a), "launch evict_select");
}

// The move, a programmatic dependent of the choice: its launch overlaps it.
template <typename W>
int launch_move(Dev *d, const Evict &a, dim3 grid, int row_words, int slices) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kMoveThreads);
    cfg.stream = d->stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return check(cudaLaunchKernelEx(&cfg, evict_move_kernel<W>, a, row_words, slices),
                 "launch evict_move");
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
        (int64_t)num_pages * page_size > 0x7fffffff || (int64_t)max_pages * page_size > kMaxTokens)
        return fail(HEXCUDA_ERR_ARG, "%s: num_pages %d page_size %d max_pages %d", name, num_pages,
                    page_size, max_pages);
    if (budget < 1 || budget > kMaxTokens || sink < 0 || recent < 0 || (int64_t)sink + recent > budget)
        return fail(HEXCUDA_ERR_ARG, "%s: budget %d sink %d recent %d", name, budget, sink, recent);
    const int width = dst_table ? dst_max_pages : max_pages;
    if (width < 1 || (int64_t)width * page_size > kMaxTokens ||
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
    const int64_t pages16 = (int64_t)num_pages * kv_heads * page_size * head_dim;
    if (overlap16(k_pages, pages16, v_pages, pages16))
        return fail(HEXCUDA_ERR_ARG, "%s: k_pages and v_pages overlap", name);
    Evict a{k_pages, v_pages, scores, block_table, dst_table ? dst_table : block_table, kv_lens,
            new_lens, kept, batch, kv_heads, head_dim, num_pages, page_size, max_pages, width,
            budget, sink, recent, -1, d->err_word};
    for (int i = 0; i < 31; i++)
        if (page_size == 1 << i) a.page_shift = i;
    launch_begin(d);
    const int bh = batch * kv_heads;
    // CTAs a sequence and key head: as many as keep the device busy, while each has
    // some thousands of places left (8 key heads of 128, the whole call, L2 flushed:
    // 1 x 32768 with several 34 us, with one 52, and with twice as many 36; 1 x 131072 50
    // and 60 with what shared memory needs; 1 x 4099 with one or two 24).  More of them
    // than SMs: of 512 threads, so that two are resident (64 x 4096: 130 us, with 1024
    // threads 147; fewer CTAs want the 1024: 1 x 131072 50 us, with 512 60).
    const int64_t longest = (int64_t)max_pages * page_size;
    int ranks = 1;
    while (ranks < kMaxCluster && (bh * 2 * ranks <= d->sms || longest > (int64_t)ranks * kSmemKeys) &&
           longest > (int64_t)ranks * 8192)
        ranks *= 2;
    const int64_t per = ((longest + ranks - 1) / ranks + 31) / 32 * 32;
    const bool half = bh * (int64_t)ranks > d->sms;
    int rc;
    if (per <= kSmemKeys)
        rc = half ? launch_select<true, 512>(d, a, ranks, (size_t)per * 4)
                  : launch_select<true, 1024>(d, a, ranks, (size_t)per * 4);
    else
        rc = launch_select<false, 512>(d, a, ranks, 0);
    if (rc) return rc;
    const bool vec = head_dim % 8 == 0 && (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15u) == 0;
    // column slices of 64 bytes, as far as CTAs are missing (in place, 1 x 131072 to
    // 8192: 97 us, unsliced 161; 64 x 4096 to 1024: unsliced 130, always sliced 149)
    int slices = 1;
    while (vec && head_dim % (64 * slices) == 0 && bh * 2 * slices < 2 * d->sms && slices < 4) slices *= 2;
    // to other pages: a chunk of tokens a CTA
    const int per_cta = kMoveRows * slices;
    const int chunks = (int)std::min<int64_t>(((int64_t)budget + per_cta - 1) / per_cta, 65535);
    const dim3 grid((unsigned)(bh * (2 * slices + 1)), (unsigned)chunks);
    rc = vec ? launch_move<uint4>(d, a, grid, head_dim / 8, slices)
             : launch_move<uint16_t>(d, a, grid, head_dim, 1);
    if (rc) return rc;
    return launch_end(d, name, 2);
}
