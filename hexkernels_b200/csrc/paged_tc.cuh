// paged_tc.cuh -- what the tensor-core kernels over the paged cache share:
// the tensor maps, the loads of a 128-key tile page by page, and the even
// split of a ragged batch over the CTAs.
//
// Split.  A work item is (sequence, key head, one or two tiles of query rows)
// and takes ceil(keys its last row sees / 128) key tiles, at least one (a row
// that sees nothing is still written).  A key tile costs one unit, or two when
// the item has two query tiles (measured 1700 and 3300 cycles at dim 64, 2600
// and 4000 at dim 128), and an item of a chunk five more for its queries, its first
// loads and its output (some 9000 cycles; when the CTAs have at least eight units:
// 40 x 40 new tokens of 3000, 16 heads of 64: 142 us without them, 108 with five, 110
// with three and 108 with eight).  The units of all items, in that order, are numbered
// 0 .. T - 1 and CTA c of C takes the key tiles that start in units c T / C ..
// (c + 1) T / C - 1: a run of items, the first and the last perhaps only in
// part.  Lengths live on the device, so each CTA derives its own run from them (a
// prefix sum over the sequences).  An item that is cut leaves one partial result
// per CTA: the unnormalised output, the reference maximum and the sum of each row.
// A second kernel joins them, in CTA order, so results do not depend on timing.
#pragma once
#include "paged.cuh"
#include "tc_common.cuh"

namespace hx {

constexpr int kKeys = 128;              // keys per tile
constexpr int kSubTile = kKeys * 128;   // 64 columns of a key tile: 128 rows x 128 bytes
constexpr int kPartRows = 256;          // rows of a partial result, at most

struct alignas(16) PartRec {            // (of the workspace's alignment, not more)
    int h, row0, ntok, nparts;          // nparts 0: the CTA's last item is not its to join
    int b, rt;                          // its sequence and place there
    int odd;                            // the CTA took values that are not finite out of a tile
};
static_assert(alignof(PartRec) <= 16, "the caller's workspace is 16-byte aligned");

// What both attention kernels get.
struct PagedTc {
    PagedSeqs s;
    int heads, kv_heads, group;
    int tok;                 // tokens of a query tile: rows / group
    int frag;                // rows of one page load: a power of two, 8 to 128
    int map_rows;            // rows of the cache: a coordinate behind the last
    int min_units;           // of a CTA's run, at least 2: then it has a key tile
    float scale_log2;        // scale * log2(e)
    const void *q, *k, *v;
    void *out;
    float *lse;
    PartRec *recs;           // [grid]
    float *part_ml;          // [grid][2][kPartRows][2]: reference maximum, sum
    float *part_o;           // [grid][2] outputs of kPartRows x D, whose rows and groups
    int part_row, part_col;  // of four columns are so many floats apart
};

// Tokens of a sequence without raising the error word (the plan has).
__device__ __forceinline__ void quiet_seq(const PagedSeqs &s, int b, int &first, int &q_len,
                                          int &kv_len) {
    first = s.q_offs[b];
    const int end = s.q_offs[b + 1];
    q_len = first >= 0 && end >= first && end <= s.total_q ? end - first : 0;
    const int n = s.kv_lens[b];
    const long long cap = (long long)s.max_pages * s.page_size;
    kv_len = n < 0 ? 0 : n > cap ? (int)cap : n;
}

// Key tiles that the tokens before `end` see.
__device__ __forceinline__ int tiles_to(const PagedSeqs &s, int kv_len, int q_len, int end) {
    const int seen = seen_by(s, kv_len, q_len, min(end, q_len) - 1);
    return max(1, (seen + kKeys - 1) / kKeys);
}

// Units of a key tile of an item (its two query tiles are 2 * a.tok tokens).
__device__ __forceinline__ int units_of(const PagedTc &a, int item_tok, int q_len, int rt) {
    return item_tok > a.tok && q_len - rt * item_tok > a.tok ? 2 : 1;
}

// A CTA's run of items, one segment (item, key tiles j0 .. j1 - 1) at a time.
// Every role of the CTA walks its own copy.
struct Walk {
    int b, h, rt, j0, j1, nt, cost, extra;
    int first, q_len, kv_len;
    long long pos, end;      // first unit of the segment, end of the run

    // the segment at (b, h, rt, j0), pos
    __device__ __forceinline__ void open(const PagedTc &a, int item_tok) {
        nt = tiles_to(a.s, kv_len, q_len, (rt + 1) * item_tok);
        cost = units_of(a, item_tok, q_len, rt);
        // (the first key tile's unit is followed by the item's extra ones)
        const long long room = end - pos - (j0 == 0 ? extra : 0);
        const long long left = room > 0 ? (room + cost - 1) / cost : 1;
        j1 = left < nt - j0 ? j0 + (int)left : nt;
    }
    __device__ __forceinline__ bool next(const PagedTc &a, int item_tok) {
        pos += (long long)(j1 - j0) * cost + (j0 == 0 ? extra : 0);
        if (pos >= end) return false;
        j0 = 0;
        if (++rt * item_tok >= q_len) {
            rt = 0;
            if (++h == a.kv_heads) {
                h = 0;
                do {
                    if (++b >= a.s.batch) return false;
                    quiet_seq(a.s, b, first, q_len, kv_len);
                } while (q_len == 0);
            }
        }
        open(a, item_tok);
        return true;
    }
};

struct PlanShared {
    long long sums[32], items[32];
    Walk start;
    int ctas;
    long long total;
};

// Whole block.  Leaves this CTA's first segment in sh.start; false when it has
// none.  item_tok: tokens of an item (one or two query tiles).
// EXTRA: units that an item costs beside its key tiles.
template <int THREADS, int EXTRA>
__device__ __forceinline__ bool plan_run(const PagedTc &a, int item_tok, PlanShared &sh) {
    const int per = (a.s.batch + THREADS - 1) / THREADS;
    const int b0 = min(a.s.batch, (int)threadIdx.x * per), b1 = min(a.s.batch, b0 + per);
    auto units = [&](int q_len, int kv_len) {       // of one key head's key tiles
        long long n = 0;
        for (int rt = 0; rt * item_tok < q_len; rt++)
            n += (long long)tiles_to(a.s, kv_len, q_len, (rt + 1) * item_tok) *
                 units_of(a, item_tok, q_len, rt);
        return n;
    };
    auto items = [&](int q_len) { return (q_len + item_tok - 1) / item_tok; };
    long long mine = 0, mine_items = 0;
    for (int b = b0; b < b1; b++) {
        int first;
        const int q_len = seq_q_len(a.s, b, first), kv_len = seq_kv_len(a.s, b);
        mine += units(q_len, kv_len) * a.kv_heads;
        if (EXTRA) mine_items += (long long)items(q_len) * a.kv_heads;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long upto = mine, upto_items = mine_items;
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, o);
        const long long z = EXTRA ? __shfl_up_sync(0xffffffffu, upto_items, o) : 0;
        if (lane >= o) {
            upto += y;
            upto_items += z;
        }
    }
    if (lane == 31) {
        sh.sums[warp] = upto;
        if (EXTRA) sh.items[warp] = upto_items;
    }
    __syncthreads();
    long long total = 0, total_items = 0;
    for (int w = 0; w < THREADS / 32; w++) {
        if (w < warp) {
            upto += sh.sums[w];
            if (EXTRA) upto_items += sh.items[w];
        }
        total += sh.sums[w];
        if (EXTRA) total_items += sh.items[w];
    }
    // (a run must be longer than a first key tile with the extra units, so that
    // some key tile starts in it)
    const int extra = total >= (EXTRA + 3LL) * gridDim.x ? EXTRA : 0;
    mine += mine_items * extra;
    upto += upto_items * extra;
    total += total_items * extra;
    const long long want = max(total / a.min_units, total > 0 ? 1LL : 0LL);
    const int ctas = want < (int)gridDim.x ? (int)want : (int)gridDim.x;
    const bool any = (int)blockIdx.x < ctas;
    if (any) {
        const long long lo = blockIdx.x * total / ctas, hi = (blockIdx.x + 1LL) * total / ctas;
        if (upto - mine <= lo && lo < upto) {
            long long at = lo - (upto - mine);
            Walk w;
            for (int b = b0; b < b1; b++) {
                quiet_seq(a.s, b, w.first, w.q_len, w.kv_len);
                const long long n = units(w.q_len, w.kv_len) + (long long)items(w.q_len) * extra;
                if (at >= n * a.kv_heads) {
                    at -= n * a.kv_heads;
                    continue;
                }
                w.b = b;
                w.h = (int)(at / n);
                at -= w.h * n;
                for (w.rt = 0;; w.rt++) {
                    const int units = tiles_to(a.s, w.kv_len, w.q_len, (w.rt + 1) * item_tok) *
                                          units_of(a, item_tok, w.q_len, w.rt) +
                                      extra;
                    if (at < units) break;
                    at -= units;
                }
                break;
            }
            // the first key tile that starts here: perhaps the next item's first
            w.cost = units_of(a, item_tok, w.q_len, w.rt);
            w.extra = extra;
            w.j0 = at == 0 ? 0 : max(1, ((int)at - extra + w.cost - 1) / w.cost);
            w.j1 = w.j0;
            w.pos = lo + (w.j0 == 0 ? 0 : w.j0 * w.cost + extra - at);
            w.end = hi;
            if (w.j0 < tiles_to(a.s, w.kv_len, w.q_len, (w.rt + 1) * item_tok))
                w.open(a, item_tok);
            else
                w.next(a, item_tok);
            sh.start = w;
            sh.ctas = ctas;
            sh.total = total;
        }
    }
    if (threadIdx.x == 0) a.recs[blockIdx.x].nparts = 0;
    __syncthreads();
    return any;
}

// One thread, once the CTA's last segment `w` is known: whether this CTA joins
// its item's parts (it holds the first of several).
__device__ __forceinline__ void note_parts(const PagedTc &a, const PlanShared &sh, const Walk &w,
                                           int item_tok) {
    PartRec r = {};
    if (w.j0 == 0 && w.j1 < w.nt) {
        // the CTA where the item's last tile starts, in unit u: the largest c with c T / C <= u
        const long long u = w.pos + (long long)(w.nt - 1) * w.cost + w.extra;
        r.h = w.h;
        r.row0 = w.first + w.rt * item_tok;
        r.ntok = min(item_tok, w.q_len - w.rt * item_tok);
        r.nparts = (int)(((u + 1) * sh.ctas - 1) / sh.total) - (int)blockIdx.x + 1;
        r.b = w.b;
        r.rt = w.rt;
    }
    a.recs[blockIdx.x] = r;
}

// ---- one warp: the page loads of a key tile ----

// Lane f's fragment of tile j of the walk's sequence: its first token (-1 when
// no cached token lies in it) and its page as the table has it.  The page is
// fetched a tile ahead and only looked at in frag_row, so that the warp does
// not wait for it.
struct Frag {
    int token, page;
};
__device__ __forceinline__ Frag frag_of(const PagedTc &a, const Walk &w, int j, int lane) {
    const int t = j * kKeys + lane * a.frag;
    if (lane * a.frag >= kKeys || t >= w.kv_len) return Frag{-1, 0};
    return Frag{t, a.s.table[(int64_t)w.b * a.s.max_pages + t / a.s.page_size]};
}
// The row of the cache where the fragment starts: one behind the last (the
// load then gives zeros) when the table names no page.
__device__ __forceinline__ int frag_row(const PagedTc &a, const Frag &f, int h) {
    if (f.token < 0) return -1;
    if (f.page >= 0 && f.page < a.s.num_pages)
        return (f.page * a.kv_heads + h) * a.s.page_size + f.token % a.s.page_size;
    flag_index(a.s.err_word);
    return a.map_rows;
}
// Fragments that hold cached tokens (the lanes with a row).
__device__ __forceinline__ int frag_count(int row) {
    return __popc(__ballot_sync(0xffffffffu, row >= 0));
}
template <int SUBS>
__device__ __forceinline__ void load_frags(const PagedTc &a, uint8_t *dst, const CUtensorMap *map,
                                           uint64_t *bar, int row, int count, int lane) {
    if (lane == 0)
        tc::mbar_arrive_expect_tx(bar, (uint32_t)(count * a.frag * 128 * SUBS));
    __syncwarp();
    if (row >= 0)
        for (int c = 0; c < SUBS; c++)
            tc::tma_load_2d(dst + c * kSubTile + lane * a.frag * 128, map, bar, c * 64, row);
    __syncwarp();
}

// ---- values that a weight of zero must not meet ----
//
// The weight of a token that a row does not see is zero, and zero times infinity or
// not-a-number is not zero.  Two kinds of rows of a value tile can hold such tokens:
// those behind the last cached token (whatever the page holds), and the tokens behind
// the item's first one, which some of its rows do not see.  Before P V reads the tile
// the former become zeros, and of the latter the elements that are not finite.  A row
// that does see one of those gets it back once it is written (mend_items, the join):
// weights are positive, so what such values add to a column is their plain sum, which
// no weight changes.  That is the work of an item's own tokens, whatever the cache
// holds.  Measured with a channel of infinities over the whole cache, 16 heads of 128
// on 4: 600 new tokens of 6000 128 us (finite values 69), 7 of 12000 41 (38).

// Whether a chunk of eight values holds one that is not finite, as bits that are not
// all zero: a product with zero keeps infinities and not-a-numbers apart from the rest.
template <typename T>
__device__ __forceinline__ uint32_t odd_bits(const uint4 &w) {
    typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type T2;
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
    const uint32_t zero = 0;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const T2 r = __hmul2(*reinterpret_cast<const T2 *>(&v[i]), *reinterpret_cast<const T2 *>(&zero));
        bits |= *reinterpret_cast<const uint32_t *>(&r);
    }
    return bits & 0x7fff7fffu;
}
// Two values, zeros for those that are not finite.
template <typename T>
__device__ __forceinline__ uint32_t finite_of(uint32_t w) {
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    if ((w & e) == e) w &= 0xffff0000u;
    if ((w >> 16 & e) == e) w &= 0xffffu;
    return w;
}

// One thread per key of a value tile: rows from `valid` on become zeros, and of those
// between `from` and them what is not finite; then odd is set.
template <typename T, int SUBS>
__device__ __forceinline__ void settle_row(uint8_t *tile, int key, int from, int valid,
                                           volatile int *odd) {
    uint4 *row = reinterpret_cast<uint4 *>(tile + key * 128);
    constexpr int kStep = kSubTile / 16;        // a 64-column piece further
    if (key >= valid) {
#pragma unroll 1
        for (int i = 0; i < 8 * SUBS; i++) row[(i >> 3) * kStep + (i & 7)] = make_uint4(0, 0, 0, 0);
        return;
    }
    if (key < from) return;
    // (short loops: this code is met once an item, when it is in no cache.  Eight
    // neighbours start at eight different chunks: no bank conflicts.)
    uint32_t bits = 0;
#pragma unroll 1
    for (int i = 0; i < 8 * SUBS; i += 4)
#pragma unroll
        for (int u = 0; u < 4; u++)
            bits |= odd_bits<T>(row[(i >> 3) * kStep + (((i + u) ^ key) & 7)]);
    if (bits == 0) return;
    *odd = 1;
#pragma unroll 1
    for (int i = 0; i < 8 * SUBS; i++) {
        uint4 &w = row[(i >> 3) * kStep + (i & 7)];
        w = make_uint4(finite_of<T>(w.x), finite_of<T>(w.y), finite_of<T>(w.z), finite_of<T>(w.w));
    }
}

// Columns `at` .. `at` + V - 1 of the values of token j of sequence b and key head h,
// zeros for those that are finite.
template <typename T, int D, int V>
__device__ __forceinline__ void odd_values(const PagedTc &a, int b, int h, int j, int at, float (&x)[V]) {
    const int page = a.s.table[(int64_t)b * a.s.max_pages + j / a.s.page_size];
    const bool there = page >= 0 && page < a.s.num_pages;
    const int64_t row = there ? ((int64_t)page * a.kv_heads + h) * a.s.page_size + j % a.s.page_size : 0;
    const uint32_t *p = reinterpret_cast<const uint32_t *>(reinterpret_cast<const T *>(a.v) + row * D + at);
#pragma unroll
    for (int i = 0; i < V / 2; i++) {
        const float2 f = unpack2<T>(p[i]);
        x[2 * i] = there && f.x * 0.0f != 0.0f ? f.x : 0.0f;
        x[2 * i + 1] = there && f.y * 0.0f != 0.0f ? f.y : 0.0f;
    }
}

// Warp `warp` of 8, once the CTA has written all its items: gives the rows of those
// that the CTA wrote alone what they see of the item's own tokens.  Lane t has columns
// t D / 32 ..; the warp walks the tokens and has their sum where a token's row ends.
template <typename T, int D>
__device__ __forceinline__ void mend_items(const PagedTc &a, const Walk &start, int item_tok, int warp) {
    constexpr int V = D / 32, U = 8;
    const int lane = threadIdx.x & 31;
    Walk w = start;
    do {
        if (w.j0 > 0 || w.j1 < w.nt) continue;
        const int t0 = w.rt * item_tok, ntok = min(item_tok, w.q_len - t0);
        const int first = w.kv_len - w.q_len + t0 + 1;      // what token t0 sees, if positive (causal)
        const int end = min(w.kv_len, first + ntok - 1);
        float sum[V];
#pragma unroll
        for (int i = 0; i < V; i++) sum[i] = 0.0f;
        for (int j = seen_by(a.s, w.kv_len, w.q_len, t0); j < end; j += U) {
            float x[U][V];
#pragma unroll
            for (int u = 0; u < U; u++) odd_values<T, D, V>(a, w.b, w.h, min(j + u, end - 1), lane * V, x[u]);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int t = j + u + 1 - first;            // the token that sees just those up to j + u
                if (j + u >= end) continue;
                bool any = false;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    sum[i] += x[u][i];
                    any |= sum[i] != 0.0f;
                }
                if (t < 0 || !__any_sync(0xffffffffu, any)) continue;
                for (int g = (warp + 8 - t % 8) % 8; g < a.group; g += 8) {
                    uint32_t *p = reinterpret_cast<uint32_t *>(
                        reinterpret_cast<T *>(a.out) +
                        ((int64_t)(w.first + t0 + t) * a.heads + w.h * a.group + g) * D + lane * V);
#pragma unroll
                    for (int i = 0; i < V / 2; i++) {
                        const float2 f = unpack2<T>(p[i]);
                        p[i] = pack2<T>(f.x + sum[2 * i], f.y + sum[2 * i + 1]);
                    }
                }
            }
        }
    } while (w.next(a, item_tok));
}

// ---- host side (paged_attn.cu) ----

// The cache's pages as a matrix [num_pages * kv_heads * page_size][dim], box
// 64 x frag; q as [total_q][heads][dim], box 64 x group x tok.  Both 128-byte
// swizzle.
int make_page_map(CUtensorMap *map, const void *base, int64_t rows, int dim, int frag);
int make_query_map(CUtensorMap *map, const void *base, int total_q, int heads, int dim, int group,
                   int tok);

// Whether the tensor-core kernels take these tensors: TMA boxes start on 16
// bytes and hold whole 8-row swizzle atoms, coordinates fit 31 bits.
bool paged_tc_fits(const void *q, const void *k, const void *v, const void *out, int heads,
                   int kv_heads, int dim, int num_pages, int page_size);

int launch_paged_dec(Dev *d, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
                     PagedTc &a, int dtype, int dim, int rows);
int launch_paged_pre(Dev *d, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
                     PagedTc &a, int dtype, int dim);

// The weights of cache_scores (scores_tc.cu), for what paged_tc_fits.
int launch_scores_tc(Dev *d, const PagedSeqs &s, int dtype, const void *q, const float *lse,
                     const void *k, float *scores, int max_q, int heads, int kv_heads, int dim,
                     float scale);

}  // namespace hx
