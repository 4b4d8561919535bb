// scores_tc.cu -- collected attention weight (cache_scores.cu) on the tensor
// cores.
//
// A column sum of the softmax matrix is a row sum when the keys are on the M
// side: S^T [128 keys x R rows] = K Q^T, one thread per key, which adds
// 2^(scale*log2e * s - lse*log2e) over the columns.  The key tile stays in
// shared memory while the query tiles that see it pass by, so a key's sum is
// made by one CTA, in a fixed order, and added to the cache once.
//
// A work item is (sequence, key head, 256 keys); it costs one unit per query
// tile that sees it (R = 16 or 32 rows when a key head has few, else 128; tok =
// R / group tokens a tile).  Items go to the CTAs whole, in order, CTA c
// taking those that start in units c T / C .. (c + 1) T / C - 1.
//
// Per CTA (one per SM), 384 threads: warps 0 and 3 TMA of the halves of the keys
// (page fragments, one lane each; 16-token pages make more loads than one warp
// can start in time), warp 1 tensor memory and MMA issue, warp 2 TMA of query
// tiles and the rows' lse * log2e (minus infinity where a row counts for
// nothing, and a flag for the tile), then a warpgroup for each half of the keys, each with two score
// tiles in tensor memory.  256 keys to a query tile, because the query tiles
// come from L2 again and again: with 128 keys they asked for more than L2
// gives.  With few rows the kernel is bound by HBM (each key once): 64 sequences of
// up to 8192 (half that on average), one new token, 32 heads of 128 over 8 key heads:
// 101 to 107 us from box to box for 563 MB, 5.2 to 5.6 TB/s.  With many it is bound by
// the exponentials, one per score: 3 sequences of up to 1000 new tokens of 6000: 130
// us, a unit of 256 keys x 128 rows taking 3000 cycles, 2048 of them the MUFU's.  Items
// are not cut (a key's sum then needs a second pass in a fixed order): there the
// busiest CTA has 71 units for 56 on average, and 4 CTAs do all of 1000 new tokens of
// 1000 with one key head.
//
// Every wait is bounded; see mbar_wait.
#include <math.h>

#include "paged_tc.cuh"

namespace hx {
namespace {

struct ScoresTc {
    PagedSeqs s;
    int heads, kv_heads, group, tok, frag, map_rows;
    float scale_log2;
    const float *lse;
    float *scores;
};

template <int D, int R>
struct ScSmem {
    static constexpr int kSubs = D / 64;
    static constexpr int kTile = kSubs * kSubTile;           // 128 keys
    // (many rows: the query tiles stream, and a load takes longer than a unit's
    // exponentials; few: the keys do)
    static constexpr int kKStages = (R == 128 ? 1 : 3) * (128 / D);
    static constexpr int kQStages = R == 32 ? 2 : 4;
    static constexpr int kQTile = kSubs * R * 128;
    static constexpr int kK = 0;
    static constexpr int kQ = kK + kKStages * 2 * kTile;
    static constexpr int kLse = kQ + kQStages * kQTile;      // [4][R]
    static constexpr int kNone = kLse + 4 * R * 4;           // [4]: a row of the tile has no weight
    static constexpr int kPlan = kNone + 16;
    static constexpr int kBar = kPlan + 512;
    // l_full, l_empty [4], s_full, s_empty [half][2], drain, q_full, q_empty,
    // k_full, k_empty [stages]
    static constexpr int kNumBars = 17 + 2 * kQStages + 2 * kKStages;
    static constexpr int kTotal = kBar + kNumBars * 8 + 16 + 1024;
};

constexpr int kItemKeys = 2 * kKeys;

// The CTA's items in order.  Every role walks its own copy.
struct KeyWalk {
    int b, h, kt, first, q_len, kv_len;
    long long pos, end;      // first unit of the item, end of the run

    __device__ __forceinline__ int row_tiles(const ScoresTc &a) const {
        return (q_len + a.tok - 1) / a.tok;
    }
    // the first query tile that sees a key of the item's half x
    __device__ __forceinline__ int first_tile(const ScoresTc &a, int x) const {
        if (!a.s.causal) return 0;
        const int t = kt * kItemKeys + x * kKeys - (kv_len - q_len);
        return t > 0 ? t / a.tok : 0;
    }
    // the same for half 1, or behind the last when no key lies in it
    __device__ __forceinline__ int first_tile_1(const ScoresTc &a) const {
        return kt * kItemKeys + kKeys < kv_len ? first_tile(a, 1) : row_tiles(a);
    }
    __device__ __forceinline__ int cost(const ScoresTc &a) const {
        return row_tiles(a) - first_tile(a, 0);
    }
    __device__ __forceinline__ bool next(const ScoresTc &a) {
        pos += cost(a);
        if (pos >= end) return false;
        if (++kt * kItemKeys >= kv_len) {
            kt = 0;
            if (++h == a.kv_heads) {
                h = 0;
                do {
                    if (++b >= a.s.batch) return false;
                    quiet_seq(a.s, b, first, q_len, kv_len);
                } while (q_len == 0 || kv_len == 0);
            }
        }
        return true;
    }
};

struct KeyPlan {
    long long sums[12];
    KeyWalk start;
    int any;
};
static_assert(sizeof(KeyPlan) <= 512, "KeyPlan");

// Units of one key head of a sequence, and of those the ones of its first
// `plain` tiles, which every query tile sees.
__device__ __forceinline__ long long head_units(const ScoresTc &a, KeyWalk &w, int &plain) {
    plain = 0;
    if (w.q_len == 0 || w.kv_len == 0) return 0;
    const int tiles = (w.kv_len + kItemKeys - 1) / kItemKeys;
    plain = tiles;
    if (a.s.causal) {
        const long long c = (long long)w.kv_len - w.q_len + a.tok;
        plain = c <= 0 ? 0 : (int)min((long long)tiles, (c + kItemKeys - 1) / kItemKeys);
    }
    long long n = (long long)plain * w.row_tiles(a);
    for (w.kt = plain; w.kt < tiles; w.kt++) n += w.cost(a);
    return n;
}

// Whole block: this CTA's first item in sh.start; false when it has none.
__device__ __forceinline__ bool plan_keys(const ScoresTc &a, KeyPlan &sh) {
    constexpr int kThreads = 384;
    const int per = (a.s.batch + kThreads - 1) / kThreads;
    const int b0 = min(a.s.batch, (int)threadIdx.x * per), b1 = min(a.s.batch, b0 + per);
    long long mine = 0;
    KeyWalk w;
    int plain;
    for (int b = b0; b < b1; b++) {
        w.q_len = seq_q_len(a.s, b, w.first);
        w.kv_len = seq_kv_len(a.s, b);
        mine += head_units(a, w, plain) * a.kv_heads;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) sh.sums[warp] = upto;
    if (threadIdx.x == 0) sh.any = 0;
    __syncthreads();
    long long total = 0;
    for (int i = 0; i < kThreads / 32; i++) {
        if (i < warp) upto += sh.sums[i];
        total += sh.sums[i];
    }
    const long long lo = blockIdx.x * total / gridDim.x, hi = (blockIdx.x + 1LL) * total / gridDim.x;
    if (lo < hi && upto - mine <= lo && lo < upto) {
        long long at = lo - (upto - mine);
        for (int b = b0; b < b1; b++) {
            quiet_seq(a.s, b, w.first, w.q_len, w.kv_len);
            const long long n = head_units(a, w, plain);
            if (at >= n * a.kv_heads) {
                at -= n * a.kv_heads;
                continue;
            }
            w.b = b;
            w.h = (int)(at / n);
            at -= w.h * n;
            const int rt = w.row_tiles(a);
            if (at < (long long)plain * rt) {
                w.kt = (int)(at / rt);
                at -= (long long)w.kt * rt;
            } else {
                at -= (long long)plain * rt;
                for (w.kt = plain; at >= w.cost(a); w.kt++) at -= w.cost(a);
            }
            w.pos = lo - at;
            w.end = hi;
            // an item that an earlier CTA's run cuts is that CTA's
            sh.any = at == 0 || w.next(a);
            sh.start = w;
            break;
        }
    }
    __syncthreads();
    return sh.any != 0;
}

// Sum over the rows lo <= r < hi of one score tile (this lane's key) of
// 2^(s * scale_log2 - z[r]); CUT: some lane's rows are not all R.
template <int R, bool CUT>
__device__ __forceinline__ float add_weights(uint32_t s_addr, const float *z, float scale_log2, int lo,
                                             int hi, float (&acc)[4]) {
    auto add = [&](const auto &r, int c0, auto count) {
#pragma unroll
        for (int e = 0; e < decltype(count)::value; e += 4) {
            const float4 zz = *reinterpret_cast<const float4 *>(z + c0 + e);
            const float zv[4] = {zz.x, zz.y, zz.z, zz.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float p = tc::ex2(fmaf(__uint_as_float(r[e + i]), scale_log2, -zv[i]));
                if (CUT && (c0 + e + i < lo || c0 + e + i >= hi)) p = 0.0f;
                acc[i] += p;
            }
        }
    };
    if constexpr (R == 16) {
        uint32_t r[16];
        tc::tmem_ld_32x32b_x16(s_addr, r);
        tc::tmem_ld_wait(r);
        add(r, 0, std::integral_constant<int, 16>());
    } else if constexpr (R == 32) {
        uint32_t r[32];
        tc::tmem_ld_32x32b_x32(s_addr, r);
        tc::tmem_ld_wait(r);
        add(r, 0, std::integral_constant<int, 32>());
    } else {
#pragma unroll
        for (int c = 0; c < R; c += 64) {
            uint32_t r0[32], r1[32];
            tc::tmem_ld_32x32b_x32(s_addr + c, r0);
            tc::tmem_ld_32x32b_x32(s_addr + c + 32, r1);
            tc::tmem_ld_wait(r0);
            tc::reg_fence(r1);
            add(r0, c, std::integral_constant<int, 32>());
            add(r1, c + 32, std::integral_constant<int, 32>());
        }
    }
    return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}

// The same where some row has no weight (z of minus infinity), whatever its score: a
// row that saw nothing, or that the caller masks.  A loop of its own, because the test
// within add_weights cost every chunk (3 x 1000 new tokens of 6000 137 us for 129; so
// 131).
template <int R>
__device__ __forceinline__ float add_weights_but(uint32_t s_addr, const float *z, float scale_log2, int lo,
                                              int hi) {
    float sum = 0.0f;
#pragma unroll 1
    for (int c = 0; c < R; c += 16) {
        uint32_t r[16];
        tc::tmem_ld_32x32b_x16(s_addr + c, r);
        tc::tmem_ld_wait(r);
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float p = tc::ex2(fmaf(__uint_as_float(r[e]), scale_log2, -z[c + e]));
            if (c + e >= lo && c + e < hi && z[c + e] != -INFINITY) sum += p;
        }
    }
    return sum;
}

template <typename T, int D, int R>
__global__ void __launch_bounds__(384, 1)
    scores_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const ScoresTc a) {
    using L = ScSmem<D, R>;
    constexpr int kSubs = L::kSubs, KS = L::kKStages, QS = L::kQStages;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBar);
    uint64_t *l_full = bars, *l_empty = bars + 4, *s_full = bars + 8, *s_empty = bars + 12;
    uint64_t *drain = bars + 16, *q_full = bars + 17, *q_empty = q_full + QS;
    uint64_t *k_full = q_empty + QS, *k_empty = k_full + KS;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::kNumBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    KeyPlan &plan = *reinterpret_cast<KeyPlan *>(smem + L::kPlan);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *err_word = a.s.err_word;

    if (threadIdx.x == 0) {
        for (int i = 0; i < 4; i++) {
            tc::mbar_init(&l_full[i], 1);
            tc::mbar_init(&l_empty[i], 8);
            tc::mbar_init(&s_full[i], 1);
            tc::mbar_init(&s_empty[i], 4);
        }
        tc::mbar_init(drain, 1);
        for (int i = 0; i < QS; i++) {
            tc::mbar_init(&q_full[i], 1);
            tc::mbar_init(&q_empty[i], 1);
        }
        for (int i = 0; i < KS; i++) {
            tc::mbar_init(&k_full[i], 2);       // a warp for each half of the keys
            tc::mbar_init(&k_empty[i], 1);
        }
        *abort_flag = 0;
        tc::fence_mbar_init();
        tc::tma_prefetch_desc(&tmQ);
        tc::tma_prefetch_desc(&tmK);
    }
    constexpr uint32_t kCols = 4 * R;
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, kCols);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    const bool any = plan_keys(a, plan);
    tc::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (!any) {
        // nothing to do but free the tensor memory
    } else if (warp == 0 || warp == 3) {
        // ------------------------------- TMA, the first and second half's keys
        const int x = warp == 0 ? 0 : 1;
        KeyWalk w = plan.start;
        int st = 0;
        uint32_t ph = 0, armed = 0, k_ph = 0;
        bool ok = true;
        // lane's fragment of an item: its first token and, as the table has
        // it, its page; the load is not waited for until the item's turn
        const int span = lane * a.frag;
        auto token = [&](const KeyWalk &v) {
            const int t = v.kt * kItemKeys + x * kKeys + span;
            return span < kKeys && t < v.kv_len ? t : -1;
        };
        auto page_of = [&](const KeyWalk &v, int t) {
            return t < 0 ? -1 : a.s.table[(int64_t)v.b * a.s.max_pages + t / a.s.page_size];
        };
        int tok = token(w), page = page_of(w, tok);
        bool more;
        do {
            const int t = tok, p = page, h = w.h;
            more = w.next(a);
            if (more) {
                tok = token(w);
                page = page_of(w, tok);
            }
            ok = tc::mbar_wait(&k_empty[st], ph ^ 1, abort_flag, err_word, kErrWaitEmpty);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            int row = -1;
            if (t >= 0) {
                row = a.map_rows;
                if (p >= 0 && p < a.s.num_pages)
                    row = (p * a.kv_heads + h) * a.s.page_size + t % a.s.page_size;
                else
                    flag_index(err_word);
            }
            const int count = frag_count(row);
            if (lane == 0)
                tc::mbar_arrive_expect_tx(&k_full[st], (uint32_t)(count * a.frag * 128 * kSubs));
            __syncwarp();
            if (row >= 0) {
                uint8_t *dst = smem + L::kK + (st * 2 + x) * L::kTile + span * 128;
                for (int c = 0; c < kSubs; c++)
                    tc::tma_load_2d(dst + c * kSubTile, &tmK, &k_full[st], c * 64, row);
            }
            __syncwarp();
            armed |= 1u << st;
            k_ph = (k_ph & ~(1u << st)) | (ph << st);
            if (++st == KS) {
                st = 0;
                ph ^= 1;
            }
        } while (more);
        if (lane == 0) {
            // drain our own loads (a no-op when every load was consumed; after an
            // abort the other half's warp may not have armed the phase: 10 ms, in
            // which any copy has landed)
            const uint64_t t0 = tc::globaltimer(), limit = ok ? kWaitBudgetNs : 10000000ull;
            for (int i = 0; i < KS; i++)
                if (armed >> i & 1)
                    while (!tc::mbar_try_wait(&k_full[i], k_ph >> i & 1) &&
                           tc::globaltimer() - t0 < limit) {
                    }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // ----------------------------------------------------------- MMA
            constexpr uint32_t idesc = tc::idesc_f16_f32(kKeys, R, false, false, kBf16);
            const uint32_t sK = tc::smem_u32(smem + L::kK), sQ = tc::smem_u32(smem + L::kQ);
            KeyWalk w = plan.start;
            int st = 0;
            uint32_t ph = 0, u = 0, n[2] = {0, 0};       // units; score tiles of each half
            bool ok = true;
            do {
                ok = tc::mbar_wait(&k_full[st], ph, abort_flag, err_word, kErrWaitFull);
                const int t_end = w.row_tiles(a), t1 = w.first_tile_1(a);
                for (int t = w.first_tile(a, 0); t < t_end && ok; t++, u++) {
                    const int qs = u % QS;
                    ok = tc::mbar_wait(&q_full[qs], (u / QS) & 1, abort_flag, err_word, kErrWaitFull);
                    const uint32_t qb = sQ + qs * L::kQTile;
                    for (int x = 0; x < 2 && ok; x++) {
                        if (x == 1 && t < t1) continue;
                        const int buf = x * 2 + (n[x] & 1);
                        ok = tc::mbar_wait(&s_empty[buf], ((n[x] >> 1) & 1) ^ 1, abort_flag, err_word,
                                           kErrWaitAccum);
                        if (!ok) break;
                        tc::tc_fence_after();
                        const uint32_t kb = sK + (st * 2 + x) * L::kTile;
#pragma unroll
                        for (int k = 0; k < D / 16; k++)
                            tc::mma_ss<tc::MmaKind::F16>(
                                tmem_base + buf * R,
                                tc::sdesc_kmajor_sw128(kb + (k >> 2) * kSubTile + (k & 3) * 32),
                                tc::sdesc_kmajor_sw128(qb + (k >> 2) * (R * 128) + (k & 3) * 32),
                                idesc, k > 0 ? 1u : 0u);
                        tc::mma_commit(&s_full[buf]);
                        n[x]++;
                    }
                    if (ok) tc::mma_commit(&q_empty[qs]);
                }
                if (!ok) break;
                tc::mma_commit(&k_empty[st]);
                if (++st == KS) {
                    st = 0;
                    ph ^= 1;
                }
            } while (w.next(a));
            if (n[0] > 0) {
                tc::mma_commit(drain);
                const uint64_t t0 = tc::globaltimer();
                while (!tc::mbar_try_wait(drain, 0) && tc::globaltimer() - t0 < kWaitBudgetNs) {
                }
            }
        }
    } else if (warp == 2) {
        // ------------------------------ query tiles, and the rows' lse * log2e
        constexpr int kPer = (R + 31) / 32;
        KeyWalk w = plan.start;
        float *sl = reinterpret_cast<float *>(smem + L::kLse);
        int *sn = reinterpret_cast<int *>(smem + L::kNone);
        uint32_t u = 0;
        // lane's rows of a tile: token and head
        int row_tok[kPer], row_at[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            row_tok[i] = (lane + 32 * i) / a.group;
            row_at[i] = row_tok[i] * a.heads + (lane + 32 * i) % a.group;
            if (lane + 32 * i >= a.tok * a.group) row_tok[i] = 0x7fffffff;   // no row
        }
        auto load = [&](int t, float (&z)[kPer]) {
            const float *base = a.lse + ((int64_t)(w.first + t * a.tok) * a.heads + w.h * a.group);
#pragma unroll
            for (int i = 0; i < kPer; i++)
                z[i] = row_tok[i] < w.q_len - t * a.tok ? base[row_at[i]] : INFINITY;
        };
        float z[kPer], zn[kPer];
        int t = w.first_tile(a, 0);
        bool more = true;
        load(t, z);
        while (more) {
            const int q_head = w.h * a.group, q_row = w.first + t * a.tok, qs = u % QS;
            // the next unit's values, while this one's place is waited for
            if (++t >= w.row_tiles(a)) {
                more = w.next(a);
                if (more) t = w.first_tile(a, 0);
            }
            if (more) load(t, zn);
            bool ok = tc::mbar_wait(&q_empty[qs], ((u / QS) & 1) ^ 1, abort_flag, err_word, kErrWaitEmpty);
            if (!__all_sync(0xffffffffu, ok)) break;
            if (lane == 0) {
                tc::mbar_arrive_expect_tx(&q_full[qs], (uint32_t)(a.tok * a.group * 128 * kSubs));
                for (int c = 0; c < kSubs; c++)
                    tc::tma_load_3d(smem + L::kQ + qs * L::kQTile + c * R * 128, &tmQ, &q_full[qs],
                                    c * 64, q_head, q_row);
            }
            u++;
            ok = tc::mbar_wait(&l_empty[(u - 1) & 3], (((u - 1) >> 2) & 1) ^ 1, abort_flag, err_word,
                               kErrWaitEmpty);
            if (!__all_sync(0xffffffffu, ok)) break;
            bool none = false;
#pragma unroll
            for (int i = 0; i < kPer; i++)
                if (lane + 32 * i < R) {
                    none |= z[i] == -INFINITY;
                    sl[((u - 1) & 3) * R + lane + 32 * i] = z[i] * 1.4426950408889634f;
                }
            none = __any_sync(0xffffffffu, none);
            if (lane == 0) sn[(u - 1) & 3] = none;
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&l_full[(u - 1) & 3]);
#pragma unroll
            for (int i = 0; i < kPer; i++) z[i] = zn[i];
        }
        if (lane == 0) {
            // drain our own loads
            const uint64_t t0 = tc::globaltimer();
            for (uint32_t i = u > QS ? u - QS : 0; i < u; i++)
                while (!tc::mbar_try_wait(&q_full[i % QS], (i / QS) & 1) &&
                       tc::globaltimer() - t0 < kWaitBudgetNs) {
                }
        }
    } else {
        // ------------------------------------------------------------- weights
        const int x = (warp - 4) >> 2, key = (warp & 3) * 32 + lane;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const float *sl = reinterpret_cast<const float *>(smem + L::kLse);
        const int *sn = reinterpret_cast<const int *>(smem + L::kNone);
        KeyWalk w = plan.start;
        uint32_t u = 0, n = 0;
        bool ok = true;
        do {
            const int t_end = w.row_tiles(a);
            const int t_mine = x == 0 ? w.first_tile(a, 0) : w.first_tile_1(a);
            const int kk = w.kt * kItemKeys + x * kKeys + key;
            const int before = a.s.causal ? kk - (w.kv_len - w.q_len) : 0;   // tokens that do not see kk
            float sum = 0.0f;
            for (int t = w.first_tile(a, 0); t < t_end; t++, u++) {
                const int lb = u & 3;
                // (also a half that skips the unit waits for its lse values: it
                // must not hand back a place that is not filled yet)
                ok = tc::mbar_wait(&l_full[lb], (u >> 2) & 1, abort_flag, err_word, kErrWaitFull);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (t >= t_mine) {
                    const int buf = x * 2 + (n & 1), none = sn[lb];
                    ok = tc::mbar_wait(&s_full[buf], (n >> 1) & 1, abort_flag, err_word, kErrWaitAccum);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc::tc_fence_after();
                    // rows lo <= r < hi of the tile count for this key
                    const int hi = min(a.tok, w.q_len - t * a.tok) * a.group;
                    const int lo = max(0, min(a.tok, before - t * a.tok)) * a.group;
                    const uint32_t s_addr = tmem_base + lane_base + buf * R;
                    const float *zl = sl + lb * R;
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (none != 0)
                        sum += add_weights_but<R>(s_addr, zl, a.scale_log2, lo, hi);
                    else if (__any_sync(0xffffffffu, lo > 0 || hi < R))
                        sum += add_weights<R, true>(s_addr, zl, a.scale_log2, lo, hi, acc);
                    else
                        sum += add_weights<R, false>(s_addr, zl, a.scale_log2, 0, R, acc);
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&s_empty[buf]);
                    n++;
                }
                if (lane == 0) tc::mbar_arrive(&l_empty[lb]);
            }
            if (!ok) break;
            if (kk < w.kv_len) {
                const int i = kk / a.s.page_size;
                const int page = a.s.table[(int64_t)w.b * a.s.max_pages + i];
                if (page >= 0 && page < a.s.num_pages)
                    atomicAdd(&a.scores[((int64_t)page * a.kv_heads + w.h) * a.s.page_size + kk -
                                        i * a.s.page_size],
                              sum);
            }
        } while (w.next(a));
    }

    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        tc::tmem_dealloc(tmem_base, kCols);
    }
}

template <typename T, int D, int R>
int launch_scores(Dev *d, const CUtensorMap &mq, const CUtensorMap &mk, const ScoresTc &a) {
    using L = ScSmem<D, R>;
    static_assert(L::kTotal <= 232448, "shared memory of one CTA");
    static bool attr_done[64] = {};
    if (!attr_done[d->ordinal & 63]) {
        if (int rc = check(cudaFuncSetAttribute(scores_tc_kernel<T, D, R>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                L::kTotal),
                           "cudaFuncSetAttribute(scores_tc)"))
            return rc;
        attr_done[d->ordinal & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)d->sms);
    cfg.blockDim = dim3(384);
    cfg.dynamicSmemBytes = L::kTotal;
    cfg.stream = d->stream;
    return check(cudaLaunchKernelEx(&cfg, scores_tc_kernel<T, D, R>, mq, mk, a), "launch scores_tc");
}

template <typename T, int D>
int launch_scores_rows(Dev *d, const CUtensorMap &mq, const CUtensorMap &mk, const ScoresTc &a, int rows) {
    if (rows == 16) return launch_scores<T, D, 16>(d, mq, mk, a);
    if (rows == 32) return launch_scores<T, D, 32>(d, mq, mk, a);
    return launch_scores<T, D, 128>(d, mq, mk, a);
}

}  // namespace

int launch_scores_tc(Dev *d, const PagedSeqs &s, int dtype, const void *q, const float *lse,
                     const void *k, float *scores, int max_q, int heads, int kv_heads, int dim,
                     float scale) {
    ScoresTc a;
    a.s = s;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.group = heads / kv_heads;
    const int64_t need = (int64_t)(max_q < 1 ? 1 : max_q) * a.group;
    // Query tiles of 16, 32 or 128 rows.  Measured (us, dim 128, 8 key heads): 64
    // sequences of 8192, 4 rows to a key head: 197 / 201 / 430; 16 of 4096, 32 rows: 48
    // / 42 / 62, 64 rows: 73 / 50 / 63, 80 rows: 85 / 64 / 63, 128 rows: 122 / 76 / 57.
    // A tile holds a token's heads.
    const int rows = need <= 16 ? 16 : need <= 64 && a.group <= 32 ? 32 : 128;
    a.tok = rows / a.group;
    const int low = s.page_size & -s.page_size;
    a.frag = low < kKeys ? low : kKeys;
    a.map_rows = s.num_pages * kv_heads * s.page_size;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.lse = lse;
    a.scores = scores;
    CUtensorMap mq, mk;
    if (int rc = make_query_map(&mq, q, s.total_q, heads, dim, a.group, a.tok)) return rc;
    if (int rc = make_page_map(&mk, k, a.map_rows, dim, a.frag)) return rc;
    note_mech(kMechTcgen05 | kMechTma);
    if (dtype == HEXCUDA_F16)
        return dim == 128 ? launch_scores_rows<__half, 128>(d, mq, mk, a, rows)
                          : launch_scores_rows<__half, 64>(d, mq, mk, a, rows);
    return dim == 128 ? launch_scores_rows<__nv_bfloat16, 128>(d, mq, mk, a, rows)
                      : launch_scores_rows<__nv_bfloat16, 64>(d, mq, mk, a, rows);
}

}  // namespace hx
