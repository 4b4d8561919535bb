// paged_pre.cu -- attention of chunks of new tokens over the paged cache
// (more than 32 query rows to a key head) on the tensor cores, queries on the
// M side.
//
// A work item is 2 x 128 query rows of one key head: with group = heads /
// kv_heads a tile holds tok = 128 / group tokens x group heads, so that the
// heads that share a key head also share its key and value loads (rows past
// tok * group are computed and dropped).  One softmax warpgroup per tile, one
// query row per thread, so the tensor pipe works for one tile while the other
// tile's warpgroup takes its exponentials; the order of the MMAs, which keeps
// the two sides half a step apart, the hand-over of P in two halves and the lazy
// reference maximum are those of the dense ping-pong kernel (attn_tc.cu).
// An item of one tile (at most 128 rows) would leave one warpgroup idle: there
// both take the key tiles in turn, each with a reference, a sum and an output
// of its own, and the first joins the two outputs, which lie side by side in
// tensor memory.
//
// A key tile is gathered page by page, one lane of a TMA warp per fragment.
// Values behind the last cached token are zeroed before they meet a weight of
// zero.  The batch is split evenly over the CTAs (paged_tc.cuh).
//
// Per CTA (one per SM), 384 threads in three warpgroups: warps 0 and 3 TMA of
// keys (and queries) and of values, warp 1 tensor memory and MMA issue,
// warpgroups 1 and 2 softmax of tiles a and b.
// TMEM: S_a [0,128), S_b [128,256), O_a [256,..), O_b behind it; P_x over S_x.
//
// Bound by the chain scores -> maximum -> exponentials -> P V of a key tile, which
// the other tile's overlaps but does not hide: 128 x 128 exponentials take 1024
// cycles of the MUFU, the two products 1024 (dim 128) of the tensor pipe.  Measured
// with the join: 4096 new tokens of 16384, 32 heads of 128 over 8 key heads: 1.00 ms,
// 960 TFLOP/s, tensor pipe 53 % busy; 11 sequences of up to 301 new tokens of up to
// 4099, 16 heads of 64: 74 us, a key tile of two query tiles taking some 3600 cycles.
//
// Every wait is bounded; see mbar_wait.
#include <math.h>

#include "paged_tc.cuh"

namespace hx {
namespace {

// The register file is split with setmaxnreg: the control warpgroup drops to
// kRegsCtl, the softmax warpgroups rise to kRegsSoftmax (a whole score row of
// 128 fp32 and its weights).
constexpr int kRegsCtl = 120;
constexpr int kRegsSoftmax = 192;
constexpr int kRegsPool = 128 * kRegsCtl + 256 * kRegsSoftmax;

template <int D>
struct PreSmem {
    static constexpr int kSubs = D / 64;
    static constexpr int kStages = D == 128 ? 2 : 4;
    static constexpr int kTile = kSubs * kSubTile;
    static constexpr int kQ = 0;                           // Q_a, Q_b
    static constexpr int kK = 2 * kTile;
    static constexpr int kV = kK + kStages * kTile;
    static constexpr int kPlan = kV + kStages * kTile;
    static constexpr int kWalk = (kPlan + (int)sizeof(PlanShared) + 15) / 16 * 16;   // a Walk per softmax warp
    static constexpr int kMl = (kWalk + 8 * (int)sizeof(Walk) + 15) / 16 * 16;       // [128][2]: tile b's, to be joined
    static constexpr int kBar = kMl + 128 * 8;
    // q_full, q_empty, s_full[2], p_full[2], p_half[2], pv_done[2], o_free[2],
    // joined, drain, k_full, k_empty, v_full, v_empty [stages]
    static constexpr int kNumBars = 14 + 4 * kStages;
    static constexpr int kTotal = kBar + kNumBars * 8 + 16 + 1024;
};

__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// What tile x does in segment w: its first token and number of tokens, and its
// key tiles start, start + step, .. < end.  `alt`: the item has one tile, whose
// key tiles the two sides take in turn.
struct Span {
    int t0, ntok, start, end, step;
    bool alt;
    __device__ __forceinline__ int count() const {
        return start < end ? (end - start + step - 1) / step : 0;
    }
};
__device__ __forceinline__ Span span_of(const PagedTc &a, const Walk &w, int x) {
    Span s;
    s.alt = w.q_len <= (2 * w.rt + 1) * a.tok;
    s.t0 = (2 * w.rt + (s.alt ? 0 : x)) * a.tok;
    s.ntok = min(a.tok, w.q_len - s.t0);
    s.start = w.j0 + (s.alt ? x : 0);
    s.step = s.alt ? 2 : 1;
    s.end = s.alt ? w.j1 : min(w.j1, tiles_to(a.s, w.kv_len, w.q_len, s.t0 + a.tok));
    return s;
}

template <typename T, int D>
__global__ void __launch_bounds__(384, 1)
    paged_pre_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const PagedTc a) {
    using L = PreSmem<D>;
    constexpr int kSubs = L::kSubs, S = L::kStages;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBar);
    uint64_t *q_full = bars, *q_empty = bars + 1, *s_full = bars + 2, *p_full = bars + 4;
    uint64_t *p_half = bars + 6, *pv_done = bars + 8, *o_free = bars + 10, *joined = bars + 12;
    uint64_t *drain = bars + 13;
    uint64_t *k_full = bars + 14, *k_empty = k_full + S, *v_full = k_empty + S, *v_empty = v_full + S;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::kNumBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int *odd_flag = abort_flag + 1;     // some value was not finite (settle_row)
    PlanShared &plan = *reinterpret_cast<PlanShared *>(smem + L::kPlan);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *err_word = a.s.err_word;
    const int item_tok = 2 * a.tok;
    tc::launch_dependents();

    if (threadIdx.x == 0) {
        tc::mbar_init(q_full, 1);
        tc::mbar_init(q_empty, 1);
        for (int x = 0; x < 2; x++) {
            tc::mbar_init(&s_full[x], 1);
            tc::mbar_init(&p_full[x], 4);
            tc::mbar_init(&p_half[x], 4);
            tc::mbar_init(&pv_done[x], 1);
            tc::mbar_init(&o_free[x], 4);
        }
        tc::mbar_init(joined, 4);
        tc::mbar_init(drain, 1);
        for (int i = 0; i < S; i++) {
            tc::mbar_init(&k_full[i], 1);
            tc::mbar_init(&k_empty[i], 1);
            tc::mbar_init(&v_full[i], 1);
            tc::mbar_init(&v_empty[i], 1);
        }
        *abort_flag = 0;
        *odd_flag = 0;
        tc::fence_mbar_init();
        tc::tma_prefetch_desc(&tmQ);
        tc::tma_prefetch_desc(&tmK);
        tc::tma_prefetch_desc(&tmV);
    }
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, 512);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    const bool any = plan_run<384, 5>(a, item_tok, plan);
    tc::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    constexpr uint32_t kColO = 256;

    if (warp < 4) {
      // warpgroup 0: one setmaxnreg for all four warps, then the roles
      tc::setmaxnreg_dec<kRegsCtl>();
      if (!any) {
        // nothing to do but free the tensor memory
      } else if (warp == 0 || warp == 3) {
        // ------------------------------------- TMA: keys and queries, values
        const bool keys = warp == 0;
        uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
        const CUtensorMap *map = keys ? &tmK : &tmV;
        uint8_t *ring = smem + (keys ? L::kK : L::kV);
        Walk w = plan.start;
        int seg = 0, st = 0;
        uint32_t ph = 0, armed = 0, last_ph = 0;
        bool ok = true, more = true;
        int j = w.j0;
        Frag f = frag_of(a, w, j, lane);
        while (more) {
            if (j == w.j0 && keys) {
                const Span sa = span_of(a, w, 0);
                ok = tc::mbar_wait(q_empty, (seg & 1) ^ 1, abort_flag, err_word, kErrWaitEmpty);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) {
                    const int tiles = sa.alt ? 1 : 2;
                    tc::mbar_arrive_expect_tx(q_full, (uint32_t)(tiles * a.tok * a.group * 128 * kSubs));
                    for (int x = 0; x < tiles; x++)
                        for (int c = 0; c < kSubs; c++)
                            tc::tma_load_3d(smem + L::kQ + x * L::kTile + c * kSubTile, &tmQ, q_full,
                                            c * 64, w.h * a.group, w.first + sa.t0 + x * a.tok);
                }
                seg++;
            }
            const Frag f_now = f;
            const int h = w.h;
            // the tile after this one, and its pages
            if (++j == w.j1) {
                more = w.next(a, item_tok);
                j = w.j0;
            }
            if (more) f = frag_of(a, w, j, lane);
            ok = tc::mbar_wait(&empty[st], ph ^ 1, abort_flag, err_word, kErrWaitEmpty);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int row = frag_row(a, f_now, h), count = frag_count(row);
            load_frags<kSubs>(a, ring + st * L::kTile, map, &full[st], row, count, lane);
            armed |= 1u << st;
            last_ph = (last_ph & ~(1u << st)) | (ph << st);
            if (++st == S) {
                st = 0;
                ph ^= 1;
            }
        }
        if (lane == 0) {
            // drain our own loads (a no-op when every load was consumed)
            const uint64_t t0 = tc::globaltimer();
            auto drain_wait = [&](uint64_t *bar, uint32_t par) {
                while (!tc::mbar_try_wait(bar, par) && tc::globaltimer() - t0 < kWaitBudgetNs) {
                }
            };
            if (seg > 0) drain_wait(q_full, (seg - 1) & 1);
            for (int i = 0; i < S; i++)
                if (armed >> i & 1) drain_wait(&full[i], last_ph >> i & 1);
        }
      } else if (warp == 1) {
        if (lane == 0) {
            // ----------------------------------------------------------- MMA
            constexpr uint32_t idesc_s = tc::idesc_f16_f32(128, kKeys, false, false, kBf16);
            constexpr uint32_t idesc_o = tc::idesc_f16_f32(128, D, true, false, kBf16);
            const uint32_t sQ = tc::smem_u32(smem + L::kQ);
            const uint32_t sK = tc::smem_u32(smem + L::kK);
            const uint32_t sV = tc::smem_u32(smem + L::kV);
            // (the thread's own instructions are on the critical path between a
            // softmax and its next scores: descriptors are made once, sides are
            // compile-time constants)
            const uint64_t dq = tc::sdesc_kmajor_sw128(sQ), dk = tc::sdesc_kmajor_sw128(sK);
            const uint64_t dv = tc::sdesc_mnmajor_sw128(sV, kSubTile, 1024);
            constexpr uint64_t kTileStep = L::kTile >> 4;
            const std::integral_constant<int, 0> A{};
            const std::integral_constant<int, 1> B{};
            Walk w = plan.start;
            int seg = 0;
            uint32_t n[2] = {0, 0}, segs[2] = {0, 0};    // key tiles and segments of each side so far
            int k_st = 0, v_st = 0;                      // the rings' next stages and phases
            uint32_t k_ph = 0, v_ph = 0;
            bool ok = true;
            auto wait_k = [&]() {
                ok = ok && tc::mbar_wait(&k_full[k_st], k_ph, abort_flag, err_word, kErrWaitFull);
                tc::tc_fence_after();
            };
            auto wait_v = [&]() {
                ok = ok && tc::mbar_wait(&v_full[v_st], v_ph, abort_flag, err_word, kErrWaitFull);
                tc::tc_fence_after();
            };
            auto done_k = [&]() {
                tc::mma_commit(&k_empty[k_st]);
                if (++k_st == S) {
                    k_st = 0;
                    k_ph ^= 1;
                }
            };
            auto done_v = [&]() {
                tc::mma_commit(&v_empty[v_st]);
                if (++v_st == S) {
                    v_st = 0;
                    v_ph ^= 1;
                }
            };
            // S_x = Q K^T of the key tile in stage k_st; q: the query tile
            auto issue_s = [&](auto X, int q) {
                constexpr int x = decltype(X)::value;
                const uint64_t da = dq + q * kTileStep, db = dk + k_st * kTileStep;
#pragma unroll
                for (int k = 0; k < D / 16; k++) {
                    constexpr int kSub4 = kSubTile >> 4;
                    tc::mma_ss<tc::MmaKind::F16>(tmem_base + x * 128, da + (k >> 2) * kSub4 + (k & 3) * 2,
                                                 db + (k >> 2) * kSub4 + (k & 3) * 2, idesc_s,
                                                 k > 0 ? 1u : 0u);
                }
                tc::mma_commit(&s_full[x]);
            };
            // O_x += P_x V of the key tile in stage v_st, in two halves of 64 keys:
            // the first runs while the softmax warps still compute the second of P
            auto issue_pv = [&](auto X, bool first) {
                constexpr int x = decltype(X)::value;
                const uint32_t c = n[x]++ & 1;
                const uint64_t db = dv + v_st * kTileStep;
                ok = ok && tc::mbar_wait(&p_half[x], c, abort_flag, err_word, kErrWaitFull) &&
                     (!first || tc::mbar_wait(&o_free[x], (segs[x] & 1) ^ 1, abort_flag, err_word,
                                              kErrWaitAccum));
                if (!ok) return;
                tc::tc_fence_after();
#pragma unroll
                for (int k = 0; k < 4; k++)
                    tc::mma_ts_f16(tmem_base + kColO + x * D, tmem_base + x * 128 + k * 8,
                                   db + k * (2048 >> 4), idesc_o, (!first || k > 0) ? 1u : 0u);
                ok = tc::mbar_wait(&p_full[x], c, abort_flag, err_word, kErrWaitFull);
                if (!ok) return;
                tc::tc_fence_after();
#pragma unroll
                for (int k = 4; k < 8; k++)
                    tc::mma_ts_f16(tmem_base + kColO + x * D, tmem_base + x * 128 + k * 8,
                                   db + k * (2048 >> 4), idesc_o, 1u);
                tc::mma_commit(&pv_done[x]);
            };
            do {
                const Span sa = span_of(a, w, 0);
                const int len = w.j1 - w.j0;
                ok = tc::mbar_wait(q_full, seg & 1, abort_flag, err_word, kErrWaitFull);
                if (sa.alt) {
                    // one query tile, the key tiles in turn
                    auto score = [&](auto X, int i) {
                        wait_k();
                        if (!ok) return;
                        issue_s(X, 0);
                        done_k();
                        if (i == len - 1) tc::mma_commit(q_empty);
                    };
                    auto step = [&](auto X, int i) {
                        wait_v();
                        issue_pv(X, i < 2);
                        if (!ok) return;
                        done_v();
                        if (i + 2 < len) score(X, i + 2);
                    };
                    score(A, 0);
                    if (len > 1) score(B, 1);
                    for (int i = 0; i < len && ok; i += 2) {
                        step(A, i);
                        if (i + 1 < len) step(B, i + 1);
                    }
                    segs[0]++;
                    if (len > 1) segs[1]++;
                } else {
                    // both query tiles; a's key tiles end first, if not together
                    // with b's
                    const int len_a = sa.end - w.j0;
                    wait_k();
                    if (ok && len_a > 0) issue_s(A, 0);
                    if (ok) {
                        issue_s(B, 1);
                        done_k();
                        if (len == 1) tc::mma_commit(q_empty);
                    }
                    for (int i = 0; i < len && ok; i++) {
                        wait_v();
                        bool k_ready = false;
                        if (i < len_a) {
                            issue_pv(A, i == 0);
                            if (i + 1 < len_a) {
                                wait_k();
                                k_ready = true;
                                if (ok) issue_s(A, 0);
                            }
                        }
                        issue_pv(B, i == 0);
                        if (!ok) break;
                        done_v();
                        if (i + 1 < len) {
                            if (!k_ready) wait_k();
                            if (!ok) break;
                            issue_s(B, 1);
                            done_k();
                            if (i + 1 == len - 1) tc::mma_commit(q_empty);
                        }
                    }
                    if (len_a > 0) segs[0]++;
                    segs[1]++;
                }
                seg++;
            } while (ok && w.next(a, item_tok));
            tc::mma_commit(drain);
            const uint64_t t0 = tc::globaltimer();
            while (!tc::mbar_try_wait(drain, 0) && tc::globaltimer() - t0 < kWaitBudgetNs) {
            }
        }
      }
    } else {
        // ------------------------------------------------------- softmax x
        tc::setmaxnreg_inc<kRegsSoftmax>();
        const int x = (warp - 4) >> 2;
        const int q = warp & 3;
        const int row = q * 32 + lane;
        const uint32_t lane_base = (uint32_t)(q * 32) << 16;
        const uint32_t s_addr = tmem_base + lane_base + x * 128;
        const uint32_t o_addr = tmem_base + lane_base + kColO + x * D;
        float2 *ml_b = reinterpret_cast<float2 *>(smem + L::kMl);
        Walk *wp = reinterpret_cast<Walk *>(smem + L::kWalk) + (warp - 4);
        uint32_t n = 0, n_other = 0, joins = 0;  // key tiles so far, of the other side; joined segments
        int g0 = 0;               // key tiles of the CTA's earlier segments (the value ring)
        bool more = any;
        if (any && lane == 0) *wp = plan.start;
        __syncwarp();
        while (more) {
            // (what the segment's end needs is worked out again there: the loop
            // has no registers to spare)
            int left, rest, rest0, step_keys;   // key tiles; keys that the row, the tile's first row still see
            {
                const Span s = span_of(a, *wp, x);
                left = s.count();
                step_keys = s.step * kKeys;
                rest = min(wp->kv_len, seen_by(a.s, wp->kv_len, wp->q_len, s.t0 + row / a.group)) -
                       s.start * kKeys;
                rest0 = min(wp->kv_len, seen_by(a.s, wp->kv_len, wp->q_len, s.t0)) - s.start * kKeys;
            }
            bool first = true;
            float m_ref = -INFINITY, l = 0.0f;
            bool ok = true;
            for (; left > 0; left--, n++, rest -= step_keys, rest0 -= step_keys, first = false) {
                ok = tc::mbar_wait(&s_full[x], n & 1, abort_flag, err_word, kErrWaitAccum);
                if (!__all_sync(0xffffffffu, ok)) break;
                tc::tc_fence_after();
                if (rest0 < kKeys) {
                    // values that no weight of zero may meet, by each side before it
                    // hands its P over (all four warps have then).  The rows that b
                    // would settle a has settled, if it takes the tile, before its own
                    // P V and then b's read it: b writes the same zeros once more, or
                    // nothing.  (Behind the scores: they were begun after the P V of the
                    // tile that had the value stage before, so that the stage's barrier
                    // is at most one phase behind and its parity is this tile's.)
                    const Span s = span_of(a, *wp, x);
                    const int j = s.start + (s.count() - left) * s.step, gk = g0 + (j - wp->j0);
                    const int valid = wp->kv_len - j * kKeys;
                    if (valid < kKeys || rest0 < valid) {
                        ok = tc::mbar_wait(&v_full[gk % S], (gk / S) & 1, abort_flag, err_word,
                                           kErrWaitFull);
                        if (!__all_sync(0xffffffffu, ok)) break;
                        settle_row<T, kSubs>(smem + L::kV + gk % S * L::kTile, row, rest0, valid,
                                             odd_flag);
                        tc::fence_proxy_async_smem();
                    }
                }
                // the whole score row into registers: four loads, one wait
                uint32_t sr[4][32];
#pragma unroll
                for (int cc = 0; cc < 4; cc++) tc::tmem_ld_32x32b_x32(s_addr + cc * 32, sr[cc]);
                tc::tmem_ld_wait(sr[0]);
                tc::reg_fence(sr[1]);
                tc::reg_fence(sr[2]);
                tc::reg_fence(sr[3]);
                if (rest0 < kKeys) {
#pragma unroll
                    for (int cc = 0; cc < 4; cc++)
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (cc * 32 + e >= rest) sr[cc][e] = __float_as_uint(-INFINITY);
                }
                // row max over the 128 raw scores (scale folded later)
                float mx[8];
#pragma unroll
                for (int u = 0; u < 8; u++) mx[u] = -INFINITY;
#pragma unroll
                for (int cc = 0; cc < 4; cc++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        mx[i & 7] = max3(mx[i & 7], __uint_as_float(sr[cc][2 * i]),
                                         __uint_as_float(sr[cc][2 * i + 1]));
                const float mt = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], mx[4], mx[5]),
                                      fmaxf(mx[6], mx[7])) *
                                 a.scale_log2;
                const float m_new = fmaxf(m_ref, mt);
                if (first) {
                    m_ref = m_new;
                } else {
                    // Lazy rescale: the reference max moves only when the row
                    // max rose by more than 8 (P stays below 2^8 otherwise).
                    const bool need = m_new > m_ref + 8.0f;
                    if (__any_sync(0xffffffffu, need)) {
                        ok = tc::mbar_wait(&pv_done[x], (n - 1) & 1, abort_flag, err_word,
                                           kErrWaitAccum);
                        if (!__all_sync(0xffffffffu, ok)) break;
                        tc::tc_fence_after();
                        const float corr = need ? tc::ex2(m_ref - m_new) : 1.0f;
#pragma unroll 1
                        for (int cc = 0; cc < D / 32; cc++) {
                            uint32_t o[32];
                            tc::tmem_ld_32x32b_x32(o_addr + cc * 32, o);
                            tc::tmem_ld_wait(o);
#pragma unroll
                            for (int e = 0; e < 32; e++)
                                o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                            tc::tmem_st_32x32b_x32(o_addr + cc * 32, o);
                        }
                        tc::tmem_st_wait();
                        if (need) {
                            l *= corr;
                            m_ref = m_new;
                        }
                    }
                }
                // P = 2^(s*scale*log2e - m_ref) from the registers, as 16-bit
                // pairs over S columns 16cc..16cc+15; the row sum in four
                // packed pairs.  A row that sees nothing yet has no reference.
                uint64_t acc2[4] = {0, 0, 0, 0};
                const float nm = m_ref == -INFINITY ? 0.0f : -m_ref;
                const uint64_t sl2 = pair(a.scale_log2, a.scale_log2), nm2 = pair(nm, nm);
#pragma unroll
                for (int cc = 0; cc < 4; cc++) {
                    if (cc == 2) {
                        // keys 0..63 of P are in TMEM: hand them to the MMA warp
                        tc::tmem_st_wait();
                        tc::tc_fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&p_half[x]);
                    }
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        float a0, a1;
                        unpair(fma_pair(pair(__uint_as_float(sr[cc][2 * e]),
                                             __uint_as_float(sr[cc][2 * e + 1])),
                                        sl2, nm2),
                               a0, a1);
                        const float p0 = tc::ex2(a0), p1 = tc::ex2(a1);
                        acc2[e & 3] = add_pair(acc2[e & 3], pair(p0, p1));
                        pk[e] = pack2<T>(p0, p1);
                    }
                    tc::tmem_st_32x32b_x16(s_addr + cc * 16, pk);
                }
                tc::tmem_st_wait();
                {
                    float s0, s1, s2, s3, s4, s5, s6, s7;
                    unpair(acc2[0], s0, s1);
                    unpair(acc2[1], s2, s3);
                    unpair(acc2[2], s4, s5);
                    unpair(acc2[3], s6, s7);
                    l += ((s0 + s1) + (s2 + s3)) + ((s4 + s5) + (s6 + s7));
                }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&p_full[x]);
            }
            if (!__all_sync(0xffffffffu, ok)) break;
            // ---- end of the segment
            const Span s = span_of(a, *wp, x);
            const int j0 = wp->j0, tok_row = row / a.group;
            const int count_other = span_of(a, *wp, x ^ 1).count();
            const bool used = s.start < s.end;
            if (used) {
                ok = tc::mbar_wait(&pv_done[x], (n - 1) & 1, abort_flag, err_word, kErrWaitAccum);
                if (!__all_sync(0xffffffffu, ok)) break;
                tc::tc_fence_after();
            }
            float m = m_ref, sum = l, w_own = 1.0f, w_b = 0.0f;
            n_other += count_other;
            bool write = true;
            if (s.alt && wp->j1 - j0 > 1) {
                if (x == 1) {
                    // (the P V it waited for had waited for o_free: the last
                    // segment's values have been read)
                    ml_b[row] = make_float2(m_ref, l);
                    tc::tc_fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(joined);
                } else {
                    ok = tc::mbar_wait(joined, joins & 1, abort_flag, err_word, kErrWaitOther) &&
                         tc::mbar_wait(&pv_done[1], (n_other - 1) & 1, abort_flag, err_word, kErrWaitAccum);
                    if (!__all_sync(0xffffffffu, ok)) break;
                    tc::tc_fence_after();
                    const float2 b = ml_b[row];
                    m = fmaxf(m_ref, b.x);
                    const float ref = m == -INFINITY ? 0.0f : m;
                    w_own = tc::ex2(m_ref - ref);
                    w_b = tc::ex2(b.x - ref);
                    sum = l * w_own + b.y * w_b;
                }
                joins++;
            }
            if (s.alt && x == 1) write = false;
            const bool whole = j0 == 0 && wp->j1 == wp->nt;
            const bool live = tok_row < s.ntok && row < a.tok * a.group;
            const size_t prow = ((size_t)blockIdx.x * 2 + (j0 == 0 ? 1 : 0)) * kPartRows + x * 128 + row;
            const int64_t orow = (int64_t)(wp->first + s.t0 + tok_row) * a.heads + wp->h * a.group +
                                 row % a.group;
            if (write && used) {
                const bool both = s.alt && wp->j1 - j0 > 1;
                const float inv = !whole ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
                const float f_own = w_own * inv, f_b = w_b * inv;
#pragma unroll 1
                for (int cc = 0; cc < D / 32; cc++) {
                    uint32_t o[32];
                    tc::tmem_ld_32x32b_x32(o_addr + cc * 32, o);
                    tc::tmem_ld_wait(o);
#pragma unroll
                    for (int e = 0; e < 32; e++)
                        o[e] = __float_as_uint(__uint_as_float(o[e]) * f_own);
                    if (both) {
                        uint32_t ob[32];
                        tc::tmem_ld_32x32b_x32(o_addr + D + cc * 32, ob);
                        tc::tmem_ld_wait(ob);
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            o[e] = __float_as_uint(__uint_as_float(o[e]) + __uint_as_float(ob[e]) * f_b);
                    }
                    if (!live) continue;
                    if (whole) {
                        uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + orow * D +
                                                               cc * 32);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            uint32_t v[4];
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                v[i] = pack2<T>(__uint_as_float(o[8 * e + 2 * i]),
                                                __uint_as_float(o[8 * e + 2 * i + 1]));
                            dst[e] = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                    } else {
                        // (a row's neighbours are four columns of the next row: a
                        // warp stores 512 bytes in one piece)
                        uint4 *dst = reinterpret_cast<uint4 *>(a.part_o) +
                                     (prow - x * 128 - row) * (D / 4) + x * 128 + row;
#pragma unroll
                        for (int e = 0; e < 8; e++)
                            dst[(cc * 8 + e) * kPartRows] =
                                make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    tc::mbar_arrive(&o_free[x]);
                    if (both) tc::mbar_arrive(&o_free[1]);
                }
            }
            if (live && write) {
                if (!whole) {
                    reinterpret_cast<float2 *>(a.part_ml)[prow] = make_float2(m, sum);
                } else if (a.lse) {
                    a.lse[orow] = sum == 0.0f ? -INFINITY : (m + log2f(sum)) * 0.6931471805599453f;
                }
            }
            g0 += wp->j1 - j0;
            __syncwarp();
            if (lane == 0) {
                const Walk last = *wp;
                more = wp->next(a, item_tok);
                if (!more && warp == 4) note_parts(a, plan, last, item_tok);
            }
            more = __shfl_sync(0xffffffffu, (int)more, 0) != 0;
            __syncwarp();
        }
    }

    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        tc::tmem_dealloc(tmem_base, 512);
    }
    if (threadIdx.x == 0) a.recs[blockIdx.x].odd = *odd_flag;
    if (warp >= 4 && *odd_flag && !*abort_flag)
        mend_items<T, D>(a, plan.start, item_tok, warp - 4);
}

template <typename T, int D>
int launch_pre(Dev *d, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
               const PagedTc &a) {
    using L = PreSmem<D>;
    static_assert(L::kTotal <= 232448, "shared memory of one CTA");
    static bool attr_done[64] = {};
    if (!attr_done[d->ordinal & 63]) {
        auto kern = paged_pre_kernel<T, D>;
        if (int rc = check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                L::kTotal),
                           "cudaFuncSetAttribute(paged_pre)"))
            return rc;
        // setmaxnreg.inc draws on the registers of the launch: a build with
        // fewer would leave it waiting, so refuse it
        cudaFuncAttributes fa;
        if (int rc = check(cudaFuncGetAttributes(&fa, kern), "cudaFuncGetAttributes(paged_pre)"))
            return rc;
        if (fa.numRegs * 384 < kRegsPool)
            return fail(HEXCUDA_ERR_CUDA, "paged_pre_kernel built with %d registers, %d needed",
                        fa.numRegs, (kRegsPool + 383) / 384);
        attr_done[d->ordinal & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)d->sms);
    cfg.blockDim = dim3(384);
    cfg.dynamicSmemBytes = L::kTotal;
    cfg.stream = d->stream;
    return check(cudaLaunchKernelEx(&cfg, paged_pre_kernel<T, D>, mq, mk, mv, a), "launch paged_pre");
}

}  // namespace

int launch_paged_pre(Dev *d, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
                     PagedTc &a, int dtype, int dim) {
    if (dtype == HEXCUDA_F16)
        return dim == 128 ? launch_pre<__half, 128>(d, mq, mk, mv, a)
                          : launch_pre<__half, 64>(d, mq, mk, mv, a);
    return dim == 128 ? launch_pre<__nv_bfloat16, 128>(d, mq, mk, mv, a)
                      : launch_pre<__nv_bfloat16, 64>(d, mq, mk, mv, a);
}

}  // namespace hx
