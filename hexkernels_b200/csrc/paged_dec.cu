// paged_dec.cu -- attention of a few new tokens per sequence over the paged
// cache (decoding: at most 32 query rows share a key head) on the tensor
// cores, keys on the M side.
//
// A decode step reads every cached key and value once and does little with
// them, so it is bound by HBM; the 128-row MMA tile is spent on keys, not on
// the few queries:
//     S^T [128 keys x N rows] = K Q^T      A = K as it lies in the pages
//     O^T [D x N rows]       += V^T P^T    A = V as it lies (MN-major)
// with N = 16 or 32 query rows (tokens x heads of one key head).  A softmax
// thread owns one key and half of the rows: it reads its N / 2 scores from
// tensor memory, subtracts the rows' reference maxima, takes 2^x, adds to its
// own partial sums and writes its half of P^T's row (N contiguous 16-bit values
// a key, the MN-major B operand) to shared memory.  Maxima over keys are only
// needed when some score exceeds its row's reference by 2^8 (or at an item's
// first tile); a vote per tile finds that out, then the reference moves and O^T is
// rescaled.  Row sums are reduced over the threads once per item.  P is rounded to
// the element type, at most 2^8 and so never infinite in fp16; the sums are of the
// weights before that rounding.
//
// Per CTA (one per SM), 384 threads: warps 0 and 3 TMA of keys and of values,
// one lane per page fragment; warps 1 and 2 issue the MMAs of S^T and of O^T
// (two warps, because one thread's waits and issues, some 90 cycles each, added
// up to more than the tile's loads); two softmax warpgroups, one for each half
// of the rows, which know nothing of one another.  Key and value tiles of 128
// tokens go through rings of 3 stages (dim 128; 6 at dim 64), 192 KB of loads in
// flight per SM.
//
// Measured with the join: 96 sequences of up to 16384 tokens, 32 heads of 128 over
// 8 key heads: 493 to 504 us from box to box for 3.26 GB, 6.5 to 6.6 TB/s, what a copy
// reaches; one sequence of 777: 14.5 to 16, the latency of a plan (4500 cycles), one chain
// of loads and MMAs, and the join.
//
// Every wait is bounded; see mbar_wait.
#include <math.h>

#include "paged_tc.cuh"

namespace hx {
namespace {

template <int D, int N>
struct PagedDecSmem {
    static constexpr int kSubs = D / 64;
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr int kTile = kSubs * kSubTile;
    static constexpr int kQTile = kSubs * N * 128;
    static constexpr int kK = 0;
    static constexpr int kV = kK + kStages * kTile;
    static constexpr int kQ = kV + kStages * kTile;        // 2 buffers
    static constexpr int kP = kQ + 2 * kQTile;             // 2 buffers of 128 x N
    static constexpr int kRed = kP + 2 * kKeys * N * 2;    // [4][N] maxima or sums, [N] 1 / sum
    static constexpr int kPlan = kRed + 5 * N * 4;
    static constexpr int kBar = (kPlan + (int)sizeof(PlanShared) + 15) / 16 * 16;
    // q_full[2], q_empty[2], s_full[2], s_empty[2], p_full[2], pv_done[2],
    // o_free, drain[2], k_full, k_empty, v_full, v_empty [stages]
    static constexpr int kNumBars = 15 + 4 * kStages;
    static constexpr int kTotal = kBar + kNumBars * 8 + 16 + 1024;
};

// Or of a condition over the 128 threads of a softmax warpgroup (its named
// barrier).
__device__ __forceinline__ bool vote_or(int barrier, bool p) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %2, 0;\n\t"
        "barrier.cta.red.or.pred q, %1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(barrier), "r"((uint32_t)p)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ void softmax_sync(int barrier) {
    asm volatile("barrier.cta.sync %0, 128;" ::"r"(barrier) : "memory");
}

// C per-lane values (8 or 16) reduced over the warp; lane l gets column l * C / 32.
template <int C, bool MAX>
__device__ __forceinline__ float reduce_columns(float (&v)[C], int lane) {
    int o = 16;
#pragma unroll
    for (int n = C / 2; n > 0; n >>= 1, o >>= 1) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int i = 0; i < n; i++) {
            const float keep = up ? v[i + n] : v[i], send = up ? v[i] : v[i + n];
            const float got = __shfl_xor_sync(0xffffffffu, send, o);
            v[i] = MAX ? fmaxf(keep, got) : keep + got;
        }
    }
    for (; o > 0; o >>= 1) {
        const float got = __shfl_xor_sync(0xffffffffu, v[0], o);
        v[0] = MAX ? fmaxf(v[0], got) : v[0] + got;
    }
    return v[0];
}

__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&r)[8]) {
    tc::tmem_ld_32x32b_x8(taddr, r);
    tc::tmem_ld_wait(r);
}
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&r)[16]) {
    tc::tmem_ld_32x32b_x16(taddr, r);
    tc::tmem_ld_wait(r);
}
__device__ __forceinline__ void store_columns(uint32_t taddr, const uint32_t (&r)[8]) {
    tc::tmem_st_32x32b_x8(taddr, r);
    tc::tmem_st_wait();
}
__device__ __forceinline__ void store_columns(uint32_t taddr, const uint32_t (&r)[16]) {
    tc::tmem_st_32x32b_x16(taddr, r);
    tc::tmem_st_wait();
}

// Waits (bounded) for every MMA that this thread has issued.
__device__ __forceinline__ void mma_drain(uint64_t *bar) {
    tc::mma_commit(bar);
    const uint64_t t0 = tc::globaltimer();
    while (!tc::mbar_try_wait(bar, 0) && tc::globaltimer() - t0 < kWaitBudgetNs) {
    }
}

template <typename T, int D, int N>
__global__ void __launch_bounds__(384, 1)
    paged_dec_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const PagedTc a) {
    using L = PagedDecSmem<D, N>;
    constexpr int kSubs = L::kSubs, S = L::kStages;
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBar);
    uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *s_empty = bars + 6;
    uint64_t *p_full = bars + 8, *pv_done = bars + 10, *o_free = bars + 12, *drain = bars + 13;
    uint64_t *k_full = bars + 15, *k_empty = k_full + S, *v_full = k_empty + S, *v_empty = v_full + S;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::kNumBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int *odd_flag = abort_flag + 1;     // some value was not finite (settle_row)
    PlanShared &plan = *reinterpret_cast<PlanShared *>(smem + L::kPlan);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *err_word = a.s.err_word;
    tc::launch_dependents();

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            tc::mbar_init(&q_full[i], 1);
            tc::mbar_init(&q_empty[i], 1);
            tc::mbar_init(&s_full[i], 1);
            tc::mbar_init(&s_empty[i], 8);
            tc::mbar_init(&p_full[i], 8);
            tc::mbar_init(&pv_done[i], 1);
        }
        tc::mbar_init(o_free, 8);
        tc::mbar_init(&drain[0], 1);
        tc::mbar_init(&drain[1], 1);
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
    constexpr uint32_t kCols = N == 16 ? 64 : 128;   // S0, S1, O of N columns each
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, kCols);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    const bool any = plan_run<384, 0>(a, a.tok, plan);
    tc::tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tmem_o = tmem_base + 2 * N;

    if (!any) {
        // nothing to do but free the tensor memory
    } else if (warp == 0 || warp == 3) {
        // ------------------------------------------ TMA: keys (and Q), values
        // (two warps, because a page of 16 tokens makes 32 loads of a tile, and
        // the loads that one warp can start were the bound)
        const bool keys = warp == 0;
        uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
        const CUtensorMap *map = keys ? &tmK : &tmV;
        uint8_t *ring = smem + (keys ? L::kK : L::kV);
        Walk w = plan.start;
        int seg = 0, st = 0;
        uint32_t ph = 0, armed_q = 0, armed = 0, q_ph = 0, last_ph = 0;     // last loads
        bool ok = true, more = true;
        int j = w.j0;
        Frag f = frag_of(a, w, j, lane);
        while (more) {
            const Frag f_now = f;
            const int h = w.h;
            const bool first = j == w.j0;
            const int q_row = w.first + w.rt * a.tok;
            // the tile after this one, and its pages
            if (++j == w.j1) {
                more = w.next(a, a.tok);
                j = w.j0;
            }
            if (more) f = frag_of(a, w, j, lane);
            if (first && keys) {
                const int qb = seg & 1;
                ok = tc::mbar_wait(&q_empty[qb], ((seg >> 1) & 1) ^ 1, abort_flag, err_word, kErrWaitEmpty);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) {
                    tc::mbar_arrive_expect_tx(&q_full[qb], (uint32_t)(a.tok * a.group * 128 * kSubs));
                    for (int c = 0; c < kSubs; c++)
                        tc::tma_load_3d(smem + L::kQ + qb * L::kQTile + c * N * 128, &tmQ, &q_full[qb],
                                        c * 64, h * a.group, q_row);
                }
                armed_q |= 1u << qb;
                q_ph = (q_ph & ~(1u << qb)) | (((uint32_t)(seg >> 1) & 1u) << qb);
                seg++;
            }
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
            for (int i = 0; i < 2; i++)
                if (armed_q >> i & 1) drain_wait(&q_full[i], q_ph >> i & 1);
            for (int i = 0; i < S; i++)
                if (armed >> i & 1) drain_wait(&full[i], last_ph >> i & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            // -------------------------------------------------- MMA, S^T = K Q^T
            constexpr uint32_t idesc = tc::idesc_f16_f32(kKeys, N, false, false, kBf16);
            const uint32_t sK = tc::smem_u32(smem + L::kK), sQ = tc::smem_u32(smem + L::kQ);
            Walk w = plan.start;
            int seg = 0, st = 0;
            uint32_t ph = 0, g = 0;
            bool ok = true;
            do {
                const int qb = seg & 1;
                ok = tc::mbar_wait(&q_full[qb], (seg >> 1) & 1, abort_flag, err_word, kErrWaitFull);
                for (int j = w.j0; j < w.j1 && ok; j++, g++) {
                    const int buf = g & 1;
                    ok = tc::mbar_wait(&k_full[st], ph, abort_flag, err_word, kErrWaitFull) &&
                         tc::mbar_wait(&s_empty[buf], ((g >> 1) & 1) ^ 1, abort_flag, err_word,
                                       kErrWaitAccum);
                    if (!ok) break;
                    tc::tc_fence_after();
                    const uint32_t kb = sK + st * L::kTile, qt = sQ + qb * L::kQTile;
#pragma unroll
                    for (int k = 0; k < D / 16; k++)
                        tc::mma_ss<tc::MmaKind::F16>(
                            tmem_base + buf * N,
                            tc::sdesc_kmajor_sw128(kb + (k >> 2) * kSubTile + (k & 3) * 32),
                            tc::sdesc_kmajor_sw128(qt + (k >> 2) * (N * 128) + (k & 3) * 32), idesc,
                            k > 0 ? 1u : 0u);
                    tc::mma_commit(&k_empty[st]);
                    tc::mma_commit(&s_full[buf]);
                    if (j == w.j1 - 1) tc::mma_commit(&q_empty[qb]);
                    if (++st == S) {
                        st = 0;
                        ph ^= 1;
                    }
                }
                seg++;
            } while (ok && w.next(a, a.tok));
            mma_drain(&drain[0]);
        }
    } else if (warp == 2) {
        if (lane == 0) {
            // ------------------------------------------------ MMA, O^T += V^T P^T
            constexpr uint32_t idesc = tc::idesc_f16_f32(128, N, true, true, kBf16);
            const uint32_t sV = tc::smem_u32(smem + L::kV), sP = tc::smem_u32(smem + L::kP);
            Walk w = plan.start;
            int seg = 0, st = 0;
            uint32_t ph = 0, g = 0;
            bool ok = true;
            do {
                for (int j = w.j0; j < w.j1 && ok; j++, g++) {
                    const int buf = g & 1;
                    const bool first = j == w.j0;
                    ok = tc::mbar_wait(&v_full[st], ph, abort_flag, err_word, kErrWaitFull) &&
                         (!first || tc::mbar_wait(o_free, (seg & 1) ^ 1, abort_flag, err_word,
                                                  kErrWaitAccum)) &&
                         tc::mbar_wait(&p_full[buf], (g >> 1) & 1, abort_flag, err_word, kErrWaitFull);
                    if (!ok) break;
                    tc::tc_fence_after();
                    const uint32_t vb = sV + st * L::kTile, pb = sP + buf * (kKeys * N * 2);
#pragma unroll
                    for (int k = 0; k < kKeys / 16; k++)
                        // (dim 64: the second 64 of the 128 rows repeat the first, unread)
                        tc::mma_ss<tc::MmaKind::F16>(
                            tmem_o, tc::sdesc_mnmajor_sw128(vb + k * 2048, D == 128 ? kSubTile : 0, 1024),
                            tc::sdesc_mnmajor_narrow<N * 2>(pb + k * 16 * N * 2), idesc,
                            (!first || k > 0) ? 1u : 0u);
                    tc::mma_commit(&v_empty[st]);
                    tc::mma_commit(&pv_done[buf]);
                    if (++st == S) {
                        st = 0;
                        ph ^= 1;
                    }
                }
                seg++;
            } while (ok && w.next(a, a.tok));
            mma_drain(&drain[1]);
        }
    } else if (warp >= 4) {
        // ----------------------------------------------------------- softmax
        // rows n0 .. n0 + C - 1 of the tile, barrier 1 + x
        constexpr int C = N / 2;
        const int x = (warp - 4) >> 2, n0 = x * C, bar = 1 + x;
        const int qw = warp & 3, key = qw * 32 + lane;
        const uint32_t lane_base = (uint32_t)(qw * 32) << 16;
        float *red = reinterpret_cast<float *>(smem + L::kRed);     // [4][N]
        float *res = red + 4 * N;                                   // [N]
        const bool col_lane = lane % (32 / C) == 0;                 // holds a reduced column
        const int col = n0 + lane / (32 / C);
        Walk w = plan.start;
        int st = 0;
        uint32_t ph = 0, g = 0;
        T *out = reinterpret_cast<T *>(a.out);
        bool run = true;
        do {
            const int t0 = w.rt * a.tok, ntok = min(a.tok, w.q_len - t0);
            const int nrows = ntok * a.group;
            const int seen0 = min(w.kv_len, seen_by(a.s, w.kv_len, w.q_len, t0));   // fewest keys
            float m[C], l[C];
#pragma unroll
            for (int n = 0; n < C; n++) {
                m[n] = -INFINITY;
                l[n] = 0.0f;
            }
            for (int j = w.j0; j < w.j1; j++, g++) {
                const int buf = g & 1;
                bool ok = true;
                if (x == 0 && j * kKeys + kKeys > seen0) {
                    // (while the scores are made; P is handed over behind it)
                    ok = tc::mbar_wait(&v_full[st], ph, abort_flag, err_word, kErrWaitFull);
                    if (ok)
                        settle_row<T, kSubs>(smem + L::kV + st * L::kTile, key, seen0 - j * kKeys,
                                             w.kv_len - j * kKeys, odd_flag);
                }
                ok = ok && tc::mbar_wait(&s_full[buf], (g >> 1) & 1, abort_flag, err_word, kErrWaitAccum);
                tc::tc_fence_after();
                float v[C];
                if (ok) {
                    uint32_t r[C];
                    load_columns(tmem_base + buf * N + n0 + lane_base, r);
#pragma unroll
                    for (int n = 0; n < C; n++) v[n] = __uint_as_float(r[n]) * a.scale_log2;
                }
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&s_empty[buf]);
                const int kk = j * kKeys + key;
                if (j * kKeys + kKeys > seen0) {
                    // the rows of token t see the keys before seen_by(t)
                    int t = t0 + n0 / a.group, i = n0 % a.group;
#pragma unroll
                    for (int n = 0; n < C; n++) {
                        if (kk >= min(w.kv_len, seen_by(a.s, w.kv_len, w.q_len, t))) v[n] = -INFINITY;
                        if (++i == a.group) {
                            i = 0;
                            t++;
                        }
                    }
                }
                bool high = j == w.j0;
#pragma unroll
                for (int n = 0; n < C; n++) high |= v[n] > m[n] + 8.0f;
                if (vote_or(bar, high || !ok)) {
                    float top[C];
#pragma unroll
                    for (int n = 0; n < C; n++) top[n] = v[n];
                    const float mine = reduce_columns<C, true>(top, lane);
                    if (col_lane) red[qw * N + col] = mine;
                    // (the tile before this one has its P V done: O is stable)
                    if (ok && j > w.j0)
                        ok = tc::mbar_wait(&pv_done[buf ^ 1], ((g - 1) >> 1) & 1, abort_flag, err_word,
                                           kErrWaitAccum);
                    if (vote_or(bar, !ok)) {
                        run = false;
                        break;
                    }
                    tc::tc_fence_after();
                    float corr[C];
                    bool moved = false;
#pragma unroll
                    for (int n = 0; n < C; n++) {
                        const float *p = red + n0 + n;
                        const float t4 = fmaxf(fmaxf(p[0], p[N]), fmaxf(p[2 * N], p[3 * N]));
                        corr[n] = 1.0f;
                        if (t4 > m[n] + 8.0f || (j == w.j0 && t4 > m[n])) {
                            corr[n] = tc::ex2(m[n] - t4);
                            m[n] = t4;
                            l[n] *= corr[n];
                            moved = true;
                        }
                    }
                    if (moved && j > w.j0) {
                        uint32_t o[C];
                        load_columns(tmem_o + n0 + lane_base, o);
#pragma unroll
                        for (int n = 0; n < C; n++)
                            o[n] = __float_as_uint(__uint_as_float(o[n]) * corr[n]);
                        store_columns(tmem_o + n0 + lane_base, o);
                    }
                }
                // P^T of this key: weights relative to the references
                uint32_t pk[C / 2];
#pragma unroll
                for (int n = 0; n < C; n += 2) {
                    const float p0 = tc::ex2(v[n] - (m[n] == -INFINITY ? 0.0f : m[n]));
                    const float p1 = tc::ex2(v[n + 1] - (m[n + 1] == -INFINITY ? 0.0f : m[n + 1]));
                    l[n] += p0;
                    l[n + 1] += p1;
                    pk[n / 2] = pack2<T>(p0, p1);
                }
                // its buffer was last read by the P V of tile g - 2
                if (ok && g >= 2)
                    ok = tc::mbar_wait(&pv_done[buf], ((g - 2) >> 1) & 1, abort_flag, err_word,
                                       kErrWaitAccum);
                if (ok) {
                    uint4 *prow = reinterpret_cast<uint4 *>(smem + L::kP + buf * (kKeys * N * 2) +
                                                            key * N * 2);
                    const int sw = N == 16 ? (key >> 2) & 1 : (key >> 1) & 3;
#pragma unroll
                    for (int c = 0; c < C / 8; c++)
                        prow[(n0 / 8 + c) ^ sw] =
                            make_uint4(pk[4 * c], pk[4 * c + 1], pk[4 * c + 2], pk[4 * c + 3]);
                }
                tc::fence_proxy_async_smem();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&p_full[buf]);
                if (++st == S) {
                    st = 0;
                    ph ^= 1;
                }
            }
            if (!run) break;
            // ---- end of the segment: row sums over the keys, O^T / l
            bool ok = tc::mbar_wait(&pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, abort_flag, err_word,
                                    kErrWaitAccum);
            const float mine = reduce_columns<C, false>(l, lane);
            if (col_lane) red[qw * N + col] = mine;
            if (vote_or(bar, !ok)) break;
            tc::tc_fence_after();
            const bool whole = w.j0 == 0 && w.j1 == w.nt;
            const int slot = blockIdx.x * 2 + (w.j0 == 0 ? 1 : 0);
            if (key < C) {
                const int n = n0 + key;
                const float sum = (red[n] + red[N + n]) + (red[2 * N + n] + red[3 * N + n]);
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < C; i++) top = key == i ? m[i] : top;
                res[n] = sum == 0.0f ? 0.0f : 1.0f / sum;
                if (n < nrows) {
                    if (!whole) {
                        float *ml = a.part_ml + ((size_t)slot * kPartRows + n) * 2;
                        ml[0] = top;
                        ml[1] = sum;
                    } else if (a.lse) {
                        const int64_t r = (int64_t)(w.first + t0 + n / a.group) * a.heads +
                                          w.h * a.group + n % a.group;
                        a.lse[r] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
                    }
                }
            }
            softmax_sync(bar);
            uint32_t o[C];
            load_columns(tmem_o + n0 + lane_base, o);
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(o_free);
            if (key < D) {
                if (whole) {
                    int t = n0 / a.group, i = n0 % a.group;
#pragma unroll
                    for (int n = 0; n < C; n++) {
                        if (n0 + n < nrows)
                            out[((int64_t)(w.first + t0 + t) * a.heads + w.h * a.group + i) * D + key] =
                                from_f32<T>(__uint_as_float(o[n]) * res[n0 + n]);
                        if (++i == a.group) {
                            i = 0;
                            t++;
                        }
                    }
                } else {
                    float *po = a.part_o + ((size_t)slot * kPartRows + n0) * D + key;
#pragma unroll
                    for (int n = 0; n < C; n++)
                        if (n0 + n < nrows) po[n * D] = __uint_as_float(o[n]);
                }
            }
            Walk last = w;
            if (!w.next(a, a.tok)) {
                if (x == 0 && key == 0) note_parts(a, plan, last, a.tok);
                break;
            }
        } while (true);
    }

    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        tc::tmem_dealloc(tmem_base, kCols);
    }
    if (threadIdx.x == 0) a.recs[blockIdx.x].odd = *odd_flag;
    if (warp >= 4 && *odd_flag && !*abort_flag)
        mend_items<T, D>(a, plan.start, a.tok, warp - 4);
}

template <typename T, int D, int N>
int launch_dec(Dev *d, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
               const PagedTc &a) {
    using L = PagedDecSmem<D, N>;
    static_assert(L::kTotal <= 232448, "shared memory of one CTA");
    static bool attr_done[64] = {};
    if (!attr_done[d->ordinal & 63]) {
        if (int rc = check(cudaFuncSetAttribute(paged_dec_kernel<T, D, N>,
                                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                L::kTotal),
                           "cudaFuncSetAttribute(paged_dec)"))
            return rc;
        attr_done[d->ordinal & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)d->sms);
    cfg.blockDim = dim3(384);
    cfg.dynamicSmemBytes = L::kTotal;
    cfg.stream = d->stream;
    return check(cudaLaunchKernelEx(&cfg, paged_dec_kernel<T, D, N>, mq, mk, mv, a), "launch paged_dec");
}

}  // namespace

int launch_paged_dec(Dev *d, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv,
                     PagedTc &a, int dtype, int dim, int rows) {
    if (dtype == HEXCUDA_F16) {
        if (dim == 128)
            return rows == 16 ? launch_dec<__half, 128, 16>(d, mq, mk, mv, a)
                              : launch_dec<__half, 128, 32>(d, mq, mk, mv, a);
        return rows == 16 ? launch_dec<__half, 64, 16>(d, mq, mk, mv, a)
                          : launch_dec<__half, 64, 32>(d, mq, mk, mv, a);
    }
    if (dim == 128)
        return rows == 16 ? launch_dec<__nv_bfloat16, 128, 16>(d, mq, mk, mv, a)
                          : launch_dec<__nv_bfloat16, 128, 32>(d, mq, mk, mv, a);
    return rows == 16 ? launch_dec<__nv_bfloat16, 64, 16>(d, mq, mk, mv, a)
                      : launch_dec<__nv_bfloat16, 64, 32>(d, mq, mk, mv, a);
}

}  // namespace hx
