// paged_attn.cu -- attention of new tokens over a paged key / value cache:
// the entry point, the choice between its kernels, the join of partial
// results, and the CUDA-core path.
//
//   out[r, h] = sum_j softmax_j(scale * q[r, h] . K[j]) V[j],
//   lse[r, h] = log sum_j exp(scale * q[r, h] . K[j])
//
// over the cached tokens j that the row sees (paged.cuh), K and V of query
// head h's key head h / (heads / kv_heads).  A row that sees nothing gets
// zeros and minus infinity.
#include <math.h>

#include "paged_tc.cuh"

namespace hx {

int check_paged(const char *name, int dtype, const void *table, const void *kv_lens,
                const void *q_offs, int batch, int total_q, int max_q, int heads, int kv_heads,
                int head_dim, int num_pages, int page_size, int max_pages, float scale) {
    if (dtype != HEXCUDA_F16 && dtype != HEXCUDA_BF16)
        return fail(HEXCUDA_ERR_ARG, "%s: dtype %d", name, dtype);
    if (batch < 0 || total_q < 0 || total_q > kMaxTokens || max_q < 0)
        return fail(HEXCUDA_ERR_ARG, "%s: batch %d total_q %d max_q %d", name, batch, total_q,
                    max_q);
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads > 65535 || head_dim < 1 ||
        head_dim > 256)
        return fail(HEXCUDA_ERR_ARG,
                    "%s: heads %d kv_heads %d (a divisor) head_dim %d (1 to 256)", name, heads,
                    kv_heads, head_dim);
    if (num_pages < 1 || page_size < 1 || max_pages < 1 ||
        (int64_t)num_pages * page_size > 0x7fffffff || (int64_t)max_pages * page_size > kMaxTokens)
        return fail(HEXCUDA_ERR_ARG, "%s: num_pages %d page_size %d max_pages %d", name, num_pages,
                    page_size, max_pages);
    if (!(scale > 0.0f) || isinf(scale * 1.4426950408889634f))
        return fail(HEXCUDA_ERR_ARG, "%s: scale %g is not positive and finite (log2(e) times it)",
                    name, (double)scale);
    if (batch > 0 && total_q > 0 && (!table || !kv_lens || !q_offs))
        return fail(HEXCUDA_ERR_ARG, "%s: null pointer", name);
    return HEXCUDA_OK;
}

namespace {

constexpr int kMaxD = 256;

// Any head size, page size and alignment: one warp per query row and head.
// Lane t scores key t of a run of 32, the warp reduces the run's maximum and
// sum with shuffles, and lane t accumulates output columns t, t + 32, ...
template <typename T>
__global__ void __launch_bounds__(128) paged_attn_any_kernel(
    const T *__restrict__ q, const T *__restrict__ kp, const T *__restrict__ vp,
    T *__restrict__ out, float *__restrict__ lse, const PagedSeqs s, int heads, int kv_heads,
    int dim, float scale) {
    __shared__ float sq[4][kMaxD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int b = blockIdx.y; b < s.batch; b += gridDim.y) {
      int first;
      const int q_len = seq_q_len(s, b, first), kv_len = seq_kv_len(s, b);
      const int64_t rows = (int64_t)q_len * heads;
      for (int64_t i = (int64_t)blockIdx.x * 4 + warp; i < rows; i += (int64_t)gridDim.x * 4) {
        const int64_t w = (int64_t)first * heads + i;
        const int h = (int)(i % heads);
        const int seen = seen_by(s, kv_len, q_len, (int)(i / heads));
        const int kvh = h / (heads / kv_heads);
        __syncwarp();
        for (int d = lane; d < dim; d += 32) sq[warp][d] = to_f32(q[w * dim + d]);
        __syncwarp();
        float acc[kMaxD / 32];
#pragma unroll
        for (int u = 0; u < kMaxD / 32; u++) acc[u] = 0.0f;
        float m = -INFINITY, l = 0.0f;
        for (int j0 = 0; j0 < seen; j0 += 32) {
            const int j = j0 + lane;
            int64_t row = -1;
            float x = -INFINITY;
            if (j < seen) {
                const int page = seq_page(s, b, j / s.page_size);
                if (page >= 0)
                    row = ((int64_t)page * kv_heads + kvh) * s.page_size + j % s.page_size;
                // (a page that is not there: keys and values of zeros, as TMA gives them)
                float a = 0.0f;
                for (int d = 0; d < dim; d++)
                    a += sq[warp][d] * (row >= 0 ? to_f32(kp[row * dim + d]) : 0.0f);
                x = a * scale;
            }
            float top = x;
            for (int o = 16; o > 0; o >>= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float m_new = fmaxf(m, top);
            const float ref = m_new == -INFINITY ? 0.0f : m_new;
            const float corr = expf(m - ref);
            const float p = j < seen ? expf(x - ref) : 0.0f;
            float sum = p;
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l = l * corr + sum;
#pragma unroll
            for (int u = 0; u < kMaxD / 32; u++) acc[u] *= corr;
            const int n = min(32, seen - j0);
            for (int e = 0; e < n; e++) {
                const float pe = __shfl_sync(0xffffffffu, p, e);
                const int64_t re = __shfl_sync(0xffffffffu, row, e);
                if (re < 0) continue;
#pragma unroll
                for (int u = 0; u < kMaxD / 32; u++) {
                    const int d = lane + 32 * u;
                    if (d < dim) acc[u] += pe * to_f32(vp[re * dim + d]);
                }
            }
            m = m_new;
        }
#pragma unroll
        for (int u = 0; u < kMaxD / 32; u++) {
            const int d = lane + 32 * u;
            // (a sum that is not a number divides too: only an empty row gives zeros)
            if (d < dim) out[w * dim + d] = from_f32<T>(l == 0.0f ? 0.0f : acc[u] / l);
        }
        if (lse && lane == 0) lse[w] = l == 0.0f ? -INFINITY : m + logf(l);
      }
    }
}

// Joins the parts of the items that several CTAs worked on: block (c, y) those
// of the item that starts in CTA c and ends in a later one, half a warp a row, so
// that two rows' groups of four columns, neighbours in a chunk's parts, make whole
// sectors.  The parts are taken in CTA order:
//   M = max m_k,  out = sum 2^(m_k - M) O_k / sum 2^(m_k - M) l_k
// Where a part's CTA took values that are not finite out of a tile, the rows that see
// them get them here (paged_tc.cuh).  Bound by latency: 10.8 us
// for 11 chunks of 301 tokens of 64 (a warp a row: 15.6), 19 us for 148 items of 256
// rows of 128, 5.3 us for one token.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedTc a, int item_tok) {
    tc::grid_dependency_wait();
    const int c = blockIdx.x, lane = threadIdx.x & 31, sub = lane >> 4, l16 = lane & 15;
    const PartRec r = a.recs[c];
    const int i0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * 2, n = r.ntok * a.group;
    if (r.nparts == 0 || i0 >= n) return;
    const bool live = i0 + sub < n;         // (the last row again for one behind it)
    const int i = live ? i0 + sub : n - 1, t = i / a.group;
    const int row = t / a.tok * 128 + (t % a.tok) * a.group + i % a.group;
    auto slot = [&](int k) { return ((size_t)(c + k) * 2 + (k == 0 ? 1 : 0)) * kPartRows; };
    const float2 *mls = reinterpret_cast<const float2 *>(a.part_ml);
    float top = -INFINITY;
    int odd = 0;
    for (int k = l16; k < r.nparts; k += 16) {
        const float2 ml = mls[slot(k) + row];
        odd |= a.recs[c + k].odd;
        if (ml.y != 0.0f) top = fmaxf(top, ml.x);
    }
    for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    constexpr int G = D / 64;               // groups of four columns of a lane
    float acc[G][4], sum = 0.0f;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int v = 0; v < 4; v++) acc[g][v] = 0.0f;
    const float *parts = a.part_o + (int64_t)row * a.part_row + l16 * a.part_col;
    // 16 parts at a time: lane k has part k's weight, then all lanes add up rows
    for (int k0 = 0; k0 < r.nparts; k0 += 16) {
        float w = 0.0f, l = 0.0f;
        if (k0 + l16 < r.nparts) {
            const float2 ml = mls[slot(k0 + l16) + row];
            // (a part without a visible key has no output)
            if (ml.y != 0.0f) w = tc::ex2(ml.x - top);
            l = w * ml.y;
        }
        for (int o = 8; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        sum += l;
        const int m = min(16, r.nparts - k0);
#pragma unroll 2
        for (int k = 0; k < m; k++) {
            const float wk = __shfl_sync(0xffffffffu, w, k, 16);
#pragma unroll
            for (int g = 0; g < G; g++) {
                const float4 x = *reinterpret_cast<const float4 *>(parts + slot(k0 + k) * D +
                                                                   16 * g * a.part_col);
                if (wk == 0.0f) continue;
                acc[g][0] += wk * x.x;
                acc[g][1] += wk * x.y;
                acc[g][2] += wk * x.z;
                acc[g][3] += wk * x.w;
            }
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t at = (int64_t)(r.row0 + t) * a.heads + r.h * a.group + i % a.group;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int v = 0; v < 4; v++) acc[g][v] *= inv;
    if (__any_sync(0xffffffffu, odd != 0)) {
        int first, q_len, kv_len;
        quiet_seq(a.s, r.b, first, q_len, kv_len);
        const int t0 = r.rt * item_tok, seen = min(kv_len, seen_by(a.s, kv_len, q_len, t0 + t));
#pragma unroll 4
        for (int j = seen_by(a.s, kv_len, q_len, t0); j < seen; j++)
#pragma unroll
            for (int g = 0; g < G; g++) {
                float x[4];
                odd_values<T, D, 4>(a, r.b, r.h, j, (l16 + 16 * g) * 4, x);
#pragma unroll
                for (int v = 0; v < 4; v++) acc[g][v] += x[v];
            }
    }
    if (!live) return;
#pragma unroll
    for (int g = 0; g < G; g++)
        *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(a.out) + at * D + (l16 + 16 * g) * 4) =
            make_uint2(pack2<T>(acc[g][0], acc[g][1]), pack2<T>(acc[g][2], acc[g][3]));
    if (a.lse && l16 == 0)
        a.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// The join (not launched when the kernel before it was refused: its records would be
// what the workspace held) starts while that kernel still runs on the stream, and
// waits for it on the device (a programmatic dependent launch).
template <typename T, int D>
int launch_join(Dev *d, const PagedTc &a, int rows, int item_tok) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)d->sms, (unsigned)((rows + 15) / 16));
    cfg.blockDim = dim3(256);
    cfg.stream = d->stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return check(cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D>, a, item_tok), "launch paged_join");
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *,
                                  const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                                  const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode_map(CUtensorMap *map, const void *base, int rank, const cuuint64_t *dims,
               const cuuint64_t *strides, const cuuint32_t *box) {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
                cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return fail(HEXCUDA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
        fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    const cuuint32_t ones[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, (cuuint32_t)rank,
                          const_cast<void *>(base), dims, strides, box, ones,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(HEXCUDA_ERR_CUDA, "cuTensorMapEncodeTiled (paged cache) failed (%d)", (int)r);
    return HEXCUDA_OK;
}

size_t round_up(size_t n, size_t to) { return (n + to - 1) / to * to; }

}  // namespace

int make_page_map(CUtensorMap *map, const void *base, int64_t rows, int dim, int frag) {
    const cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)dim * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)frag};
    return encode_map(map, base, 2, dims, strides, box);
}

int make_query_map(CUtensorMap *map, const void *base, int total_q, int heads, int dim, int group,
                   int tok) {
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)total_q};
    const cuuint64_t strides[2] = {(cuuint64_t)dim * 2, (cuuint64_t)heads * dim * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)tok};
    return encode_map(map, base, 3, dims, strides, box);
}

bool paged_tc_fits(const void *q, const void *k, const void *v, const void *out, int heads,
                   int kv_heads, int dim, int num_pages, int page_size) {
    const uintptr_t bits = (uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out;
    return (dim == 64 || dim == 128) && page_size % 8 == 0 && (bits & 15u) == 0 &&
           heads / kv_heads <= 128 &&
           (int64_t)num_pages * kv_heads * page_size <= 0x7fffff00;
}

}  // namespace hx

using namespace hx;

HX_EXPORT int hexcuda_paged_attn_workspace(int dev, size_t *bytes) {
    Dev *d = get_dev(dev);
    if (!d) return HEXCUDA_ERR_NODEV;
    if (!bytes) return fail(HEXCUDA_ERR_ARG, "paged_attn_workspace: null pointer");
    // one record and two partial results per CTA, one CTA per SM
    *bytes = round_up(sizeof(PartRec) * d->sms, 256) +
             (size_t)d->sms * 2 * kPartRows * (128 + 2) * sizeof(float);
    return HEXCUDA_OK;
}

HX_EXPORT int hexcuda_paged_attn(int dev, int dtype, const void *q, const void *k_pages,
                                 const void *v_pages, const int32_t *block_table,
                                 const int32_t *kv_lens, const int32_t *q_offs, void *out,
                                 float *lse, void *workspace, size_t workspace_bytes, int batch,
                                 int total_q, int max_q, int heads, int kv_heads, int head_dim,
                                 int num_pages, int page_size, int max_pages, float scale,
                                 int causal) {
    if (int rc = check_paged("paged_attn", dtype, block_table, kv_lens, q_offs, batch, total_q,
                             max_q, heads, kv_heads, head_dim, num_pages, page_size, max_pages,
                             scale))
        return rc;
    if (batch == 0 || total_q == 0) return HEXCUDA_OK;
    if (!q || !k_pages || !v_pages || !out || !workspace)
        return fail(HEXCUDA_ERR_ARG, "paged_attn: null pointer");
    Dev *d = get_dev(dev);
    if (!d) return HEXCUDA_ERR_NODEV;
    size_t need = 0;
    if (int rc = hexcuda_paged_attn_workspace(dev, &need)) return rc;
    const int64_t rows16 = (int64_t)total_q * heads * head_dim;
    const int64_t pages16 = (int64_t)num_pages * kv_heads * page_size * head_dim;
    if (overlap16(out, rows16, q, rows16) || overlap16(out, rows16, k_pages, pages16) ||
        overlap16(out, rows16, v_pages, pages16))
        return fail(HEXCUDA_ERR_ARG, "paged_attn: out is q or overlaps an input");
    if (workspace_bytes < need || ((uintptr_t)workspace & 15u))
        return fail(HEXCUDA_ERR_ARG,
                    "paged_attn: workspace of %zu bytes, %zu needed, 16-byte aligned",
                    workspace_bytes, need);
    PagedSeqs s{block_table, kv_lens, q_offs, batch, total_q, num_pages, page_size,
                max_pages, causal, d->err_word};
    const int group = heads / kv_heads;
    // Up to 32 query rows share a key head: the decoding kernel, of 16 or 32 rows.
    // More: 128-row tiles.  Measured with tiles of 16 / 32 / 128 rows (dim 128, 8 key
    // heads, L2 flushed): 4 sequences of 1000, 8 rows: 21.5 / 21.5 / 25.6 us, 32 rows:
    // 25.6 / 23.6 / 27.6, 40 rows: 25.6 / 25.6 / 27.7, 128 rows: 37.9 / 29.7 / 29.7; 32
    // of 8192, 16 rows: 198 / 198 / 200, 32 rows: 364 / 202 / 202, 40 rows: 517 / 360 /
    // 202.  (Two tiles of rows read the keys twice.)
    const int64_t rows = (int64_t)(max_q < 1 ? 1 : max_q) * group;
    if (paged_tc_fits(q, k_pages, v_pages, out, heads, kv_heads, head_dim, num_pages, page_size)) {
        const bool few = rows <= 32;
        const int n = rows <= 16 ? 16 : few ? 32 : 128;
        PagedTc a;
        a.s = s;
        a.heads = heads;
        a.kv_heads = kv_heads;
        a.group = group;
        a.tok = n / group;
        const int low = page_size & -page_size;
        a.frag = low < kKeys ? low : kKeys;
        a.map_rows = num_pages * kv_heads * page_size;
        a.min_units = 2;        // (4: one sequence of 777 in 16.8 us for 14.5, longer ones the same)
        a.scale_log2 = scale * 1.4426950408889634f;
        a.q = q;
        a.k = k_pages;
        a.v = v_pages;
        a.out = out;
        a.lse = lse;
        uint8_t *p = reinterpret_cast<uint8_t *>(workspace);
        a.recs = reinterpret_cast<PartRec *>(p);
        p += round_up(sizeof(PartRec) * d->sms, 256);
        a.part_ml = reinterpret_cast<float *>(p);
        a.part_o = a.part_ml + (size_t)d->sms * 2 * kPartRows * 2;
        // single tokens: the columns are in a warp's lanes; chunks: the rows are
        a.part_row = few ? head_dim : 4;
        a.part_col = few ? 4 : 4 * kPartRows;
        CUtensorMap mq, mk, mv;
        if (int rc = make_query_map(&mq, q, total_q, heads, head_dim, group, a.tok)) return rc;
        if (int rc = make_page_map(&mk, k_pages, a.map_rows, head_dim, a.frag)) return rc;
        if (int rc = make_page_map(&mv, v_pages, a.map_rows, head_dim, a.frag)) return rc;
        launch_begin(d);
        if (int rc = few ? launch_paged_dec(d, mq, mk, mv, a, dtype, head_dim, n)
                         : launch_paged_pre(d, mq, mk, mv, a, dtype, head_dim))
            return rc;
        const bool half = dtype == HEXCUDA_F16;
        const int join_rows = few ? n : 2 * n;      // of one item
        const int item_tok = few ? a.tok : 2 * a.tok;
        if (int rc = head_dim == 128
                         ? (half ? launch_join<__half, 128>(d, a, join_rows, item_tok)
                                 : launch_join<__nv_bfloat16, 128>(d, a, join_rows, item_tok))
                         : (half ? launch_join<__half, 64>(d, a, join_rows, item_tok)
                                 : launch_join<__nv_bfloat16, 64>(d, a, join_rows, item_tok)))
            return rc;
        note_mech(kMechTcgen05 | kMechTma);
        return launch_end(d, "paged_attn", 2);
    }
    launch_begin(d);
    const int ny = batch < 1024 ? batch : 1024;
    const dim3 grid((unsigned)((d->sms * 16 + ny - 1) / ny), (unsigned)ny);
    if (dtype == HEXCUDA_F16)
        paged_attn_any_kernel<__half><<<grid, 128, 0, d->stream>>>(
            (const __half *)q, (const __half *)k_pages, (const __half *)v_pages, (__half *)out, lse,
            s, heads, kv_heads, head_dim, scale);
    else
        paged_attn_any_kernel<__nv_bfloat16><<<grid, 128, 0, d->stream>>>(
            (const __nv_bfloat16 *)q, (const __nv_bfloat16 *)k_pages,
            (const __nv_bfloat16 *)v_pages, (__nv_bfloat16 *)out, lse, s, heads, kv_heads, head_dim,
            scale);
    return launch_end(d, "paged_attn");
}
