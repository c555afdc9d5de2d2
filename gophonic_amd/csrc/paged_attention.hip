// gphq_paged_attention: argument checks, the cut of a batch into tiles and splits, and the
// join of split results. Kernels: paged_rows.hip and paged_chunk.hip.
#include <math.h>

#include <new>

#include "lm_model.h"
#include "paged_attention.h"

namespace gphq {

int paged_args(const gphq_paged_kv *kv, const gphq_paged_batch *b, PagedPool &pool, PagedBatch &batch) {
    if (!kv || !b) return GPHQ_ERR_PAGED_SHAPE;
    if (kv->dtype != GPHQ_DTYPE_F32 && kv->dtype != GPHQ_DTYPE_F16 && kv->dtype != GPHQ_DTYPE_BF16)
        return GPHQ_ERR_UNSUPPORTED;
    if (kv->head_dim != 64 && kv->head_dim != 128) return GPHQ_ERR_UNSUPPORTED;
    if (kv->page_tokens < 16 || kv->page_tokens > GPHQ_PAGED_MAX_PAGE_TOKENS ||
        (kv->page_tokens & (kv->page_tokens - 1)))
        return GPHQ_ERR_UNSUPPORTED;
    if (kv->pages < 1 || kv->pages > INT32_MAX || kv->kv_heads < 1 || kv->kv_heads > GPHQ_PAGED_MAX_HEADS)
        return GPHQ_ERR_PAGED_SHAPE;
    const int64_t size = kv->dtype == GPHQ_DTYPE_F32 ? 4 : 2, unit = 16 / size;
    for (const int64_t s : {kv->page_stride, kv->token_stride, kv->head_stride})
        if (s < kv->head_dim || s % unit || s > INT64_MAX / (size * kv->pages)) return GPHQ_ERR_PAGED_SHAPE;
    if (kv->token_stride > INT32_MAX / (kv->page_tokens * size)) return GPHQ_ERR_PAGED_SHAPE;  // a page under 2 GiB
    if (!kv->k_dev || !kv->v_dev || (uintptr_t)kv->k_dev % 16 || (uintptr_t)kv->v_dev % 16)
        return GPHQ_ERR_PAGED_SHAPE;
    if (b->seqs < 0 || b->seqs > GPHQ_PAGED_MAX_SEQS || b->rows < 0 || b->rows > GPHQ_PAGED_MAX_ROWS ||
        b->max_rows < 0 || b->max_len < 0 || b->max_len > GPHQ_PAGED_MAX_LEN || b->table_stride < 0)
        return GPHQ_ERR_PAGED_SHAPE;
    if (b->table_stride < (b->max_len + kv->page_tokens - 1) / kv->page_tokens || b->table_stride > INT32_MAX)
        return GPHQ_ERR_PAGED_SHAPE;
    if (b->seqs && (!b->starts_dev || !b->lens_dev || (b->table_stride && !b->table_dev))) return GPHQ_ERR_PAGED_SHAPE;
    if (((uintptr_t)b->starts_dev | (uintptr_t)b->lens_dev | (uintptr_t)b->table_dev | (uintptr_t)b->bad_dev) % 4)
        return GPHQ_ERR_PAGED_SHAPE;
    pool = PagedPool{kv->k_dev,       kv->v_dev,
                     kv->page_stride, kv->token_stride,
                     kv->head_stride, (int)kv->pages,
                     __builtin_ctzll((uint64_t)kv->page_tokens), (int)kv->kv_heads};
    batch = PagedBatch{b->starts_dev, b->lens_dev,  b->table_dev, b->bad_dev,
                       b->table_stride, (int)b->seqs, (int)b->rows, (int)std::min(b->max_rows, b->rows),
                       (int)b->max_len};
    if (batch.seqs == 0 || batch.max_rows == 0) batch.rows = 0;  // nothing to do
    return GPHQ_OK;
}

namespace {

constexpr int64_t kMaxBlocks = (1 << 23) - 1;  // of a launch: 2^32 threads at 512 a block are one too many

// How a call is cut: which kernels run, over how many tiles and splits.
struct AttnPlan {
    int small_cols, small_tiles, small_splits, small_len;  // small_tiles per sequence; 0: the row kernel is not run
    int big_tiles, big_splits, big_len;                    // big_tiles in all; 0: the chunk kernel is not run
    int small_rows;  // rows that a sequence of the row kernel may have; 0: split results kept by row
    int row_tiles;   // tiles of a row; 0: the row kernel's grid is by sequence, small_tiles each
    int64_t small_units;  // tiles of the row kernel's grid
};

// Keys per split of `span` keys and how many splits that makes, for about `want` of them.
void cut(int64_t span, int64_t want, int &len, int &splits) {
    const int64_t steps = std::max<int64_t>(1, (span + 127) / 128);
    const int64_t n = std::min(std::max<int64_t>(want, 1), steps);
    len = (int)((steps + n - 1) / n * 128);
    splits = (int)((span + len - 1) / len);
    if (splits < 1) splits = 1;
}

// wide: fp32 pages. From host numbers alone, so a captured call keeps its cut whatever the lengths become.
AttnPlan attn_plan(const PagedBatch &b, int kv_heads, int group, int window, int big_tile, bool wide) {
    AttnPlan p{};
    const int64_t cus = device_cus(), rows = b.rows, cols = (int64_t)b.max_rows * group;
    // Sequences of up to 64 columns run in the row kernel, in tiles of 16 that each read the
    // keys; a call of one sequence runs in one kernel only. 64 columns over 6000 tokens, eight
    // KV heads, row kernel and chunk kernel: one sequence bfloat16 14.9 and 19.0 us, fp32 27.8 and
    // 48.5; eight sequences 68 and 64, fp32 146 and 297. 80 columns, eight sequences: 125 and 69,
    // fp32 rows over FP16 pages 126 and 78.
    constexpr int kSmallCols = 64;
    p.small_cols = cols > kSmallCols && b.seqs == 1 ? 0 : kSmallCols;
    auto span = [&](int64_t tile) {  // keys a tile of that many columns may see, from a multiple of 64
        return window > 0 ? std::min<int64_t>(b.max_len, (int64_t)window + tile / group + 65) : (int64_t)b.max_len;
    };
    if (p.small_cols && group <= p.small_cols) {
        p.small_rows = std::min(p.small_cols / group, b.max_rows);
        p.small_tiles = (int)((std::min<int64_t>(cols, p.small_cols) + kSmallTile - 1) / kSmallTile);
        const int64_t units = std::min<int64_t>(b.seqs, rows) * p.small_tiles * kv_heads;
        // As many splits as leave one block on a CU: its four wavefronts keep enough loads in
        // flight, and a round more, begun or whole, costs more than it hides (16 bfloat16 rows of
        // 2000 to 4095 tokens, eight KV heads: 39.4 us with one block a CU, 41.4 with two, 46.8
        // with one and a half; fp32: 71.5, 74.7, 89.7). Short rows take no split: the second
        // launch costs more than the steps it saves up to 512 keys of 16 bits (one row: 8.2 us,
        // split 9.4; 768 keys: 10.3 and 9.3) and 256 of 32 (10.6 and 11.0; 384: 13.4 and 11.1).
        const bool brief = span(kSmallTile) <= (wide ? 256 : 512);
        // Beside longer sequences, which are the chunk kernel's, only some of the sequences are
        // this kernel's, in one tile mostly: twice as many splits of one tile each. Whole calls,
        // so and with the rule above: twelve sequences (three single rows) over up to 4000
        // bfloat16 tokens 233 and 241 us, twenty (ten) up to 8000 274 and 355, six (five), FP16,
        // up to 6000 106 and 149, thirty (fifteen) up to 3000 FP16 tokens 123 and 136.
        const bool mixed = cols > p.small_cols;
        const int64_t want = mixed ? 2 * cus / (units / p.small_tiles) : cus / units;
        // The grid is by sequence, or by row where a batch has more room for sequences than rows (one
        // row of 40000 bfloat16 tokens, alone 26 us, among 2047 idle sequences 26 by row and 544 by
        // sequence). No more splits than a launch takes.
        const int64_t row_tiles = (group + kSmallTile - 1) / kSmallTile;
        p.small_units = (int64_t)b.seqs * p.small_tiles;
        if (rows * row_tiles < p.small_units) {
            p.small_units = rows * row_tiles;
            p.row_tiles = (int)row_tiles;
        }
        const int64_t most = kMaxBlocks / (p.small_units * kv_heads);
        cut(span(kSmallTile), brief ? 1 : std::min(want, most), p.small_len, p.small_splits);
        if ((int64_t)b.seqs * p.small_rows > rows) p.small_rows = 0;  // at most `rows` sequences have any
    }
    if (cols > p.small_cols) {
        const int64_t all = rows * group;
        // Tiles of s sequences of `all` columns: the sum of their ceilings, at most.
        const int64_t s = std::min<int64_t>(b.seqs, all / (p.small_cols + 1));
        p.big_tiles = (int)((all + s * (big_tile - 1)) / big_tile);
        const int64_t units = (int64_t)p.big_tiles * kv_heads;
        const int64_t slots = big_tile == 256 ? cus : 2 * cus;  // blocks that run at once
        // Tiles enough for the chip are not split (three chunks of 300 to 1300 fp32 rows over
        // FP16 pages: 106 us, split in three 133). Fewer tiles of one sequence take as many splits
        // as fill it (512 FP16 rows over 7512 tokens: 84 us, twice as many 100); of several, whose
        // lengths differ, three times as many, so that the long ones do not come last alone: the
        // twelve sequences above 233 us, 302 with one round (261 with four times, 240 with three, at
        // that time), the twenty 274 and 535, the thirty 123 and 154. That loses where the chunks are
        // alike or one alone: three of 83 to 234 FP16 rows over 6000 tokens 106 us, 94 with one
        // round, the six (one chunk) 106 and 88.
        const int64_t want = units >= slots ? 1 : (b.seqs == 1 ? 1 : 3) * slots / units;
        cut(span(big_tile), want, p.big_len, p.big_splits);
    }
    return p;
}

// Split results that the workspace holds for each kernel.
int64_t small_count(const AttnPlan &p, const PagedBatch &b, int64_t heads) {
    const int64_t places = p.small_rows ? (int64_t)b.seqs * p.small_rows : b.rows;
    return p.small_tiles && p.small_splits > 1 ? places * heads * p.small_splits : 0;
}
int64_t big_count(const AttnPlan &p, const PagedBatch &b, int64_t heads) {
    return p.big_tiles && p.big_splits > 1 ? b.rows * heads * p.big_splits : 0;
}

// Adds the split results of every (row, head): with M = max m_i,
//   o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i,
// over the splits in order, eight at a time against the largest m so far. HD / 4 lanes take
// a head, a wavefront 256 / HD heads of one row. W = 4: the four wavefronts of a block take
// every fourth eight and are added in order, for calls of many splits, whose time is that of
// reading one row's splits one after another (two 40k-token rows of 32 heads, 32 splits:
// 11.4 us with W = 1). Rows whose tile had one split were written by the tile itself.
template <typename RT, int HD, int W>
__global__ __launch_bounds__(256) void paged_join_kernel(const AttnArgs a) {
    constexpr int LH = HD / 4, HW = 64 / LH;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int groups = (a.heads + HW - 1) / HW;
    const int unit = W == 4 ? (int)blockIdx.x : (int)blockIdx.x * 4 + wave;
    const int row = unit / groups, head = (unit - row * groups) * HW + lane / LH;
    if (row >= a.b.rows) return;
    const SeqRow s = find_seq(a.b, row);
    if (row < s.start || row >= s.end || !seq_ok(a.b, s.start, s.end, s.len)) return;
    const int n = s.end - s.start, i = row - s.start, cols = n * a.group;
    const bool small = cols <= a.small_cols;
    const int tm = small ? kSmallTile : a.big_tile, c0 = (i * a.group + head % a.group) / tm * tm;
    const TileKeys k = tile_keys(n, s.len, c0 / a.group, min((c0 + tm - 1) / a.group, n - 1), a.window);
    const int all = head < a.heads ? tile_splits(k, small ? a.split_small : a.split_big) : 1;
    const int splits = all > 1 ? all : 0;  // (heads of a row may lie in different tiles)
    const int hc = min(head, a.heads - 1);
    const int64_t at = small ? (small_place(a, s.seq, s.start, i) * a.heads + hc) * a.small_parts
                             : ((int64_t)row * a.heads + hc) * a.parts;
    const float *part_o = small ? a.small_o : a.part_o, *part_ml = small ? a.small_ml : a.part_ml;
    const int d = 4 * (lane % LH);
    float M = -INFINITY, L = 0.0f;
    f32x4 o{};
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    for (int j0 = W == 4 ? 8 * wave : 0; j0 < splits; j0 += 8 * W) {
        f32x2 ml[8];
        f32x4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int64_t e = at + min(j0 + u, splits - 1);
            ml[u] = *(const f32x2 *)(part_ml + 2 * e);
            v[u] = *(const f32x4 *)(part_o + e * HD + d);
        }
        float mx = M;
#pragma unroll
        for (int u = 0; u < 8; ++u) mx = fmaxf(mx, ml[u].x);
        const float ref = mx == -INFINITY ? 0.0f : mx, c = __builtin_amdgcn_exp2f(M - ref);
        M = mx;
        L *= c;
        o *= c;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (j0 + u < splits) {
                const float w = __builtin_amdgcn_exp2f(ml[u].x - ref);
                L += w * ml[u].y;
                o += w * v[u];
            }
    }
    if (W == 4) {
        __shared__ float sm[4][64], sl[4][64];
        __shared__ f32x4 so[4][64];
        sm[wave][lane] = M;
        sl[wave][lane] = L;
        so[wave][lane] = o;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int w = 1; w < 4; ++w) M = fmaxf(M, sm[w][lane]);
        const float ref = M == -INFINITY ? 0.0f : M;
        const float c = __builtin_amdgcn_exp2f(sm[0][lane] - ref);
        L *= c;
        o *= c;
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            const float e = __builtin_amdgcn_exp2f(sm[w][lane] - ref);
            L += e * sl[w][lane];
            o += e * so[w][lane];
        }
    }
    if (!splits) return;
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = M == -INFINITY ? 0.0f : o[e] / L;
    store_vec((RT *)a.out + (int64_t)row * a.out_stride + head * HD + d, r);
}

// Takes the bits that were reported out of a batch's word; one that another stream has set since stays.
__global__ void paged_clear_kernel(int32_t *bad, int32_t reported) { atomicAnd(bad, ~reported); }

int64_t join_units(const PagedBatch &b, int64_t heads, int hd) { return b.rows * ((heads * hd + 255) / 256); }

template <typename RT, int HD>
int join_launch(const AttnArgs &a, hipStream_t st) {
    const int64_t units = join_units(a.b, a.heads, HD);
    if (std::max(a.parts, a.small_parts) > 8 && units <= kMaxBlocks)
        hipLaunchKernelGGL((paged_join_kernel<RT, HD, 4>), dim3((unsigned)units), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((paged_join_kernel<RT, HD, 1>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, a);
    return launch_status();
}

template <typename RT, typename CT>
int attend(const AttnArgs &a, const AttnPlan &p, int hd, hipStream_t st) {
    if (p.big_tiles) GPHQ_TRY((attn_chunk_launch<RT, CT>(a, hd, p.big_splits, p.big_tiles, st)));
    if (p.small_tiles) GPHQ_TRY((attn_rows_launch<RT, CT>(a, hd, p.small_splits, p.small_tiles, st)));
    if (!small_count(p, a.b, a.heads) && !big_count(p, a.b, a.heads)) return GPHQ_OK;
    return hd == 128 ? join_launch<RT, 128>(a, st) : join_launch<RT, 64>(a, st);
}

// The call's cut, refused where a launch would have too many blocks.
int plan_of(const AttnArgs &a, const gphq_paged_kv *kv, AttnPlan &p) {
    const int64_t kvh = a.pool.kv_heads;
    p = attn_plan(a.b, (int)kvh, a.group, a.window, a.big_tile, kv->dtype == GPHQ_DTYPE_F32);
    if (p.small_units * p.small_splits * kvh > kMaxBlocks ||
        (int64_t)p.big_tiles * p.big_splits * kvh > kMaxBlocks)
        return GPHQ_ERR_PAGED_SHAPE;
    const bool join = small_count(p, a.b, a.heads) || big_count(p, a.b, a.heads);
    // (The join's blocks take 256 threads, and four units where there are many.)
    return join && join_units(a.b, a.heads, (int)kv->head_dim) / 8 > kMaxBlocks ? GPHQ_ERR_PAGED_SHAPE : GPHQ_OK;
}

// The checks that the attention and its workspace size share.
int attn_args(const gphq_paged_kv *kv, const gphq_paged_batch *b, int row_dtype, int64_t heads, int64_t window,
              AttnArgs &a) {
    GPHQ_TRY(paged_args(kv, b, a.pool, a.b));
    if (row_dtype != GPHQ_DTYPE_F32 && row_dtype != kv->dtype) return GPHQ_ERR_UNSUPPORTED;
    if (heads < 1 || heads > GPHQ_PAGED_MAX_HEADS || heads % kv->kv_heads || window < 0) return GPHQ_ERR_PAGED_SHAPE;
    a.heads = (int)heads;
    a.group = (int)(heads / kv->kv_heads);
    a.window = window >= b->max_len ? 0 : (int)window;  // a window as long as any sequence hides nothing
    const bool f16c = kv->dtype == GPHQ_DTYPE_F16;
    a.big_tile = 32 * (kv->dtype == GPHQ_DTYPE_F32 ? kChunkWaves<float, float>
                       : row_dtype == kv->dtype    ? (f16c ? kChunkWaves<f16, f16> : kChunkWaves<bf16, bf16>)
                                                   : (f16c ? kChunkWaves<float, f16> : kChunkWaves<float, bf16>));
    return GPHQ_OK;
}

}  // namespace
}  // namespace gphq

using namespace gphq;

extern "C" {

int64_t gphq_paged_attention_workspace_bytes(const gphq_paged_kv *kv, const gphq_paged_batch *batch, int row_dtype,
                                             int64_t heads, int64_t window) {
    AttnArgs a{};
    GPHQ_TRY(attn_args(kv, batch, row_dtype, heads, window, a));
    if (a.b.rows == 0) return 0;
    AttnPlan p;
    GPHQ_TRY(plan_of(a, kv, p));
    return (small_count(p, a.b, heads) + big_count(p, a.b, heads)) * (kv->head_dim + 2) * 4;
}

int gphq_paged_attention(const gphq_paged_kv *kv, const gphq_paged_batch *batch, int row_dtype, const void *q,
                         int64_t q_stride, int64_t heads, double scale, int64_t window, void *out, int64_t out_stride,
                         void *work, int64_t work_bytes, void *stream) {
    AttnArgs a{};
    GPHQ_TRY(attn_args(kv, batch, row_dtype, heads, window, a));
    const int64_t hd = kv->head_dim, size = row_dtype == GPHQ_DTYPE_F32 ? 4 : 2;
    if (!(fabs(scale) <= 1e30) || q_stride < heads * hd || out_stride < heads * hd || q_stride * size % 16 || out_stride * size % 16)
        return GPHQ_ERR_PAGED_SHAPE;
    if (a.b.rows == 0) return GPHQ_OK;
    if (!q || !out || ((uintptr_t)q | (uintptr_t)out) % 16) return GPHQ_ERR_PAGED_SHAPE;
    if (spans_overlap(q, span_bytes(a.b.rows, q_stride, heads * hd, size), out,
                      span_bytes(a.b.rows, out_stride, heads * hd, size)))
        return GPHQ_ERR_OVERLAP;
    AttnPlan p;
    GPHQ_TRY(plan_of(a, kv, p));
    const int64_t big = big_count(p, a.b, heads), small = small_count(p, a.b, heads);
    if (big + small && (!work || (uintptr_t)work % 16 || work_bytes < (big + small) * (hd + 2) * 4))
        return GPHQ_ERR_PAGED_SHAPE;
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.parts = big ? p.big_splits : 1;
    a.small_parts = small ? p.small_splits : 1;
    a.small_rows = p.small_rows;
    a.row_tiles = p.row_tiles;
    a.part_o = (float *)work;
    a.small_o = a.part_o + big * hd;
    a.part_ml = a.small_o + small * hd;
    a.small_ml = a.part_ml + 2 * big;
    a.small_cols = p.small_cols;
    a.split_small = p.small_len;
    a.split_big = p.big_len;
    a.q_sign = scale > 0 ? 1.0f : scale < 0 ? -1.0f : 0.0f;
    a.scale_log2 = scale == 0 ? 1.0f : (float)(fabs(scale) * 1.4426950408889634);
    hipStream_t st = (hipStream_t)stream;
    if (row_dtype == GPHQ_DTYPE_F32) {
        if (kv->dtype == GPHQ_DTYPE_F32) return attend<float, float>(a, p, (int)hd, st);
        if (kv->dtype == GPHQ_DTYPE_F16) return attend<float, f16>(a, p, (int)hd, st);
        return attend<float, bf16>(a, p, (int)hd, st);
    }
    if (kv->dtype == GPHQ_DTYPE_F16) return attend<f16, f16>(a, p, (int)hd, st);
    return attend<bf16, bf16>(a, p, (int)hd, st);
}

int gphq_paged_pool_new(const gphq_lm *lm, int64_t pages, int64_t page_tokens, int dtype, gphq_paged_pool **out) {
    if (!out) return GPHQ_ERR_DIMENSIONS;
    *out = nullptr;
    if (!lm) return GPHQ_ERR_WORKSPACE;
    if (dtype != GPHQ_DTYPE_F32 && dtype != GPHQ_DTYPE_F16 && dtype != GPHQ_DTYPE_BF16) return GPHQ_ERR_UNSUPPORTED;
    if (page_tokens < 16 || page_tokens > GPHQ_PAGED_MAX_PAGE_TOKENS || (page_tokens & (page_tokens - 1)))
        return GPHQ_ERR_UNSUPPORTED;
    if (pages < 1 || pages > INT32_MAX) return GPHQ_ERR_PAGED_SHAPE;
    const gphq_lm_config &c = lm->cfg;
    const int64_t token = lm->kvd * (dtype == GPHQ_DTYPE_F32 ? 4 : 2);
    if (pages > INT64_MAX / (token * page_tokens * c.layers)) return GPHQ_ERR_PAGED_SHAPE;
    gphq_paged_pool *p = new (std::nothrow) gphq_paged_pool();
    if (!p) return GPHQ_ERR_SCRATCH_LIMIT;
    p->lm = lm;
    p->pages = pages;
    p->page_tokens = page_tokens;
    p->dtype = dtype;
    p->layer_bytes = token * page_tokens * pages;
    hipError_t e = hipMalloc((void **)&p->k, (size_t)(p->layer_bytes * c.layers));
    if (e == hipSuccess) e = hipMalloc((void **)&p->v, (size_t)(p->layer_bytes * c.layers));
    if (e != hipSuccess) {
        gphq_paged_pool_free(p);
        return hip_status(e);
    }
    *out = p;
    return GPHQ_OK;
}

void gphq_paged_pool_free(gphq_paged_pool *p) {
    if (!p) return;
    if (p->k) (void)hipFree(p->k);
    if (p->v) (void)hipFree(p->v);
    delete p;
}

int gphq_paged_pool_layer(const gphq_paged_pool *p, int64_t layer, gphq_paged_kv *out) {
    if (!p || !out) return GPHQ_ERR_PAGED_SHAPE;
    const gphq_lm_config &c = p->lm->cfg;
    if (layer < 0 || layer >= c.layers) return GPHQ_ERR_PAGED_SHAPE;
    out->k_dev = p->k + layer * p->layer_bytes;
    out->v_dev = p->v + layer * p->layer_bytes;
    out->token_stride = c.head_dim;
    out->head_stride = p->page_tokens * c.head_dim;
    out->page_stride = c.kv_heads * p->page_tokens * c.head_dim;
    out->pages = p->pages;
    out->page_tokens = p->page_tokens;
    out->kv_heads = c.kv_heads;
    out->head_dim = c.head_dim;
    out->dtype = p->dtype;
    out->reserved = 0;
    return GPHQ_OK;
}

int gphq_paged_check(int32_t *bad_dev, void *stream) {
    if (!bad_dev) return GPHQ_ERR_PAGED_SHAPE;
    // All on the caller's stream: a call that follows on it finds the word cleared, not about to be.
    hipStream_t st = (hipStream_t)stream;
    int32_t bad = 0;
    GPHQ_TRY(hip_status(hipMemcpyAsync(&bad, bad_dev, 4, hipMemcpyDeviceToHost, st)));
    GPHQ_TRY(hip_status(hipStreamSynchronize(st)));
    if (!bad) return GPHQ_OK;
    hipLaunchKernelGGL(paged_clear_kernel, dim3(1), dim3(1), 0, st, bad_dev, bad);
    GPHQ_TRY(launch_status());
    return GPHQ_ERR_PAGED_BATCH;
}

}  // extern "C"
