// gphq_paged_append: a batch's fused QKV rows [heads | KV heads | KV heads] to
// prepared queries and to keys and values in the pages of their sequences.
//
// Per row of sequence s at position p = lens[s] - (rows of s behind it) and
// per query or key head x of hd values, in fp32:
//   a = x * (1 / sqrt(sum(x^2) / hd + eps)) * w       (w given)
//   y[l]        = a[l] cos[p][l] - a[l + hd/2] sin[p][l]
//   y[l + hd/2] = a[l + hd/2] cos[p][l] + a[l] sin[p][l]   (cos, sin given)
// and a query is multiplied by q_scale at last; each result is rounded once, to
// the type it is stored in.
#include "paged.h"

namespace gphq {

struct AppendArgs {
    PagedBatch b;
    PagedPool pool;
    const void *qkv;
    void *q;
    const float *qn, *kn, *cos, *sin;
    int64_t qkv_stride, q_stride;
    int rope_rows, heads, parts;
    float eps, qscale;
};

// One wavefront takes the head items part, part + parts, ... of a row, four at
// a time: 16 lanes to an item, lane j holding values (HD/32) j .. of both
// halves, so a rotary pair is in one lane. For HD = 128 and fp32 rows the
// arithmetic and its order are those of the batched pass's and of the decode
// step's own kernels, so a key row stored in an fp32 page equals, bit for bit,
// the row that a private prefix would hold.
//
// Bound by memory in long calls: every value is read once and written once, 3417 fp32 rows of
// 32 + 16 heads to fp32 pages 37.3 us (170 MB, 4.6 TB/s, where a plain copy makes 5.1); by its
// chain of loads (sequence, page, then the stores) in short ones, one row 3 us. A wavefront
// of four items, the next four loaded while these are worked on, keeps 2 KB a wavefront on
// its way at 60 registers, eight wavefronts a SIMD.
template <typename RT, typename CT, int HD>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendArgs a) {
    constexpr int E = HD / 32;  // values of each half per lane
    const int lane = threadIdx.x & 63, j = lane & 15, slot = lane >> 4;
    const int unit = uniform((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int row = unit / a.parts, part = unit - row * a.parts;
    if (row >= a.b.rows) return;
    const int kvh = a.pool.kv_heads, rot = a.heads + kvh, items = rot + kvh;
    const RT *src = (const RT *)a.qkv + (int64_t)row * a.qkv_stride + E * j;
    const int stride = 4 * a.parts;
    int h = 4 * part + slot;
    int hc = min(h, items - 1);  // every lane takes part in the lane exchanges
    float x0[E], x1[E];
    load_vec(src + (int64_t)hc * HD, x0);
    load_vec(src + (int64_t)hc * HD + HD / 2, x1);

    const SeqRow s = find_seq(a.b, row);
    if (row < s.start || row >= s.end) {
        // Before the first sequence or behind the last: left alone. Else in none by bad starts.
        if (row >= a.b.starts[0] && row < a.b.starts[a.b.seqs] && lane == 0) paged_flag(a.b, PAGED_BAD_SEQ);
        return;
    }
    const int pos = s.len - (s.end - row);
    if (!seq_ok(a.b, s.start, s.end, s.len) || pos < 0) {
        if (lane == 0) paged_flag(a.b, PAGED_BAD_SEQ);
        return;
    }
    if (a.cos && pos >= a.rope_rows) {
        if (lane == 0) paged_flag(a.b, PAGED_BAD_POSITION);
        return;
    }
    const int page = a.b.table[s.seq * a.b.table_stride + (pos >> a.pool.shift)];
    const bool stored = page >= 0 && page < a.pool.pages;
    if (!stored && lane == 0) paged_flag(a.b, PAGED_BAD_PAGE);
    const int64_t place = (int64_t)(stored ? page : 0) * a.pool.page_stride +
                          (int64_t)(pos & ((1 << a.pool.shift) - 1)) * a.pool.token_stride + E * j;
    float cs[E], sn[E];
    if (a.cos) {
        load_vec(a.cos + (int64_t)pos * (HD / 2) + E * j, cs);
        load_vec(a.sin + (int64_t)pos * (HD / 2) + E * j, sn);
    }
    while (true) {
        const int hn = h + stride;
        float y0[E], y1[E];
#pragma unroll
        for (int i = 0; i < E; ++i) y0[i] = x0[i], y1[i] = x1[i];
        const int hcur = hc;
        const bool more = uniform(hn - slot) < items;
        if (more) {  // the next items' values, while these are worked on
            hc = min(hn, items - 1);
            load_vec(src + (int64_t)hc * HD, x0);
            load_vec(src + (int64_t)hc * HD + HD / 2, x1);
        }
        const bool isQ = hcur < a.heads, isV = hcur >= rot;
        const float *w = isQ ? a.qn : a.kn;
        if (w) {
            float p[E];
#pragma unroll
            for (int i = 0; i < E; ++i) p[i] = y0[i] * y0[i] + y1[i] * y1[i];
            float v = E == 4 ? (p[0] + p[1]) + (p[E / 2] + p[E - 1]) : p[0] + p[E - 1];
            v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
            v += __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
            v += __shfl_xor(v, 4);
            v += __shfl_xor(v, 8);
            const float inv = 1.0f / sqrtf(v / (float)HD + a.eps);
            if (!isV) {
                float w0[E], w1[E];
                load_vec(w + E * j, w0);
                load_vec(w + HD / 2 + E * j, w1);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    y0[i] *= inv * w0[i];
                    y1[i] *= inv * w1[i];
                }
            }
        }
        if (a.cos && !isV) {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float u = y0[i], v = y1[i];
                y0[i] = u * cs[i] - v * sn[i];
                y1[i] = v * cs[i] + u * sn[i];
            }
        }
        if (h < items) {
            if (isQ) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    y0[i] *= a.qscale;
                    y1[i] *= a.qscale;
                }
                RT *d = (RT *)a.q + (int64_t)row * a.q_stride + (int64_t)hcur * HD + E * j;
                store_vec(d, y0);
                store_vec(d + HD / 2, y1);
            } else if (stored) {
                CT *d = (CT *)(isV ? a.pool.v : a.pool.k) + place +
                        (int64_t)(hcur - (isV ? rot : a.heads)) * a.pool.head_stride;
                store_vec(d, y0);
                store_vec(d + HD / 2, y1);
            }
        }
        if (!more) break;
        h = hn;
    }
}

template <typename RT, typename CT>
int append_hd(const AppendArgs &a, int hd, unsigned blocks, hipStream_t st) {
    if (hd == 128)
        hipLaunchKernelGGL((paged_append_kernel<RT, CT, 128>), dim3(blocks), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((paged_append_kernel<RT, CT, 64>), dim3(blocks), dim3(256), 0, st, a);
    return launch_status();
}

}  // namespace gphq

using namespace gphq;

extern "C" int gphq_paged_append(const gphq_paged_kv *kv, const gphq_paged_batch *batch, int row_dtype,
                                 const void *qkv, int64_t qkv_stride, int64_t heads, const float *q_norm,
                                 const float *k_norm, double eps, const float *cos, const float *sin,
                                 int64_t rope_rows, double q_scale, void *q, int64_t q_stride, void *stream) {
    AppendArgs a{};
    GPHQ_TRY(paged_args(kv, batch, a.pool, a.b));
    const int64_t hd = kv->head_dim, rb = row_dtype == GPHQ_DTYPE_F32 ? 4 : 2;
    if (row_dtype != GPHQ_DTYPE_F32 && row_dtype != kv->dtype) return GPHQ_ERR_UNSUPPORTED;
    if (heads < 1 || heads > GPHQ_PAGED_MAX_HEADS || heads % kv->kv_heads) return GPHQ_ERR_PAGED_SHAPE;
    const int64_t items = heads + 2 * kv->kv_heads;
    if (qkv_stride < items * hd || q_stride < heads * hd || qkv_stride * rb % 16 || q_stride * rb % 16)
        return GPHQ_ERR_PAGED_SHAPE;
    if (!cos != !sin || (cos && rope_rows < 1)) return GPHQ_ERR_PAGED_SHAPE;
    if ((q_norm || k_norm) && !(eps >= 0)) return GPHQ_ERR_PAGED_SHAPE;
    if (a.b.rows == 0) return GPHQ_OK;
    const uintptr_t bits = (uintptr_t)qkv | (uintptr_t)q | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)cos |
                           (uintptr_t)sin;
    if (!qkv || !q || bits % 16) return GPHQ_ERR_PAGED_SHAPE;
    // Queries may replace the rows' own (a lane writes back what it alone has read), not lie over them otherwise.
    if (!(q == qkv && q_stride == qkv_stride) &&
        spans_overlap(qkv, span_bytes(a.b.rows, qkv_stride, items * hd, rb), q, span_bytes(a.b.rows, q_stride, heads * hd, rb)))
        return GPHQ_ERR_OVERLAP;
    a.qkv = qkv;
    a.q = q;
    a.qn = q_norm;
    a.kn = k_norm;
    a.cos = cos;
    a.sin = sin;
    a.qkv_stride = qkv_stride;
    a.q_stride = q_stride;
    a.rope_rows = (int)std::min<int64_t>(rope_rows, INT32_MAX);
    a.heads = (int)heads;
    a.eps = (float)eps;
    a.qscale = (float)q_scale;
    // Wavefronts per row: all of a row's items at once while that leaves the
    // chip short of wavefronts, else fewer, each over several groups of four.
    const int64_t groups = (items + 3) / 4, want = 32ll * device_cus();
    a.parts = (int)std::min<int64_t>(groups, std::max<int64_t>(1, (want + a.b.rows - 1) / a.b.rows));
    const unsigned blocks = (unsigned)(((int64_t)a.b.rows * a.parts + 3) / 4);
    hipStream_t st = (hipStream_t)stream;
    if (row_dtype == GPHQ_DTYPE_F32) {
        if (kv->dtype == GPHQ_DTYPE_F32) return append_hd<float, float>(a, (int)hd, blocks, st);
        if (kv->dtype == GPHQ_DTYPE_F16) return append_hd<float, f16>(a, (int)hd, blocks, st);
        return append_hd<float, bf16>(a, (int)hd, blocks, st);
    }
    if (kv->dtype == GPHQ_DTYPE_F16) return append_hd<f16, f16>(a, (int)hd, blocks, st);
    return append_hd<bf16, bf16>(a, (int)hd, blocks, st);
}
