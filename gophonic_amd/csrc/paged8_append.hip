// gphq_paged8_append: a batch's fused QKV rows [heads | KV heads | KV heads] to prepared queries
// and to 8-bit codes of keys and values in the pages of their sequences, with a scale for every
// block of 16 tokens and KV head.
//
// Queries as paged_append.hip has them, in fp32. Keys (norm and rotation) and codes in 64 bits,
// so that a code does not hang on the order of a sum: what lies within fp32's rounding of the
// border between two codes would come out one way or the other. With m the largest magnitude of
// a block's new values and s the block's scale before them:
//   no earlier token in the block (or s no positive finite number): s' = m / top
//   else s' = 2^k s, the least k >= 0 with m <= over s', and earlier codes become round(c / 2^k)
//   code = round(y / s')
// A doubling costs an int8 code at most half a step, the next one half a step of half the size:
// together less than one step of s', however often the block grows.
#include "paged8.h"

namespace gphq {
namespace {

struct Append8Args {
    PagedBatch b;
    PagedPool pool;
    Paged8Scales s;
    const void *qkv;
    void *q;
    const float *qn, *kn, *cos, *sin;
    int64_t qkv_stride, q_stride;
    int rope_rows, heads;
    int span;          // rows whose blocks one wavefront of the key and value part looks for
    int q_parts;       // wavefronts of a row in the query part
    unsigned kv_blocks;  // blocks of the key and value part; the query part's come behind them
    double eps;
    float qscale;
};

__device__ __forceinline__ double shfl_xor_f64(double v, int mask) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __shfl_xor((int)(uint32_t)u, mask), hi = __shfl_xor((int)(uint32_t)(u >> 32), mask);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Four (or two) codes of values in units of their scale, in the low bytes.
template <typename C, int E>
__device__ __forceinline__ int encode(const double (&y)[E]) {
    int w = 0;
    if constexpr (std::is_same<C, CodesI8>::value) {
#pragma unroll
        for (int i = 0; i < E; ++i)
            w |= ((int)fmin(fmax(__builtin_rint(y[i]), -127.0), 127.0) & 255) << (8 * i);
    } else {
        float f[E];
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = fminf(fmaxf((float)y[i], -448.0f), 448.0f);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], w, false);
        if constexpr (E == 4) w = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
    }
    return w;
}

template <typename C, int E>
__device__ __forceinline__ void decode(int w, double (&y)[E]) {
    if constexpr (std::is_same<C, CodesI8>::value) {
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = (double)(int8_t)(w >> (8 * i));
    } else {
        const int r = C::ready(w);
        const f16x2 lo = __builtin_bit_cast(f16x2, C::template along<0>(r));
        y[0] = (double)(float)lo[0] * 256.0;
        y[1] = (double)(float)lo[1] * 256.0;
        if constexpr (E == 4) {
            const f16x2 hi = __builtin_bit_cast(f16x2, C::template along<2>(r));
            y[2] = (double)(float)hi[0] * 256.0;
            y[3] = (double)(float)hi[1] * 256.0;
        }
    }
}

template <int E>
__device__ __forceinline__ int load_codes(const char *p) {
    return E == 4 ? *(const int *)p : (int)*(const uint16_t *)p;
}
template <int E>
__device__ __forceinline__ void store_codes(char *p, int w) {
    if (E == 4)
        *(int *)p = w;
    else
        *(uint16_t *)p = (uint16_t)w;
}

// The new tokens [n0, n1) of one block of a sequence, which stand in rows row .. of the batch,
// for one KV head's keys or values. 16 lanes to a token, lane j holding values E j .. of both
// halves (a rotary pair is in one lane), four tokens at a time: tokens 4 i + lane / 16.
template <typename RT, typename C, int HD>
__device__ __forceinline__ void append_block(const Append8Args &a, int row, int n0, int n1, int page, bool key,
                                             int head) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 63, j = lane & 15, slot = lane >> 4;
    const int b0 = n0 & ~(kBlockTokens - 1), kvh = a.pool.kv_heads;
    const RT *src = (const RT *)a.qkv + (int64_t)(a.heads + (key ? 0 : kvh) + head) * HD + E * j;
    const float *w = key ? a.kn : nullptr;
    const bool rotate = key && a.cos;
    float w0[E], w1[E];
    if (w) {
        load_vec(w + E * j, w0);
        load_vec(w + HD / 2 + E * j, w1);
    }
    double y[4][2 * E];
    double most = 0.0;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pos = b0 + 4 * i + slot;
        const bool mine = pos >= n0 && pos < n1;
        const int p = mine ? pos : n0;
        const RT *x = src + (int64_t)(row + p - n0) * a.qkv_stride;
        float x0[E], x1[E];
        load_vec(x, x0);
        load_vec(x + HD / 2, x1);
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            y[i][e] = x0[e];
            y[i][E + e] = x1[e];
            sum += y[i][e] * y[i][e] + y[i][E + e] * y[i][E + e];
        }
        if (w) {
#pragma unroll
            for (int d = 1; d < 16; d *= 2) sum += shfl_xor_f64(sum, d);
            const double inv = 1.0 / sqrt(sum / HD + a.eps);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                y[i][e] *= inv * w0[e];
                y[i][E + e] *= inv * w1[e];
            }
        }
        if (rotate) {
            float cs[E], sn[E];
            load_vec(a.cos + (int64_t)p * (HD / 2) + E * j, cs);
            load_vec(a.sin + (int64_t)p * (HD / 2) + E * j, sn);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double u = y[i][e], v = y[i][E + e];
                y[i][e] = u * cs[e] - v * sn[e];
                y[i][E + e] = v * cs[e] + u * sn[e];
            }
        }
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) {
            const bool fine = fabs(y[i][e]) < (double)INFINITY;
            odd |= mine && !fine;
            if (!fine) y[i][e] = 0.0;
            most = mine ? fmax(most, fabs(y[i][e])) : most;
        }
    }
    if (odd) paged_flag(a.b, PAGED_BAD_VALUE);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) most = fmax(most, shfl_xor_f64(most, d));

    const int in = b0 & ((1 << a.pool.shift) - 1);
    char *codes = (char *)(key ? a.pool.k : a.pool.v) + (int64_t)page * a.pool.page_stride +
                  (int64_t)head * a.pool.head_stride + (int64_t)in * a.pool.token_stride + E * j;
    float *at = (key ? a.s.k : a.s.v) + (int64_t)page * a.s.page_stride + (int64_t)head * a.s.head_stride +
                in / kBlockTokens;
    float scale = most > 0.0 ? fmaxf((float)(most / C::kTop), 0x1p-126f) : 0.0f;
    scale = fminf(scale, FLT_MAX);
    if (n0 > b0) {
        const float old = *at;
        if (old > 0.0f && old < INFINITY) {
            const double r = most / ((double)C::kOver * old);
            int k = 0;
            if (r > 1.0) {
                const int e = __builtin_amdgcn_frexp_exp(r);
                k = __builtin_amdgcn_frexp_mant(r) == 0.5 ? e - 1 : e;
            }
            scale = __builtin_amdgcn_ldexpf(old, k);
            if (k) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (b0 + 4 * i + slot >= n0) continue;
                    char *p = codes + (int64_t)(4 * i + slot) * a.pool.token_stride;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        double c[E];
                        decode<C>(load_codes<E>(p + h * (HD / 2)), c);
#pragma unroll
                        for (int e = 0; e < E; ++e) c[e] = ldexp(c[e], -k);
                        store_codes<E>(p + h * (HD / 2), encode<C>(c));
                    }
                }
            }
        }
    }
    if (lane == 0) *at = scale;
    const double inv = scale > 0.0f ? 1.0 / (double)scale : 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int pos = b0 + 4 * i + slot;
        if (pos < n0 || pos >= n1) continue;
        char *p = codes + (int64_t)(4 * i + slot) * a.pool.token_stride;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            double c[E];
#pragma unroll
            for (int e = 0; e < E; ++e) c[e] = y[i][h * E + e] * inv;
            store_codes<E>(p + h * (HD / 2), encode<C>(c));
        }
    }
}

// What find_seq says of a row, checked: false (and flagged) for a row that no sequence brings.
__device__ __forceinline__ bool row_of(const PagedBatch &b, int row, SeqRow &s) {
    const bool lane0 = (threadIdx.x & 63) == 0;
    s = find_seq(b, row);
    if (row < s.start || row >= s.end) {
        // Before the first sequence or behind the last: left alone. Else in none by bad starts.
        if (row >= b.starts[0] && row < b.starts[b.seqs] && lane0) paged_flag(b, PAGED_BAD_SEQ);
        return false;
    }
    if (!seq_ok(b, s.start, s.end, s.len)) {
        if (lane0) paged_flag(b, PAGED_BAD_SEQ);
        return false;
    }
    return true;
}

// One grid for both parts. Keys and values: a wavefront takes one head's keys or values of the
// blocks whose first new token lies in `span` rows of the batch. Queries: a wavefront takes every
// q_parts-th four heads of a row.
template <typename RT, typename C, int HD>
__global__ __launch_bounds__(256) void paged8_append_kernel(const Append8Args a) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 63, j = lane & 15, slot = lane >> 4;
    const int kvh = a.pool.kv_heads;
    if (blockIdx.x < a.kv_blocks) {
        const int unit = uniform((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
        const int group = unit / (2 * kvh), item = unit - group * 2 * kvh;
        const int r1 = min((group + 1) * a.span, a.b.rows);
        for (int row = group * a.span; row < r1;) {
            SeqRow s;
            if (!row_of(a.b, row, s)) {
                ++row;
                continue;
            }
            const int pos = s.len - (s.end - row), first = max(s.len - (s.end - s.start), 0);
            const int n1 = min((pos & ~(kBlockTokens - 1)) + kBlockTokens, a.cos ? min(s.len, a.rope_rows) : s.len);
            const bool lead = pos == first || pos % kBlockTokens == 0;
            if (pos < 0 || pos >= n1) {  // a row before token 0, or past the rotary table: flagged below
                ++row;
                continue;
            }
            if (lead) {
                const int page = a.b.table[s.seq * a.b.table_stride + (pos >> a.pool.shift)];
                if (page >= 0 && page < a.pool.pages)
                    append_block<RT, C, HD>(a, row, pos, n1, page, item < kvh, item < kvh ? item : item - kvh);
                else if (lane == 0)
                    paged_flag(a.b, PAGED_BAD_PAGE);
            }
            row += n1 - pos;
        }
        return;
    }
    const int unit = uniform((int)((blockIdx.x - a.kv_blocks) * 4 + (threadIdx.x >> 6)));
    const int row = unit / a.q_parts, part = unit - row * a.q_parts;
    if (row >= a.b.rows) return;
    SeqRow s;
    if (!row_of(a.b, row, s)) return;
    const int pos = s.len - (s.end - row);
    if (pos < 0) {
        if (lane == 0) paged_flag(a.b, PAGED_BAD_SEQ);
        return;
    }
    if (a.cos && pos >= a.rope_rows) {
        if (lane == 0) paged_flag(a.b, PAGED_BAD_POSITION);
        return;
    }
    float cs[E], sn[E], w0[E], w1[E];
    if (a.cos) {
        load_vec(a.cos + (int64_t)pos * (HD / 2) + E * j, cs);
        load_vec(a.sin + (int64_t)pos * (HD / 2) + E * j, sn);
    }
    if (a.qn) {
        load_vec(a.qn + E * j, w0);
        load_vec(a.qn + HD / 2 + E * j, w1);
    }
    const RT *src = (const RT *)a.qkv + (int64_t)row * a.qkv_stride + E * j;
    RT *dst = (RT *)a.q + (int64_t)row * a.q_stride + E * j;
    for (int h0 = 4 * part; h0 < a.heads; h0 += 4 * a.q_parts) {
        const int h = h0 + slot, hc = min(h, a.heads - 1);  // every lane takes part in the lane exchanges
        float y0[E], y1[E];
        load_vec(src + (int64_t)hc * HD, y0);
        load_vec(src + (int64_t)hc * HD + HD / 2, y1);
        if (a.qn) {
            float v = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) v += y0[e] * y0[e] + y1[e] * y1[e];
            v = row16_sum(v);
            const float inv = 1.0f / sqrtf(v / (float)HD + (float)a.eps);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                y0[e] *= inv * w0[e];
                y1[e] *= inv * w1[e];
            }
        }
        if (a.cos) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float u = y0[e], v = y1[e];
                y0[e] = u * cs[e] - v * sn[e];
                y1[e] = v * cs[e] + u * sn[e];
            }
        }
        if (h < a.heads) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                y0[e] *= a.qscale;
                y1[e] *= a.qscale;
            }
            store_vec(dst + (int64_t)h * HD, y0);
            store_vec(dst + (int64_t)h * HD + HD / 2, y1);
        }
    }
}

template <typename RT, typename C>
int append8_hd(const Append8Args &a, int hd, unsigned blocks, hipStream_t st) {
    if (hd == 128)
        hipLaunchKernelGGL((paged8_append_kernel<RT, C, 128>), dim3(blocks), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((paged8_append_kernel<RT, C, 64>), dim3(blocks), dim3(256), 0, st, a);
    return launch_status();
}

}  // namespace
}  // namespace gphq

using namespace gphq;

extern "C" int gphq_paged8_append(const gphq_paged8_kv *kv, const gphq_paged_batch *batch, int row_dtype,
                                  const void *qkv, int64_t qkv_stride, int64_t heads, const float *q_norm,
                                  const float *k_norm, double eps, const float *cos, const float *sin,
                                  int64_t rope_rows, double q_scale, void *q, int64_t q_stride, void *stream) {
    Append8Args a{};
    GPHQ_TRY(paged8_args(kv, batch, a.pool, a.s, a.b));
    const int64_t hd = kv->codes.head_dim, kvh = kv->codes.kv_heads, rb = row_dtype == GPHQ_DTYPE_F32 ? 4 : 2;
    if (row_dtype != GPHQ_DTYPE_F32 && row_dtype != GPHQ_DTYPE_F16 && row_dtype != GPHQ_DTYPE_BF16)
        return GPHQ_ERR_UNSUPPORTED;
    if (heads < 1 || heads > GPHQ_PAGED_MAX_HEADS || heads % kvh) return GPHQ_ERR_PAGED_SHAPE;
    const int64_t items = heads + 2 * kvh;
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
        spans_overlap(qkv, span_bytes(a.b.rows, qkv_stride, items * hd, rb), q,
                      span_bytes(a.b.rows, q_stride, heads * hd, rb)))
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
    a.eps = eps;
    a.qscale = (float)q_scale;
    const int64_t rows = a.b.rows;
    // Rows that a wavefront looks through for blocks, and no more than 2^22 wavefronts.
    a.span = (int)std::max<int64_t>(a.b.max_rows == 1 ? 1 : 4, (rows * 2 * kvh + (1 << 22) - 1) >> 22);
    const int64_t kv_units = (rows + a.span - 1) / a.span * 2 * kvh;
    // Wavefronts per row of queries: all of a row's heads at once while that leaves the chip
    // short of wavefronts, else fewer, each over several groups of four.
    const int64_t groups = (heads + 3) / 4, want = 32ll * device_cus();
    a.q_parts = (int)std::min<int64_t>(groups, std::max<int64_t>(1, (want + rows - 1) / rows));
    a.kv_blocks = (unsigned)((kv_units + 3) / 4);
    const unsigned blocks = a.kv_blocks + (unsigned)((rows * a.q_parts + 3) / 4);
    hipStream_t st = (hipStream_t)stream;
    const bool i8 = kv->codes.dtype == GPHQ_DTYPE_I8;
    if (row_dtype == GPHQ_DTYPE_F32)
        return i8 ? append8_hd<float, CodesI8>(a, (int)hd, blocks, st) : append8_hd<float, CodesE4M3>(a, (int)hd, blocks, st);
    if (row_dtype == GPHQ_DTYPE_F16)
        return i8 ? append8_hd<f16, CodesI8>(a, (int)hd, blocks, st) : append8_hd<f16, CodesE4M3>(a, (int)hd, blocks, st);
    return i8 ? append8_hd<bf16, CodesI8>(a, (int)hd, blocks, st) : append8_hd<bf16, CodesE4M3>(a, (int)hd, blocks, st);
}
