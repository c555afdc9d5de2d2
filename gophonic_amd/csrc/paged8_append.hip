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
//   code = round(y / s'), of the true quotient: y (1 / s') and one step on its remainder
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
    int by_row;          // a block of the key and value part takes the 16-token block that a row begins, not a numbered one
    int kv_parts;        // blocks that share a 16-token block's heads
    int q_parts;         // wavefronts of a row in the query part
    unsigned kv_blocks;  // blocks of the key and value part; the query part's come behind them
    double eps;
    float qscale;
};

// Another lane's value, by a DPP control that exchanges lanes of a row of 16.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)u, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
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
        for (int i = 0; i < E; ++i) {
            // Cut to 20 bits of fraction, the last of them set where others were: one rounding, not two.
            const uint64_t u = __builtin_bit_cast(uint64_t, y[i]);
            const uint32_t hi = (uint32_t)(u >> 32) | ((uint32_t)u ? 1u : 0u);
            f[i] = fminf(fmaxf((float)__builtin_bit_cast(double, (uint64_t)hi << 32), -448.0f), 448.0f);
        }
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

// The new tokens [n0, n1) of one block of a sequence, which stand in rows row .. of the batch:
// keys and values of every kv_parts-th KV head from `part` on. A block's 256 threads take the 16
// tokens, 16 lanes each, lane j of them holding values E j .. of both halves (a rotary pair is in one
// lane); the wavefronts' largest magnitudes meet in LDS, in two places in turn, so that one barrier
// a head is enough.
template <typename RT, typename C, int HD>
__device__ __forceinline__ void append_block(const Append8Args &a, int row, int n0, int n1, int page, int part) {
    constexpr int E = HD / 32;
    __shared__ double tops[2][4];
    const int lane = threadIdx.x & 63, j = lane & 15, wave = threadIdx.x >> 6;
    const int b0 = n0 & ~(kBlockTokens - 1), kvh = a.pool.kv_heads;
    const int pos = b0 + (threadIdx.x >> 4);
    const bool mine = pos >= n0 && pos < n1, earlier = pos < n0;
    const int p = mine ? pos : n0;
    const RT *src = (const RT *)a.qkv + (int64_t)(row + p - n0) * a.qkv_stride + (int64_t)a.heads * HD + E * j;
    const int in = b0 & ((1 << a.pool.shift) - 1);
    const int64_t code_at = (int64_t)page * a.pool.page_stride + (int64_t)(in + pos - b0) * a.pool.token_stride + E * j;
    const int64_t scale_at = (int64_t)page * a.s.page_stride + in / kBlockTokens;
    float x0[E], x1[E], w0[E], w1[E], cs[E], sn[E];
    load_vec(src + (int64_t)part * HD, x0);
    load_vec(src + (int64_t)part * HD + HD / 2, x1);
    if (a.kn) {
        load_vec(a.kn + E * j, w0);
        load_vec(a.kn + HD / 2 + E * j, w1);
    }
    if (a.cos) {
        load_vec(a.cos + (int64_t)p * (HD / 2) + E * j, cs);
        load_vec(a.sin + (int64_t)p * (HD / 2) + E * j, sn);
    }
    int turn = 0;
    for (int item = part; item < 2 * kvh; item += a.kv_parts, turn ^= 1) {
        const bool key = item < kvh;
        const int head = key ? item : item - kvh;
        char *codes = (char *)(key ? a.pool.k : a.pool.v) + code_at + (int64_t)head * a.pool.head_stride;
        float *at = (key ? a.s.k : a.s.v) + scale_at + (int64_t)head * a.s.head_stride;
        const float old = n0 > b0 ? *at : 0.0f;  // read by all before the barrier, written behind it
        double y[2 * E], sum = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            y[e] = x0[e];
            y[E + e] = x1[e];
            sum += y[e] * y[e] + y[E + e] * y[E + e];
        }
        if (item + a.kv_parts < 2 * kvh) {  // the next head's values, while these are worked on
            load_vec(src + (int64_t)(item + a.kv_parts) * HD, x0);
            load_vec(src + (int64_t)(item + a.kv_parts) * HD + HD / 2, x1);
        }
        if (key && a.kn) {
            sum += dpp_f64<0xB1>(sum);
            sum += dpp_f64<0x4E>(sum);
            sum += dpp_f64<0x141>(sum);
            sum += dpp_f64<0x140>(sum);
            const double inv = 1.0 / sqrt(sum / HD + a.eps);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                y[e] *= inv * w0[e];
                y[E + e] *= inv * w1[e];
            }
        }
        if (key && a.cos) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double u = y[e], v = y[E + e];
                y[e] = u * cs[e] - v * sn[e];
                y[E + e] = v * cs[e] + u * sn[e];
            }
        }
        double most = 0.0;
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) {
            const bool fine = fabs(y[e]) <= (double)FLT_MAX;
            odd |= mine && !fine;
            if (!fine) y[e] = 0.0;
            most = mine ? fmax(most, fabs(y[e])) : most;
        }
        if (odd) paged_flag(a.b, PAGED_BAD_VALUE);
        most = fmax(most, dpp_f64<0xB1>(most));
        most = fmax(most, dpp_f64<0x4E>(most));
        most = fmax(most, dpp_f64<0x141>(most));
        most = fmax(most, dpp_f64<0x140>(most));
        most = fmax(most, shfl_xor_f64(most, 16));
        most = fmax(most, shfl_xor_f64(most, 32));
        if (lane == 0) tops[turn][wave] = most;
        __syncthreads();
        most = fmax(fmax(tops[turn][0], tops[turn][1]), fmax(tops[turn][2], tops[turn][3]));

        float scale = most > 0.0 ? fminf(fmaxf((float)(most / C::kTop), 0x1p-126f), FLT_MAX) : 0.0f;
        if (old > 0.0f && old < INFINITY) {
            const double r = most / ((double)C::kOver * old);
            int k = 0;
            if (r > 1.0) {
                const int e = __builtin_amdgcn_frexp_exp(r);
                k = __builtin_amdgcn_frexp_mant(r) == 0.5 ? e - 1 : e;
            }
            scale = __builtin_amdgcn_ldexpf(old, k);
            if (k && earlier) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    double c[E];
                    decode<C>(load_codes<E>(codes + h * (HD / 2)), c);
#pragma unroll
                    for (int e = 0; e < E; ++e) c[e] = ldexp(c[e], -k);
                    store_codes<E>(codes + h * (HD / 2), encode<C>(c));
                }
            }
        }
        if (threadIdx.x == 0) *at = scale;
        const double inv = scale > 0.0f ? 1.0 / (double)scale : 0.0;
        if (mine) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                double c[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    // The quotient or a step beside it, then the nearest to it (these signs keep that of a zero).
                    const double v = y[h * E + e], near = v * inv;
                    c[e] = fma(-fma(near, (double)scale, -v), inv, near);
                }
                store_codes<E>(codes + h * (HD / 2), encode<C>(c));
            }
        }
    }
    __syncthreads();  // the last heads' tops have been read
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

// The 16-token blocks of a batch by numbers: a sequence's n tokens touch n / 16 + 2 of them at most
// (rounded down), so those of sequence s get the numbers from starts[s] / 16 + 2 s on. False for a number
// that no block has. Its first new token is in row `row`, at position pos, the block's last before n1.
__device__ __forceinline__ bool block_of(const Append8Args &a, int number, SeqRow &s, int &row, int &pos, int &n1) {
    const PagedBatch &b = a.b;
    const int lane = threadIdx.x & 63;
    int lo = 0, cnt = b.seqs;
    while (cnt > 64) {
        const int step = (cnt + 63) / 64, i = min(lane * step, cnt - 1);
        const int at = last_lane(__ballot(lane * step < cnt && (b.starts[lo + i] >> 4) + 2 * (lo + i) <= number)) * step;
        lo += at;
        cnt = min(step, cnt - at);
    }
    const int i = lo + min(lane, cnt - 1);
    const int s0 = b.starts[i], s1 = b.starts[i + 1], len = b.lens[i];
    const int at = last_lane(__ballot(lane < cnt && (s0 >> 4) + 2 * i <= number));
    s = SeqRow{lo + at, __builtin_amdgcn_readlane(s0, at), __builtin_amdgcn_readlane(s1, at),
               __builtin_amdgcn_readlane(len, at)};
    if (!seq_ok(b, s.start, s.end, s.len)) return false;  // (flagged by its rows' queries)
    const int shift = s.len - (s.end - s.start), first = max(shift, 0), k = number - ((s.start >> 4) + 2 * s.seq);
    const int end = a.cos ? min(s.len, a.rope_rows) : s.len;
    if (k < 0) return false;
    pos = k == 0 ? first : (first & ~(kBlockTokens - 1)) + k * kBlockTokens;
    n1 = min((pos & ~(kBlockTokens - 1)) + kBlockTokens, end);
    row = s.start + pos - shift;
    return pos < end && find_seq(b, row).seq == s.seq;  // (not so where starts descend)
}

// The same by the row: false where it is not the first new one of a 16-token block, or cannot be placed.
__device__ __forceinline__ bool block_at(const Append8Args &a, int row, SeqRow &s, int &pos, int &n1) {
    if (!row_of(a.b, row, s)) return false;
    const int shift = s.len - (s.end - s.start), end = a.cos ? min(s.len, a.rope_rows) : s.len;
    pos = row - s.start + shift;
    n1 = min((pos & ~(kBlockTokens - 1)) + kBlockTokens, end);
    return pos >= 0 && pos < end && (pos == max(shift, 0) || pos % kBlockTokens == 0);
}

// One grid for both parts. Keys and values: a block takes every kv_parts-th head's keys or values of
// one 16-token block. Queries: a wavefront takes every q_parts-th four heads of a row.
//
// Bound by memory, and by the chain of loads before it where rows are few: five fp32 prompts of
// 3417 rows in all, 32 heads and 8 KV heads, 28.2 us with two sets of inputs, which the last-level cache
// keeps in part (144 MB, 5.1 TB/s); 64 single tokens 7.1 us. The 64-bit quotients cost 1.9 us of the former.
// A wavefront a block and head, with all its 16 tokens in registers, took 54.0 us when this took 37.9.
// Registers for more wavefronts a CU spilled: bounds of 5, 6 and 8 to a SIMD unit 39.6, 55.4 and 72.6 us
// beside those 37.9.
template <typename RT, typename C, int HD>
__global__ __launch_bounds__(256) void paged8_append_kernel(const Append8Args a) {
    constexpr int E = HD / 32;
    const int lane = threadIdx.x & 63, j = lane & 15, slot = lane >> 4;
    if (blockIdx.x < a.kv_blocks) {
        const int group = blockIdx.x / a.kv_parts, part = blockIdx.x - group * a.kv_parts;
        SeqRow s;
        int row = group, pos, n1;
        if (a.by_row ? !block_at(a, row, s, pos, n1) : !block_of(a, group, s, row, pos, n1)) return;
        const int page = a.b.table[s.seq * a.b.table_stride + (pos >> a.pool.shift)];
        if (page >= 0 && page < a.pool.pages)
            append_block<RT, C, HD>(a, row, pos, n1, page, part);
        else if (lane == 0)
            paged_flag(a.b, PAGED_BAD_PAGE);
        return;
    }
    const int unit = uniform((int)((blockIdx.x - a.kv_blocks) * 4 + (threadIdx.x >> 6)));
    const int row = unit / a.q_parts, part = unit - row * a.q_parts;
    if (row >= a.b.rows) return;
    const RT *src = (const RT *)a.qkv + (int64_t)row * a.qkv_stride + E * j;
    RT *dst = (RT *)a.q + (int64_t)row * a.q_stride + E * j;
    int h = 4 * part + slot, hc = min(h, a.heads - 1);  // every lane takes part in the lane exchanges
    float x0[E], x1[E];
    load_vec(src + (int64_t)hc * HD, x0);
    load_vec(src + (int64_t)hc * HD + HD / 2, x1);
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
    for (;;) {
        float y0[E], y1[E];
#pragma unroll
        for (int e = 0; e < E; ++e) y0[e] = x0[e], y1[e] = x1[e];
        const int now = h;
        h += 4 * a.q_parts;
        const bool more = uniform(h - slot) < a.heads;
        if (more) {  // the next heads' values, while these are worked on
            hc = min(h, a.heads - 1);
            load_vec(src + (int64_t)hc * HD, x0);
            load_vec(src + (int64_t)hc * HD + HD / 2, x1);
        }
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
        if (now < a.heads) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                y0[e] *= a.qscale;
                y1[e] *= a.qscale;
            }
            store_vec(dst + (int64_t)now * HD, y0);
            store_vec(dst + (int64_t)now * HD + HD / 2, y1);
        }
        if (!more) break;
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
    // Blocks by their numbers, or by rows, each looking whether it is the first of one, where there are
    // fewer rows (idle sequences have numbers, two each): 64 single tokens 7.8 us by rows, 7.9 by numbers;
    // five sequences of four rows 5.8 and 5.0. Before numbers, with a block for every four rows, 3417 rows took
    // 39.5 us (now 28.2), 512 rows 11.5 (7.1).
    const int64_t numbers = rows / kBlockTokens + 2 * (int64_t)a.b.seqs;
    a.by_row = rows <= numbers;
    // Blocks that share a 16-token block's heads: all while that leaves the chip short of wavefronts, else
    // fewer. With 8, 16, 24 and 32 wavefronts a CU wanted: 3417 rows 26.5, 28.2, 29.9, 32.5 us, forty
    // sequences of up to 80 rows 15.2, 12.3, 13.0, 14.4, 32 of five 8.3, 7.6, 7.5, 7.2.
    const int64_t spans = std::min(rows, numbers), want = 16ll * device_cus();
    a.kv_parts = (int)std::min<int64_t>(2 * kvh, std::max<int64_t>(1, want / 4 / spans));
    // Wavefronts per row of queries, likewise: of its heads four at a time.
    const int64_t groups = (heads + 3) / 4;
    a.q_parts = (int)std::min<int64_t>(groups, std::max<int64_t>(1, (want + rows - 1) / rows));
    a.kv_blocks = (unsigned)(spans * a.kv_parts);
    const unsigned blocks = a.kv_blocks + (unsigned)((rows * a.q_parts + 3) / 4);
    hipStream_t st = (hipStream_t)stream;
    const bool i8 = kv->codes.dtype == GPHQ_DTYPE_I8;
    if (row_dtype == GPHQ_DTYPE_F32)
        return i8 ? append8_hd<float, CodesI8>(a, (int)hd, blocks, st) : append8_hd<float, CodesE4M3>(a, (int)hd, blocks, st);
    if (row_dtype == GPHQ_DTYPE_F16)
        return i8 ? append8_hd<f16, CodesI8>(a, (int)hd, blocks, st) : append8_hd<f16, CodesE4M3>(a, (int)hd, blocks, st);
    return i8 ? append8_hd<bf16, CodesI8>(a, (int)hd, blocks, st) : append8_hd<bf16, CodesE4M3>(a, (int)hd, blocks, st);
}
