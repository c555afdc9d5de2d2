// gphq_probabilities and gphq_verify_drafts: from a head's logits to the tokens that a step keeps.
#include <float.h>

#include "paged.h"

namespace gphq {
namespace {

constexpr int kThreads = 256, kPer = 16, kTile = kThreads * kPer;  // values of a row that a block takes at once

// N neighbouring values from i on of a row of n: 16 bytes at a time where rows allow it (VEC).
template <bool VEC, int N>
__device__ __forceinline__ void load_row(const float *x, int i, int n, float fill, float (&v)[N]) {
    if (VEC && i + N <= n) {
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const f32x4 q = *(const f32x4 *)(x + i + k);
            v[k] = q.x, v[k + 1] = q.y, v[k + 2] = q.z, v[k + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = i + k < n ? x[i + k] : fill;
    }
}

// ---- probabilities --------------------------------------------------------------

struct ProbArgs {
    const float *x, *temperatures;
    float *out;
    float2 *part;  // [rows][parts]: (largest, sum of exponentials against it), or (largest, its index) at t = 0
    int64_t x_stride, out_stride;
    int rows, n, parts, len;  // len: values of a part, a multiple of kTile
};

// log2(e) / t in two floats, 0 for a row that takes its largest value alone.
struct Rate {
    float hi, lo;
};
__device__ __forceinline__ Rate rate_of(const ProbArgs &a, int row) {
    const float t = a.temperatures ? a.temperatures[row] : 1.0f;
    if (!(t > 0.0f)) return Rate{0.0f, 0.0f};
    constexpr float hi = 1.44269504088896340736f, lo = (float)(1.44269504088896340736 - (double)hi);
    const float q = hi / t;
    if (!(q >= FLT_MIN && q <= FLT_MAX)) return Rate{q < 1.0f ? FLT_MIN : FLT_MAX, 0.0f};
    return Rate{q, (fmaf(-q, t, hi) + lo) / t};
}
// exp(d / t), d at most 0. The exponent's rounding, up to 2^-24 of it, is put back as a factor: one row of
// 151936 is 1.3e-7 off its 64-bit values with it and 2.1e-7 without, which saves 0.6 of 5.0 us of a kernel
// on one row and 2.8 of 48.8 us on 160.
__device__ __forceinline__ float power(float d, Rate r) {
    const float e = d * r.hi, rest = e > -160.0f ? fmaf(d, r.lo, fmaf(d, r.hi, -e)) : 0.0f;
    const float p = __builtin_amdgcn_exp2f(e);
    return fmaf(p, rest * 0.693147180559945309417f, p);
}

// Joins two (largest, sum) pairs.
__device__ __forceinline__ void join_sums(float &m, float &s, float m2, float s2, Rate rate) {
    const float mx = fmaxf(m, m2), ref = mx == -INFINITY ? 0.0f : mx;
    s = s * power(m - ref, rate) + s2 * power(m2 - ref, rate);
    m = mx;
}
// Joins two (largest, first index of it) pairs.
__device__ __forceinline__ void join_first(float &m, int &i, float m2, int i2) {
    if (m2 > m || (m2 == m && i2 < i)) m = m2, i = i2;
}

// A block's pairs to one, in a fixed order; the same in every thread.
__device__ __forceinline__ void block_join(float &m, float &s, int &first, Rate rate) {
    __shared__ float sm[4], ss[4];
    __shared__ int si[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const float m2 = __shfl_xor(m, d), s2 = __shfl_xor(s, d);
        const int i2 = __shfl_xor(first, d);
        if (rate.hi > 0.0f)
            join_sums(m, s, m2, s2, rate);
        else
            join_first(m, first, m2, i2);
    }
    if (lane == 0) sm[wave] = m, ss[wave] = s, si[wave] = first;
    __syncthreads();
    m = sm[0], s = ss[0], first = si[0];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
        if (rate.hi > 0.0f)
            join_sums(m, s, sm[w], ss[w], rate);
        else
            join_first(m, first, sm[w], si[w]);
    }
}

// Two passes over a row: its parts' pairs, then all of them joined by every block, and the values. Bound by
// memory, read twice and written once: 160 rows of 151936 (97 MB) 19.8 and 29.0 us, 55.1 in calls one behind
// the other. One row 4.2 and 5.0 us, all latency: 38 blocks of 4096 values.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void prob_parts_kernel(const ProbArgs a) {
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const float *x = a.x + (int64_t)row * a.x_stride;
    const Rate rate = rate_of(a, row);
    const int end = min(a.n, (part + 1) * a.len);
    float m = -INFINITY, s = 0.0f;
    int first = INT32_MAX;
    for (int i0 = part * a.len; i0 < end; i0 += kTile) {
        float v[kPer];
#pragma unroll
        for (int k = 0; k < kPer; k += 4) {
            float q[4];
            load_row<VEC>(x, i0 + k * kThreads + 4 * threadIdx.x, end, -INFINITY, q);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[k + e] = q[e];
        }
        if (rate.hi > 0.0f) {
            float mx = m, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < kPer; ++k) mx = fmaxf(mx, v[k]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int k = 0; k < kPer; ++k) sum += power(v[k] - ref, rate);
            s = s * power(m - ref, rate) + sum;
            m = mx;
        } else {
#pragma unroll
            for (int k = 0; k < kPer; ++k)
                if (v[k] > m) m = v[k], first = i0 + k / 4 * 4 * kThreads + 4 * threadIdx.x + k % 4;
        }
    }
    block_join(m, s, first, rate);
    if (threadIdx.x == 0) a.part[blockIdx.x] = make_float2(m, rate.hi > 0.0f ? s : __builtin_bit_cast(float, first));
}

template <bool VEC>
__global__ __launch_bounds__(kThreads) void prob_write_kernel(const ProbArgs a) {
    const int row = blockIdx.x / a.parts, part = blockIdx.x - row * a.parts;
    const float *x = a.x + (int64_t)row * a.x_stride;
    float *out = a.out + (int64_t)row * a.out_stride;
    const Rate rate = rate_of(a, row);
    float m = -INFINITY, s = 0.0f;
    int first = INT32_MAX;
    for (int p = threadIdx.x; p < a.parts; p += kThreads) {
        const float2 q = a.part[(int64_t)row * a.parts + p];
        if (rate.hi > 0.0f)
            join_sums(m, s, q.x, q.y, rate);
        else
            join_first(m, first, q.x, __builtin_bit_cast(int, q.y));
    }
    block_join(m, s, first, rate);
    const float ref = m == -INFINITY ? 0.0f : m, inv = s == 0.0f ? 0.0f : 1.0f / s;
    const int end = min(a.n, (part + 1) * a.len);
    for (int i0 = part * a.len; i0 < end; i0 += kTile) {
#pragma unroll
        for (int k = 0; k < kPer; k += 4) {
            const int i = i0 + k * kThreads + 4 * threadIdx.x;
            float q[4];
            if (rate.hi > 0.0f) {
                load_row<VEC>(x, i, end, 0.0f, q);
#pragma unroll
                for (int e = 0; e < 4; ++e) q[e] = power(q[e] - ref, rate) * inv;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) q[e] = i + e == first ? 1.0f : 0.0f;
            }
            if (VEC && i + 4 <= end) {
                *(f32x4 *)(out + i) = f32x4{q[0], q[1], q[2], q[3]};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < end) out[i + e] = q[e];
            }
        }
    }
}

// Parts of a row: about 2048 blocks in all. 160 rows with 512, 1024, 2048 and 4096: 50.4, 48.2, 45.9 and
// 45.1 us in the two kernels (with exponents of one float), 40 rows 15.7, 15.8, 16.3 and 16.0; one row has
// 38 in any case.
void prob_cut(int64_t rows, int64_t n, int &len, int &parts) {
    const int64_t tiles = (n + kTile - 1) / kTile, per = std::max<int64_t>(1, tiles * rows / 2048);
    len = (int)(std::min(per, tiles) * kTile);
    parts = (int)((n + len - 1) / len);
}

// ---- drafts ---------------------------------------------------------------------

constexpr int kStretch = 64 * kPer;  // values of a row whose weights a wavefront sums

struct VerifyArgs {
    const int32_t *starts, *drafts, *lens;
    const float *target, *draft, *accept_u, *sample_u;
    int32_t *tokens, *accepted, *kept;
    int2 *decided;   // [seqs]: the row that a sequence's token is taken from, and the draft not to be taken
    double2 *sums;   // [seqs][stretches]: of w, and of the target's row
    int64_t target_stride, draft_stride;
    int seqs, rows, n, stretches;
};

template <int CTRL>
__device__ __forceinline__ double shifted(double v) {  // 0 where the row of 16 lanes has no such lane
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Sum over the lanes up to this one of a wavefront, and over all, in a fixed order.
__device__ __forceinline__ double wave_scan(double v, double &total) {
    v += shifted<0x111>(v);
    v += shifted<0x112>(v);
    v += shifted<0x114>(v);
    v += shifted<0x118>(v);
    const double a = lane_f64(v, 15), b = lane_f64(v, 31), c = lane_f64(v, 47);
    const int row = (threadIdx.x & 63) >> 4;
    v += row == 0 ? 0.0 : row == 1 ? a : row == 2 ? a + b : (a + b) + c;
    total = lane_f64(v, 63);
    return v;
}

__device__ __forceinline__ double weight(double v) { return v > 0.0 ? v : 0.0; }

// The rows that a sequence's token is taken from.
struct Row {
    const float *p, *q;  // q NULL: certain of x
    int x;               // the draft; -1: w is the target's row
};
__device__ __forceinline__ Row row_at(const VerifyArgs &a, int row, int x) {
    return Row{a.target + (int64_t)row * a.target_stride,
               x >= 0 && a.draft ? a.draft + (int64_t)row * a.draft_stride : nullptr, x};
}

// This lane's kPer neighbouring weights of a stretch: w, and the target's alone.
template <bool VEC>
__device__ __forceinline__ void stretch_weights(const VerifyArgs &a, const Row &r, int stretch, double (&w)[kPer],
                                                double (&t)[kPer]) {
    const int i = stretch * kStretch + kPer * (threadIdx.x & 63);
    float p[kPer], q[kPer];
    load_row<VEC>(r.p, i, a.n, 0.0f, p);
    if (r.q) load_row<VEC>(r.q, i, a.n, 0.0f, q);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        t[k] = weight(p[k]);
        w[k] = r.x < 0 ? t[k] : r.q ? weight((double)p[k] - (double)q[k]) : i + k == r.x ? 0.0 : t[k];
    }
}
__device__ __forceinline__ double lane_sum(const double (&w)[kPer]) {
    double s[kPer / 2];
#pragma unroll
    for (int k = 0; k < kPer / 2; ++k) s[k] = w[2 * k] + w[2 * k + 1];
#pragma unroll
    for (int n = kPer / 4; n > 0; n /= 2)
#pragma unroll
        for (int k = 0; k < n; ++k) s[k] = s[2 * k] + s[2 * k + 1];
    return s[0];
}

// A sequence's rows [first, last]; false for one that has none or whose starts are bad.
__device__ __forceinline__ bool rows_of(const VerifyArgs &a, int s, int &first, int &last) {
    first = a.starts[s];
    last = a.starts[s + 1] - 1;
    return first >= 0 && last >= first && last < a.rows;
}

// The first row of [first, last) whose draft is not accepted, last if there is none, and that
// draft (-1: none of the vocabulary); by each wavefront.
__device__ __forceinline__ int2 decide(const VerifyArgs &a, int first, int last) {
    const int lane = threadIdx.x & 63;
    for (int r0 = first; r0 < last; r0 += 64) {
        const int r = r0 + lane;
        bool fails = false;
        int x = -1;
        if (r < last) {
            x = a.drafts[r];
            const bool in = x >= 0 && x < a.n;
            const double p = in ? a.target[(int64_t)r * a.target_stride + x] : 0.0;
            const double q = !a.draft ? 1.0 : in ? a.draft[(int64_t)r * a.draft_stride + x] : 0.0;
            fails = !in || !((double)a.accept_u[r] * q < p);
            x = in ? x : -1;
        }
        const uint64_t b = __ballot(fails);
        if (b) {
            const int at = __builtin_ctzll(b);
            return int2{r0 + at, __builtin_amdgcn_readlane(x, at)};
        }
    }
    return int2{last, -1};
}

// Four stretches of a sequence's row to a block, whose wavefronts have nothing to say to each
// other. Bound by memory for many sequences, two rows of the vocabulary each: 64 of 151936, 78 MB, 14.6
// us (5.3 TB/s); one sequence 3.5 us.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void verify_sums_kernel(const VerifyArgs a) {
    const int blocks = (a.stretches + 3) / 4, s = blockIdx.x / blocks;
    const int stretch = uniform((int)(blockIdx.x - s * blocks) * 4 + (int)(threadIdx.x >> 6));
    int first, last;
    if (stretch >= a.stretches || !rows_of(a, s, first, last)) return;
    const int2 at = decide(a, first, last);
    double w[kPer], t[kPer], wt, tt;
    stretch_weights<VEC>(a, row_at(a, at.x, at.y), stretch, w, t);
    wave_scan(lane_sum(w), wt);
    wave_scan(lane_sum(t), tt);
    if ((threadIdx.x & 63) == 0) {
        a.sums[(int64_t)s * a.stretches + stretch] = double2{wt, tt};
        if (stretch == 0) a.decided[s] = at;
    }
}

// One wavefront a sequence: the stretch in which the sum passes the number, then the token in it.
// All latency: the stretches' sums 64 at a time, then one stretch's weights. 5.8 us for 64 sequences,
// 4.2 for one; a block of 256 threads, with its barriers, 12.0 and 10.6.
template <bool VEC>
__global__ __launch_bounds__(64) void verify_pick_kernel(const VerifyArgs a) {
    const int s = blockIdx.x, lane = threadIdx.x;
    int first, last;
    if (!rows_of(a, s, first, last)) {
        if (lane == 0) {
            a.accepted[s] = first >= 0 && last == first - 1 && first <= a.rows ? 0 : -1;
            if (a.kept) a.kept[s] = a.lens[s];
        }
        return;
    }
    const int2 at = a.decided[s];
    const float u = a.sample_u[s];
    const double2 *sums = a.sums + (int64_t)s * a.stretches;
    double ws = 0.0, ts = 0.0, wt, tt;
    for (int i = lane; i < a.stretches; i += 64) ws += sums[i].x, ts += sums[i].y;
    wave_scan(ws, wt);
    wave_scan(ts, tt);
    Row r = row_at(a, at.x, at.y);
    if (wt == 0.0) {  // no weight left: the target's row
        r = row_at(a, at.x, -1);
        wt = tt;
    }
    const double goal = (double)(u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f) * wt;
    // The first stretch with a weight behind which the sum is over goal, else the last with a weight.
    int stretch = -1;
    bool any = false;
    double before = 0.0, at_stretch = 0.0;
    for (int i0 = 0; i0 < a.stretches && !any; i0 += 64) {
        const int i = i0 + lane;
        const double v = i < a.stretches ? (r.x < 0 ? sums[i].y : sums[i].x) : 0.0;
        double total;
        const double c = before + wave_scan(v, total);
        const uint64_t over = __ballot(v > 0.0 && c > goal), some = __ballot(v > 0.0);
        any = over != 0;
        if (some) {
            const int n = any ? __builtin_ctzll(over) : last_lane(some);
            stretch = i0 + n;
            at_stretch = lane_f64(c, n) - lane_f64(v, n);
        }
        before += total;
    }
    int token = 0;
    if (stretch >= 0) {
        double w[kPer], t[kPer], total;
        stretch_weights<VEC>(a, r, stretch, w, t);
        const double mine = lane_sum(w);
        double c = at_stretch + (wave_scan(mine, total) - mine);
        int hit = -1, end = -1;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            c += w[k];
            if (w[k] > 0.0) {
                end = k;
                if (hit < 0 && c > goal) hit = k;
            }
        }
        const uint64_t hits = __ballot(any && hit >= 0), ends = __ballot(end >= 0);
        const int n = hits ? __builtin_ctzll(hits) : last_lane(ends);
        token = stretch * kStretch + kPer * n + max(__builtin_amdgcn_readlane(hits ? hit : end, n), 0);
    }
    for (int i = first + lane; i <= last; i += 64) {
        const int v = i < at.x ? a.drafts[i] : i == at.x ? token : -1;
        a.tokens[i] = v;
    }
    if (lane == 0) {
        a.accepted[s] = at.x - first;
        if (a.kept) a.kept[s] = a.lens[s] - (last - at.x);
    }
}

int verify_stretches(int64_t n) { return (int)((n + kStretch - 1) / kStretch); }
int64_t verify_blocks(int64_t seqs, int64_t n) { return seqs * ((verify_stretches(n) + 3) / 4); }

bool rows16(const void *p, int64_t stride) { return (uintptr_t)p % 16 == 0 && stride % 4 == 0; }

}  // namespace
}  // namespace gphq

using namespace gphq;

extern "C" {

int64_t gphq_probabilities_workspace_bytes(int64_t rows, int64_t vocab) {
    if (rows < 0 || rows > GPHQ_SAMPLE_MAX_ROWS || vocab < 0 || vocab > GPHQ_SAMPLE_MAX_VOCAB)
        return GPHQ_ERR_DIMENSIONS;
    if (rows == 0 || vocab == 0) return 0;
    int len, parts;
    prob_cut(rows, vocab, len, parts);
    return (rows * parts * (int64_t)sizeof(float2) + 15) / 16 * 16;
}

int gphq_probabilities(const float *x, int64_t x_stride, const float *temperatures, float *out, int64_t out_stride,
                       int64_t rows, int64_t vocab, void *work, int64_t work_bytes, void *stream) {
    const int64_t need = gphq_probabilities_workspace_bytes(rows, vocab);
    if (need < 0) return (int)need;
    if (x_stride < vocab || out_stride < vocab || x_stride > INT64_MAX / 8 / GPHQ_SAMPLE_MAX_ROWS ||
        out_stride > INT64_MAX / 8 / GPHQ_SAMPLE_MAX_ROWS)
        return GPHQ_ERR_DIMENSIONS;
    if (need == 0) return GPHQ_OK;
    if (!x || !out || ((uintptr_t)x | (uintptr_t)out | (uintptr_t)temperatures) % 4) return GPHQ_ERR_DIMENSIONS;
    if (!work || (uintptr_t)work % 16 || work_bytes < need) return GPHQ_ERR_DIMENSIONS;
    if (!(x == out && x_stride == out_stride) &&
        spans_overlap(x, span_bytes(rows, x_stride, vocab, 4), out, span_bytes(rows, out_stride, vocab, 4)))
        return GPHQ_ERR_OVERLAP;
    ProbArgs a{x, temperatures, out, (float2 *)work, x_stride, out_stride, (int)rows, (int)vocab, 0, 0};
    prob_cut(rows, vocab, a.len, a.parts);
    const dim3 grid((unsigned)(rows * a.parts));
    hipStream_t st = (hipStream_t)stream;
    const bool vec = rows16(x, x_stride) && rows16(out, out_stride);
    if (vec)
        hipLaunchKernelGGL(prob_parts_kernel<true>, grid, dim3(kThreads), 0, st, a);
    else
        hipLaunchKernelGGL(prob_parts_kernel<false>, grid, dim3(kThreads), 0, st, a);
    GPHQ_TRY(launch_status());
    if (vec)
        hipLaunchKernelGGL(prob_write_kernel<true>, grid, dim3(kThreads), 0, st, a);
    else
        hipLaunchKernelGGL(prob_write_kernel<false>, grid, dim3(kThreads), 0, st, a);
    return launch_status();
}

int64_t gphq_verify_drafts_workspace_bytes(int64_t seqs, int64_t vocab) {
    if (seqs < 0 || seqs > GPHQ_PAGED_MAX_SEQS || vocab < 1 || vocab > GPHQ_SAMPLE_MAX_VOCAB ||
        verify_blocks(seqs, vocab) > (1 << 23) - 1)
        return GPHQ_ERR_DIMENSIONS;
    return seqs * verify_stretches(vocab) * (int64_t)sizeof(double2) + (seqs * (int64_t)sizeof(int2) + 15) / 16 * 16;
}

int gphq_verify_drafts(const int32_t *starts, const int32_t *drafts, const float *target, int64_t target_stride,
                       const float *draft, int64_t draft_stride, const float *accept_u, const float *sample_u,
                       int64_t seqs, int64_t rows, int64_t vocab, int32_t *tokens, int32_t *accepted,
                       const int32_t *lens, int32_t *kept, void *work, int64_t work_bytes, void *stream) {
    const int64_t need = gphq_verify_drafts_workspace_bytes(seqs, vocab);
    if (need < 0) return (int)need;
    if (rows < 0 || rows > GPHQ_SAMPLE_MAX_ROWS || target_stride < vocab || (draft && draft_stride < vocab) ||
        target_stride > INT64_MAX / 8 / GPHQ_SAMPLE_MAX_ROWS || draft_stride > INT64_MAX / 8 / GPHQ_SAMPLE_MAX_ROWS)
        return GPHQ_ERR_DIMENSIONS;
    if (seqs == 0) return GPHQ_OK;
    if (!starts || !accepted || !sample_u || (kept && !lens)) return GPHQ_ERR_DIMENSIONS;
    if (rows && (!drafts || !target || !accept_u || !tokens)) return GPHQ_ERR_DIMENSIONS;
    const uintptr_t bits = (uintptr_t)starts | (uintptr_t)drafts | (uintptr_t)target | (uintptr_t)draft |
                           (uintptr_t)accept_u | (uintptr_t)sample_u | (uintptr_t)tokens | (uintptr_t)accepted |
                           (uintptr_t)lens | (uintptr_t)kept;
    if (bits % 4 || !work || (uintptr_t)work % 16 || work_bytes < need) return GPHQ_ERR_DIMENSIONS;
    const int stretches = verify_stretches(vocab);
    double2 *sums = (double2 *)work;
    VerifyArgs a{starts, drafts, lens, target, draft, accept_u, sample_u, tokens, accepted, kept,
                 (int2 *)(sums + seqs * stretches), sums, target_stride, draft_stride, (int)seqs, (int)rows, (int)vocab,
                 stretches};
    const dim3 grid((unsigned)verify_blocks(seqs, vocab));
    hipStream_t st = (hipStream_t)stream;
    const bool vec = rows16(target, target_stride) && (!draft || rows16(draft, draft_stride));
    if (vec)
        hipLaunchKernelGGL(verify_sums_kernel<true>, grid, dim3(kThreads), 0, st, a);
    else
        hipLaunchKernelGGL(verify_sums_kernel<false>, grid, dim3(kThreads), 0, st, a);
    GPHQ_TRY(launch_status());
    if (vec)
        hipLaunchKernelGGL(verify_pick_kernel<true>, dim3((unsigned)seqs), dim3(64), 0, st, a);
    else
        hipLaunchKernelGGL(verify_pick_kernel<false>, dim3((unsigned)seqs), dim3(64), 0, st, a);
    return launch_status();
}

}  // extern "C"
