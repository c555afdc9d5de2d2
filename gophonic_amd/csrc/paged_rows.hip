// Paged attention of few query rows: the row kernel of gphq_paged_attention
// (single tokens, and sequences of a few rows). See paged_attention.h for the
// mathematics and the tiling.
#include "paged_rows.h"

namespace gphq {
namespace {

// One 32-key step's exponentials: s[0], s[1] are the scores (fac times them in log2) of keys
// kt + 4 g4 + r and kt + 16 + 4 g4 + r; those that the lane's column does not see are left
// out. p[8] are 2^(x - m + lift), m and l the running reference and this lane's running sum;
// returns what o is to be multiplied by, and whether any lane's reference moved.
template <typename CT>
__device__ __forceinline__ float softmax_step(const RowTile &t, const f32x4 (&s)[2], float fac, bool masked, int kt,
                                              unsigned ok, float (&p)[8], float &m, float &l, bool &moved) {
    const int g4 = (threadIdx.x & 63) >> 4;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = s[i >> 2][i & 3];
    float mx = kLeast;
    if (masked) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int key = kt + 16 * (i >> 2) + 4 * g4 + (i & 3);
            const bool sees = key <= t.pos && key >= t.first && (ok >> (i >> 2) & 1);
            if (!sees) x[i] = -INFINITY;
            any |= sees;
        }
        mx = any ? kLeast : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, x[i]);
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    mx = mx == -INFINITY ? mx : fmaxf(mx * fac, kLeast);
    const bool grew = mx > m + kLag;
    const float mn = grew ? mx : m;
    const float ref = mn == -INFINITY ? 0.0f : mn - kLift<CT>;
    const float corr = __builtin_amdgcn_exp2f((m == -INFINITY ? m : m - kLift<CT>) - ref);
    m = mn;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(x[i], fac, -ref));
        sum += p[i];
    }
    l = l * corr + sum;
    moved = __any(grew);
    return corr;
}

// Adds what was taken out of a step's values: odd has a bit for each of the lane's eight keys.
template <typename CT, int HD>
__device__ __forceinline__ void add_not_finite(const RowTile &t, const char *v, const int64_t (&at)[2], int ts,
                                               int kt, unsigned odd, f32x4 (&o)[HD / 16]) {
    constexpr int VD = HD / 16;
    const int g4 = (threadIdx.x & 63) >> 4;
#pragma unroll 1
    for (int n = 0; n < 32; ++n) {  // key kt + n is key 4 (n / 16) + n % 4 of the lanes of group n / 4 % 4
        if (!(__ballot(odd >> (4 * (n >> 4) + (n & 3)) & 1) >> (16 * (n >> 2 & 3)) & 0xFFFF)) continue;
        const CT *row = (const CT *)(v + (n < 16 ? at[0] : at[1]) + (n & 15) * ts) + VD * 4 * g4;
        const bool sees = kt + n <= t.pos && kt + n >= t.first;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < VD; d += 4) {
                float x[4];
                load_vec(row + VD * r + d, x);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[d + e][r] += sees ? not_finite(x[e]) : 0.0f;
                asm volatile("" ::: "memory");  // few values at a time: this must not cost registers
            }
    }
}

// 16-bit pages. Four wavefronts take the tile's 32-key steps in turn, each on its own:
// everything goes from memory to registers, nothing through LDS. On
// v_mfma_f32_16x16x32:
//   S^T (16 keys x 16 columns) = K . Q^T, K's fragment as it lies in the page;
//   O^T (16 dims x 16 columns) += V^T . P^T: the score registers are P^T's fragment as they
//     stand (keys 4 g4 + 0..3 of both 16-key tiles); a lane loads those eight keys of V at
//     HD/16 neighbouring dims, and 16-bit halves exchanged between the eight registers make
//     the fragments of V^T for HD/16 tiles of dims HD/16 apart.
// Bound by memory: a 32-key step takes 512 cycles of the matrix cores a piece (HD = 128) and
// brings 16 KB, at any rate of the memory less than half of a SIMD's time. K of the next step
// is loaded as soon as this one's scores are made, V as soon as it is multiplied, so a block's
// four wavefronts keep 64 KB on their way; 16 columns, not more, because one row of a group of
// up to 16 heads needs no more and every column costs registers. Probabilities of 16-bit rows
// take two pieces, 2^-16 (bfloat16) or 2^-22 of one lost: the matrix cores have the time (59.7 us
// either way in the case that follows). Two rows over 36286 and 39946
// tokens, eight KV heads, bfloat16: 59.5 us with the join (312 MB, 5.25 TB/s; a kernel that
// only reads makes 6.2).
template <typename RT, typename CT, int HD, bool BY_ROW>
__global__ __launch_bounds__(256, 2) void attn_rows16_kernel(const AttnArgs a, int tiles, int splits) {
    typedef Half<CT> H;
    typedef typename H::vec8 vec8;
    constexpr int NP = kPieces<RT, CT>, KC = HD / 32, VD = HD / 16, VW = VD / 2;  // VW: dwords of V per key
    constexpr int PP = NP == 1 ? 2 : NP;  // pieces of a probability
    RowTile t;
    if (!row_tile<BY_ROW>(a, tiles, splits, t)) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g4 = lane >> 4;
    const char *kp = (const char *)a.pool.k, *vp = (const char *)a.pool.v;
    const int ts = (int)(a.pool.token_stride * sizeof(CT));
    const unsigned ko = c * ts + 16 * g4, vo = 4 * g4 * ts + 2 * VD * c;  // this lane's bytes within 16 keys

    float fac = score_factor(a.scale_log2);
    vec8 qf[NP][KC];
    {
        const RT *q = (const RT *)a.q + (int64_t)(t.start + t.row) * a.q_stride + t.head * HD + 8 * g4;
        float x[KC][8], inverse = 1.0f, up = 1.0f;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            float lo[4], hi[4];
            load_vec(q + 32 * i, lo);
            load_vec(q + 32 * i + 4, hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = lo[e], x[i][4 + e] = hi[e];
        }
        if (NP == 2) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < KC; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[i][e]));
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            up = f16_scale(m, inverse);
            fac = score_factor(fac * inverse);
        }
        up *= a.q_sign;
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                CT pc[NP];
                split_pieces(x[i][e] * up, pc);
#pragma unroll
                for (int k = 0; k < NP; ++k) qf[k][i][e] = pc[k];
            }
    }
    f32x4 o[VD];
#pragma unroll
    for (int i = 0; i < VD; ++i) o[i] = f32x4{};
    float m = -INFINITY, l = 0.0f;
    typedef int vrow __attribute__((ext_vector_type(VW)));
    vec8 kf[2][KC];
    vrow v[8];
    int64_t at[2];
    PageWalk w;
    auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            kf[0][i] = *(const vec8 *)(kp + at[0] + (ko + 64 * i));
            kf[1][i] = *(const vec8 *)(kp + at[1] + (ko + 64 * i));
        }
    };
    auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *(const vrow *)(vp + at[i >> 2] + (i & 3) * ts + vo);
    };
    // One step, of keys kt .. kt + 31, whose K and V are in registers; more: the step after it
    // is loaded into them as they become free.
    auto step = [&](int kt, unsigned &ok, auto more) __attribute__((always_inline)) {
        f32x4 s[2] = {f32x4{}, f32x4{}};
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                s[0] = H::mfma16(kf[0][i], qf[k][i], s[0]);
                s[1] = H::mfma16(kf[1][i], qf[k][i], s[1]);
            }
        const unsigned okc = ok;
        const int64_t now[2] = {at[0], at[1]};
        if (more) {
            ok = pages_step<CT>(a, w, t.seq, t.g, kt + 128, at);
            load_k();
        }
        // Whether some column does not see some key of the step.
        const bool masked = kt + 31 > t.p0 || kt < t.lo || (a.window > 0 && kt < t.p1 - a.window + 1) || okc != 3;
        float p[8];
        bool moved;
        const float corr = softmax_step<CT>(t, s, fac, masked, kt, okc, p, m, l, moved);
        unsigned odd = 0;  // of this lane's eight keys, those with a value that is not finite
        if (masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = kt + 16 * (i >> 2) + 4 * g4 + (i & 3);
                if (key >= t.hi || key < t.lo || !(okc >> (i >> 2) & 1)) v[i] = vrow{};  // no row of the tile sees it
                int any = 0;
#pragma unroll
                for (int u = 0; u < VW; ++u) {
                    const int out = pair_not_finite<CT>(v[i][u]);
                    v[i][u] &= ~out;
                    any |= out;
                }
                odd |= any ? 1u << i : 0u;
            }
        }
        vec8 pf[PP];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            CT pc[PP];
            split_pieces(p[i], pc);
#pragma unroll
            for (int k = 0; k < PP; ++k) pf[k][i] = pc[k];
        }
        if (moved) {
#pragma unroll
            for (int i = 0; i < VD; ++i) o[i] *= corr;
        }
#pragma unroll
        for (int d = 0; d < VD; ++d) {
            i32x4 f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                f[j] = __builtin_amdgcn_perm(v[2 * j + 1][d / 2], v[2 * j][d / 2], d % 2 ? 0x07060302 : 0x05040100);
#pragma unroll
            for (int k = 0; k < PP; ++k) o[d] = H::mfma16(__builtin_bit_cast(vec8, f), pf[k], o[d]);
        }
        if (more) load_v();
        if (__any(odd)) add_not_finite<CT, HD>(t, vp, now, ts, kt, odd, o);
    };
    int kt = t.k0 + 32 * wave;
    if (kt < t.k1) {
        pages_start<CT>(a, w, t.seq, t.g, t.lo, t.hi, kt);
        unsigned ok = pages_step<CT>(a, w, t.seq, t.g, kt, at);
        load_k();
        load_v();
        for (; kt + 128 < t.k1; kt += 128) step(kt, ok, std::true_type{});
        step(kt, ok, std::false_type{});
    }
    rows_finish<RT, HD>(a, t, m, l, o);
}

// fp32 pages, the same walk on v_mfma_f32_16x16x4_f32: its operands are one fp32 value a
// lane, so V needs no exchange between registers, and a lane's 16-byte pieces of K and Q
// hold the same dims (16 i + 4 g4 ..), in whatever order they are multiplied.
// 16 rows of 2000 to 4095 tokens, eight KV heads: 72 us with the join (364 MB, 5.1 TB/s). A
// 32-key step's 128 instructions take 4096 cycles for 32 KB, so the memory stays the bound;
// one block a CU with all the registers it asks for measured faster than two with 256 a lane
// (kernel alone 72.7 and 78.7 us).
template <int HD, bool BY_ROW>
__global__ __launch_bounds__(256) void attn_rows32_kernel(const AttnArgs a, int tiles, int splits) {
    constexpr int KC = HD / 16, VD = HD / 16;
    RowTile t;
    if (!row_tile<BY_ROW>(a, tiles, splits, t)) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g4 = lane >> 4;
    const char *kp = (const char *)a.pool.k, *vp = (const char *)a.pool.v;
    const int ts = (int)(a.pool.token_stride * sizeof(float));
    const unsigned ko = c * ts + 16 * g4, vo = 4 * g4 * ts + 4 * VD * c;  // this lane's bytes within 16 keys
    f32x4 qf[KC];
    {
        const float *q = (const float *)a.q + (int64_t)(t.start + t.row) * a.q_stride + t.head * HD + 4 * g4;
#pragma unroll
        for (int i = 0; i < KC; ++i) qf[i] = *(const f32x4 *)(q + 16 * i) * a.q_sign;
    }
    f32x4 o[VD];
#pragma unroll
    for (int i = 0; i < VD; ++i) o[i] = f32x4{};
    float m = -INFINITY, l = 0.0f;
    f32x4 kf[2][KC], v[8][VD / 4];
    int64_t at[2];
    PageWalk w;
    auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < KC; ++i) kf[h][i] = *(const f32x4 *)(kp + at[h] + (ko + 64 * i));
    };
    auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int u = 0; u < VD / 4; ++u)
                v[i][u] = *(const f32x4 *)(vp + at[i >> 2] + (i & 3) * ts + (vo + 16 * u));
    };
    auto step = [&](int kt, unsigned &ok, auto more) __attribute__((always_inline)) {
        f32x4 s[2] = {f32x4{}, f32x4{}};
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[0][i][e], qf[i][e], s[0], 0, 0, 0);
                s[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[1][i][e], qf[i][e], s[1], 0, 0, 0);
            }
        const unsigned okc = ok;
        const int64_t now[2] = {at[0], at[1]};
        if (more) {
            ok = pages_step<float>(a, w, t.seq, t.g, kt + 128, at);
            load_k();
        }
        const bool masked = kt + 31 > t.p0 || kt < t.lo || (a.window > 0 && kt < t.p1 - a.window + 1) || okc != 3;
        float p[8];
        bool moved;
        const float corr = softmax_step<float>(t, s, score_factor(a.scale_log2), masked, kt, okc, p, m, l, moved);
        unsigned odd = 0;  // of this lane's eight keys, those with a value that is not finite
        if (masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = kt + 16 * (i >> 2) + 4 * g4 + (i & 3);
                const bool none = key >= t.hi || key < t.lo || !(okc >> (i >> 2) & 1);  // no row of the tile sees it
#pragma unroll
                for (int u = 0; u < VD / 4; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool out = !(fabsf(v[i][u][e]) < INFINITY);
                        if (out || none) v[i][u][e] = 0.0f;
                        odd |= out && !none ? 1u << i : 0u;
                    }
            }
        }
        if (moved) {
#pragma unroll
            for (int i = 0; i < VD; ++i) o[i] *= corr;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int d = 0; d < VD; ++d)
                o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][d / 4][d % 4], p[i], o[d], 0, 0, 0);
        if (more) load_v();
        if (__any(odd)) add_not_finite<float, HD>(t, vp, now, ts, kt, odd, o);
    };
    int kt = t.k0 + 32 * wave;
    if (kt < t.k1) {
        pages_start<float>(a, w, t.seq, t.g, t.lo, t.hi, kt);
        unsigned ok = pages_step<float>(a, w, t.seq, t.g, kt, at);
        load_k();
        load_v();
        for (; kt + 128 < t.k1; kt += 128) step(kt, ok, std::true_type{});
        step(kt, ok, std::false_type{});
    }
    rows_finish<float, HD>(a, t, m, l, o);
}

}  // namespace

template <typename RT, typename CT>
int attn_rows_launch(const AttnArgs &a, int hd, int splits, int tiles, hipStream_t st) {
    const unsigned units = a.row_tiles ? (unsigned)(a.b.rows * a.row_tiles) : (unsigned)(a.b.seqs * tiles);
    const unsigned blocks = units * (unsigned)splits * (unsigned)a.pool.kv_heads;
    auto launch = [&](auto dim, auto by_row) {
        constexpr int HD = decltype(dim)::value;
        constexpr bool BY_ROW = decltype(by_row)::value;
        if constexpr (std::is_same<CT, float>::value)
            hipLaunchKernelGGL((attn_rows32_kernel<HD, BY_ROW>), dim3(blocks), dim3(256), 0, st, a, tiles, splits);
        else
            hipLaunchKernelGGL((attn_rows16_kernel<RT, CT, HD, BY_ROW>), dim3(blocks), dim3(256), 0, st, a, tiles, splits);
    };
    auto pick = [&](auto by_row) {
        hd == 128 ? launch(std::integral_constant<int, 128>{}, by_row) : launch(std::integral_constant<int, 64>{}, by_row);
    };
    a.row_tiles ? pick(std::true_type{}) : pick(std::false_type{});
    return launch_status();
}

template int attn_rows_launch<float, float>(const AttnArgs &, int, int, int, hipStream_t);
template int attn_rows_launch<float, f16>(const AttnArgs &, int, int, int, hipStream_t);
template int attn_rows_launch<float, bf16>(const AttnArgs &, int, int, int, hipStream_t);
template int attn_rows_launch<f16, f16>(const AttnArgs &, int, int, int, hipStream_t);
template int attn_rows_launch<bf16, bf16>(const AttnArgs &, int, int, int, hipStream_t);

}  // namespace gphq
