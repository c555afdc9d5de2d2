// Paged attention over 8-bit pages, few query rows: the row kernel of gphq_paged8_attention
// (single tokens, and sequences of a few rows). See paged_attention.h for the mathematics and
// the tiling, paged8.h for the codes.
#include "paged8.h"
#include "paged_rows.h"

namespace gphq {
namespace {

// Four wavefronts take the tile's 64-key steps in turn, each on its own: everything goes from
// memory to registers, nothing through LDS. On v_mfma_f32_16x16x32_f16, per block of 16 keys:
//   S^T (16 keys x 16 columns) = K . Q^T; a lane loads 16 neighbouring codes of a key at once,
//     so its two fragments hold other dims than the instruction's order has, and Q's hold the same;
//   O^T (16 dims x 16 columns) += V^T . P^T over two blocks: the score registers are P^T's
//     fragment as they stand; a lane loads its keys of V at HD/16 neighbouring dims, and bytes
//     taken from two keys' dwords make the fragments of V^T for HD/16 tiles of dims HD/16 apart.
template <typename RT, typename C, int HD, bool BY_ROW>
__global__ __launch_bounds__(256, 2) void attn8_rows_kernel(const Attn8Args e, int tiles, int splits) {
    typedef Half<f16> H;
    constexpr int NB = 4, STEP = 16 * NB, KQ = HD / 64, VD = HD / 16, VW = VD / 4;
    constexpr int NP = kPieces<RT, f16>, PP = 2;  // pieces of a query value, of a probability
    const AttnArgs &a = e.a;
    RowTile t;
    if (!row_tile<BY_ROW>(a, tiles, splits, t)) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g4 = lane >> 4;
    const char *kp = (const char *)a.pool.k, *vp = (const char *)a.pool.v;
    const int ts = (int)a.pool.token_stride;
    const unsigned ko = c * ts + 16 * g4, vo = 4 * g4 * ts + VD * c;  // this lane's bytes within 16 keys

    float fac = a.scale_log2;
    f16x8 qf[NP][2 * KQ];
    {
        const RT *q = (const RT *)a.q + (int64_t)(t.start + t.row) * a.q_stride + t.head * HD + 16 * g4;
        float x[2 * KQ][8], inverse = 1.0f, up = 1.0f;
#pragma unroll
        for (int i = 0; i < 2 * KQ; ++i) {
            float lo[4], hi[4];
            load_vec(q + 64 * (i >> 1) + 8 * (i & 1), lo);
            load_vec(q + 64 * (i >> 1) + 8 * (i & 1) + 4, hi);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i][k] = lo[k], x[i][4 + k] = hi[k];
        }
        if (!std::is_same<RT, f16>::value) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * KQ; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(x[i][k]));
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            up = f16_scale(m, inverse);
        }
        fac = score_factor(fac * inverse * (float)(1 << C::kExp));
        up *= a.q_sign;
#pragma unroll
        for (int i = 0; i < 2 * KQ; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                f16 pc[NP];
                query_pieces(x[i][k] * up, pc);
#pragma unroll
                for (int n = 0; n < NP; ++n) qf[n][i][k] = pc[n];
            }
    }
    f32x4 o[VD];
#pragma unroll
    for (int i = 0; i < VD; ++i) o[i] = f32x4{};
    float m = -INFINITY, l = 0.0f;
    int ve = kNoExp;
    typedef int vrow __attribute__((ext_vector_type(VW)));
    i32x4 kc[NB][KQ];
    vrow vc[4 * NB];
    float ks[NB], vs[NB];
    Page8Walk w;
    // Loads a step's codes and scales; its blocks' bits.
    auto load = [&](int kt) __attribute__((always_inline)) -> unsigned {
        int64_t at[NB], sat[NB];
        const unsigned ok = pages8_step(e, w, t.seq, t.g, kt, at, sat);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int i = 0; i < KQ; ++i) kc[b][i] = *(const i32x4 *)(kp + at[b] + (ko + 64 * i));
            ks[b] = uniform_scale(e.s.k, sat[b]);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int r = 0; r < 4; ++r) vc[4 * b + r] = *(const vrow *)(vp + at[b] + r * ts + vo);
            vs[b] = uniform_scale(e.s.v, sat[b]);
        }
        return ok;
    };
    int kt = t.k0 + STEP * wave;
    if (kt < t.k1) pages8_start(a, w, t.seq, t.lo, t.hi, kt);
    for (; kt < t.k1; kt += 4 * STEP) {
        const unsigned ok = load(kt);
        float x[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f32x4 s[NP] = {};
#pragma unroll
            for (int i = 0; i < KQ; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const f16x8 kf = codes8<C>(C::ready(kc[b][i][2 * j]), C::ready(kc[b][i][2 * j + 1]));
#pragma unroll
                    for (int n = 0; n < NP; ++n) s[n] = H::mfma16(kf, qf[n][2 * i + j], s[n]);
                }
            const float f = fac * ks[b];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[b][r] = (NP == 1 ? s[0][r] : s[0][r] + s[NP - 1][r]) * f;
        }
        // Whether some column does not see some key of the step.
        const bool masked =
            kt + STEP - 1 > t.p0 || kt < t.lo || (a.window > 0 && kt < t.p1 - a.window + 1) || ok != (1u << NB) - 1;
        float mx = kLeast;
        int vn = ve;
        unsigned some = (1u << NB) - 1;  // the blocks of which the column sees any key
        if (masked) {
            some = 0;
            bool any = false;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = kt + 16 * b + 4 * g4 + r;
                    if (!(key <= t.pos && key >= t.first && (ok >> b & 1))) x[b][r] = -INFINITY;
                }
                const bool sees = kt + 16 * b <= t.pos && kt + 16 * b + 15 >= t.first && (ok >> b & 1);
                some |= sees ? 1u << b : 0u;
                any |= sees;
            }
            mx = any ? kLeast : -INFINITY;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int v = scale_exp(vs[b]);
            vn = some >> b & 1 ? max(vn, v) : vn;
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[b][r]);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const bool grew = mx > m + kLag || vn != ve;
        const float mn = mx > m + kLag ? mx : m;
        const float ref = mn == -INFINITY ? 0.0f : mn - kLift<f16>;
        float corr = __builtin_amdgcn_exp2f((m == -INFINITY ? m : m - kLift<f16>) - ref);
        m = mn;
        float sum = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                x[b][r] = __builtin_amdgcn_exp2f(x[b][r] - ref);
                sum += x[b][r];
            }
        l = l * corr + sum;
        if (__any(grew)) {
            corr = __builtin_amdgcn_ldexpf(corr, ve - vn);
#pragma unroll
            for (int i = 0; i < VD; ++i) o[i] *= corr;
            ve = vn;
        }
#pragma unroll
        for (int b = 0; b < NB; b += 2) {
            f16x8 pf[PP];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float scale = some >> (b + h) & 1 ? __builtin_amdgcn_ldexpf(vs[b + h], -ve) : 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    f16 pc[PP];
                    weight_pieces(x[b + h][r], scale, pc);
#pragma unroll
                    for (int n = 0; n < PP; ++n) pf[n][4 * h + r] = pc[n];
                }
            }
#pragma unroll
            for (int u = 0; u < VW; ++u) {
                int v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = C::ready(vc[4 * b + i][u]);
                auto dim = [&](auto byte) __attribute__((always_inline)) {
                    constexpr int B = decltype(byte)::value;
                    const i32x4 f = {C::template across<B>(v[1], v[0]), C::template across<B>(v[3], v[2]),
                                     C::template across<B>(v[5], v[4]), C::template across<B>(v[7], v[6])};
#pragma unroll
                    for (int n = 0; n < PP; ++n)
                        o[4 * u + B] = H::mfma16(__builtin_bit_cast(f16x8, f), pf[n], o[4 * u + B]);
                };
                dim(std::integral_constant<int, 0>{});
                dim(std::integral_constant<int, 1>{});
                dim(std::integral_constant<int, 2>{});
                dim(std::integral_constant<int, 3>{});
            }
        }
    }
    const int down = ve - kDrop + C::kExp;
#pragma unroll
    for (int i = 0; i < VD; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[i][r] = __builtin_amdgcn_ldexpf(o[i][r], down);
    rows_finish<RT, HD>(a, t, m, __builtin_amdgcn_ldexpf(l, -kDrop), o);
}

}  // namespace

template <typename RT, typename C>
int attn8_rows_launch(const Attn8Args &e, int hd, int splits, int tiles, hipStream_t st) {
    const AttnArgs &a = e.a;
    const unsigned units = a.row_tiles ? (unsigned)(a.b.rows * a.row_tiles) : (unsigned)(a.b.seqs * tiles);
    const unsigned blocks = units * (unsigned)splits * (unsigned)a.pool.kv_heads;
    auto launch = [&](auto dim, auto by_row) {
        constexpr int HD = decltype(dim)::value;
        constexpr bool BY_ROW = decltype(by_row)::value;
        hipLaunchKernelGGL((attn8_rows_kernel<RT, C, HD, BY_ROW>), dim3(blocks), dim3(256), 0, st, e, tiles, splits);
    };
    auto pick = [&](auto by_row) {
        hd == 128 ? launch(std::integral_constant<int, 128>{}, by_row) : launch(std::integral_constant<int, 64>{}, by_row);
    };
    a.row_tiles ? pick(std::true_type{}) : pick(std::false_type{});
    return launch_status();
}

#define GPHQ_ROWS8(RT)                                                                          \
    template int attn8_rows_launch<RT, CodesI8>(const Attn8Args &, int, int, int, hipStream_t); \
    template int attn8_rows_launch<RT, CodesE4M3>(const Attn8Args &, int, int, int, hipStream_t)
GPHQ_ROWS8(float);
GPHQ_ROWS8(f16);
GPHQ_ROWS8(bf16);
#undef GPHQ_ROWS8

}  // namespace gphq
