// Paged attention over 8-bit pages, few query rows: the row kernel of gphq_paged8_attention
// (single tokens, and sequences of a few rows). See paged_attention.h for the mathematics and
// the tiling, paged8.h for the codes.
#include "paged8.h"
#include "paged_rows.h"

namespace gphq {
namespace {

constexpr int row8_waves(int sets) { return sets == 1 ? 4 : 8; }

// Four wavefronts, or eight with two sets, take the tile's 32-key steps in turn, each on its own: everything goes from
// memory to registers, nothing through LDS. NC sets of 16 columns share what is loaded and made
// FP16 of a step. On v_mfma_f32_16x16x32_f16, per block of 16 keys:
//   S^T (16 keys x 16 columns) = K . Q^T; a lane loads 16 neighbouring codes of a key at once,
//     so its two fragments hold other dims than the instruction's order has, and Q's hold the same;
//   O^T (16 dims x 16 columns) += V^T . P^T over two blocks: the score registers are P^T's
//     fragment as they stand; a lane loads its keys of V at HD/16 neighbouring dims, and bytes
//     taken from two keys' dwords make the fragments of V^T for HD/16 tiles of dims HD/16 apart.
// K of the next step is loaded as soon as this one's scores are made, V as soon as it is
// multiplied; a step's scales come with them, a lane each, so that no wait of the loop is for
// anything but loads in their order.
//
// Bound by memory where a tile has one set of columns: two single rows over 36286 and 39946 tokens,
// eight KV heads, bfloat16 rows: 27.2 us (141 MB, 5.2 TB/s). With two sets by what is done to the
// codes between memory and the matrix instructions, about 200 vector instructions a step for
// the codes and 220 a set for its softmax: five rows each over the same caches 35.6 us. Loading a
// step further ahead gained nothing (28.7 and 37.8 us); two sets as wavefronts of their own, each
// loading and converting: 44.9 us. What four and eight wavefronts cost is
// said at the host's rule for their splits.
template <typename RT, typename C, int HD, int NC, bool BY_ROW>
__global__ __launch_bounds__(row8_waves(NC) * 64) void attn8_rows_kernel(const Attn8Args e, int tiles, int splits) {
    typedef Half<f16> H;
    constexpr int NB = 2, NW = row8_waves(NC), STEP = 16 * NB, ROUND = NW * STEP, KQ = HD / 64, VD = HD / 16, VW = VD / 4;
    constexpr int NP = kPieces<RT, f16>, PP = 2;  // pieces of a query value, of a probability
    const AttnArgs &a = e.a;
    RowTile t;
    if (!row_tile<BY_ROW, 16 * NC, 64 * NW>(a, tiles, splits, t)) return;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g4 = lane >> 4;
    const char *kp = (const char *)a.pool.k, *vp = (const char *)a.pool.v;
    const int ts = (int)a.pool.token_stride;
    const unsigned ko = c * ts + 16 * g4, vo = 4 * g4 * ts + VD * c;  // this lane's bytes within 16 keys

    float fac[NC], m[NC], l[NC];
    int pos[NC], first[NC], ve[NC];
    f16x8 qf[NC][NP][2 * KQ];
    f32x4 o[NC][VD];
#pragma unroll
    for (int u = 0; u < NC; ++u) {
        row_column(a, t, t.c0 + 16 * u + c);
        pos[u] = t.pos;
        first[u] = t.first;
        m[u] = -INFINITY;
        l[u] = 0.0f;
        ve[u] = kNoExp;
#pragma unroll
        for (int i = 0; i < VD; ++i) o[u][i] = f32x4{};
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
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * KQ; ++i)
#pragma unroll
                for (int k = 0; k < 8; ++k) big = fmaxf(big, fabsf(x[i][k]));
            up = f16_scale(column_max(big), inverse);
        }
        fac[u] = score_factor(a.scale_log2 * inverse * (float)(1 << C::kExp));
        up *= a.q_sign;
#pragma unroll
        for (int i = 0; i < 2 * KQ; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                f16 pc[NP];
                query_pieces(x[i][k] * up, pc);
#pragma unroll
                for (int n = 0; n < NP; ++n) qf[u][n][i][k] = pc[n];
            }
    }
    typedef int vrow __attribute__((ext_vector_type(VW)));
    i32x4 kc[NB][KQ];
    vrow vc[4 * NB];
    float ks, vs;  // lane l: of block l % NB
    int64_t at[NB], sat;
    unsigned ok;
    Page8Walk w;
    auto load_k = [&](int kt) __attribute__((always_inline)) {
        int64_t s[NB];
        ok = pages8_step(e, w, t.seq, t.g, kt, at, s);
        sat = lane_scale(s);
        ks = e.s.k[sat];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const __amdgpu_buffer_rsrc_t from = buffer_at(kp + at[b]);
#pragma unroll
            for (int i = 0; i < KQ; ++i)
                kc[b][i] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(from, ko, 64 * i, 0));
        }
    };
    auto load_v = [&]() __attribute__((always_inline)) {
        vs = e.s.v[sat];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const __amdgpu_buffer_rsrc_t from = buffer_at(vp + at[b]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (VW == 2)
                    vc[4 * b + r] = __builtin_bit_cast(vrow, __builtin_amdgcn_raw_buffer_load_b64(from, vo, r * ts, 0));
                else
                    vc[4 * b + r] = __builtin_bit_cast(vrow, __builtin_amdgcn_raw_buffer_load_b32(from, vo, r * ts, 0));
            }
        }
    };
    // One step, of keys kt .. kt + 31, whose codes are in registers; more: the step after it is
    // loaded into them as they become free.
    auto step = [&](int kt, auto more) __attribute__((always_inline)) {
        float x[NC][NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f32x4 s[NC][NP] = {};
#pragma unroll
            for (int i = 0; i < KQ; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const f16x8 kf = codes8<C>(C::ready(kc[b][i][2 * j]), C::ready(kc[b][i][2 * j + 1]));
#pragma unroll
                    for (int u = 0; u < NC; ++u)
#pragma unroll
                        for (int n = 0; n < NP; ++n) s[u][n] = H::mfma16(kf, qf[u][n][2 * i + j], s[u][n]);
                }
            const float kb = lane_value(ks, b);
#pragma unroll
            for (int u = 0; u < NC; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    x[u][b][r] = (NP == 1 ? s[u][0][r] : s[u][0][r] + s[u][NP - 1][r]) * (fac[u] * kb);
        }
        const unsigned okc = ok;
        if (more) load_k(kt + ROUND);
        // Whether some column does not see some key of the step.
        const bool masked =
            kt + STEP - 1 > t.p0 || kt < t.lo || (a.window > 0 && kt < t.p1 - a.window + 1) || okc != (1u << NB) - 1;
        f16x8 pf[NC][NB / 2][PP];
#pragma unroll
        for (int u = 0; u < NC; ++u) {
            float mx = kLeast;
            int vn = ve[u];
            unsigned some = (1u << NB) - 1;  // the blocks of which the column sees any key
            if (masked) {
                some = 0;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = kt + 16 * b + 4 * g4 + r;
                        if (!(key <= pos[u] && key >= first[u] && (okc >> b & 1))) x[u][b][r] = -INFINITY;
                    }
                    some |= kt + 16 * b <= pos[u] && kt + 16 * b + 15 >= first[u] && (okc >> b & 1) ? 1u << b : 0u;
                }
                mx = some ? kLeast : -INFINITY;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int v = scale_exp(lane_value(vs, b));
                vn = some >> b & 1 ? max(vn, v) : vn;
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[u][b][r]);
            }
            mx = column_max(mx);
            const bool up = mx > m[u] + kLag;
            const float mn = up ? mx : m[u];
            const float ref = mn == -INFINITY ? 0.0f : mn - kLift<f16>;
            float corr = __builtin_amdgcn_exp2f((m[u] == -INFINITY ? m[u] : m[u] - kLift<f16>) - ref);
            m[u] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[u][b][r] = __builtin_amdgcn_exp2f(x[u][b][r] - ref);
                    sum += x[u][b][r];
                }
            l[u] = l[u] * corr + sum;
            if (__any(up || vn != ve[u])) {
                corr = __builtin_amdgcn_ldexpf(corr, ve[u] - vn);
#pragma unroll
                for (int i = 0; i < VD; ++i) o[u][i] *= corr;
                ve[u] = vn;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {  // the scale of V in units of 2^ve
                const float g = some >> b & 1 ? __builtin_amdgcn_ldexpf(lane_value(vs, b), -ve[u]) : 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    f16 pc[PP];
                    weight_pieces(x[u][b][r], g, pc);
#pragma unroll
                    for (int n = 0; n < PP; ++n) pf[u][b / 2][n][4 * (b & 1) + r] = pc[n];
                }
            }
        }
#pragma unroll
        for (int b = 0; b < NB; b += 2) {
#pragma unroll
            for (int d = 0; d < VW; ++d) {
                int v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = C::ready(vc[4 * b + i][d]);
                auto dim = [&](auto byte) __attribute__((always_inline)) {
                    constexpr int B = decltype(byte)::value;
                    const i32x4 f = {C::template across<B>(v[1], v[0]), C::template across<B>(v[3], v[2]),
                                     C::template across<B>(v[5], v[4]), C::template across<B>(v[7], v[6])};
#pragma unroll
                    for (int u = 0; u < NC; ++u)
#pragma unroll
                        for (int n = 0; n < PP; ++n)
                            o[u][4 * d + B] = H::mfma16(__builtin_bit_cast(f16x8, f), pf[u][b / 2][n], o[u][4 * d + B]);
                };
                dim(std::integral_constant<int, 0>{});
                dim(std::integral_constant<int, 1>{});
                dim(std::integral_constant<int, 2>{});
                dim(std::integral_constant<int, 3>{});
            }
        }
        if (more) load_v();
    };
    int kt = t.k0 + STEP * wave;
    if (kt < t.k1) {
        pages8_start(a, w, t.seq, t.lo, t.hi, kt);
        load_k(kt);
        load_v();
        for (; kt + ROUND < t.k1; kt += ROUND) step(kt, std::true_type{});
        step(kt, std::false_type{});
    }
#pragma unroll
    for (int u = 0; u < NC; ++u) {
        if (u > 0) {
            if (t.c0 + 16 * u >= t.n * a.group) break;
            __syncthreads();  // the last columns' results have been read
        }
        const int down = ve[u] - kDrop + C::kExp;
#pragma unroll
        for (int i = 0; i < VD; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[u][i][r] = __builtin_amdgcn_ldexpf(o[u][i][r], down);
        row_column(a, t, t.c0 + 16 * u + c);
        rows_finish<RT, HD, NW>(a, t, m[u], __builtin_amdgcn_ldexpf(l[u], -kDrop), o[u]);
    }
}

}  // namespace

template <typename RT, typename C>
int attn8_rows_launch(const Attn8Args &e, int hd, int splits, int tiles, hipStream_t st) {
    const AttnArgs &a = e.a;
    const unsigned units = a.row_tiles ? (unsigned)(a.b.rows * a.row_tiles) : (unsigned)(a.b.seqs * tiles);
    const unsigned blocks = units * (unsigned)splits * (unsigned)a.pool.kv_heads;
    auto launch = [&](auto dim, auto sets, auto by_row) {
        constexpr int HD = decltype(dim)::value, NC = decltype(sets)::value;
        constexpr bool BY_ROW = decltype(by_row)::value;
        hipLaunchKernelGGL((attn8_rows_kernel<RT, C, HD, NC, BY_ROW>), dim3(blocks), dim3(64 * row8_waves(NC)), 0, st, e, tiles, splits);
    };
    auto pick = [&](auto dim, auto sets) {
        a.row_tiles ? launch(dim, sets, std::true_type{}) : launch(dim, sets, std::false_type{});
    };
    auto size = [&](auto dim) {
        a.small_tile == 16 ? pick(dim, std::integral_constant<int, 1>{}) : pick(dim, std::integral_constant<int, 2>{});
    };
    hd == 128 ? size(std::integral_constant<int, 128>{}) : size(std::integral_constant<int, 64>{});
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
