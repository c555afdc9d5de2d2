// Paged attention over 8-bit pages, many query rows: the chunk kernel of gphq_paged8_attention
// (prompt chunks). See paged_attention.h for the mathematics and the tiling, paged8.h for the
// codes.
#include "paged8.h"
#include "paged_chunk.h"

namespace gphq {
namespace {

// The walk of the 16-bit chunk kernel: each step's 64 keys are brought to LDS once for the
// block's 32 NW columns, K and V as rows of FP16 whose 16-byte pieces are permuted so that the
// fragment reads fall on all banks; two LDS buffers, one barrier a step; S^T = K . Q^T and
// O^T += V^T . P^T on v_mfma_f32_32x32x16_f16, V^T's fragments by transposing LDS reads. But a
// step's codes come through registers, a step ahead, and are made FP16 once, on their way to LDS;
// and a step is multiplied 32 keys at a time, which leaves the registers for the pieces of fp32 rows
// (64 at a time they spilled: one prompt of 4096 fp32 rows 402 us, 350 with this).
//
// With c the code, an exponent is s ks fac - m + log2(vs / 2^ve): V's scales are in the
// exponents of the weights, and a block's sum of them is brought back by 2^-log for the
// denominator.
//
// Bound by the vector instructions beside the matrix instructions, which overlap little: per 64 keys
// and 32 columns a wavefront has about 360 of the first (1850 cycles with the exponentials) and 1024 cycles
// of the second a piece. 512 FP16 rows of 32 heads over 16512 tokens: 195 us with the join, 0.70
// PFLOP/s (the 16-bit kernel over FP16 pages 0.73); twelve sequences of up to 300 fp32 rows 104 us.
// The next half's scores beside this half's exponentials in one wavefront's instructions, with V's
// buffer tripled, took more registers than there are (340 and 331 us).
template <typename RT, typename C, int HD, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn8_chunk_kernel(const Attn8Args e, int tiles, int splits) {
    typedef Half<f16> H;
    constexpr int NT = 64 * NW, NP = kPieces<RT, f16>, KB = 64, NB = KB / 16, QC = HD / 16, DT = HD / 32;
    constexpr int KP = HD / 16, PT = 2 * KB * KP / NT;  // 16-code pieces per key; per thread and step, K's first
    __shared__ __attribute__((aligned(16))) f16 Ks[2][KB * HD];
    __shared__ __attribute__((aligned(16))) f16 Vs[2][KB * HD];
    const AttnArgs &a = e.a;
    ChunkTile t;
    if (!chunk_tile<32 * NW>(a, tiles, splits, t)) return;
    const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, q = lane & 31, hi = lane >> 5;
    const char *kp = (const char *)a.pool.k, *vp = (const char *)a.pool.v;
    const int ts = (int)a.pool.token_stride;

    float fac = a.scale_log2;
    f16x8 qf[NP][QC];
    {
        const RT *src = (const RT *)a.q + (int64_t)(t.start + t.row) * a.q_stride + t.head * HD + 8 * hi;
        float inverse = 1.0f, up = 1.0f;
        if (!std::is_same<RT, f16>::value) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * QC; ++i) {
                float x[4];
                load_vec(src + 16 * (i >> 1) + 4 * (i & 1), x);
#pragma unroll
                for (int k = 0; k < 4; ++k) m = fmaxf(m, fabsf(x[k]));
            }
            m = fmaxf(m, __shfl_xor(m, 32));
            up = f16_scale(m, inverse);
        }
        fac = score_factor(fac * inverse * (float)(1 << C::kExp));
        up *= a.q_sign;
#pragma unroll
        for (int i = 0; i < 2 * QC; ++i) {
            float x[4];
            load_vec(src + 16 * (i >> 1) + 4 * (i & 1), x);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                f16 pc[NP];
                query_pieces(x[k] * up, pc);
#pragma unroll
                for (int n = 0; n < NP; ++n) qf[n][i >> 1][4 * (i & 1) + k] = pc[n];
            }
        }
    }

    auto k_swz = [](int row) { return HD == 128 ? row & 15 : row >> 1 & 7; };
    auto v_swz = [](int row) { return HD == 128 ? 4 * (row & 3) : 4 * (row >> 1 & 1); };
    Page8Walk w;
    i32x4 code[PT];  // piece tid + i NT of the step: K's KB * KP, then V's
    float ks[NB], vs[NB];
    auto load = [&](int kt) __attribute__((always_inline)) -> unsigned {
        int64_t at[NB], sat[NB];
        const unsigned ok = pages8_step(e, w, t.seq, t.g, kt, at, sat);
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const int first = wave * 64 + i * NT;  // the same for a wavefront: K's or V's, and one block
            const int row = (first + lane) / KP % KB, n = uniform(first / KP % KB >> 4);
            const int64_t base = n == 0 ? at[0] : n == 1 ? at[1] : n == 2 ? at[2] : at[3];
            code[i] = *(const i32x4 *)((first < KB * KP ? kp : vp) + base + ((row & 15) * ts + 16 * ((first + lane) % KP)));
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            ks[b] = uniform_scale(e.s.k, sat[b]);
            vs[b] = uniform_scale(e.s.v, sat[b]);
        }
        return ok;
    };
    auto store = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const int first = wave * 64 + i * NT, row = (first + lane) / KP % KB, pc = (first + lane) % KP;
            const bool isK = first < KB * KP;
            f16 *dst = (isK ? Ks[buf] : Vs[buf]) + row * HD;
            const int swz = isK ? k_swz(row & 15) : v_swz(row);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                *(f16x8 *)(dst + 8 * ((2 * pc + j) ^ swz)) =
                    codes8<C>(C::ready(code[i][2 * j]), C::ready(code[i][2 * j + 1]));
        }
    };

    // This lane's part of the transposing reads, for each 32 dims.
    const int s16 = lane & 15;
    int v_at[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        const int row = 4 * hi + (s16 >> 2), pc = 4 * d + 2 * (lane >> 4 & 1) + (s16 >> 1 & 1);
        v_at[d] = row * HD + 8 * (pc ^ v_swz(row)) + 4 * (s16 & 1);
    }
    auto v_frag = [&](int buf, int k16, int d) __attribute__((always_inline)) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 lds_s4;
        union {
            s4 h[2];
            f16x8 v;
        } f;
        f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(Vs[buf] + v_at[d] + 16 * k16 * HD));
        f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(Vs[buf] + v_at[d] + (16 * k16 + 8) * HD));
        return f.v;
    };

    f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    int ve = kNoExp;

    // Scores of the 32 keys of half h of K's buffer: s[r] is key 8 (r / 4) + 4 hi + r % 4 of them.
    auto scores = [&](int buf, int h, f32x16 &s) __attribute__((always_inline)) {
        f32x16 low{};
        s = f32x16{};
#pragma unroll
        for (int i = 0; i < QC; ++i) {
            const int row = 32 * h + q;
            const f16x8 kf = *(const f16x8 *)(Ks[buf] + row * HD + 8 * ((2 * i + hi) ^ k_swz(row & 15)));
            s = H::mfma32(kf, qf[0][i], s);
            if (NP == 2) low = H::mfma32(kf, qf[NP - 1][i], low);
        }
        if (NP == 2) s += low;
    };
    // The exponentials of 32 keys from kt on, whose blocks have the scales kb and vb and the bits ok;
    // o is brought to their units. pf are the probabilities times V's scales in those units.
    auto weigh = [&](f32x16 &s, int kt, const float *kb, const float *vb, unsigned ok, bool masked,
                     f16x8 (&pf)[2][NP]) __attribute__((always_inline)) {
        unsigned some = 3;  // the blocks of which the column sees any key
        if (masked) {
            some = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = kt + 8 * (r >> 2) + 4 * hi + (r & 3);
                if (!(key <= t.pos && key >= t.first && (ok >> (r >> 3) & 1))) s[r] = -INFINITY;
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
                some |= kt + 16 * b <= t.pos && kt + 16 * b + 15 >= t.first && (ok >> b & 1) ? 1u << b : 0u;
        }
        float mx = some ? kLeast : -INFINITY, f[2];
        int vx = ve;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            // (The factor of a block that the column does not see: any, so long as -inf times it stays that.)
            const bool sees = !masked || (some >> b & 1);
            f[b] = fac * kb[b];
            f[b] = !sees ? 1.0f : f[b] < FLT_MIN ? FLT_MIN : f[b];  // (not a maximum: what is not a number stays that)
            const int v = scale_exp(vb[b]);
            vx = sees ? max(vx, v) : vx;
            float big = s[8 * b];
#pragma unroll
            for (int r = 1; r < 8; ++r) big = fmaxf(big, s[8 * b + r]);
            mx = fmaxf(mx, big * f[b]);
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const bool up = mx > m + kLag, grew = up || vx != ve;
        const float mn = up ? mx : m;
        const float ref = mn == -INFINITY ? 0.0f : mn - kLift<f16>;
        float corr = __builtin_amdgcn_exp2f((m == -INFINITY ? m : m - kLift<f16>) - ref);
        m = mn;
        l *= corr;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const float raise = !masked || (some >> b & 1) ? scale_log(vb[b], vx) : 0.0f, from = raise - ref;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[8 * b + i], f[b], from));
                sum += p;
                f16 pc[NP];
                split_pieces(p, pc);
#pragma unroll
                for (int n = 0; n < NP; ++n) pf[b][n][i] = pc[n];
            }
            l = fmaf(sum, __builtin_amdgcn_exp2f(-raise), l);
        }
        if (__any(grew)) {
            corr = __builtin_amdgcn_ldexpf(corr, ve - vx);
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= corr;
            ve = vx;
        }
    };
    auto outputs = [&](int vbuf, int h, const f16x8 (&pf)[2][NP]) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const f16x8 f = v_frag(vbuf, 2 * h + b, d);
#pragma unroll
                for (int n = 0; n < NP; ++n) o[d] = H::mfma32(f, pf[b][n], o[d]);
            }
    };
    unsigned ok = 0;
    if (t.k0 < t.k1) {
        pages8_start(a, w, t.seq, t.lo, t.hi, t.k0);
        ok = load(t.k0);
    }
    int buf = 0;
    for (int kt = t.k0; kt < t.k1; kt += KB, buf ^= 1) {
        store(buf);
        __syncthreads();  // the step is here, and the other buffer has been read
        const unsigned okc = ok;
        float kn[NB], vn[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) kn[b] = ks[b], vn[b] = vs[b];
        if (kt + KB < t.k1) ok = load(kt + KB);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int kh = kt + 32 * h;
            if (kh >= t.w_hi || kh + 32 <= t.w_lo) continue;
            const unsigned okh = okc >> (2 * h) & 3;
            f32x16 s;
            f16x8 pf[2][NP];
            __builtin_amdgcn_s_setprio(1);
            scores(buf, h, s);
            __builtin_amdgcn_s_setprio(0);
            const bool masked = kh + 31 > t.p0 || kh < t.w_lo || (a.window > 0 && kh < t.p1 - a.window + 1) || okh != 3;
            weigh(s, kh, kn + 2 * h, vn + 2 * h, okh, masked, pf);
            outputs(buf, h, pf);
        }
    }
    const int down = ve - kDrop + C::kExp;
    chunk_finish<RT, HD>(a, t, m, __builtin_amdgcn_ldexpf(l, -kDrop), [&](int i) {
        const f32x16 &v = o[i / 4];
        const int r = 4 * (i % 4);
        return f32x4{__builtin_amdgcn_ldexpf(v[r], down), __builtin_amdgcn_ldexpf(v[r + 1], down),
                     __builtin_amdgcn_ldexpf(v[r + 2], down), __builtin_amdgcn_ldexpf(v[r + 3], down)};
    });
}

}  // namespace

template <typename RT, typename C>
int attn8_chunk_launch(const Attn8Args &e, int hd, int splits, int tiles, hipStream_t st) {
    const unsigned blocks = (unsigned)tiles * (unsigned)splits * (unsigned)e.a.pool.kv_heads;
    auto launch = [&](auto dim, auto waves) {
        constexpr int HD = decltype(dim)::value, NW = decltype(waves)::value;
        hipLaunchKernelGGL((attn8_chunk_kernel<RT, C, HD, NW>), dim3(blocks), dim3(64 * NW), 0, st, e, tiles, splits);
    };
    auto pick = [&](auto dim) {
        if constexpr (kPieces<RT, f16> == 1)
            if (e.a.big_tile == 256) return launch(dim, std::integral_constant<int, 8>{});
        launch(dim, std::integral_constant<int, 4>{});
    };
    hd == 128 ? pick(std::integral_constant<int, 128>{}) : pick(std::integral_constant<int, 64>{});
    return launch_status();
}

#define GPHQ_CHUNK8(RT)                                                                          \
    template int attn8_chunk_launch<RT, CodesI8>(const Attn8Args &, int, int, int, hipStream_t); \
    template int attn8_chunk_launch<RT, CodesE4M3>(const Attn8Args &, int, int, int, hipStream_t)
GPHQ_CHUNK8(float);
GPHQ_CHUNK8(f16);
GPHQ_CHUNK8(bf16);
#undef GPHQ_CHUNK8

}  // namespace gphq
