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
// step's codes come through registers, a step ahead, and are made FP16 once, on their way to LDS.
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
        if (kt >= t.w_hi || kt + KB <= t.w_lo) continue;
        f32x16 s[2];
        __builtin_amdgcn_s_setprio(1);
        if (NP == 1) {
            s[0] = s[1] = f32x16{};
#pragma unroll
            for (int i = 0; i < QC; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int row = 32 * h + q;
                    const f16x8 kf = *(const f16x8 *)(Ks[buf] + row * HD + 8 * ((2 * i + hi) ^ k_swz(row & 15)));
                    s[h] = H::mfma32(kf, qf[0][i], s[h]);
                }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                f32x16 p[2] = {f32x16{}, f32x16{}};
#pragma unroll
                for (int i = 0; i < QC; ++i) {
                    const int row = 32 * h + q;
                    const f16x8 kf = *(const f16x8 *)(Ks[buf] + row * HD + 8 * ((2 * i + hi) ^ k_swz(row & 15)));
                    p[0] = H::mfma32(kf, qf[0][i], p[0]);
                    p[1] = H::mfma32(kf, qf[NP - 1][i], p[1]);
                }
                s[h] = p[0] + p[1];
            }
        }
        __builtin_amdgcn_s_setprio(0);
        // s[h][r] is key kt + 32 h + 8 (r / 4) + 4 hi + r % 4, of block 2 h + r / 8.
        const bool masked =
            kt + KB - 1 > t.p0 || kt < t.w_lo || (a.window > 0 && kt < t.p1 - a.window + 1) || okc != 15;
        float mx = kLeast;
        unsigned some = 15;  // the blocks of which the column sees any key
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[h][r] *= fac * kn[2 * h + (r >> 3)];
        if (masked) {
            some = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = kt + 32 * h + 8 * (r >> 2) + 4 * hi + (r & 3);
                    if (!(key <= t.pos && key >= t.first && (okc >> (2 * h + (r >> 3)) & 1))) s[h][r] = -INFINITY;
                }
#pragma unroll
            for (int b = 0; b < NB; ++b)
                some |= kt + 16 * b <= t.pos && kt + 16 * b + 15 >= t.first && (okc >> b & 1) ? 1u << b : 0u;
            mx = some ? kLeast : -INFINITY;
        }
        int vx = ve;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int v = scale_exp(vn[b]);
            vx = some >> b & 1 ? max(vx, v) : vx;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[h][r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const bool grew = mx > m + kLag || vx != ve;
        const float mn = mx > m + kLag ? mx : m;
        const float ref = mn == -INFINITY ? 0.0f : mn - kLift<f16>;
        float corr = __builtin_amdgcn_exp2f((m == -INFINITY ? m : m - kLift<f16>) - ref);
        m = mn;
        float sum = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[h][r] = __builtin_amdgcn_exp2f(s[h][r] - ref);
                sum += s[h][r];
            }
        l = l * corr + sum;
        if (__any(grew)) {
            corr = __builtin_amdgcn_ldexpf(corr, ve - vx);
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= corr;
            ve = vx;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float scale = some >> b & 1 ? __builtin_amdgcn_ldexpf(vn[b], -ve) : 0.0f;
            f16x8 pf[NP];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f16 pc[NP];
                weight_pieces(s[b >> 1][8 * (b & 1) + i], scale, pc);
#pragma unroll
                for (int n = 0; n < NP; ++n) pf[n][i] = pc[n];
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const f16x8 f = v_frag(buf, b, d);
#pragma unroll
                for (int n = 0; n < NP; ++n) o[d] = H::mfma32(f, pf[n], o[d]);
            }
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
    constexpr int NW = kChunkWaves<RT, f16>;
    if (hd == 128)
        hipLaunchKernelGGL((attn8_chunk_kernel<RT, C, 128, NW>), dim3(blocks), dim3(64 * NW), 0, st, e, tiles, splits);
    else
        hipLaunchKernelGGL((attn8_chunk_kernel<RT, C, 64, NW>), dim3(blocks), dim3(64 * NW), 0, st, e, tiles, splits);
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
