// Paged attention of many query rows: the chunk kernel of gphq_paged_attention (prompt
// chunks). See paged_attention.h for the mathematics and the tiling.
#include "paged_attention.h"

namespace gphq {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// One block's tile: TM columns of a sequence and KV head, 32 to each wavefront, over the keys [k0, k1).
struct ChunkTile {
    int seq, g, n, len, start, splits, split;
    int lo, hi, k0, k1;
    int b_p0, b_p1;  // positions of the tile's first and last row
    // this wavefront's rows and their keys [w_lo, w_hi)
    int r0, r1, p0, p1, w_lo, w_hi;
    // this lane's column
    int row, head, pos, first;
    bool live;
};

// The block's tile among those of the sequences that are not the row kernel's, counted by
// 64 lanes over 64 sequences at a time. Tiles are dealt out from the back: a sequence's last
// rows see most keys, so the long tiles start first. False where there is no such tile.
template <int TM>
__device__ __forceinline__ bool chunk_tile(const AttnArgs &a, int tiles, int splits, ChunkTile &t) {
    int u = blockIdx.x;
    t.g = u % a.pool.kv_heads;
    u /= a.pool.kv_heads;
    t.split = u % splits;
    const int want = tiles - 1 - u / splits;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    int before = 0, tile = -1;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 64) {
        const int s = min(s0 + lane, a.b.seqs - 1);
        const int start = a.b.starts[s], end = a.b.starts[s + 1], len = a.b.lens[s];
        const bool ok = seq_ok(a.b, start, end, len);
        if (!ok) paged_flag(a.b, PAGED_BAD_SEQ);
        const int cols = ok ? (end - start) * a.group : 0;
        const int mine = s0 + lane < a.b.seqs && cols > a.small_cols ? (cols + TM - 1) / TM : 0;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int v = __shfl_up(sum, d);
            sum += lane >= d ? v : 0;
        }
        const int total = __builtin_amdgcn_readlane(sum, 63);
        if (want < before + total) {
            const int at = __builtin_ctzll(__ballot(want < before + sum));
            t.seq = s0 + at;
            tile = want - before - __builtin_amdgcn_readlane(sum - mine, at);
            t.start = __builtin_amdgcn_readlane(start, at);
            t.n = __builtin_amdgcn_readlane(end, at) - t.start;
            t.len = __builtin_amdgcn_readlane(len, at);
            break;
        }
        before += total;
    }
    if (tile < 0) return false;
    const int cols = t.n * a.group, c0 = tile * TM, off = t.len - t.n;
    const TileKeys k =
        tile_keys(t.n, t.len, c0 / a.group, min((c0 + TM - 1) / a.group, t.n - 1), a.window);
    t.lo = k.lo;
    t.hi = k.hi;
    t.b_p0 = off + c0 / a.group;
    t.b_p1 = off + min((c0 + TM - 1) / a.group, t.n - 1);
    t.splits = tile_splits(k, a.split_big);
    if (t.split >= t.splits) return false;
    t.k0 = k.from + t.split * a.split_big;
    t.k1 = min(t.k0 + a.split_big, k.hi);
    const int w0 = c0 + 32 * wave;
    t.r0 = min(w0 / a.group, t.n - 1);
    t.r1 = min((w0 + 31) / a.group, t.n - 1);
    t.p0 = off + t.r0;
    t.p1 = off + t.r1;
    const TileKeys w = tile_keys(t.n, t.len, t.r0, t.r1, a.window);
    t.w_lo = w.lo;
    t.w_hi = w0 < cols ? w.hi : 0;  // a wavefront without columns sees no key
    const int col = w0 + (lane & 31);
    t.live = col < cols;
    t.row = t.live ? col / a.group : t.r1;
    t.head = t.g * a.group + (t.live ? col - t.row * a.group : 0);
    t.pos = off + t.row;
    t.first = a.window > 0 ? t.pos - a.window + 1 : 0;
    return true;
}

// A step that holds keys which some row of the tile does not see.
__device__ __forceinline__ bool chunk_edge(const AttnArgs &a, const ChunkTile &t, int kt, int keys) {
    return kt + keys - 1 > t.b_p0 || kt < t.lo || (a.window > 0 && kt < t.b_p1 - a.window + 1);
}

// One step's exponentials over N 32-key score tiles: s[h][r] is key kt + 32 h + 8 (r / 4) +
// 4 hi + r % 4; as the row kernel's softmax_step. ok: a bit per 16 keys.
template <typename CT, int N>
__device__ __forceinline__ float chunk_softmax(const ChunkTile &t, f32x16 (&s)[N], float fac, bool masked, int kt,
                                               unsigned ok, float &m, float &l, bool &moved) {
    const int hi = (threadIdx.x & 63) >> 5;
    float mx = kLeast;
    if (masked) {
        bool any = false;
#pragma unroll
        for (int h = 0; h < N; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int key = kt + 32 * h + 8 * (r >> 2) + 4 * hi + (r & 3);
                const bool sees = key <= t.pos && key >= t.first && (ok >> (2 * h + (r >> 3)) & 1);
                if (!sees) s[h][r] = -INFINITY;
                any |= sees;
            }
        mx = any ? kLeast : -INFINITY;
    }
#pragma unroll
    for (int h = 0; h < N; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[h][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    mx = mx == -INFINITY ? mx : fmaxf(mx * fac, kLeast);
    const bool grew = mx > m + kLag;
    const float mn = grew ? mx : m;
    const float ref = mn == -INFINITY ? 0.0f : mn - kLift<CT>;
    const float corr = __builtin_amdgcn_exp2f((m == -INFINITY ? m : m - kLift<CT>) - ref);
    m = mn;
    float sum = 0.0f;
#pragma unroll
    for (int h = 0; h < N; ++h)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[h][r] = __builtin_amdgcn_exp2f(fmaf(s[h][r], fac, -ref));
            sum += s[h][r];
        }
    l = l * corr + sum;
    moved = __any(grew);
    return corr;
}

// Writes a lane's column, or its split result: o(d0) gives four values of consecutive dims
// from d0 on, the lane holding the dims of every 8 that start at 4 hi.
template <typename RT, int HD, typename F>
__device__ __forceinline__ void chunk_finish(const AttnArgs &a, const ChunkTile &t, float m, float l, F &&o) {
    const int hi = (threadIdx.x & 63) >> 5;
    l += __shfl_xor(l, 32);
    if (!t.live) return;
    if (t.splits == 1) {
        const float inv = 1.0f / l;
        const bool empty = m == -INFINITY;
        RT *out = (RT *)a.out + (int64_t)(t.start + t.row) * a.out_stride + t.head * HD;
#pragma unroll
        for (int d = 0; d < HD; d += 8) {
            const f32x4 v = o(d / 8);
            const float w[4] = {empty ? 0.0f : v[0] * inv, empty ? 0.0f : v[1] * inv,
                                empty ? 0.0f : v[2] * inv, empty ? 0.0f : v[3] * inv};
            store_vec(out + d + 4 * hi, w);
        }
        return;
    }
    const int64_t at = ((int64_t)(t.start + t.row) * a.heads + t.head) * a.parts + t.split;
#pragma unroll
    for (int d = 0; d < HD; d += 8) *(f32x4 *)(a.part_o + at * HD + d + 4 * hi) = o(d / 8);
    if (hi == 0) {
        a.part_ml[2 * at] = m;
        a.part_ml[2 * at + 1] = l;
    }
}

// 16-bit pages. Each step's 64 keys are brought from the pages straight to LDS, once for the
// block's 32 NW columns, both K and V as rows. A row's 16-byte pieces are permuted (by the
// source address: the LDS side of such a load is linear), so that the fragment reads below
// fall on all banks. On v_mfma_f32_32x32x16:
//   S^T (32 keys x 32 columns) = K . Q^T;
//   O^T (32 dims x 32 columns) += V^T . P^T, the score registers being P^T's fragment: in
//     each 16 keys a lane of the lower half holds keys 0-3 and 8-11, of the upper half 4-7
//     and 12-15; V^T's fragment comes from two transposing LDS reads, in each of which 16
//     lanes read 4 keys x 16 dims and a lane gets the 4 keys of one dim.
// Two LDS buffers, one barrier a step: step u + 1 is on its way while step u is multiplied.
//
// Bound by the matrix cores and, beside them, the exponentials: per 64 keys and 32 columns a
// wavefront has 1024 cycles of matrix instructions a piece and about 1100 of softmax, on two
// wavefronts a SIMD (four a block and two blocks a CU where rows and pages have one type, eight
// a block where rows are split in pieces and Q's pieces take the registers). 512 FP16 rows of
// 32 heads over 7512 tokens: 84 us with the join, 0.73 PFLOP/s; 4096 fp32 rows, FP16 pages: 258
// us, 0.53 PFLOP/s and twice that in pieces, the rate at which a large FP16 library product
// runs on this card (1.1). 16-bit rows take their probabilities in one piece, rounded to the
// rows' type: a second one, as the row kernel has, makes the 84 us 108. Half-step offsets
// between the wavefronts of a SIMD, to set one's
// exponentials beside the other's products, measured the same or slower (268 us before, 273
// to 275 with them).
template <typename RT, typename CT, int HD, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attn_chunk16_kernel(const AttnArgs a, int tiles, int splits) {
    typedef Half<CT> H;
    typedef typename H::vec8 vec8;
    constexpr int NT = 64 * NW, NP = kPieces<RT, CT>, KB = 64, QC = HD / 16, DT = HD / 32;
    constexpr int KP = HD / 8, RI = 64 / KP, KI = KB / RI / NW;  // pieces per key; keys per load, loads per wavefront
    __shared__ __attribute__((aligned(16))) CT Ks[2][KB * HD];
    __shared__ __attribute__((aligned(16))) CT Vs[2][KB * HD];
    // Of three pieces of Q the last stays in LDS, read again each step: three do not fit the registers.
    constexpr int NR = HD == 128 && NP == 3 ? 2 : NP;
    __shared__ vec8 ql[NR < NP ? NW : 1][QC][NR < NP ? 64 : 1];
    __shared__ int odd[2][KB];  // for each key of a buffer, the step (its first key) whose V[key] is not all finite
    ChunkTile t;
    if (!chunk_tile<32 * NW>(a, tiles, splits, t)) return;
    const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, q = lane & 31, hi = lane >> 5;
    const char *kp = (const char *)a.pool.k, *vp = (const char *)a.pool.v;
    const int ts = (int)(a.pool.token_stride * sizeof(CT));

    float fac = score_factor(a.scale_log2);
    vec8 qf[NR][QC];
    {
        const RT *src = (const RT *)a.q + (int64_t)(t.start + t.row) * a.q_stride + t.head * HD + 8 * hi;
        float inverse = 1.0f, up = 1.0f;
        if (NP == 2) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * QC; ++i) {
                float x[4];
                load_vec(src + 16 * (i >> 1) + 4 * (i & 1), x);
#pragma unroll
                for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(x[e]));
            }
            m = fmaxf(m, __shfl_xor(m, 32));
            up = f16_scale(m, inverse);
            fac = score_factor(fac * inverse);
        }
        up *= a.q_sign;
#pragma unroll
        for (int i = 0; i < 2 * QC; ++i) {
            float x[4];
            load_vec(src + 16 * (i >> 1) + 4 * (i & 1), x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                CT pc[NP];
                split_pieces(x[e] * up, pc);
#pragma unroll
                for (int k = 0; k < NR; ++k) qf[k][i >> 1][4 * (i & 1) + e] = pc[k];
                if (NR < NP) ql[wave][i >> 1][lane][4 * (i & 1) + e] = pc[NP - 1];
            }
        }
    }

    // Load j of a wavefront brings keys row0 + RI j .. of the step, lane l piece l % KP of key l / KP.
    const int row0 = wave * KI * RI, lrow = lane / KP, lpc = lane % KP;
    auto k_swz = [](int row) { return HD == 128 ? row & 15 : row >> 1 & 7; };
    auto v_swz = [](int row) { return HD == 128 ? 4 * (row & 3) : 4 * (row >> 1 & 1); };
    PageWalk w;
    auto load = [&](int kt, int buf) __attribute__((always_inline)) -> unsigned {
        int64_t at[4];
        const unsigned ok = pages_step<CT>(a, w, t.seq, t.g, kt, at);
#pragma unroll
        for (int j = 0; j < KI; ++j) {
            const int row = row0 + RI * j, n = row >> 4, r = (row & 15) + lrow;
            const int64_t base = n == 0 ? at[0] : n == 1 ? at[1] : n == 2 ? at[2] : at[3];
            dma16(kp + base, r * ts + 16 * (lpc ^ k_swz(r)), Ks[buf] + row * HD);
            dma16(vp + base, r * ts + 16 * (lpc ^ v_swz(r)), Vs[buf] + row * HD);
        }
        return ok;
    };
    // In a step with keys that some row of the tile does not see: what no row sees becomes 0
    // (it may hold anything, and 0 times it must stay 0), what is not finite is taken out.
    // Each wavefront mends what it has loaded itself.
    auto mend = [&](int kt, unsigned ok, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < KI; ++j) {
            const int row = row0 + RI * j + lrow, key = kt + row;
            i32x4 *p = (i32x4 *)(Vs[buf] + (row0 + RI * j) * HD) + lane;
            i32x4 v = *p;
            if (key < t.lo || key >= t.hi || !(ok >> (row >> 4) & 1)) v = i32x4{};
            int any = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int out = pair_not_finite<CT>(v[e]);
                v[e] &= ~out;
                any |= out;
            }
            if (any) odd[buf][row] = kt;
            *p = v;
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
    auto v_frag = [&](int buf, int ks, int d) __attribute__((always_inline)) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 lds_s4;
        union {
            s4 h[2];
            vec8 v;
        } f;
        f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(Vs[buf] + v_at[d] + 16 * ks * HD));
        f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(Vs[buf] + v_at[d] + (16 * ks + 8) * HD));
        return f.v;
    };

    f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    if (tid < 2 * KB) (&odd[0][0])[tid] = -1;
    __syncthreads();
    unsigned ok = 0;
    if (t.k0 < t.k1) {
        pages_start<CT>(a, w, t.seq, t.g, t.lo, t.hi, t.k0);
        ok = load(t.k0, 0);
    }
    int buf = 0;
    for (int kt = t.k0; kt < t.k1; kt += KB, buf ^= 1) {
        wait_vm_lgkm0<0>();
        asm volatile("" ::: "memory");  // the wait is no memory operation: mend's reads stay behind it
        const unsigned okc = ok;
        const bool edge = chunk_edge(a, t, kt, KB) || okc != 15;
        if (edge) mend(kt, okc, buf);
        __syncthreads();  // the step is here, and the other buffer has been read
        if (kt + KB < t.k1) ok = load(kt + KB, buf ^ 1);
        if (kt >= t.w_hi || kt + KB <= t.w_lo) continue;
        f32x16 s[2] = {f32x16{}, f32x16{}};
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < QC; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = 32 * h + q;
                const vec8 kf = *(const vec8 *)(Ks[buf] + row * HD + 8 * ((2 * i + hi) ^ k_swz(row & 15)));
#pragma unroll
                for (int k = 0; k < NR; ++k) s[h] = H::mfma32(kf, qf[k][i], s[h]);
                if (NR < NP) s[h] = H::mfma32(kf, ql[wave][i][lane], s[h]);
            }
        __builtin_amdgcn_s_setprio(0);
        const bool masked =
            kt + KB - 1 > t.p0 || kt < t.w_lo || (a.window > 0 && kt < t.p1 - a.window + 1) || okc != 15;
        bool moved;
        const float corr = chunk_softmax<CT>(t, s, fac, masked, kt, okc, m, l, moved);
        if (moved) {
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= corr;
        }
#pragma unroll
        for (int ks = 0; ks < KB / 16; ++ks) {
            vec8 pf[NP];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                CT pc[NP];
                split_pieces(s[ks >> 1][8 * (ks & 1) + i], pc);
#pragma unroll
                for (int k = 0; k < NP; ++k) pf[k][i] = pc[k];
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const vec8 f = v_frag(buf, ks, d);
#pragma unroll
                for (int k = 0; k < NP; ++k) o[d] = H::mfma32(f, pf[k], o[d]);
            }
        }
        if (!edge) continue;
        for (uint64_t left = __ballot(odd[buf][lane] == kt); left; left &= left - 1) {
            const int key = kt + __builtin_ctzll(left);
            const int page = a.b.table[t.seq * a.b.table_stride + (key >> a.pool.shift)];  // a good one: V was kept
            const CT *v = (const CT *)a.pool.v + page * a.pool.page_stride +
                          (key & ((1 << a.pool.shift) - 1)) * a.pool.token_stride + t.g * a.pool.head_stride;
            const bool sees = key <= t.pos && key >= t.first;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x[4];
                    load_vec(v + 32 * d + 8 * j + 4 * hi, x);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d][4 * j + e] += sees ? not_finite(x[e]) : 0.0f;
                    asm volatile("" ::: "memory");  // few values at a time: this must not cost registers
                }
        }
    }
    chunk_finish<RT, HD>(a, t, m, l, [&](int i) {
        const f32x16 &v = o[i / 4];
        const int r = 4 * (i % 4);
        return f32x4{v[r], v[r + 1], v[r + 2], v[r + 3]};
    });
}

// Bound by the fp32 matrix instructions, a sixteenth of the 16-bit ones' rate: 512 rows over
// 7512 tokens 524 us, 117 TFLOP/s where a large fp32 library product makes 153.
// fp32 pages, the same walk in 32-key steps on v_mfma_f32_32x32x2_f32. Its operands are one
// fp32 value a lane, so V is staged as rows; a lane takes HD / 32 neighbouring dims of V at
// once, one for each of its output tiles: tile d holds dims HD/32 * i + d.
template <int HD, int NW>
__global__ __launch_bounds__(64 * NW) void attn_chunk32_kernel(const AttnArgs a, int tiles, int splits) {
    constexpr int NT = 64 * NW, KB = 32, QC = HD / 8, DT = HD / 32;
    constexpr int KP = HD / 4, KI = KB * KP / NT;  // 16-byte pieces per key, per thread
    __shared__ float Ks[2][KB * HD];
    __shared__ float Vs[2][KB * HD];
    __shared__ int odd[2][KB];  // for each key of a buffer, the step (its first key) whose V[key] is not all finite
    ChunkTile t;
    if (!chunk_tile<32 * NW>(a, tiles, splits, t)) return;
    const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, q = lane & 31, hi = lane >> 5;
    const char *kp = (const char *)a.pool.k, *vp = (const char *)a.pool.v;
    const int ts = (int)(a.pool.token_stride * sizeof(float));
    f32x4 qf[QC];
    {
        const float *src = (const float *)a.q + (int64_t)(t.start + t.row) * a.q_stride + t.head * HD + 4 * hi;
#pragma unroll
        for (int i = 0; i < QC; ++i) qf[i] = *(const f32x4 *)(src + 8 * i) * a.q_sign;
    }
    typedef float vdim __attribute__((ext_vector_type(DT)));
    f32x4 kr[KI], vr[KI];
    const int krow = tid / KP, kpc = tid % KP;
    PageWalk w;
    auto load = [&](int kt) __attribute__((always_inline)) -> unsigned {
        int64_t at[2];
        const unsigned ok = pages_step<float>(a, w, t.seq, t.g, kt, at);
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            const int64_t base = (wave * 64 + i * NT) / KP < 16 ? at[0] : at[1];  // the same for a wavefront's rows
            const unsigned off = (krow + i * (NT / KP)) % 16 * ts + 16 * kpc;
            kr[i] = *(const f32x4 *)(kp + base + off);
            vr[i] = *(const f32x4 *)(vp + base + off);
        }
        return ok;
    };
    auto store = [&](int kt, unsigned ok, int buf) __attribute__((always_inline)) {
        const bool edge = chunk_edge(a, t, kt, KB) || ok != 3;
#pragma unroll
        for (int i = 0; i < KI; ++i) {
            const int row = krow + i * (NT / KP), key = kt + row;
            *(f32x4 *)(Ks[buf] + row * HD + 4 * (kpc ^ (row & 15))) = kr[i];
            if (edge) {
                if (key < t.lo || key >= t.hi || !(ok >> (row >> 4) & 1)) vr[i] = f32x4{};  // no row of the tile sees it
                bool any = false;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!(fabsf(vr[i][e]) < INFINITY)) vr[i][e] = 0.0f, any = true;
                if (any) odd[buf][row] = kt;
            }
            *(f32x4 *)(Vs[buf] + row * HD + 4 * kpc) = vr[i];
        }
    };
    f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = f32x16{};
    float m = -INFINITY, l = 0.0f;
    if (tid < 2 * KB) (&odd[0][0])[tid] = -1;
    unsigned ok = 0;
    if (t.k0 < t.k1) {
        pages_start<float>(a, w, t.seq, t.g, t.lo, t.hi, t.k0);
        ok = load(t.k0);
    }
    int buf = 0;
    __syncthreads();
    for (int kt = t.k0; kt < t.k1; kt += KB, buf ^= 1) {
        store(kt, ok, buf);
        __syncthreads();
        const unsigned okc = ok;
        if (kt + KB < t.k1) ok = load(kt + KB);
        if (kt >= t.w_hi || kt + KB <= t.w_lo) continue;
        f32x16 s[1] = {f32x16{}};
#pragma unroll
        for (int i = 0; i < QC; ++i) {
            const f32x4 kf = *(const f32x4 *)(Ks[buf] + q * HD + 4 * ((2 * i + hi) ^ (q & 15)));
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[e], qf[i][e], s[0], 0, 0, 0);
        }
        const bool masked =
            kt + KB - 1 > t.p0 || kt < t.w_lo || (a.window > 0 && kt < t.p1 - a.window + 1) || okc != 3;
        bool moved;
        const float corr = chunk_softmax<float>(t, s, score_factor(a.scale_log2), masked, kt, okc, m, l, moved);
        if (moved) {
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= corr;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const vdim v = *(const vdim *)(Vs[buf] + (8 * (r >> 2) + 4 * hi + (r & 3)) * HD + DT * q);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[d], s[0][r], o[d], 0, 0, 0);
        }
        if (!chunk_edge(a, t, kt, KB) && okc == 3) continue;
        for (uint64_t left = __ballot(lane < KB && odd[buf][lane % KB] == kt); left; left &= left - 1) {
            const int key = kt + __builtin_ctzll(left);
            const int page = a.b.table[t.seq * a.b.table_stride + (key >> a.pool.shift)];  // a good one: V was kept
            const float *v = (const float *)a.pool.v + page * a.pool.page_stride +
                             (key & ((1 << a.pool.shift) - 1)) * a.pool.token_stride + t.g * a.pool.head_stride;
            const bool sees = key <= t.pos && key >= t.first;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const vdim x = *(const vdim *)(v + DT * (8 * (r >> 2) + 4 * hi + (r & 3)));
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d][r] += sees ? not_finite(x[d]) : 0.0f;
                asm volatile("" ::: "memory");  // few values at a time: this must not cost registers
            }
        }
    }
    // Output register r of tile d is dim DT * (8 (r / 4) + 4 hi + r % 4) + d: DT rows of four
    // consecutive registers hold 4 DT consecutive dims, starting at 4 DT (2 (r / 4) + hi).
    l += __shfl_xor(l, 32);
    if (!t.live) return;
    const float inv = 1.0f / l;
    float *out = (float *)a.out + (int64_t)(t.start + t.row) * a.out_stride + t.head * HD;
    const int64_t at = ((int64_t)(t.start + t.row) * a.heads + t.head) * a.parts + t.split;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int d0 = DT * (8 * (r >> 2) + 4 * hi + (r & 3));
        vdim v;
#pragma unroll
        for (int d = 0; d < DT; ++d) v[d] = t.splits > 1 ? o[d][r] : m == -INFINITY ? 0.0f : o[d][r] * inv;
        *(vdim *)((t.splits > 1 ? a.part_o + at * HD : out) + d0) = v;
    }
    if (t.splits > 1 && hi == 0) {
        a.part_ml[2 * at] = m;
        a.part_ml[2 * at + 1] = l;
    }
}

}  // namespace

template <typename RT, typename CT>
int attn_chunk_launch(const AttnArgs &a, int hd, int splits, int tiles, hipStream_t st) {
    const unsigned blocks = (unsigned)tiles * (unsigned)splits * (unsigned)a.pool.kv_heads;
    constexpr int NW = kChunkWaves<RT, CT>;
    if constexpr (std::is_same<CT, float>::value) {
        if (hd == 128)
            hipLaunchKernelGGL((attn_chunk32_kernel<128, NW>), dim3(blocks), dim3(64 * NW), 0, st, a, tiles, splits);
        else
            hipLaunchKernelGGL((attn_chunk32_kernel<64, NW>), dim3(blocks), dim3(64 * NW), 0, st, a, tiles, splits);
    } else {
        if (hd == 128)
            hipLaunchKernelGGL((attn_chunk16_kernel<RT, CT, 128, NW>), dim3(blocks), dim3(64 * NW), 0, st, a, tiles,
                               splits);
        else
            hipLaunchKernelGGL((attn_chunk16_kernel<RT, CT, 64, NW>), dim3(blocks), dim3(64 * NW), 0, st, a, tiles,
                               splits);
    }
    return launch_status();
}

template int attn_chunk_launch<float, float>(const AttnArgs &, int, int, int, hipStream_t);
template int attn_chunk_launch<float, f16>(const AttnArgs &, int, int, int, hipStream_t);
template int attn_chunk_launch<float, bf16>(const AttnArgs &, int, int, int, hipStream_t);
template int attn_chunk_launch<f16, f16>(const AttnArgs &, int, int, int, hipStream_t);
template int attn_chunk_launch<bf16, bf16>(const AttnArgs &, int, int, int, hipStream_t);

}  // namespace gphq
