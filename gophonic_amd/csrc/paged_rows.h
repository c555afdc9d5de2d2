// What the row kernels of paged attention share (paged_rows.hip, paged8_rows.hip): a block's tile
// of a few query rows, and the join of its four wavefronts.
#pragma once
#include "paged_attention.h"

namespace gphq {
namespace {

// One block's tile: 16 (or TM) columns of a sequence and KV head over the keys [k0, k1).
struct RowTile {
    int seq, g, n, len, start, r0, r1, splits, split;
    int lo, hi, k0, k1, p0, p1;  // p0, p1: positions of the tile's first and last row
    int c0;                      // the tile's first column
    // this lane's column
    int row, head, pos, first;
    bool live;
};

// Makes `col` this lane's column.
__device__ __forceinline__ void row_column(const AttnArgs &a, RowTile &t, int col) {
    t.live = col < t.n * a.group;
    t.row = t.live ? col / a.group : t.r1;
    t.head = t.g * a.group + (t.live ? col - t.row * a.group : 0);
    t.pos = t.len - t.n + t.row;
    t.first = a.window > 0 ? t.pos - a.window + 1 : 0;
}

// False where this block has nothing to do. BY_ROW: the grid has row_tiles tiles for every row (a
// kernel of its own: both ways in one took 110 us instead of 108 in a call by sequence of one FP16
// chunk and five single tokens over up to 6000 tokens).
template <bool BY_ROW, int TM = kSmallTile, int NT = 256>
__device__ __forceinline__ bool row_tile(const AttnArgs &a, int tiles, int splits, RowTile &t) {
    int u = blockIdx.x;
    t.g = u % a.pool.kv_heads;
    u /= a.pool.kv_heads;
    t.split = u % splits;
    u /= splits;
    int ct, end;
    if (BY_ROW) {
        // A row of group columns has up to row_tiles tiles of its own: n rows as many as their sequence
        // has, or more. The blocks share the check of all sequences, idle ones too.
        for (unsigned s = blockIdx.x * NT + threadIdx.x; s < (unsigned)a.b.seqs; s += gridDim.x * NT)
            if (!seq_ok(a.b, a.b.starts[s], a.b.starts[s + 1], a.b.lens[s])) paged_flag(a.b, PAGED_BAD_SEQ);
        const int row = u / a.row_tiles;
        const SeqRow s = find_seq(a.b, row);
        if (row < s.start || row >= s.end || !seq_ok(a.b, s.start, s.end, s.len)) return false;
        ct = (row - s.start) * a.row_tiles + u % a.row_tiles;
        t.seq = uniform(s.seq);
        t.start = s.start;
        end = s.end;
        t.len = s.len;
    } else {
        ct = u % tiles;
        t.seq = u / tiles;
        t.start = a.b.starts[t.seq];
        end = a.b.starts[t.seq + 1];
        t.len = a.b.lens[t.seq];
        if (!seq_ok(a.b, t.start, end, t.len)) {
            if (threadIdx.x == 0) paged_flag(a.b, PAGED_BAD_SEQ);
            return false;
        }
    }
    t.n = end - t.start;
    const int cols = t.n * a.group;
    if (cols > a.small_cols || ct * TM >= cols) return false;
    t.c0 = ct * TM;
    t.r0 = t.c0 / a.group;
    t.r1 = min((t.c0 + TM - 1) / a.group, t.n - 1);
    const TileKeys k = tile_keys(t.n, t.len, t.r0, t.r1, a.window);
    t.lo = k.lo;
    t.hi = k.hi;
    t.splits = tile_splits(k, a.split_small);
    if (t.split >= t.splits) return false;
    t.k0 = k.from + t.split * a.split_small;
    t.k1 = min(t.k0 + a.split_small, k.hi);
    t.p0 = t.len - t.n + t.r0;
    t.p1 = t.len - t.n + t.r1;
    row_column(a, t, t.c0 + (threadIdx.x & 15));
    return true;
}

// Joins the (m, l, o) of the NW wavefronts that have the same 16 columns, NS such sets of them in a
// block, and writes the columns' rows, or their split results. o[t][r] is column lane % 16, dim
// VD * (4 g4 + r) + t. All threads take part.
template <typename RT, int HD, int NW = 4, int NS = 1>
__device__ __forceinline__ void rows_finish(const AttnArgs &a, const RowTile &t, float m, float l,
                                            const f32x4 (&o)[HD / 16]) {
    constexpr int VD = HD / 16, LD = HD + 4;
    __shared__ float set_o[NS][NW][16][LD];
    __shared__ float set_m[NS][NW][16], set_l[NS][NW][16];
    const int set = NS == 1 ? 0 : threadIdx.x / (64 * NW), tid = NS == 1 ? threadIdx.x : threadIdx.x % (64 * NW);
    float(&so)[NW][16][LD] = set_o[set];
    float(&sm)[NW][16] = set_m[set], (&sl)[NW][16] = set_l[set];
    const int wave = tid >> 6, lane = threadIdx.x & 63, c = lane & 15, g4 = lane >> 4;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g4 == 0) {
        sm[wave][c] = m;
        sl[wave][c] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int v = 0; v < VD; v += 4)
            *(f32x4 *)&so[wave][c][VD * (4 * g4 + r) + v] =
                f32x4{o[v][r], o[v + 1][r], o[v + 2][r], o[v + 3][r]};
    // The column of thread i is i / 16: this lane's own numbers come from the lane holding it.
    const int col = tid >> 4 & 15, d = (tid & 15) * VD;
    const int from = col;  // lanes 0..15 of any wavefront hold columns 0..15
    const int row = __shfl(t.row, from), head = __shfl(t.head, from);
    const bool live = __shfl((int)t.live, from) != 0;
    __syncthreads();
    if (!live || (NW > 4 && tid >= 256)) return;
    float M = sm[0][col];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, sm[w][col]);
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f, v[VD];
#pragma unroll
    for (int i = 0; i < VD; ++i) v[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float e = __builtin_amdgcn_exp2f(sm[w][col] - ref);
        L += e * sl[w][col];
#pragma unroll
        for (int i = 0; i < VD; ++i) v[i] += e * so[w][col][d + i];
    }
    if (t.splits == 1) {
        const float inv = 1.0f / L;
        RT *out = (RT *)a.out + (int64_t)(t.start + row) * a.out_stride + head * HD + d;
#pragma unroll
        for (int i = 0; i < VD; i += 4) {
            float w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = M == -INFINITY ? 0.0f : v[i + k] * inv;
            store_vec(out + i, w);
        }
        return;
    }
    const int64_t at = (small_place(a, t.seq, t.start, row) * a.heads + head) * a.small_parts + t.split;
#pragma unroll
    for (int i = 0; i < VD; i += 4) *(f32x4 *)(a.small_o + at * HD + d + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    if (d == 0) {
        a.small_ml[2 * at] = M;
        a.small_ml[2 * at + 1] = L;
    }
}

}  // namespace
}  // namespace gphq
