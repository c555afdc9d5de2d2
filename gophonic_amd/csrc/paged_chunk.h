// What the chunk kernels of paged attention share (paged_chunk.hip, paged8_chunk.hip): a block's
// tile of many query rows, and how a column is written.
#pragma once
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

}  // namespace
}  // namespace gphq
