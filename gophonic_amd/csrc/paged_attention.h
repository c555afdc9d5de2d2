// What the kernels of gphq_paged_attention share: the arguments, how a batch
// is cut into tiles and splits, and where split results go.
//
// The mathematics, per query row i of head h at position p: over the keys j its
// mask leaves (j <= p, and j > p - window where there is one),
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),  x_j = scale log2(e) q.k_j,
// one pass over the keys with a running reference m: x is exponentiated against
// m, and m moves to a larger x only when that passes it by more than 8, so most
// steps rescale nothing. Scores, sums and outputs are fp32. m is -inf until the row sees a key,
// then kLeast or more, whatever that key's score: a row whose m is -inf at the end has seen none
// and is 0, one that saw scores of -inf or NaN alone is 0 / 0 or NaN.
//
// A query tile is TM columns of one sequence and one KV head: column c is query
// row c / group, query head KV head * group + c % group, so all heads that share
// the KV head, and rows behind one another, share one read of its keys. A tile's
// keys start at a multiple of 64 (tile_keys) and are cut every split_len keys;
// where that gives more than one piece, each writes its unnormalized output, its
// reference and its sum, and paged_join_kernel adds them in order.
#pragma once
#include <float.h>

#include "paged.h"

namespace gphq {

struct AttnArgs {
    PagedBatch b;
    PagedPool pool;
    const void *q;
    void *out;
    // Split results, output and (reference, sum): the chunk kernel's by [row][head][parts], the
    // row kernel's, whose splits may be many, by [sequence][small_rows][head][small_parts], or by
    // [row][head][small_parts] (small_rows 0) where the batch has fewer rows than that has places.
    float *part_o, *part_ml, *small_o, *small_ml;
    int64_t q_stride, out_stride;
    int heads, group, window;
    int parts, small_parts, small_rows;
    int row_tiles;         // the row kernel's grid has this many tiles for every row; 0: all tiles for every sequence
    int small_cols;        // sequences of at most this many columns are the row kernel's
    int big_tile;          // columns of the chunk kernel's tiles
    float q_sign;          // the sign of scale (0 if scale is 0), applied to the queries
    int split_small, split_big;  // keys per split in each kernel, multiples of 128
    float scale_log2;      // |scale| log2(e) (1 if scale is 0): positive, so the largest score stays the largest
};

constexpr int kSmallTile = 16;
constexpr float kLag = 8.0f;  // the reference maximum may be passed by this much (in log2)
constexpr float kLeast = -FLT_MAX;  // the least reference of a row that has seen a key

// Exponentials are 2^(x - m + lift). FP16 probabilities reach 2^15, so that they keep 2^-24 of a
// 2^7 .. 2^15 maximum, not of 1 (and FP16 values, up to 2^16, stay far inside fp32). Elsewhere none
// passes 1: a sum over finite values leaves fp32's range only where that of their magnitudes,
// each times a probability of at most 1, does.
template <typename CT>
constexpr float kLift = std::is_same<CT, f16>::value ? 7.0f : -kLag;

// The keys [lo, hi) that rows r0 .. r1 of a sequence of n rows and len keys see, and the
// key, a multiple of 64, that its splits count from.
struct TileKeys {
    int lo, hi, from;
};
__device__ __forceinline__ TileKeys tile_keys(int n, int len, int r0, int r1, int window) {
    TileKeys t;
    t.hi = max(len - n + r1 + 1, 0);
    t.lo = window > 0 ? max(len - n + r0 - window + 1, 0) : 0;
    t.lo = min(t.lo, t.hi);
    t.from = t.lo & ~63;
    return t;
}
__device__ __forceinline__ int tile_splits(const TileKeys &t, int split_len) {
    return t.hi > t.lo ? (t.hi - t.from + split_len - 1) / split_len : 1;
}

// The place of row i of a sequence that starts at row `start` among the row kernel's split results.
__device__ __forceinline__ int64_t small_place(const AttnArgs &a, int seq, int start, int i) {
    return a.small_rows ? (int64_t)seq * a.small_rows + i : start + i;
}

// The pages of a tile's keys [lo, hi): lane i of a wavefront holds where entry first + i of
// the sequence's table lies, so that a step finds its pages without waiting for memory.
// Entries no row of the tile needs may be unset: numbers outside lo .. hi stand for the
// nearest that is needed. An entry that names no page of the pool is flagged and becomes
// page 0, which can be read; its keys are bad (a bit per lane) and are masked.
struct PageWalk {
    int first, lo_entry, hi_entry;
    uint64_t bad;
    int at_lo, at_hi;  // byte offset of the entry's page and KV head, in two halves
};

template <typename CT>
__device__ __forceinline__ void pages_fill(const AttnArgs &a, PageWalk &w, int seq, int g, int first) {
    const int lane = threadIdx.x & 63;
    w.first = first;
    const int e = min(max(first + lane, w.lo_entry), w.hi_entry);
    int page = a.b.table[seq * a.b.table_stride + e];
    const bool bad = page < 0 || page >= a.pool.pages;
    if (bad) {
        paged_flag(a.b, PAGED_BAD_PAGE);
        page = 0;
    }
    w.bad = __ballot(bad);
    const int64_t at = (page * a.pool.page_stride + g * a.pool.head_stride) * (int64_t)sizeof(CT);
    w.at_lo = (int)at;
    w.at_hi = (int)(at >> 32);
}

template <typename CT>
__device__ __forceinline__ void pages_start(const AttnArgs &a, PageWalk &w, int seq, int g, int lo, int hi, int kt) {
    w.lo_entry = lo >> a.pool.shift;
    w.hi_entry = (hi - 1) >> a.pool.shift;
    pages_fill<CT>(a, w, seq, g, kt >> a.pool.shift);
}

// Byte offsets of the 16-key groups kt, kt + 16, ... of a step; a bit per group that is not bad.
template <typename CT, int N>
__device__ __forceinline__ unsigned pages_step(const AttnArgs &a, PageWalk &w, int seq, int g, int kt,
                                               int64_t (&at)[N]) {
    const int shift = a.pool.shift, ts = (int)(a.pool.token_stride * sizeof(CT)), mask = (1 << shift) - 1;
    if (((kt + 16 * N - 1) >> shift) - w.first >= 64) pages_fill<CT>(a, w, seq, g, kt >> shift);
    auto get = [&](int key, bool &bad) {
        const int i = (key >> shift) - w.first;
        bad = w.bad >> i & 1;
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane(w.at_hi, i) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane(w.at_lo, i)) + (int64_t)((key & mask) * ts);
    };
    unsigned ok = 0;
    bool bad;
    if (16 * N <= mask + 1) {  // steps of 16 N keys start at multiples of 16 N: one page
        at[0] = get(kt, bad);
#pragma unroll
        for (int i = 1; i < N; ++i) at[i] = at[0] + (int64_t)i * 16 * ts;
        return bad ? 0 : (1u << N) - 1;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        at[i] = get(kt + 16 * i, bad);
        ok |= bad ? 0 : 1u << i;
    }
    return ok;
}

// One 16-byte-per-lane load straight to LDS, lane l's from base + off to lds + 16 l. Unlike
// lds_dma16 the compiler does not know of it, and so does not wait for it at the next LDS
// read, whatever that reads: the caller waits (vmcnt) and has a barrier before the data's use.
__device__ __forceinline__ void dma16(const char *base, unsigned off, void *lds) {
    const int at = uniform((int)(uintptr_t)(__attribute__((address_space(3))) void *)lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(base)
                 : "memory", "m0");
}

// A key that some rows of a tile see and others do not may hold values that are not finite,
// and a masked probability times one is NaN, not 0. So in a step with such keys V's values
// that are not finite are taken out of the products, and added to the columns that do see
// their key (a probability is positive) in a loop over the keys that have any.

// 16-bit types: conversion, matrix instructions, packed tests.
template <typename T>
struct Half;
template <>
struct Half<f16> {
    typedef f16 vec8 __attribute__((ext_vector_type(8)));
    static constexpr int kExp = 0x7C00;
    static __device__ __forceinline__ f32x4 mfma16(vec8 a, vec8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    typedef float f32x16 __attribute__((ext_vector_type(16)));
    static __device__ __forceinline__ f32x16 mfma32(vec8 a, vec8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Half<bf16> {
    typedef bf16 vec8 __attribute__((ext_vector_type(8)));
    static constexpr int kExp = 0x7F80;
    static __device__ __forceinline__ f32x4 mfma16(vec8 a, vec8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    typedef float f32x16 __attribute__((ext_vector_type(16)));
    static __device__ __forceinline__ f32x16 mfma32(vec8 a, vec8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

// Pieces of a 16-bit type that a value of the row type is split into for the matrix
// instructions: one where they are the same type; an fp32 value as two FP16 pieces
// (22 bits, the value scaled into FP16's range) or three bfloat16 ones (24 bits). Products
// of pieces with the cache's values are exact in fp32, so an fp32 row loses at most 2^-22
// of its largest value. Probabilities of fp32 rows are split alike.
template <typename RT, typename CT>
constexpr int kPieces = sizeof(RT) == 2 ? 1 : (std::is_same<CT, f16>::value ? 2 : 3);

template <typename CT, int NP>
__device__ __forceinline__ void split_pieces(float v, CT (&out)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        out[i] = (CT)v;
        v -= (float)out[i];
    }
}

// A positive factor of the scores that -inf times it stays -inf.
__device__ __forceinline__ float score_factor(float f) { return fmaxf(f, 0x1p-126f); }

// 2^e that brings a largest magnitude m into [2^13, 2^14) (1 for 0, Inf and NaN), with
// both it and its inverse normal.
__device__ __forceinline__ float f16_scale(float m, float &inverse) {
    const int e = m > 0.0f && m < INFINITY ? min(max(14 - __builtin_amdgcn_frexp_expf(m), -120), 120) : 0;
    inverse = __builtin_amdgcn_ldexpf(1.0f, -e);
    return __builtin_amdgcn_ldexpf(1.0f, e);
}

// A value that is not finite, 0 for one that is.
__device__ __forceinline__ float not_finite(float v) { return fabsf(v) < INFINITY ? 0.0f : v; }

// Of a packed pair, the halves with an all-ones exponent (Inf or NaN), as a mask.
template <typename T>
__device__ __forceinline__ int pair_not_finite(int x) {
    constexpr int e = Half<T>::kExp;
    return ((x & e) == e ? 0xFFFF : 0) | ((x & (e << 16)) == (e << 16) ? 0xFFFF0000 : 0);
}

// Wavefronts, of 32 columns each, in a block of the chunk kernel.
template <typename RT, typename CT>
constexpr int kChunkWaves = kPieces<RT, CT> > 1 ? 8 : 4;

template <typename RT, typename CT>
int attn_rows_launch(const AttnArgs &a, int hd, int splits, int tiles, hipStream_t st);
template <typename RT, typename CT>
int attn_chunk_launch(const AttnArgs &a, int hd, int splits, int tiles, hipStream_t st);

}  // namespace gphq
