// What the kernels of gphq_paged_attention share: the arguments, how a batch
// is cut into tiles and splits, and where split results go.
//
// The mathematics, per query row i of head h at position p: over the keys j its
// mask leaves (j <= p, and j > p - window where there is one),
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),  x_j = scale log2(e) q.k_j,
// one pass over the keys with a running reference m: x is exponentiated against
// m, and m moves to a larger x only when that passes it by more than 8, so most
// steps rescale nothing. Scores, sums and outputs are fp32.
//
// A query tile is TM columns of one sequence and one KV head: column c is query
// row c / group, query head KV head * group + c % group, so all heads that share
// the KV head, and rows behind one another, share one read of its keys. A tile's
// keys start at a multiple of 32 (tile_keys) and are cut every split_len keys;
// where that gives more than one piece, each writes its unnormalized output, its
// reference and its sum, and paged_join_kernel adds them in order.
#pragma once
#include "paged.h"

namespace gphq {

struct AttnArgs {
    PagedBatch b;
    PagedPool pool;
    const void *q;
    void *out;
    float *part_o;   // [row][head][parts][hd]
    float *part_ml;  // [row][head][parts][2]: reference, sum
    int64_t q_stride, out_stride;
    int heads, group, window;
    int parts;             // split slots per (row, head) in the workspace
    int small_cols;        // sequences of at most this many columns are the row kernel's
    int big_tile;          // columns of the chunk kernel's tiles
    float q_sign;          // the sign of scale (0 if scale is 0), applied to the queries
    int split_small, split_big;  // keys per split in each kernel, multiples of 128
    float scale_log2;      // |scale| log2(e) (1 if scale is 0): positive, so the largest score stays the largest
};

constexpr int kSmallTile = 16;
constexpr float kLag = 8.0f;    // the reference maximum may be passed by this much (in log2)
constexpr float kLift = 7.0f;   // exponentials are 2^(x - m + 7): at most 2^15, so that FP16
                                // probabilities keep 2^-24 of a 2^7 .. 2^15 maximum, not of 1

// The keys [lo, hi) that rows r0 .. r1 of a sequence of n rows and len keys see, and the
// 32-aligned key that its splits count from.
struct TileKeys {
    int lo, hi, from;
};
__device__ __forceinline__ TileKeys tile_keys(int n, int len, int r0, int r1, int window) {
    TileKeys t;
    t.hi = max(len - n + r1 + 1, 0);
    t.lo = window > 0 ? max(len - n + r0 - window + 1, 0) : 0;
    t.lo = min(t.lo, t.hi);
    t.from = t.lo & ~31;
    return t;
}
__device__ __forceinline__ int tile_splits(const TileKeys &t, int split_len) {
    return t.hi > t.lo ? (t.hi - t.from + split_len - 1) / split_len : 1;
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
// of its largest value.
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
