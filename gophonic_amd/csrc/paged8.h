// The paged cache held in 8 bits: its device view, its codes, and the walk over its pages that
// the row and the chunk kernel of gphq_paged8_attention share (paged8_rows.hip,
// paged8_chunk.hip).
//
// A value is scale[block] * code, a block being 16 neighbouring tokens of one KV head in one
// page. Codes are taken into FP16, where every one of them is exact, and multiplied on the FP16
// matrix instructions; a block's scale of K multiplies its scores, its scale of V its
// probabilities, so neither is rounded beyond fp32.
#pragma once
#include "paged_attention.h"

namespace gphq {

constexpr int kBlockTokens = GPHQ_PAGED_BLOCK_TOKENS;

// Scale of block b of (page, head): page * page_stride + head * head_stride + b.
struct Paged8Scales {
    float *k, *v;
    int64_t page_stride, head_stride;
};

// Checks of a gphq_paged8_kv and a batch (paged_attention.hip).
int paged8_args(const gphq_paged8_kv *kv, const gphq_paged_batch *b, PagedPool &pool, Paged8Scales &scales,
                PagedBatch &batch);

struct Attn8Args {
    AttnArgs a;
    Paged8Scales s;
};

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef Half<f16>::vec8 f16x8;

// int8 codes -127 .. 127, whole: code c of a byte as FP16 1024 + (c + 128) by putting the byte
// under the exponent of 1024, less 1152.
struct CodesI8 {
    static constexpr float kTop = 127.0f, kOver = 127.5f;  // the largest code; what still rounds to it
    static constexpr int kExp = 0;                         // FP16 values are 2^-kExp of what they stand for
    // Once per dword of four codes, before pairs are taken out of it.
    static __device__ __forceinline__ int ready(int w) { return w ^ (int)0x80808080; }
    // Codes at byte B of `lo` and byte B of `hi`; bytes B and B + 1 of one dword.
    template <int B>
    static __device__ __forceinline__ int across(int hi, int lo) {
        return offset(__builtin_amdgcn_perm(hi, lo, 0x0C000C00 | B | (4 + B) << 16) | 0x64006400);
    }
    template <int B>
    static __device__ __forceinline__ int along(int w) {
        return offset(__builtin_amdgcn_perm(0x64646464, w, 0x04000400 | B | (B + 1) << 16));
    }
    static __device__ __forceinline__ int offset(int x) {
        const f16x2 v = __builtin_bit_cast(f16x2, x) - f16x2{(f16)1152.0f, (f16)1152.0f};
        return __builtin_bit_cast(int, v);
    }
};

// e4m3 codes: the seven bits under the sign, one to the right, are the FP16 number 2^-8 times
// the value, those below its normal range too. The two codes that stand for no number, which
// append never writes, read as 480 and -480.
struct CodesE4M3 {
    static constexpr float kTop = 448.0f, kOver = 464.0f;
    static constexpr int kExp = 8;
    static __device__ __forceinline__ int ready(int w) { return w; }
    template <int B>
    static __device__ __forceinline__ int across(int hi, int lo) {
        return half(__builtin_amdgcn_perm(hi, lo, 0x000C000C | B << 8 | (4 + B) << 24));
    }
    template <int B>
    static __device__ __forceinline__ int along(int w) {
        return half(__builtin_amdgcn_perm(0, w, 0x000C000C | B << 8 | (B + 1) << 24));
    }
    // Codes in the upper bytes of both halves: shifted right with their sign, whose second copy is taken out.
    static __device__ __forceinline__ int half(int x) {
        typedef short s16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(int, __builtin_bit_cast(s16x2, x) >> (short)1) & (int)0xBFFFBFFF;
    }
};

// Eight neighbouring codes (two ready dwords) as FP16.
template <typename C>
__device__ __forceinline__ f16x8 codes8(int w0, int w1) {
    const i32x4 x = {C::template along<0>(w0), C::template along<2>(w0), C::template along<0>(w1),
                     C::template along<2>(w1)};
    return __builtin_bit_cast(f16x8, x);
}

// Pieces of a query value x, its row brought into FP16's range by f16_scale (the largest in 2^13
// .. 2^14): of a 16-bit row x itself; of an fp32 row a multiple of 8, and the rest. The first
// pieces' products with int8 codes are whole multiples of 8 below 2^21, and sums of 128 of them
// exact (the matrix instructions cut off what lies 2^-25 below the largest term, which cost a
// row's output 8e-7 when each piece had 11 bits of its own and both went into one sum; the
// sums of the pieces are kept apart). FP32 rows keep 22 bits of the row's largest value.
template <int NP>
__device__ __forceinline__ void query_pieces(float x, f16 (&out)[NP]) {
    out[0] = NP == 1 ? (f16)x : (f16)(__builtin_rintf(x * 0.125f) * 8.0f);
    if constexpr (NP == 2) out[1] = (f16)(x - (float)out[0]);
}

// Pieces of a probability times its block's scale. The product is rounded to fp32 before anything
// else looks at it: left to itself the compiler makes the first piece from the unrounded product
// and the rest from the rounded one, and where a tie lies between them one FP16 step (2^-10 of the
// probability) is lost.
template <int NP>
__device__ __forceinline__ void weight_pieces(float p, float scale, f16 (&out)[NP]) {
    float w = p * scale;
    asm("" : "+v"(w));
    split_pieces(w, out);
}

// As PageWalk, for codes and scales: lane i of a wavefront holds the page of entry first + i of
// the sequence's table; an entry that names no page of the pool is flagged and becomes page 0,
// its keys bad.
struct Page8Walk {
    int first, lo_entry, hi_entry, page;
    uint64_t bad;
};

__device__ __forceinline__ void pages8_fill(const AttnArgs &a, Page8Walk &w, int seq, int first) {
    const int lane = threadIdx.x & 63;
    w.first = first;
    const int e = min(max(first + lane, w.lo_entry), w.hi_entry);
    w.page = a.b.table[seq * a.b.table_stride + e];
    const bool bad = w.page < 0 || w.page >= a.pool.pages;
    if (bad) {
        paged_flag(a.b, PAGED_BAD_PAGE);
        w.page = 0;
    }
    w.bad = __ballot(bad);
}

__device__ __forceinline__ void pages8_start(const AttnArgs &a, Page8Walk &w, int seq, int lo, int hi, int kt) {
    w.lo_entry = lo >> a.pool.shift;
    w.hi_entry = (hi - 1) >> a.pool.shift;
    pages8_fill(a, w, seq, kt >> a.pool.shift);
}

// Offsets of the codes (bytes) and the scales (floats) of the blocks kt, kt + 16, ... of a step,
// for KV head g; a bit per block that is not bad.
template <int N>
__device__ __forceinline__ unsigned pages8_step(const Attn8Args &e, Page8Walk &w, int seq, int g, int kt,
                                                int64_t (&at)[N], int64_t (&sat)[N]) {
    const AttnArgs &a = e.a;
    const int shift = a.pool.shift, mask = (1 << shift) - 1, ts = (int)a.pool.token_stride;
    if (((kt + 16 * N - 1) >> shift) - w.first >= 64) pages8_fill(a, w, seq, kt >> shift);
    auto get = [&](int key, int i) {
        const int n = (key >> shift) - w.first, page = __builtin_amdgcn_readlane(w.page, n), in = key & mask;
        at[i] = (int64_t)page * a.pool.page_stride + g * a.pool.head_stride + (int64_t)(in * ts);
        sat[i] = (int64_t)page * e.s.page_stride + g * e.s.head_stride + in / kBlockTokens;
        return (unsigned)(~w.bad >> n & 1);
    };
    if (16 * N <= mask + 1) {  // steps of 16 N keys start at multiples of 16 N: one page
        const unsigned ok = get(kt, 0);
#pragma unroll
        for (int i = 1; i < N; ++i) {
            at[i] = at[0] + (int64_t)i * 16 * ts;
            sat[i] = sat[0] + i;
        }
        return ok ? (1u << N) - 1 : 0;
    }
    unsigned ok = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) ok |= get(kt + 16 * i, i) << i;
    return ok;
}

// Memory from p on, for loads whose places are a lane's 32-bit offset and a wavefront's.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, 0x7FFFFFFF, 0x00020000);
}

// Lane l's place among a step's N scales: block l % N's.
template <int N>
__device__ __forceinline__ int64_t lane_scale(const int64_t (&sat)[N]) {
    const int b = threadIdx.x & (N - 1);
    int64_t at = sat[0];
#pragma unroll
    for (int i = 1; i < N; ++i) at = b == i ? sat[i] : at;
    return at;
}
// log2 of a block's scale of V in units of 2^ve, by which the exponents of its probabilities are
// raised: 2^-60 for less (a scale of 0 among them), where FP16 probabilities become 0 and their
// fp32 sum, taken back by 2^-log, still counts them.
__device__ __forceinline__ float scale_log(float s, int ve) {
    const float l = __builtin_amdgcn_logf(__builtin_amdgcn_ldexpf(s, -ve));
    return l < -60.0f ? -60.0f : l;  // (not a maximum: a scale that is not a number stays one)
}

// What lane i holds, wavefront-uniform.
__device__ __forceinline__ float lane_value(float v, int i) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i));
}

// A scale at a wavefront-uniform place, by the scalar unit (nothing writes scales while attention reads them).
__device__ __forceinline__ float uniform_scale(const float *p, int64_t at) {
    return *(const __attribute__((address_space(4))) float *)(uintptr_t)(p + at);
}

// The exponent e of a scale, 2^e above it: -149 for 0 and what is not a number.
__device__ __forceinline__ int scale_exp(float s) { return s > 0.0f ? __builtin_amdgcn_frexp_expf(s) : -149; }

// Sums of probabilities times codes are kept in units of 2^ve, ve the largest exponent among the
// scales of the blocks that the column has seen, so that FP16 probabilities times scale / 2^ve
// stay below 2^15; none is seen before kNoExp. What leaves the kernel has probabilities of at most 1.
constexpr int kNoExp = -1000;
constexpr int kDrop = 15;

// Largest of a column's values, which lie in the four lanes lane % 16 + 16 i of a wavefront: rows
// of 16 lanes, then halves, exchanged between two registers (the waits are those that the exchange
// needs behind a vector instruction's result).
__device__ __forceinline__ float column_max(float v) {
    float w = v;
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(v), "+v"(w));
    w = v = fmaxf(v, w);
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(v), "+v"(w));
    return fmaxf(v, w);
}

template <typename RT, typename C>
int attn8_rows_launch(const Attn8Args &a, int hd, int splits, int tiles, hipStream_t st);
template <typename RT, typename C>
int attn8_chunk_launch(const Attn8Args &a, int hd, int splits, int tiles, hipStream_t st);

}  // namespace gphq
