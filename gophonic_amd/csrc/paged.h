// The paged K/V cache's device view, shared by the append (paged_append.hip)
// and the attention (paged_rows.hip, paged_chunk.hip, paged_attention.hip).
#pragma once
#include "common.h"

namespace gphq {

// Bits a kernel sets in a batch's bad word.
enum { PAGED_BAD_SEQ = 1, PAGED_BAD_PAGE = 2, PAGED_BAD_POSITION = 4 };

typedef __bf16 bf16;
typedef _Float16 f16;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// gphq_paged_batch as the kernels take it.
struct PagedBatch {
    const int32_t *starts, *lens, *table;
    int32_t *bad;
    int64_t table_stride;
    int seqs, rows, max_rows, max_len;
};

// A pool's geometry: element (page, token, head, dim) of k and v is at
// page * page_stride + token * token_stride + head * head_stride + dim.
struct PagedPool {
    void *k, *v;
    int64_t page_stride, token_stride, head_stride;
    int pages, shift, kv_heads;  // 1 << shift tokens a page
};

// Argument checks of the two structs (paged_attention.hip); GPHQ_OK fills the
// device views.
int paged_args(const gphq_paged_kv *kv, const gphq_paged_batch *b, PagedPool &pool, PagedBatch &batch);

// Bytes from the first to the last of `rows` rows of `width` values, `stride` apart; whether two such runs meet.
inline uintptr_t span_bytes(int64_t rows, int64_t stride, int64_t width, int64_t size) {
    return (uintptr_t)(((rows - 1) * stride + width) * size);
}
inline bool spans_overlap(const void *a, uintptr_t na, const void *b, uintptr_t nb) {
    return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

// A wavefront-uniform value, told to the compiler.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ void paged_flag(const PagedBatch &b, int bit) {
    if (b.bad) atomicOr(b.bad, bit);
}

// What a sequence's three numbers must satisfy for its rows to be touched.
__device__ __forceinline__ bool seq_ok(const PagedBatch &b, int start, int end, int len) {
    return start >= 0 && end >= start && end <= b.rows && end - start <= b.max_rows && len >= 0 && len <= b.max_len;
}

struct SeqRow {
    int seq, start, end, len;
};

// The highest lane of a ballot (0 for none).
__device__ __forceinline__ int last_lane(unsigned long long m) { return m ? 63 - __builtin_clzll(m) : 0; }

// The sequence holding `row`: the last s with starts[s] <= row, by ballots of
// 64 starts at a time (one round trip up to 64 sequences, two up to 4096). All
// 64 lanes take part and all get the result. The caller checks it: with starts
// that do not ascend, or a row outside all sequences, it does not hold the row.
__device__ __forceinline__ SeqRow find_seq(const PagedBatch &b, int row) {
    const int lane = threadIdx.x & 63;
    int lo = 0, cnt = b.seqs;
    while (cnt > 64) {
        const int step = (cnt + 63) / 64;
        const int i = min(lane * step, cnt - 1);
        const int at = last_lane(__ballot(lane * step < cnt && b.starts[lo + i] <= row)) * step;
        lo += at;
        cnt = min(step, cnt - at);
    }
    const int i = lo + min(lane, cnt - 1);
    const int s0 = b.starts[i], s1 = b.starts[i + 1], len = b.lens[i];
    const int at = last_lane(__ballot(lane < cnt && s0 <= row));
    return SeqRow{lo + at, __builtin_amdgcn_readlane(s0, at), __builtin_amdgcn_readlane(s1, at),
                  __builtin_amdgcn_readlane(len, at)};
}

// N consecutive values of type T as floats; N * sizeof(T) bytes, aligned to them.
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T *p, float (&v)[N]) {
    typedef T vec __attribute__((ext_vector_type(N)));
    const vec x = *(const vec *)p;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)x[i];
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[N]) {
    typedef T vec __attribute__((ext_vector_type(N)));
    vec x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (T)v[i];
    *(vec *)p = x;
}

}  // namespace gphq
