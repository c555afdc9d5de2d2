// gphq_lora_add: low-rank adapters of many requests beside one shared projection,
//   y[r] += scale[s] * B[s] (A[s] x[r]),  s = row_slots[r],
// for the rows that have an adapter; A[s] is [rank][k], B[s] [n][rank].
//
// Two launches. The shrink makes t[r] = A[s] x[r] (rank values a row) over ranges of k, one
// partial sum each; the expand adds the partial sums in order, scales them and adds B[s] t[r]
// into y. Both work on tiles of rows (32; 16 in the expand of a call of up to 16) and pass over a tile once for every
// distinct adapter among its rows: rows of one request stand side by side, so a tile of a
// prompt mostly has one, a tile of decode lanes many.
//
// Products are to fp32 accuracy whatever the weights' type. 16-bit weights are multiplied on
// the bfloat16 matrix instructions: an fp32 value is exactly three bfloat16 pieces (8 of its
// 24 bits each), an FP16 weight two, a bfloat16 weight one; of the products of pieces only
// that of the two smallest (2^-24 of the whole) is left out. fp32 weights take
// v_mfma_f32_16x16x4_f32.
#include "paged.h"

namespace gphq {
namespace {

constexpr int kFewRows = 256;  // up to here a tile's adapters go to blocks of their own
constexpr int kShrinkRows = 32;  // two 16-row tiles share the weights' fragments

struct LoraArgs {
    const void *a, *b;
    const int32_t *ranks, *row_slots;
    const float *scales, *x;
    float *y, *t;  // t: [splits][rows][max_rank]
    int64_t x_stride, y_stride;
    int slots, max_rank, rows, k, n;
    int splits, k_split;  // ranges of k, and the k of each (a multiple of 128)
    int passes;           // blocks that share a tile's distinct adapters
    int n_block;          // columns of y per block of the expand (a multiple of 256)
    bool vec;             // y's rows may be read four values at a time
};

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Row r's adapter; -1: none.
__device__ __forceinline__ int lora_slot(const LoraArgs &a, int r) {
    const int s = r < a.rows ? a.row_slots[r] : -1;
    return s >= 0 && s < a.slots ? s : -1;
}

__device__ __forceinline__ int lora_rank(const LoraArgs &a, int s) {
    return a.ranks ? min(max(a.ranks[s], 0), a.max_rank) : a.max_rank;
}

// Runs f(slot, rows) for the distinct adapters of a tile, number first, first + step, ...:
// lane i holds row i's slot, rows has a bit for each row of that slot.
template <typename F>
__device__ __forceinline__ void each_slot(int slot, int first, int step, F &&f) {
    unsigned long long left = __ballot(slot >= 0);
    for (int i = 0; left; ++i) {
        const int s = __builtin_amdgcn_readlane(slot, __builtin_ctzll(left));
        const unsigned long long mine = __ballot(slot == s);
        left &= ~mine;
        if (i % step == first) f(s, mine);
    }
}

// Eight values as a fragment of the matrix instructions: fp32 as they are, bfloat16 in NP
// pieces, each the leading 8 bits of what those before it leave.
template <int NP>
struct Pieces {
    bf16x8 p[NP];
};
template <int NP>
__device__ __forceinline__ Pieces<NP> pieces_of(const float (&v)[8]) {
    Pieces<NP> out;
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
        i32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (int)__builtin_amdgcn_perm(__builtin_bit_cast(unsigned, r[2 * i + 1]),
                                              __builtin_bit_cast(unsigned, r[2 * i]), 0x07060302);
        out.p[k] = __builtin_bit_cast(bf16x8, w);
        if (k + 1 < NP) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                r[i] -= __builtin_bit_cast(float, __builtin_bit_cast(unsigned, r[i]) & 0xFFFF0000u);
        }
    }
    return out;
}

template <typename W>
__device__ __forceinline__ void load8(const W *p, float (&v)[8]) {
    typedef W vec __attribute__((ext_vector_type(sizeof(W) == 2 ? 8 : 4)));
    constexpr int N = sizeof(W) == 2 ? 8 : 4;
#pragma unroll
    for (int h = 0; h < 8 / N; ++h) {
        const vec x = *(const vec *)(p + N * h);
#pragma unroll
        for (int i = 0; i < N; ++i) v[N * h + i] = (float)x[i];
    }
}

// The fragment types of weights and of fp32 values beside them, and their product.
template <typename W>
struct Frag {  // 16-bit weights
    static constexpr int WP = std::is_same<W, f16>::value ? 2 : 1;
    typedef Pieces<WP> weight;
    typedef Pieces<3> value;
    static __device__ __forceinline__ weight weights(const float (&v)[8]) { return pieces_of<WP>(v); }
    static __device__ __forceinline__ value values(const float (&v)[8]) { return pieces_of<3>(v); }
};
template <>
struct Frag<float> {
    struct weight {
        float v[8];
    };
    typedef weight value;
    static __device__ __forceinline__ weight weights(const float (&v)[8]) {
        weight w;
#pragma unroll
        for (int i = 0; i < 8; ++i) w.v[i] = v[i];
        return w;
    }
    static __device__ __forceinline__ value values(const float (&v)[8]) { return weights(v); }
};
template <int NA, int NB>
__device__ __forceinline__ f32x4 product(const Pieces<NA> &a, const Pieces<NB> &b, f32x4 c) {
#pragma unroll
    for (int i = NA - 1; i >= 0; --i)
#pragma unroll
        for (int j = NB - 1; j >= 0; --j)
            if (i + j < 3) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x4 product(const Frag<float>::weight &a, const Frag<float>::weight &b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[e], b.v[e], c, 0, 0, 0);
    return c;
}

// t[split][r][0 .. max_rank) of a tile's rows, over k of one split: D (16 ranks x 16 rows)
// = A . X^T per 16 ranks and 16 rows. The four wavefronts take every fourth 32 k and are
// added in order. Bound by reading x and A in long calls (4814 rows of 4096, one adapter of rank 64: 25 us,
// 79 MB of x), by one wavefront's chain of loads in short ones, where k is cut into as many
// ranges as leave a block two steps (32 rows of eight adapters: 7 us).
template <typename W, int RT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(const LoraArgs a) {
    typedef Frag<W> F;
    __shared__ f32x4 sum[4][2][RT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    int u = blockIdx.x;
    const int pass = u % a.passes;
    u /= a.passes;
    const int split = u % a.splits, r0 = u / a.splits * kShrinkRows;
    const int slot = lane < kShrinkRows ? lora_slot(a, r0 + lane) : -1;
    const float *x[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) x[h] = a.x + (int64_t)min(r0 + 16 * h + c, a.rows - 1) * a.x_stride + 8 * g;
    const int k0 = split * a.k_split, k1 = min(k0 + a.k_split, a.k);
    each_slot(slot, pass, a.passes, [&](int s, unsigned long long mine) {
        const int rank = lora_rank(a, s);
        const bool use[2] = {(mine & 0xFFFF) != 0, (mine & 0xFFFF0000) != 0};
        f32x4 acc[2][RT];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[h][i] = f32x4{};
        const W *w[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i)
            w[i] = (const W *)a.a + ((int64_t)s * a.max_rank + min(16 * i + c, max(rank, 1) - 1)) * a.k + 8 * g;
        auto run = [&](auto both) __attribute__((always_inline)) {
            const int only = use[0] ? 0 : 1;
#pragma unroll 2
            for (int k = k0 + 32 * wave; k < k1; k += 128) {
                // Ranks past the last are the last again (and become 0 below), so no load waits for a test.
                float v0[8], v1[8], u[RT][8];
                load8(both ? x[0] + k : x[only] + k, v0);
                if (both) load8(x[1] + k, v1);
#pragma unroll
                for (int i = 0; i < RT; ++i) load8(w[i] + k, u[i]);
                const typename F::value x0 = F::values(v0), x1 = F::values(both ? v1 : v0);
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const typename F::weight wv = F::weights(u[i]);
                    acc[0][i] = product(wv, x0, acc[0][i]);
                    if (both) acc[1][i] = product(wv, x1, acc[1][i]);
                }
            }
            if (!both && only == 1) {
#pragma unroll
                for (int i = 0; i < RT; ++i) acc[1][i] = acc[0][i];
            }
        };
        if (use[0] && use[1])
            run(std::true_type{});
        else
            run(std::false_type{});
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < RT; ++i) sum[wave][h][i][lane] = acc[h][i];
        __syncthreads();
        // Lane (c, g) of tile (h, i) holds ranks 16 i + 4 g .. + 3 of row r0 + 16 h + c.
        for (int n = wave; n < 2 * RT; n += 4) {
            const int h = n / RT, i = n % RT, r = 16 * i + 4 * g;
            f32x4 v = ((sum[0][h][i][lane] + sum[1][h][i][lane]) + sum[2][h][i][lane]) + sum[3][h][i][lane];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r + e >= rank) v[e] = 0.0f;
            if (mine >> (16 * h + c) & 1 && r < a.max_rank)
                *(f32x4 *)(a.t + ((int64_t)split * a.rows + r0 + 16 * h + c) * a.max_rank + r) = v;
        }
        __syncthreads();
    });
}

// y[r][n0 .. n0 + n_block) += scale * B t[r] of the tile's 16 RH rows: D (16 rows x 16
// columns) = T . B^T, four column tiles at once, tile j holding columns 4 i + j, so that a
// lane has four neighbouring columns of y. Bound by reading and writing y in long calls (4814
// rows of 6144: 56 us, 237 MB), by the chain t, B, y in short ones (32 rows of eight adapters
// beside 24576 columns: 13 us). EARLY: y is read before the products, so that the
// two reads are on their way together, at the price of registers and so of wavefronts at once
// (4814 rows beside 6144 columns: 106 us, 125 without; 32 rows of eight adapters beside 24576
// columns, whose blocks have one adapter each and are many: 25 us, 21 without).
template <typename W, int RH, bool EARLY>
__global__ __launch_bounds__(256) void lora_expand_kernel(const LoraArgs a) {
    typedef Frag<W> F;
    extern __shared__ char lds[];  // T's fragments: [row tile][32 ranks][piece][lane], 16 bytes each
    constexpr int TP = sizeof(W) == 2 ? 3 : 2;
    i32x4 *ts = (i32x4 *)lds;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int nb = (a.n + a.n_block - 1) / a.n_block, chunks = (a.max_rank + 31) / 32;
    const int pass = blockIdx.x % a.passes, b = blockIdx.x / a.passes;
    const int r0 = b / nb * (16 * RH), n0 = b % nb * a.n_block, n1 = min(n0 + a.n_block, a.n);
    int slot = lane < 16 * RH ? lora_slot(a, r0 + lane) : -1;
    unsigned long long live = 0;  // the rows of this block's adapters
    each_slot(slot, pass, a.passes, [&](int, unsigned long long mine) { live |= mine; });
    if (!live) return;
    if (!(live >> lane & 1)) slot = -1;
    for (int u = wave; u < RH * chunks; u += 4) {
        const int h = u / chunks, r = u % chunks * 32 + 8 * g, row = r0 + 16 * h + c;
        const int s = __shfl(slot, 16 * h + c);
        float v[8] = {};
        if (s >= 0 && r < a.max_rank) {
            const float *t = a.t + (int64_t)row * a.max_rank + r;
            f32x4 lo{}, hi{};
#pragma unroll 8
            for (int p = 0; p < a.splits; ++p) {
                lo += *(const f32x4 *)(t + (int64_t)p * a.rows * a.max_rank);
                hi += *(const f32x4 *)(t + (int64_t)p * a.rows * a.max_rank + 4);
            }
            const float scale = a.scales ? a.scales[s] : 1.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = scale * lo[e], v[4 + e] = scale * hi[e];
        }
        const typename F::value f = F::values(v);
#pragma unroll
        for (int p = 0; p < TP; ++p) {
            if constexpr (sizeof(W) == 2)
                ts[(u * TP + p) * 64 + lane] = __builtin_bit_cast(i32x4, f.p[p]);
            else
                ts[(u * TP + p) * 64 + lane] = *(const i32x4 *)(f.v + 4 * p);
        }
    }
    __syncthreads();
    for (int n = n0 + 64 * wave; n < n1; n += 256) {
        const int at = n + 4 * c;  // lane (c, g) holds rows r0 + 16 h + 4 g + i at columns at .. at + 3
        each_slot(slot, 0, 1, [&](int s, unsigned long long mine) {
            const int rank = lora_rank(a, s);
            const W *w = (const W *)a.b + (int64_t)s * a.n * a.max_rank;
            f32x4 d[RH][4];
#pragma unroll
            for (int h = 0; h < RH; ++h)
#pragma unroll
                for (int j = 0; j < 4; ++j) d[h][j] = f32x4{};
            auto own = [&](int h, int i) { return (mine >> (16 * h + 4 * g + i) & 1) != 0; };
            auto y_of = [&](int h, int i) { return a.y + (int64_t)(r0 + 16 * h + 4 * g + i) * a.y_stride + at; };
            const bool whole = a.vec && at + 4 <= n1;
            f32x4 y[RH][4];
            auto load_y = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int h = 0; h < RH; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (!own(h, i)) continue;
                        if (whole)
                            y[h][i] = *(const f32x4 *)y_of(h, i);
                        else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) y[h][i][j] = at + j < n1 ? y_of(h, i)[j] : 0.0f;
                        }
                    }
            };
            if (EARLY) load_y();
#pragma unroll 2
            for (int r = 0; r < rank; r += 32) {
                typename F::weight wv[4];
                const int rr = min(r + 8 * g, a.max_rank - 8);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float v[8];
                    load8(w + (int64_t)min(n + 4 * c + j, a.n - 1) * a.max_rank + rr, v);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (r + 8 * g + e >= rank) v[e] = 0.0f;  // past the rank, B may hold anything
                    wv[j] = F::weights(v);
                }
#pragma unroll
                for (int h = 0; h < RH; ++h) {
                    if (!(mine >> (16 * h) & 0xFFFF)) continue;
                    typename F::value tv;
                    const i32x4 *t = ts + (h * chunks + r / 32) * TP * 64 + lane;
#pragma unroll
                    for (int p = 0; p < TP; ++p) {
                        if constexpr (sizeof(W) == 2)
                            tv.p[p] = __builtin_bit_cast(bf16x8, t[64 * p]);
                        else
                            *(i32x4 *)(tv.v + 4 * p) = t[64 * p];
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) d[h][j] = product(tv, wv[j], d[h][j]);
                }
            }
            if (!EARLY) load_y();
            // Rows of other adapters are left out here: a row has one adapter, so each is written once.
#pragma unroll
            for (int h = 0; h < RH; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (!own(h, i)) continue;
                    y[h][i] += f32x4{d[h][0][i], d[h][1][i], d[h][2][i], d[h][3][i]};
                    if (whole)
                        *(f32x4 *)y_of(h, i) = y[h][i];
                    else {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (at + j < n1) y_of(h, i)[j] = y[h][i][j];
                    }
                }
        });
    }
}

// Rows of a block of the expand.
int expand_rows(int64_t rows) { return rows <= 16 ? 16 : 32; }

// How a call of `rows` rows is cut.
void lora_plan(int64_t rows, int64_t k, int64_t n, LoraArgs &a) {
    const int64_t cus = device_cus(), tiles = (rows + kShrinkRows - 1) / kShrinkRows;
    const int64_t steps = (k + 127) / 128;  // a block's four wavefronts take 128 k a step
    const int64_t want = std::min<int64_t>((steps + 1) / 2, std::max<int64_t>(1, 2 * cus / tiles));
    const int64_t per = (steps + want - 1) / want;
    a.k_split = (int)(per * 128);
    a.splits = (int)std::max<int64_t>(1, (steps + per - 1) / per);
    // Blocks of the expand: enough of them to fill the chip, no wider than 1024 columns.
    const int64_t etiles = (rows + expand_rows(rows) - 1) / expand_rows(rows);
    const int64_t blocks = std::max<int64_t>(1, 4 * cus / etiles);
    a.n_block = (int)std::min<int64_t>(1024, std::max<int64_t>(256, ((n + blocks - 1) / blocks + 255) / 256 * 256));
}

template <typename W, int RH, bool EARLY>
int expand_launch(const LoraArgs &a, hipStream_t st) {
    const unsigned tiles = (unsigned)((a.rows + 16 * RH - 1) / (16 * RH)), nb = (unsigned)((a.n + a.n_block - 1) / a.n_block);
    const unsigned lds = (unsigned)(RH * ((a.max_rank + 31) / 32) * (sizeof(W) == 2 ? 3 : 2) * 1024);
    hipLaunchKernelGGL((lora_expand_kernel<W, RH, EARLY>), dim3(tiles * nb * (unsigned)a.passes), dim3(256), lds, st, a);
    return launch_status();
}

template <typename W>
int lora_run(const LoraArgs &a, hipStream_t st) {
    const unsigned tiles = (unsigned)((a.rows + kShrinkRows - 1) / kShrinkRows);
    const dim3 grid(tiles * (unsigned)a.splits * (unsigned)a.passes);
    if (a.max_rank <= 16)
        hipLaunchKernelGGL((lora_shrink_kernel<W, 1>), grid, dim3(256), 0, st, a);
    else if (a.max_rank <= 32)
        hipLaunchKernelGGL((lora_shrink_kernel<W, 2>), grid, dim3(256), 0, st, a);
    else if (a.max_rank <= 64)
        hipLaunchKernelGGL((lora_shrink_kernel<W, 4>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((lora_shrink_kernel<W, 8>), grid, dim3(256), 0, st, a);
    GPHQ_TRY(launch_status());
    const int rows = expand_rows(a.rows);
    if (rows == 16) return expand_launch<W, 1, false>(a, st);
    return a.rows <= kFewRows ? expand_launch<W, 2, false>(a, st) : expand_launch<W, 2, true>(a, st);
}

}  // namespace
}  // namespace gphq

using namespace gphq;

extern "C" {

int64_t gphq_lora_workspace_bytes(int64_t rows, int64_t k, int64_t max_rank) {
    if (rows < 0 || rows > GPHQ_PAGED_MAX_ROWS || k < 0 || k > 1 << 30 || k % 32 || max_rank < 0 ||
        max_rank > GPHQ_LORA_MAX_RANK || max_rank % 8)
        return GPHQ_ERR_DIMENSIONS;
    if (rows == 0 || k == 0) return 0;
    LoraArgs a{};
    lora_plan(rows, k, 1, a);
    return a.splits * rows * max_rank * 4;
}

int gphq_lora_add(int dtype, const void *a_dev, const void *b_dev, const int32_t *ranks, const float *scales,
                  int64_t slots, int64_t max_rank, const int32_t *row_slots, const float *x, int64_t x_stride,
                  float *y, int64_t y_stride, int64_t rows, int64_t k, int64_t n, void *work, int64_t work_bytes,
                  void *stream) {
    if (dtype != GPHQ_DTYPE_F32 && dtype != GPHQ_DTYPE_F16 && dtype != GPHQ_DTYPE_BF16) return GPHQ_ERR_UNSUPPORTED;
    const int64_t need = gphq_lora_workspace_bytes(rows, k, max_rank);
    if (need < 0) return (int)need;
    if (n < 0 || n > INT32_MAX - 1024 || slots < 0 || slots > INT32_MAX) return GPHQ_ERR_DIMENSIONS;
    if (x_stride < k || x_stride % 4 || y_stride < n) return GPHQ_ERR_DIMENSIONS;
    if (rows == 0 || n == 0 || k == 0 || slots == 0 || max_rank == 0) return GPHQ_OK;
    if (!a_dev || !b_dev || !row_slots || !x || !y || !work) return GPHQ_ERR_DIMENSIONS;
    if (((uintptr_t)a_dev | (uintptr_t)b_dev | (uintptr_t)x | (uintptr_t)work) % 16 ||
        ((uintptr_t)y | (uintptr_t)ranks | (uintptr_t)scales | (uintptr_t)row_slots) % 4)
        return GPHQ_ERR_DIMENSIONS;
    if (work_bytes < need) return GPHQ_ERR_DIMENSIONS;
    if (spans_overlap(x, span_bytes(rows, x_stride, k, 4), y, span_bytes(rows, y_stride, n, 4))) return GPHQ_ERR_OVERLAP;
    LoraArgs p{};
    p.a = a_dev;
    p.b = b_dev;
    p.ranks = ranks;
    p.row_slots = row_slots;
    p.scales = scales;
    p.x = x;
    p.y = y;
    p.t = (float *)work;
    p.x_stride = x_stride;
    p.y_stride = y_stride;
    p.slots = (int)slots;
    p.max_rank = (int)max_rank;
    p.rows = (int)rows;
    p.k = (int)k;
    p.n = (int)n;
    p.vec = y_stride % 4 == 0 && (uintptr_t)y % 16 == 0;
    lora_plan(rows, k, n, p);
    // Few tiles: the adapters of a tile go to blocks of their own.
    p.passes = rows <= kFewRows ? (int)std::min<int64_t>(std::min<int64_t>(slots, rows), 16) : 1;
    const int64_t tiles = (rows + 15) / 16, per = (n + p.n_block - 1) / p.n_block;
    if (tiles * std::max<int64_t>(per, p.splits) * p.passes > (1 << 24) - 1)  // blocks of 256, under 2^32 threads
        return GPHQ_ERR_DIMENSIONS;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GPHQ_DTYPE_F32) return lora_run<float>(p, st);
    if (dtype == GPHQ_DTYPE_F16) return lora_run<f16>(p, st);
    return lora_run<bf16>(p, st);
}

}  // extern "C"
