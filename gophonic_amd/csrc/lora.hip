// gphq_lora_add: low-rank adapters of many requests beside one shared projection,
//   y[r] += scale[s] * B[s] (A[s] x[r]),  s = row_slots[r],
// for the rows that have an adapter; A[s] is [rank][k], B[s] [n][rank].
//
// Two launches. The shrink makes t[r] = A[s] x[r] (rank values a row) over ranges of k,
// one partial sum each; the expand adds the partial sums in order, scales them and adds
// B[s] t[r] into y. Both work on tiles of 16 rows and pass over the tile once for every
// distinct adapter among its rows: rows of one request stand side by side, so a tile of a
// prompt has one, a tile of decode lanes at most 16. All products are fp32 on
// v_mfma_f32_16x16x4_f32 (16-bit weights widened, exactly).
#include "paged.h"

namespace gphq {
namespace {

constexpr int kLoraRows = 16;

struct LoraArgs {
    const void *a, *b;
    const int32_t *ranks, *row_slots;
    const float *scales, *x;
    float *y, *t;  // t: [splits][rows][max_rank]
    int64_t x_stride, y_stride;
    int slots, max_rank, rows, k, n;
    int splits, k_split;  // ranges of k, and the k of each (a multiple of 128)
    int passes;           // blocks that share a tile's distinct adapters
    int n_block;          // columns of y per block of the expand
    bool vec;             // y's rows may be read four values at a time
};

// The tile's rows: this lane's row (lane % 16) and its adapter (-1: none).
__device__ __forceinline__ int lora_slot(const LoraArgs &a, int r0) {
    const int r = r0 + (threadIdx.x & 15);
    const int s = r < a.rows ? a.row_slots[r] : -1;
    return s >= 0 && s < a.slots ? s : -1;
}

__device__ __forceinline__ int lora_rank(const LoraArgs &a, int s) {
    return a.ranks ? min(max(a.ranks[s], 0), a.max_rank) : a.max_rank;
}

// Runs f(slot) for the tile's distinct adapters number first, first + step, ...
template <typename F>
__device__ __forceinline__ void each_slot(int slot, int first, int step, F &&f) {
    unsigned long long left = __ballot(slot >= 0) & 0xFFFF;
    for (int i = 0; left; ++i) {
        const int s = __builtin_amdgcn_readlane(slot, __builtin_ctzll(left));
        left &= ~__ballot(slot == s);
        if (i % step == first) f(s);
    }
}

template <typename W>
__device__ __forceinline__ void load8(const W *p, float (&v)[8]) {
    float lo[4], hi[4];
    load_vec(p, lo);
    load_vec(p + 4, hi);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
}

// t[split][r][0 .. max_rank) of a tile's rows, over k of one split: D (16 ranks x 16 rows)
// = A . X^T per 16 ranks. The four wavefronts take every fourth 32 k and are added in order.
template <typename W, int RT>
__global__ __launch_bounds__(256) void lora_shrink_kernel(const LoraArgs a) {
    __shared__ f32x4 sum[4][RT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    int u = blockIdx.x;
    const int pass = u % a.passes;
    u /= a.passes;
    const int split = u % a.splits, r0 = u / a.splits * kLoraRows;
    const int slot = lora_slot(a, r0);
    const float *x = a.x + (int64_t)min(r0 + c, a.rows - 1) * a.x_stride;
    const int k0 = split * a.k_split, k1 = min(k0 + a.k_split, a.k);
    each_slot(slot, pass, a.passes, [&](int s) {
        const int rank = lora_rank(a, s);
        f32x4 acc[RT];
#pragma unroll
        for (int i = 0; i < RT; ++i) acc[i] = f32x4{};
        const W *w = (const W *)a.a + (int64_t)s * a.max_rank * a.k;
        for (int k = k0 + 32 * wave; k < k1; k += 128) {
            float xv[8];
            load8(x + k + 8 * g, xv);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                if (16 * i >= rank) break;
                float wv[8];
                load8(w + (int64_t)min(16 * i + c, rank - 1) * a.k + k + 8 * g, wv);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[e], xv[e], acc[i], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) sum[wave][i][lane] = acc[i];
        __syncthreads();
        // Lane (c, g) of tile i holds ranks 16 i + 4 g .. + 3 of row r0 + c.
        for (int i = wave; 16 * i < a.max_rank; i += 4) {
            f32x4 v = ((sum[0][i][lane] + sum[1][i][lane]) + sum[2][i][lane]) + sum[3][i][lane];
            const int r = 16 * i + 4 * g;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (r + e >= rank) v[e] = 0.0f;
            if (slot == s && r < a.max_rank)
                *(f32x4 *)(a.t + ((int64_t)split * a.rows + r0 + c) * a.max_rank + r) = v;
        }
        __syncthreads();
    });
}

// y[r][n0 .. n0 + n_block) += scale * B t[r] of a tile's rows: D (16 rows x 16 columns) =
// T . B^T, four column tiles at once, tile j holding columns 4 i + j, so that a lane has
// four neighbouring columns of y.
template <typename W>
__global__ __launch_bounds__(256) void lora_expand_kernel(const LoraArgs a) {
    extern __shared__ float ts[];  // [16][max_rank + 4]: the tile's t, summed and scaled
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int nb = (a.n + a.n_block - 1) / a.n_block;
    const int r0 = blockIdx.x / nb * kLoraRows, n0 = blockIdx.x % nb * a.n_block, n1 = min(n0 + a.n_block, a.n);
    const int slot = lora_slot(a, r0);
    if (!__any(slot >= 0)) return;
    const int ld = a.max_rank + 4;
    for (int i = threadIdx.x; i < kLoraRows * a.max_rank / 4; i += 256) {
        const int r = i / (a.max_rank / 4), e = i % (a.max_rank / 4) * 4;
        const int s = r0 + r < a.rows ? a.row_slots[r0 + r] : -1;
        f32x4 v{};
        if (s >= 0 && s < a.slots) {
            for (int p = 0; p < a.splits; ++p)
                v += *(const f32x4 *)(a.t + ((int64_t)p * a.rows + r0 + r) * a.max_rank + e);
            if (a.scales) v *= a.scales[s];
        }
        *(f32x4 *)(ts + r * ld + e) = v;
    }
    __syncthreads();
    for (int n = n0 + 64 * wave; n < n1; n += 256) {
        each_slot(slot, 0, 1, [&](int s) {
            const int rank = lora_rank(a, s);
            f32x4 acc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = f32x4{};
            const W *w = (const W *)a.b + (int64_t)s * a.n * a.max_rank;
            for (int r = 0; r < rank; r += 32) {
                float tv[8], wv[4][8];
                const bool in = r + 8 * g < a.max_rank;
                const int rr = in ? r + 8 * g : 0;
                load8(ts + c * ld + rr, tv);
#pragma unroll
                for (int j = 0; j < 4; ++j) load8(w + (int64_t)min(n + 4 * c + j, a.n - 1) * a.max_rank + rr, wv[j]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool live = r + 8 * g + e < rank;  // past the rank, B may hold anything
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(live ? tv[e] : 0.0f, live ? wv[j][e] : 0.0f,
                                                                      acc[j], 0, 0, 0);
                }
            }
            // Lane (c, g) holds rows r0 + 4 g + i at columns n + 4 c .. + 3.
            const int at = n + 4 * c;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (__shfl(slot, 4 * g + i) != s) continue;
                float *y = a.y + (int64_t)(r0 + 4 * g + i) * a.y_stride + at;
                if (a.vec && at + 4 <= n1) {
                    f32x4 v = *(const f32x4 *)y;
                    v += f32x4{acc[0][i], acc[1][i], acc[2][i], acc[3][i]};
                    *(f32x4 *)y = v;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (at + j < n1) y[j] += acc[j][i];
                }
            }
        });
    }
}

// How a call of `rows` rows is cut.
void lora_plan(int64_t rows, int64_t k, int64_t n, LoraArgs &a) {
    const int64_t cus = device_cus(), tiles = (rows + kLoraRows - 1) / kLoraRows;
    const int64_t steps = (k + 127) / 128;
    const int64_t want = std::min<int64_t>(steps, std::max<int64_t>(1, 2 * cus / tiles));
    const int64_t per = (steps + want - 1) / want;
    a.k_split = (int)(per * 128);
    a.splits = (int)std::max<int64_t>(1, (steps + per - 1) / per);
    // Blocks of the expand: enough of them to fill the chip, no wider than 1024 columns.
    const int64_t blocks = std::max<int64_t>(1, 4 * cus / tiles);
    a.n_block = (int)std::min<int64_t>(1024, std::max<int64_t>(256, (n + blocks - 1) / blocks + 255) / 256 * 256);
}

template <typename W>
int lora_run(const LoraArgs &a, hipStream_t st) {
    const unsigned tiles = (unsigned)((a.rows + kLoraRows - 1) / kLoraRows);
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
    const unsigned nb = (unsigned)((a.n + a.n_block - 1) / a.n_block);
    hipLaunchKernelGGL((lora_expand_kernel<W>), dim3(tiles * nb), dim3(256), kLoraRows * (a.max_rank + 4) * 4, st, a);
    return launch_status();
}

}  // namespace
}  // namespace gphq

using namespace gphq;

extern "C" {

int64_t gphq_lora_workspace_bytes(int64_t rows, int64_t k, int64_t max_rank) {
    if (rows < 0 || rows > GPHQ_PAGED_MAX_ROWS || k < 0 || k > INT32_MAX || k % 32 || max_rank < 0 ||
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
    p.passes = rows <= 256 ? (int)std::min<int64_t>(std::min<int64_t>(slots, rows), kLoraRows) : 1;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == GPHQ_DTYPE_F32) return lora_run<float>(p, st);
    if (dtype == GPHQ_DTYPE_F16) return lora_run<f16>(p, st);
    return lora_run<bf16>(p, st);
}

}  // extern "C"
