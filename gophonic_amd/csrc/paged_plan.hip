// gphq_paged_plan: a step's pages, row starts and slots from the requests' lengths.
//
// With T tokens a page, of every sequence
//   need = ceil((held + count) / T)
//   gives = entries max(need, min(shared, taken)) .. taken - 1, wants = need - taken
// and of all sequences, in order, the prefix sums of gives and wants: a given page goes to place
// free_count + (gives before it), a wanted one comes from place total - 1 - (wants before it) of
// the list, total = free_count + all gives. starts are the prefix sums of count over the
// sequences whose pages are there.
#include "paged.h"

namespace gphq {
namespace {

constexpr int kPlanFew = 256, kPlanMany = 1024;  // threads of the block, for up to as many sequences and for more

struct PlanArgs {
    const int32_t *held, *count, *taken, *shared, *free_count;
    int32_t *table, *free, *starts, *lens, *taken_out, *free_count_out, *positions, *sequences, *bad;
    int64_t *slots;
    int64_t table_stride, free_len;
    int seqs, rows, max_rows, max_len, shift;
};

__device__ __forceinline__ void plan_flag(const PlanArgs &a, int bit) {
    if (a.bad) atomicOr(a.bad, bit);
}

// Sum over the threads before this one, and over all, of a block of 64 NW.
template <int NW>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t &total, int64_t (&lds)[NW]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t sum = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t lo = __shfl_up((int)(uint32_t)sum, d), hi = __shfl_up((int)(sum >> 32), d);
        if (lane >= d) sum += (int64_t)((uint64_t)hi << 32 | lo);
    }
    __syncthreads();  // lds of the last scan has been read
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < NW; ++w) {
        before += w < wave ? lds[w] : 0;
        total += lds[w];
    }
    return before + sum - v;
}

struct Request {
    int held, count, need, keep, taken;  // keep: entries that stay or are taken
    bool ok;
};

__device__ __forceinline__ Request request(const PlanArgs &a, int s) {
    Request r{0, 0, 0, 0, 0, true};
    if (s >= a.seqs) return r;
    r.held = a.held[s];
    r.count = a.count[s];
    r.taken = a.taken[s];
    const int shared = a.shared ? a.shared[s] : 0;
    r.ok = r.held >= 0 && r.count >= 0 && r.count <= a.max_rows && r.taken >= 0 && r.taken <= a.table_stride &&
           shared >= 0 && r.held <= a.max_len - r.count;
    if (!r.ok) {
        r.count = 0;
        r.need = r.keep = r.taken;
        return r;
    }
    r.need = (int)(((int64_t)r.held + r.count + (1 << a.shift) - 1) >> a.shift);
    r.keep = max(r.need, min(shared, r.taken));
    return r;
}

// The last thread whose first place, of `first` (ascending), is at most k.
template <int NT>
__device__ __forceinline__ int owner(const int64_t (&first)[NT], int64_t k) {
    int at = 0;
#pragma unroll
    for (int d = NT / 2; d > 0; d /= 2)
        if (first[at + d] <= k) at += d;
    return at;
}

// Positions, sequences and slots of 64 rows from row0 on, by one wavefront: the sequence of the
// first by ballots, of the others by where they lie among the next 64 starts.
__device__ __forceinline__ void map_rows(const PlanArgs &a, int row0) {
    const int lane = threadIdx.x & 63, row = row0 + lane;
    int lo = 0, cnt = a.seqs + 1;  // starts[seqs] is where the rows of none begin
    while (cnt > 64) {
        const int step = (cnt + 63) / 64;
        const int i = min(lane * step, cnt - 1);
        const int at = last_lane(__ballot(lane * step < cnt && a.starts[lo + i] <= row0)) * step;
        lo += at;
        cnt = min(step, cnt - at);
    }
    lo += last_lane(__ballot(lane < cnt && a.starts[lo + min(lane, cnt - 1)] <= row0));
    int seq = lo;
    for (int base = lo + 1; base <= a.seqs; base += 64) {
        const int start = base + lane <= a.seqs ? a.starts[base + lane] : INT32_MAX;
        int n = 0;
#pragma unroll
        for (int d = 32; d > 0; d /= 2)
            if (__shfl(start, n + d - 1) <= row) n += d;
        const int last = __builtin_amdgcn_readlane(start, 63);
        seq += n + (n == 63 && last <= row ? 1 : 0);
        if (last > row0 + 63) break;
    }
    if (row >= a.rows) return;
    const bool live = seq < a.seqs;
    int pos = -1;
    int64_t slot = -1;
    if (live) {
        pos = a.lens[seq] - (a.starts[seq + 1] - row);
        slot = ((int64_t)a.table[seq * a.table_stride + (pos >> a.shift)] << a.shift) + (pos & ((1 << a.shift) - 1));
    }
    if (a.positions) a.positions[row] = pos;
    if (a.sequences) a.sequences[row] = live ? seq : -1;
    if (a.slots) a.slots[row] = slot;
}

// One block: the prefix sums run over all sequences, NT at a time, and the pages of those are
// moved by all threads, each finding the sequence of its page in the sums. With MAP it also maps
// the rows. All latency, a chain of loads, sums and barriers: 32 requests 4.5 us (8.4 with 1024
// threads and a sum for each case that may come), 1000 requests 9.0, and 3.3 for the rows in a grid of
// their own.
template <bool MAP, int NT>
__global__ __launch_bounds__(NT) void paged_plan_kernel(const PlanArgs a) {
    __shared__ int64_t lds[NT / 64];
    __shared__ int64_t first[NT];
    __shared__ int entry[NT];
    const int tid = threadIdx.x;
    int64_t have = *a.free_count;
    if (have < 0 || have > a.free_len) {
        if (tid == 0) plan_flag(a, PAGED_BAD_PAGE);
        have = have < 0 ? 0 : a.free_len;
    }
    Request r{};
    for (int s0 = 0; s0 < a.seqs; s0 += NT) {
        r = request(a, s0 + tid);
        int64_t total;
        const int64_t gives = max(r.taken - r.keep, 0), at = block_scan(gives, total, lds);
        if (total) {
            first[tid] = at;
            entry[tid] = r.keep;
            __syncthreads();
            const int64_t fit = min(total, a.free_len - have);
            if (fit < total && tid == 0) plan_flag(a, PAGED_BAD_PAGE);
            for (int64_t k = tid; k < fit; k += NT) {
                const int i = owner(first, k);
                a.free[have + k] = a.table[(s0 + i) * a.table_stride + entry[i] + (k - first[i])];
            }
            have += fit;
            __syncthreads();
        }
    }
    int64_t wanted = 0, used = 0, row_sum = 0, rows = 0;
    for (int s0 = 0; s0 < a.seqs; s0 += NT) {
        const int s = s0 + tid;
        const bool mine = s < a.seqs;
        if (a.seqs > NT) r = request(a, s);
        int64_t total;
        const int64_t wants = max(r.need - r.taken, 0), at = block_scan(wants, total, lds);
        const bool served = wants == 0 || wanted + at + wants <= have;
        first[tid] = at;
        entry[tid] = r.taken;
        __syncthreads();
        // Those served are the first with wants: the pages taken are the first of all wanted.
        int64_t got = total;
        if (wanted + total > have) block_scan(served ? wants : 0, got, lds);
        for (int64_t k = tid; k < got; k += NT) {
            const int i = owner(first, k);
            a.table[(s0 + i) * a.table_stride + entry[i] + (k - first[i])] = a.free[have - 1 - wanted - k];
        }
        used += got;
        wanted += total;
        __syncthreads();  // first and entry have been read
        int count = served ? r.count : 0;
        int64_t brought;
        const int64_t row_before = block_scan(count, brought, lds), row_at = row_sum + row_before;
        row_sum += brought;
        const bool fits = !count || row_at + count <= a.rows;
        if (mine) {
            if (!r.ok || !fits) plan_flag(a, PAGED_BAD_SEQ);
            if (!served) plan_flag(a, PAGED_NO_PAGES);
        }
        count = fits ? count : 0;
        int64_t start = rows + row_before;
        if (row_sum > a.rows) start = rows + block_scan(count, brought, lds);  // some do not
        rows += brought;
        if (mine) {
            a.starts[s + 1] = (int)(start + count);
            a.lens[s] = r.held + count;
            a.taken_out[s] = served ? r.keep : r.taken;
        }
    }
    if (tid == 0) {
        a.starts[0] = 0;
        *a.free_count_out = (int)(have - used);
    }
    if (MAP) {
        __syncthreads();  // starts, lens and tables are written
        for (int row0 = tid & ~63; row0 < a.rows; row0 += NT) map_rows(a, row0);
    }
}

__global__ __launch_bounds__(256) void paged_map_kernel(const PlanArgs a) {
    const int row0 = (int)(blockIdx.x * 256 + (threadIdx.x & ~63));
    if (row0 < a.rows) map_rows(a, row0);
}

}  // namespace
}  // namespace gphq

using namespace gphq;

extern "C" int gphq_paged_plan(const gphq_paged_requests *r, void *stream) {
    if (!r) return GPHQ_ERR_PAGED_SHAPE;
    if (r->page_tokens < 16 || r->page_tokens > GPHQ_PAGED_MAX_PAGE_TOKENS || (r->page_tokens & (r->page_tokens - 1)))
        return GPHQ_ERR_UNSUPPORTED;
    if (r->seqs < 0 || r->seqs > GPHQ_PAGED_MAX_SEQS || r->rows < 0 || r->rows > GPHQ_PAGED_MAX_ROWS ||
        r->max_rows < 0 || r->max_len < 0 || r->max_len > GPHQ_PAGED_MAX_LEN || r->free_len < 0 ||
        r->free_len > INT32_MAX || r->table_stride < 0 || r->table_stride > INT32_MAX ||
        r->table_stride < (r->max_len + r->page_tokens - 1) / r->page_tokens)
        return GPHQ_ERR_PAGED_SHAPE;
    if (!r->starts_dev || !r->free_count_dev || !r->free_count_out_dev || (r->free_len && !r->free_dev))
        return GPHQ_ERR_PAGED_SHAPE;
    if (r->seqs && (!r->held_dev || !r->count_dev || !r->taken_dev || !r->lens_dev || !r->taken_out_dev ||
                    (r->table_stride && !r->table_dev)))
        return GPHQ_ERR_PAGED_SHAPE;
    const uintptr_t bits = (uintptr_t)r->held_dev | (uintptr_t)r->count_dev | (uintptr_t)r->taken_dev |
                           (uintptr_t)r->shared_dev | (uintptr_t)r->table_dev | (uintptr_t)r->free_dev |
                           (uintptr_t)r->free_count_dev | (uintptr_t)r->starts_dev | (uintptr_t)r->lens_dev |
                           (uintptr_t)r->taken_out_dev | (uintptr_t)r->free_count_out_dev |
                           (uintptr_t)r->positions_dev | (uintptr_t)r->sequences_dev | (uintptr_t)r->bad_dev;
    if (bits % 4 || (uintptr_t)r->slots_dev % 8) return GPHQ_ERR_PAGED_SHAPE;
    PlanArgs a{};
    a.held = r->held_dev;
    a.count = r->count_dev;
    a.taken = r->taken_dev;
    a.shared = r->shared_dev;
    a.free_count = r->free_count_dev;
    a.table = r->table_dev;
    a.free = r->free_dev;
    a.starts = r->starts_dev;
    a.lens = r->lens_dev;
    a.taken_out = r->taken_out_dev;
    a.free_count_out = r->free_count_out_dev;
    a.positions = r->positions_dev;
    a.sequences = r->sequences_dev;
    a.slots = r->slots_dev;
    a.bad = r->bad_dev;
    a.table_stride = r->table_stride;
    a.free_len = r->free_len;
    a.seqs = (int)r->seqs;
    a.rows = (int)r->rows;
    a.max_rows = (int)std::min<int64_t>(r->max_rows, INT32_MAX);
    a.max_len = (int)r->max_len;
    a.shift = __builtin_ctzll((uint64_t)r->page_tokens);
    hipStream_t st = (hipStream_t)stream;
    const bool map = a.rows && (a.positions || a.sequences || a.slots);
    // A few rows are mapped by the block itself, more by a grid of their own, whose launch costs less than
    // the passes over them: 32 sequences of 32 rows 7.0 us and 3.6 + 2.8, of 64 rows 10.3 and 3.8 + 3.2, 500 of
    // four 10.2 and 6.3 + 3.2, of one, 300, 8.1 and 6.2 + 2.6. Up to 256 sequences need 256 threads only: 256
    // of one row 5.1 us, with 1024 threads 7.8.
    const bool few = a.seqs <= kPlanFew, self = map && a.rows <= 1024;
    if (few && self)
        hipLaunchKernelGGL((paged_plan_kernel<true, kPlanFew>), dim3(1), dim3(kPlanFew), 0, st, a);
    else if (few)
        hipLaunchKernelGGL((paged_plan_kernel<false, kPlanFew>), dim3(1), dim3(kPlanFew), 0, st, a);
    else if (self)
        hipLaunchKernelGGL((paged_plan_kernel<true, kPlanMany>), dim3(1), dim3(kPlanMany), 0, st, a);
    else
        hipLaunchKernelGGL((paged_plan_kernel<false, kPlanMany>), dim3(1), dim3(kPlanMany), 0, st, a);
    GPHQ_TRY(launch_status());
    if (self) return GPHQ_OK;
    if (!map) return GPHQ_OK;
    hipLaunchKernelGGL(paged_map_kernel, dim3((unsigned)((a.rows + 255) / 256)), dim3(256), 0, st, a);
    return launch_status();
}
