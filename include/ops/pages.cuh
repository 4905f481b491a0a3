#pragma once

// ops::page_take, ops::page_give — block tables and slot maps of a paged cache,
// built on the GPU from the requests' lengths, so that a step's lengths need not
// come back to the host. The reference has no pages; the Llama runtime's
// BlockAllocator (runtime/kv_cache.cuh) hands them out on the host.
//
// Sequence b holds lens[b] tokens in the pages ceil(lens[b] / 16) at the head of
// its table row, and gets the rows row_start[b] .. row_start[b + 1] - 1. The free
// pages are a stack of *free_count block ids. With need[b] = ceil((lens[b] + n) /
// 16) - ceil(lens[b] / 16):
//   table[b][ceil(lens[b] / 16) + k] = free[count - 1 - (sum of need before b) - k]
//   positions[r] = lens[b] + r - row_start[b]
//   slots[r] = 16 * table[b][positions[r] / 16] + positions[r] % 16
// All or nothing: where pages are missing, or a sequence does not fit its table
// row, the status says so, nothing is taken and every slot is -1. Giving back is
// the same the other way round: the pages ceil(new / 16) .. ceil(old / 16) - 1 of
// each sequence go onto the stack, in order.
//
// Both are bound by latency: a launch, and in this design three dependent rounds of
// loads (counts, ids, the table) with barriers between them. One cluster does it all, since
// the sums over the sequences come before everything else: every CTA repeats them
// (they are short) and takes its share of the pages and rows, and a cluster
// barrier stands where a second launch would. So the count may be updated in
// place: it is written after every CTA has read it. Measured (kernel time, one B200):
// one token more for 32 sequences 3.3 us; 79,000 rows of 48 prompts 12.2; 32,000 pages
// of 512 sequences given back 8.6.

#include <cstdint>

#include "../core/cuda_utils.cuh"
#include "kv_quant.cuh"
#include "tree_attention_common.cuh"

namespace opworks {

// What a step asks for, and where the answers go (device pointers).
struct PageTake {
    const int *lens;       // [batch]
    const int *row_start;  // [batch + 1]
    int batch, rows;       // rows: room in positions and slots; those past the last sequence's get slot -1
    int *block_table;      // [batch][table_stride]
    int table_stride;
    const int *free_blocks; // null: the table has all pages already, only positions and slots are wanted
    const int *free_count;
    int *positions;  // [rows]
    int64_t *slots;  // [rows]
    int *free_left;  // may be free_count; unused where free_blocks is null
    int *status;     // 0; the number of pages missing; -1: a sequence is longer than its table row, or below zero
};

struct PageGive {
    const int *old_lens, *new_lens; // [batch]
    int batch;
    const int *block_table;
    int table_stride;
    int *free_blocks; // [capacity]
    int capacity;
    const int *free_count;
    int *free_left; // may be free_count
    int *status;    // 0; -1: a length below zero or longer than the table row, or a stack without room
};

namespace detail {

constexpr int kPageFew = 256, kPageMany = 1024; // threads of a CTA that is alone; of one of a cluster
constexpr int kPageStarts = 4096; // row starts that are kept in shared memory to be searched

__device__ __forceinline__ int64_t pages_of(int64_t tokens) { return (tokens + kKvPage - 1) / kKvPage; }

// The pages [first, first + n) of a table row that a sequence takes or gives;
// n = -1: its lengths are no good.
struct PageSpan {
    int first, n;
};
__device__ __forceinline__ PageSpan page_span(const PageTake &a, int b) {
    const int64_t len = a.lens[b], n = static_cast<int64_t>(a.row_start[b + 1]) - a.row_start[b];
    const int64_t have = pages_of(len), need = pages_of(len + n);
    if (len < 0 || n < 0 || need > a.table_stride || a.row_start[b] < 0 || a.row_start[b + 1] > a.rows)
        return {0, -1};
    return {static_cast<int>(have), a.free_blocks != nullptr ? static_cast<int>(need - have) : 0};
}
__device__ __forceinline__ PageSpan page_span(const PageGive &a, int b) {
    const int64_t from = pages_of(a.new_lens[b]), to = pages_of(a.old_lens[b]);
    if (a.new_lens[b] < 0 || a.old_lens[b] < 0 || to > a.table_stride)
        return {0, -1};
    return {static_cast<int>(from < to ? from : to), static_cast<int>(to > from ? to - from : 0)};
}

// Sum over the block, known to all threads. `room`: a number for each warp.
template <int kThreadsOf> __device__ __forceinline__ int64_t page_block_sum(int64_t x, int64_t *room) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
        x += __shfl_xor_sync(kFullWarpMask, x, off);
    __syncthreads();
    if ((threadIdx.x & 31) == 0)
        room[threadIdx.x >> 5] = x;
    __syncthreads();
    int64_t sum = 0;
#pragma unroll
    for (int i = 0; i < kThreadsOf / 32; ++i)
        sum += room[i];
    return sum;
}

// Calls each(b, first, before, n) from whole warps for the sequences that have
// pages to move, shared out among all warps of the grid; before: the pages of the
// sequences ahead of b. The lengths are good.
template <int kThreadsOf, typename A, typename F> __device__ __forceinline__ void each_page_span(const A &a, int64_t *room, int2 *spans, F &&each) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int64_t done = 0;
    for (int base = 0; base < a.batch; base += kThreadsOf) {
        const int b = base + tid;
        const PageSpan s = b < a.batch ? page_span(a, b) : PageSpan{0, 0};
        int upto = s.n;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int other = __shfl_up_sync(kFullWarpMask, upto, off);
            upto += lane >= off ? other : 0;
        }
        __syncthreads(); // the round before has read room and spans
        if (lane == 31)
            room[warp] = upto;
        spans[tid] = make_int2(s.first, s.n);
        __syncthreads();
        int64_t all = 0, ahead = 0;
#pragma unroll
        for (int i = 0; i < kThreadsOf / 32; ++i) {
            ahead += i < warp ? room[i] : 0;
            all += room[i];
        }
        // sequence base + i is the grid's warp i's, so a batch of prompts spreads out
        const int64_t mine = done + ahead + upto - s.n;
        __shared__ int64_t before_s[kThreadsOf];
        before_s[tid] = mine;
        __syncthreads();
        const int left = min(kThreadsOf, a.batch - base);
        for (int i = warp * gridDim.x + blockIdx.x; i < left; i += kThreadsOf / 32 * gridDim.x) {
            const int2 span = spans[i];
            if (span.y > 0)
                each(base + i, span.x, before_s[i], span.y);
        }
        done += all;
    }
}

template <int kThreadsOf> static __global__ void __launch_bounds__(kThreadsOf) page_take_kernel(PageTake a) {
    __shared__ int64_t room[kThreadsOf / 32];
    __shared__ int2 spans[kThreadsOf];
    __shared__ int starts[kPageStarts];
    const int tid = threadIdx.x, lane = tid & 31;
    pdl_trigger();
    pdl_wait();
    int64_t need = 0;
    int bad = 0;
    for (int b = tid; b < a.batch; b += kThreadsOf) {
        const PageSpan s = page_span(a, b);
        if (b < kPageStarts)
            starts[b] = a.row_start[b];
        need += s.n > 0 ? s.n : 0;
        bad |= s.n < 0;
    }
    const int64_t count = a.free_blocks != nullptr ? max(0, *a.free_count) : 0;
    need = page_block_sum<kThreadsOf>(need, room);
    bad = __syncthreads_or(bad);
    const bool good = !bad && need <= count;
    if (good && need > 0)
        each_page_span<kThreadsOf>(a, room, spans, [&](int b, int first, int64_t before, int n) {
            int *row = a.block_table + static_cast<int64_t>(b) * a.table_stride + first;
            const int *top = a.free_blocks + (count - 1 - before);
            for (int k = lane; k < n; k += 32)
                row[k] = top[-k];
        });
    if (gridDim.x > 1)
        cluster_sync_all();
    else
        __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        *a.status = bad ? -1 : static_cast<int>(good ? 0 : min(need - count, static_cast<int64_t>(INT32_MAX)));
        if (a.free_blocks != nullptr)
            *a.free_left = static_cast<int>(good ? count - need : count);
    }
    const int first = a.row_start[0], last = good ? a.row_start[a.batch] : 0;
    const int *begins = a.batch <= kPageStarts ? starts : a.row_start;
    // a warp takes 128 rows in a row: mostly of one sequence, which is searched for once
    constexpr int kRows = 4;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreadsOf * kRows;
    for (int64_t base = (static_cast<int64_t>(blockIdx.x) * kThreadsOf + tid - lane) * kRows; base < a.rows; base += stride) {
        const int r0 = static_cast<int>(base) + lane, room_left = a.rows - r0; // row r0 + 32 i is there for 32 i < room_left
        int of = -1, end = 0, pos[kRows], id[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const int r = r0 + 32 * i;
            pos[i] = 0, id[i] = -1;
            if (32 * i >= room_left || r < first || r >= last)
                continue;
            if (of < 0 || r >= end) {
                int lo = max(of, 0), hi = a.batch; // the last sequence that starts at or before r
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (begins[mid] <= r)
                        lo = mid;
                    else
                        hi = mid;
                }
                of = lo, end = lo + 1 < a.batch ? begins[lo + 1] : last;
            }
            pos[i] = a.lens[of] + (r - begins[of]);
            id[i] = __ldcg(a.block_table + static_cast<int64_t>(of) * a.table_stride + pos[i] / kKvPage);
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (32 * i < room_left) {
                a.positions[r0 + 32 * i] = pos[i];
                a.slots[r0 + 32 * i] = id[i] < 0 ? -1 : static_cast<int64_t>(id[i]) * kKvPage + pos[i] % kKvPage;
            }
    }
}

template <int kThreadsOf> static __global__ void __launch_bounds__(kThreadsOf) page_give_kernel(PageGive a) {
    __shared__ int64_t room[kThreadsOf / 32];
    __shared__ int2 spans[kThreadsOf];
    const int tid = threadIdx.x, lane = tid & 31;
    pdl_trigger();
    pdl_wait();
    int64_t given = 0;
    int bad = 0;
    for (int b = tid; b < a.batch; b += kThreadsOf) {
        const PageSpan s = page_span(a, b);
        given += s.n > 0 ? s.n : 0;
        bad |= s.n < 0;
    }
    const int64_t count = *a.free_count;
    given = page_block_sum<kThreadsOf>(given, room);
    bad = __syncthreads_or(bad || count < 0 || count + given > a.capacity);
    if (!bad && given > 0)
        each_page_span<kThreadsOf>(a, room, spans, [&](int b, int first, int64_t before, int n) {
            const int *row = a.block_table + static_cast<int64_t>(b) * a.table_stride + first;
            int *to = a.free_blocks + count + before;
            for (int k = lane; k < n; k += 32)
                to[k] = row[k];
        });
    if (gridDim.x > 1)
        cluster_sync_all();
    else
        __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        *a.status = bad ? -1 : 0;
        *a.free_left = static_cast<int>(bad ? count : count + given);
    }
}

// One CTA for what it does in a few rounds, else a cluster as large as the device
// launches (79,000 rows of 48 prompts: 45.5 us with one CTA, 14.5 with 8, 12.2 with
// 16; 32,000 pages of 512 sequences given back: 18.2, 9.7, 8.6).
template <typename A> inline void page_launch(void (*few)(A), void (*many)(A), int64_t items, const A &a, cudaStream_t stream) {
    if (items <= 4 * kPageFew) {
        launch_ex(few, dim3(1), dim3(kPageFew), 0, stream, a);
        return;
    }
    const int ctas = allow_shared_bytes(many, kPageMany, 0);
    launch_ex_cluster(many, dim3(ctas), dim3(ctas), dim3(kPageMany), 0, stream, a);
}

} // namespace detail

namespace ops {

inline void page_take(const PageTake &a, cudaStream_t stream = nullptr) {
    detail::require(a.batch >= 0 && a.rows >= 0, "page_take: batch and rows must be nonnegative");
    detail::require(a.table_stride > 0 && a.table_stride <= INT32_MAX / detail::kKvPage,
                    "page_take: table_stride must be positive, and 16 * table_stride an int");
    detail::require(a.status && a.row_start, "page_take: null pointer");
    detail::require(a.batch == 0 || (a.lens && a.block_table), "page_take: null pointer");
    detail::require(a.rows == 0 || (a.positions && a.slots), "page_take: null pointer");
    detail::require(a.free_blocks == nullptr || (a.free_count && a.free_left), "page_take: a stack without its count");
    detail::page_launch(detail::page_take_kernel<detail::kPageFew>, detail::page_take_kernel<detail::kPageMany>,
                        static_cast<int64_t>(a.rows) + a.batch, a, stream);
}

inline void page_give(const PageGive &a, cudaStream_t stream = nullptr) {
    detail::require(a.batch >= 0 && a.capacity >= 0, "page_give: batch and capacity must be nonnegative");
    detail::require(a.table_stride > 0 && a.table_stride <= INT32_MAX / detail::kKvPage,
                    "page_give: table_stride must be positive, and 16 * table_stride an int");
    detail::require(a.status && a.free_count && a.free_left, "page_give: null pointer");
    detail::require(a.batch == 0 || (a.old_lens && a.new_lens && a.block_table && a.free_blocks), "page_give: null pointer");
    detail::page_launch(detail::page_give_kernel<detail::kPageFew>, detail::page_give_kernel<detail::kPageMany>, 16 * static_cast<int64_t>(a.batch),
                        a, stream);
}

} // namespace ops
} // namespace opworks
