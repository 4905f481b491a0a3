#pragma once

// ops::tree_commit — after a step over drafted tokens: compares each tree with
// what the model answered, finds the accepted path, and moves the path's cache
// rows to where the context goes on. No reference counterpart (the reference
// decodes one token per step).
//
// The drafted tokens of sequence b are nodes 0 .. n - 1 (rows row_start[b] ..
// row_start[b + 1]); their K/V rows lie at positions ctx + node. Node 0 is the
// root: the token that the step before this one chose, so it is accepted
// always. parent[j] < j is the node that j follows (-1: none), draft[j] its
// token, target[j] the token that the model chose after node j. The walk goes
// from a node i to its child j with draft[j] == target[i], the lowest j where
// several have it, until there is none. Results per sequence: the path's nodes
// (count of them, then -1), count, the model's next token target[last] and the
// new context length ctx + count. Row path[i] moves to row i in every layer
// and kv head; paths ascend, so a row is always read before the place that it
// lies in is written.
//
// The kernel is bound by latency: a few kilobytes per (layer, head). Every CTA
// of a sequence repeats the walk (a scatter of each node to its parent with a
// shared-memory minimum, then one dependent shared load per accepted token)
// instead of a second launch that would wait for the first one's answer. Measured
// (kernel time): a tree of 26 nodes, 16 layers of fp32 pools 3.2 us; 64 trees of
// up to 64 nodes, 16 layers of 8 bits 6.5 us, of which the bytes account for 1.0.

#include <climits>
#include <cstdint>

#include "../core/cuda_utils.cuh"
#include "kv4.cuh"
#include "kv_quant.cuh"

namespace opworks {

// The drafted trees of a batch, and where the results go (device pointers).
struct TreeVerify {
    const int *draft, *target, *parent; // [rows]
    const int *row_start;               // [batch + 1]
    const int *ctx_lens;                // [batch]
    int batch, max_rows;
    int *path;                       // [rows]
    int *count, *next, *new_lens;    // [batch]
};

namespace detail {

constexpr int kCommitThreads = 256;
constexpr int kCommitMaxRows = 2048; // per sequence: 4 ints of shared memory each
constexpr int kCommitBatch = 4;      // rows that a warp reads before it writes them

// The caches of all layers in one form: K row of (block, head, slot) at k +
// (block * kvh + head) * head_bytes + slot * row bytes, V the same from v,
// fp32 scales (8-bit pools) at scales + slot * 4 and 64 bytes further.
struct CommitCache {
    uint8_t *k, *v, *scales;
    int64_t head_bytes, layer_bytes;
    int layers, kvh;
    const int *table;
    int table_stride;
};

template <int kBytes> struct LaneBytes { // what a lane moves of one row: kBytes of 16 lanes
    uint32_t w[kBytes / 4];
    __device__ void load(const uint8_t *p) {
        if constexpr (kBytes == 4)
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        else if constexpr (kBytes == 8)
            *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(p);
        else
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i)
                reinterpret_cast<uint4 *>(w)[i] = reinterpret_cast<const uint4 *>(p)[i * 16];
    }
    __device__ void store(uint8_t *p) const {
        if constexpr (kBytes == 4)
            *reinterpret_cast<uint32_t *>(p) = w[0];
        else if constexpr (kBytes == 8)
            *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(w);
        else
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i)
                reinterpret_cast<uint4 *>(p)[i * 16] = reinterpret_cast<const uint4 *>(w)[i];
    }
};

// The walk of sequence blockIdx.y, by the whole block: its results (from block x =
// 0), the accepted nodes' count, and the blocks that path row i is moved from and
// to, -1 for a row that stays or lies outside the table. (A block and its slot are no
// one int: 16 times an id is above one from 2^27 blocks on.)
struct CommitMoves {
    const int *from, *to, *path;
    int ctx, count;
    __device__ int from_slot(int i) const { return static_cast<int>((static_cast<unsigned>(ctx) + path[i]) % kKvPage); }
    __device__ int to_slot(int i) const { return static_cast<int>((static_cast<unsigned>(ctx) + i) % kKvPage); }
};
__device__ __forceinline__ CommitMoves commit_walk(const TreeVerify &t, const CommitCache &c) {
    extern __shared__ int commit_smem[]; // succ | target | path | block of each path row
    __shared__ int count_s;
    int *succ = commit_smem, *target = succ + t.max_rows, *path = target + t.max_rows, *block = path + t.max_rows;
    const int b = blockIdx.y, tid = threadIdx.x;
    const int row0 = t.row_start[b], ctx = t.ctx_lens[b];
    const int n = min(t.row_start[b + 1] - row0, t.max_rows);
    for (int j = tid; j < n; j += kCommitThreads) {
        succ[j] = INT_MAX;
        target[j] = t.target[row0 + j];
    }
    __syncthreads();
    for (int j = tid; j < n; j += kCommitThreads) {
        const int p = t.parent[row0 + j];
        if (p >= 0 && p < j && t.draft[row0 + j] == target[p])
            atomicMin(&succ[p], j);
    }
    __syncthreads();
    if (tid == 0) {
        int cur = 0, count = 0;
        while (cur < n) { // succ[cur] > cur or INT_MAX
            path[count++] = cur;
            cur = succ[cur];
        }
        count_s = count;
    }
    __syncthreads();
    const int count = count_s;
    const int64_t tokens = static_cast<int64_t>(c.table_stride) * kKvPage;
    const int *table = c.table + static_cast<int64_t>(b) * c.table_stride;
    // block of path row i, and over succ, which is done, the block that it moves to
    for (int i = tid; i < count; i += kCommitThreads) {
        const int64_t from = static_cast<int64_t>(ctx) + path[i], to = static_cast<int64_t>(ctx) + i;
        const bool in = to >= 0 && from < tokens && from != to;
        const int from_block = in ? table[from / kKvPage] : -1, to_block = in ? table[to / kKvPage] : -1;
        block[i] = to_block < 0 ? -1 : from_block;
        succ[i] = from_block < 0 ? -1 : to_block;
    }
    if (blockIdx.x == 0) {
        for (int i = tid; i < n; i += kCommitThreads)
            t.path[row0 + i] = i < count ? path[i] : -1;
        if (tid == 0) {
            t.count[b] = count;
            t.next[b] = count ? target[path[count - 1]] : -1;
            t.new_lens[b] = ctx + count;
        }
    }
    __syncthreads();
    return {block, succ, path, ctx, count};
}

// kRowBytes: a K or V row of one head. Lanes 0-15 move K, 16-31 V. A lane reads
// and writes the same bytes of every row, so its own program order is enough.
template <int kRowBytes, bool kScales>
static __global__ void __launch_bounds__(kCommitThreads) tree_commit_kernel(TreeVerify t, CommitCache c) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    const CommitMoves moves = commit_walk(t, c);
    const int count = moves.count;
    constexpr int kLane = kRowBytes / 16; // bytes per lane
    const int units = c.layers * c.kvh;
    for (int u = blockIdx.x * (kCommitThreads / 32) + warp; u < units; u += gridDim.x * (kCommitThreads / 32)) {
        const int64_t base = (u / c.kvh) * c.layer_bytes + (u % c.kvh) * c.head_bytes;
        uint8_t *rows = (lane < 16 ? c.k : c.v) + base;
        uint8_t *scales = c.scales + base + (lane & 1) * 4 * kKvPage;
        for (int i0 = 1; i0 < count; i0 += kCommitBatch) {
            LaneBytes<kLane> x[kCommitBatch];
            float s[kCommitBatch];
#pragma unroll
            for (int i = 0; i < kCommitBatch; ++i) {
                const int from = i0 + i < count ? moves.from[i0 + i] : -1;
                if (from < 0)
                    continue;
                const int64_t at = static_cast<int64_t>(from) * c.kvh * c.head_bytes;
                const int slot = moves.from_slot(i0 + i);
                x[i].load(rows + at + slot * kRowBytes + (lane & 15) * min(kLane, 16));
                if (kScales && lane < 2)
                    s[i] = *reinterpret_cast<const float *>(scales + at + 4 * slot);
            }
#pragma unroll
            for (int i = 0; i < kCommitBatch; ++i) {
                const int to = i0 + i < count ? moves.to[i0 + i] : -1;
                if (to < 0)
                    continue;
                const int64_t at = static_cast<int64_t>(to) * c.kvh * c.head_bytes;
                const int slot = moves.to_slot(i0 + i);
                x[i].store(rows + at + slot * kRowBytes + (lane & 15) * min(kLane, 16));
                if (kScales && lane < 2)
                    *reinterpret_cast<float *>(scales + at + 4 * slot) = s[i];
            }
        }
    }
}

// Records of ops/kv4.cuh, from c.k: a row is 2 G pieces of 16 bytes (K's groups,
// then V's) and as many fp16 scales, a lane each, so a warp moves a row of 4 (D = 64)
// or 2 heads at a time. The same bytes of every row again.
template <int D> static __global__ void __launch_bounds__(kCommitThreads) tree_commit_q4_kernel(TreeVerify t, CommitCache c) {
    using R = Kv4Record<D>;
    constexpr int kPieces = 2 * R::kGroups, kLanes = 2 * kPieces;
    const int tid = threadIdx.x, part = tid % kLanes;
    pdl_wait();
    const CommitMoves moves = commit_walk(t, c);
    const bool codes = part < kPieces;
    const int64_t at0 = codes ? part * kKvPage * 16 : R::kKScale + (part - kPieces) * kKvPage * 2, step = codes ? 16 : 2;
    const int units = c.layers * c.kvh;
    for (int u = (blockIdx.x * kCommitThreads + tid) / kLanes; u < units; u += gridDim.x * kCommitThreads / kLanes) {
        uint8_t *base = c.k + (u / c.kvh) * c.layer_bytes + (u % c.kvh) * c.head_bytes + at0;
        for (int i0 = 1; i0 < moves.count; i0 += kCommitBatch) {
            uint4 x[kCommitBatch];
#pragma unroll
            for (int i = 0; i < kCommitBatch; ++i) {
                const int from = i0 + i < moves.count ? moves.from[i0 + i] : -1;
                if (from < 0)
                    continue;
                const uint8_t *src = base + static_cast<int64_t>(from) * c.kvh * c.head_bytes + moves.from_slot(i0 + i) * step;
                if (codes)
                    x[i] = *reinterpret_cast<const uint4 *>(src);
                else
                    x[i].x = *reinterpret_cast<const uint16_t *>(src);
            }
#pragma unroll
            for (int i = 0; i < kCommitBatch; ++i) {
                const int to = i0 + i < moves.count ? moves.to[i0 + i] : -1;
                if (to < 0)
                    continue;
                uint8_t *dst = base + static_cast<int64_t>(to) * c.kvh * c.head_bytes + moves.to_slot(i0 + i) * step;
                if (codes)
                    *reinterpret_cast<uint4 *>(dst) = x[i];
                else
                    *reinterpret_cast<uint16_t *>(dst) = static_cast<uint16_t>(x[i].x);
            }
        }
    }
}

inline void validate_commit(const TreeVerify &t, const CommitCache &c, int head_dim, int64_t layer_stride) {
    require(t.batch >= 0 && t.batch <= 65535, "tree_commit: batch must be 0 to 65535");
    require(t.max_rows >= 0 && t.max_rows <= kCommitMaxRows, "tree_commit: at most 2048 nodes per sequence");
    require(c.layers > 0 && c.kvh > 0 && c.table_stride > 0, "tree_commit: layers, kv heads and table_stride must be positive");
    require(head_dim == 64 || head_dim == 128, "tree_commit: head_dim must be 64 or 128");
    require(c.layers == 1 || layer_stride > 0, "tree_commit: layer_stride must be positive");
    if (t.batch == 0)
        return;
    require(t.row_start && t.ctx_lens && t.count && t.next && t.new_lens && c.table, "tree_commit: null pointer");
    require(t.max_rows == 0 || (t.draft && t.target && t.parent && t.path), "tree_commit: null pointer");
    require(c.k && c.v, "tree_commit: null pointer");
    require(t.new_lens != t.ctx_lens, "tree_commit: new_lens must not be ctx_lens (other blocks still read it)");
    require(aligned16(c.k) && aligned16(c.v) && c.layer_bytes % 16 == 0, "tree_commit: pools must be 16-byte aligned");
}

template <int kRowBytes, bool kScales>
inline void commit_launch(const TreeVerify &t, const CommitCache &c, cudaStream_t stream) {
    // one (layer, head) per warp while that fills at most four blocks per SM
    const int units = c.layers * c.kvh, warps = kCommitThreads / 32;
    const int want = (units + warps - 1) / warps;
    const int room = (4 * device_facts().sm_count + t.batch - 1) / t.batch;
    launch_ex(tree_commit_kernel<kRowBytes, kScales>, dim3(want < room ? want : room, t.batch), dim3(kCommitThreads),
              sizeof(int) * 4 * static_cast<size_t>(t.max_rows), stream, t, c);
}

} // namespace detail

namespace ops {

// Over fp32 pools [layers][blocks][kvh][16][head_dim]; layer_stride in floats.
inline void tree_commit(const TreeVerify &t, float *kpool, float *vpool, int64_t layer_stride, int layers,
                        const int *block_table, int table_stride, int kv_heads, int head_dim,
                        cudaStream_t stream = nullptr) {
    const detail::CommitCache c{reinterpret_cast<uint8_t *>(kpool), reinterpret_cast<uint8_t *>(vpool), nullptr,
                                static_cast<int64_t>(detail::kKvPage) * head_dim * 4, layer_stride * 4,
                                layers, kv_heads, block_table, table_stride};
    detail::validate_commit(t, c, head_dim, layer_stride);
    if (t.batch == 0)
        return;
    head_dim == 64 ? detail::commit_launch<256, false>(t, c, stream) : detail::commit_launch<512, false>(t, c, stream);
}

// Over 8-bit pools [layers][blocks][kvh][record]; layer_stride in bytes.
inline void tree_commit_q8(const TreeVerify &t, uint8_t *pool, int64_t layer_stride, int layers,
                           const int *block_table, int table_stride, int kv_heads, int head_dim,
                           cudaStream_t stream = nullptr) {
    const int64_t codes = static_cast<int64_t>(detail::kKvPage) * head_dim;
    const detail::CommitCache c{pool, pool ? pool + codes : nullptr, pool ? pool + 2 * codes : nullptr,
                                2 * codes + 8 * detail::kKvPage, layer_stride,
                                layers, kv_heads, block_table, table_stride};
    detail::validate_commit(t, c, head_dim, layer_stride);
    if (t.batch == 0)
        return;
    head_dim == 64 ? detail::commit_launch<64, true>(t, c, stream) : detail::commit_launch<128, true>(t, c, stream);
}

// Over 4-bit pools [layers][blocks][kvh][record]; layer_stride in bytes.
inline void tree_commit_q4(const TreeVerify &t, uint8_t *pool, int64_t layer_stride, int layers, const int *block_table,
                           int table_stride, int kv_heads, int head_dim, cudaStream_t stream = nullptr) {
    const detail::CommitCache c{pool, pool, pool, 18 * static_cast<int64_t>(head_dim), layer_stride, layers, kv_heads, block_table, table_stride};
    detail::validate_commit(t, c, head_dim, layer_stride);
    if (t.batch == 0)
        return;
    const int units = layers * kv_heads, per_block = detail::kCommitThreads / (head_dim == 64 ? 8 : 16);
    const int want = (units + per_block - 1) / per_block, room = (4 * detail::device_facts().sm_count + t.batch - 1) / t.batch;
    launch_ex(head_dim == 64 ? detail::tree_commit_q4_kernel<64> : detail::tree_commit_q4_kernel<128>,
              dim3(want < room ? want : room, t.batch), dim3(detail::kCommitThreads), sizeof(int) * 4 * static_cast<size_t>(t.max_rows),
              stream, t, c);
}

} // namespace ops
} // namespace opworks
