#pragma once

// What the tree attention kernels share: the arguments, the span of a
// sequence, the tree mask, cluster helpers (ops/tree_attention.cuh has the
// operator).

#include <algorithm>
#include <cstdint>
#include <cuda_bf16.h>
#include <mutex>
#include <utility>
#include <vector>

#include "../core/cuda_utils.cuh"
#include "attention_kernels.cuh"
#include "kv_quant.cuh"

namespace opworks {

// A batch of trees over a cache (device pointers).
struct TreeBatch {
    const int *block_table; // [batch][table_stride]
    int table_stride;
    const int *ctx_lens;    // [batch]
    const int *row_start;   // [batch + 1]
    const uint32_t *mask;   // [rows][mask_words], or null: a chain
    int mask_words;
    int batch, rows, max_rows; // max_rows: the most rows of one sequence
    int max_ctx;               // an upper bound of ctx_lens; plans the launch only
};

namespace detail {

struct TreeArgs {
    TreeBatch t;
    const void *k; // fp32 K pool, or the 8-bit pool
    const void *v; // fp32 V pool
    int qh, kvh;
    float scale_log2; // scale * log2(e): scores in log2 units
    int64_t q_stride, out_stride;
};

// Lets `kernel` have `bytes` of dynamic shared memory and clusters of up to 16
// CTAs on the current device
// (set once per kernel and device; setting it twice does no harm).
template <typename... P> inline void allow_shared_bytes(void (*kernel)(P...), int bytes) {
    static std::mutex mu;
    static std::vector<std::pair<const void *, int>> set;
    static thread_local std::vector<std::pair<const void *, int>> seen; // no lock once a thread knows
    const std::pair<const void *, int> key{reinterpret_cast<const void *>(kernel), device_facts().device};
    if (std::find(seen.begin(), seen.end(), key) != seen.end())
        return;
    const std::lock_guard<std::mutex> lock(mu);
    if (std::find(set.begin(), set.end(), key) == set.end()) {
        OPWORKS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        OPWORKS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        set.push_back(key);
    }
    seen.push_back(key);
}

// Keys and rows of a sequence, held inside the table and the row count.
struct TreeSpan {
    int row0, n, ctx, keys;
    __device__ TreeSpan(const TreeBatch &t, int b) {
        row0 = max(0, t.row_start[b]);
        n = max(0, min(min(t.row_start[b + 1], t.rows) - row0, t.max_rows));
        const int64_t places = static_cast<int64_t>(t.table_stride) * kKvPage;
        ctx = static_cast<int>(min(static_cast<int64_t>(max(0, t.ctx_lens[b])), places));
        keys = static_cast<int>(min(static_cast<int64_t>(ctx) + n, places));
    }
};

// Bit i: node `node` (row `row` of the mask) sees the key j0 + i, i < 16, where
// keys below 0 are context and there are none from `limit` on. j0 > -32.
__device__ __forceinline__ uint32_t tree_sees16(const TreeBatch &t, int row, int node, int j0, int limit) {
    uint32_t bits;
    if (t.mask == nullptr) {
        limit = min(limit, node + 1);
        bits = 0xffffu;
    } else {
        const uint32_t *w = t.mask + static_cast<int64_t>(row) * t.mask_words;
        if (j0 < 0) {
            bits = (w[0] << -j0) | ((1u << -j0) - 1u);
        } else {
            const int i = j0 >> 5;
            const uint32_t lo = i < t.mask_words ? w[i] : 0u, hi = i + 1 < t.mask_words ? w[i + 1] : 0u;
            bits = __funnelshift_r(lo, hi, j0 & 31);
        }
    }
    const int left = limit - j0;
    return left >= 16 ? bits & 0xffffu : left <= 0 ? 0u : bits & ((1u << left) - 1u);
}

__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A float at the address of `p` in the shared memory of CTA `rank` of the cluster.
__device__ __forceinline__ float peer_load(const float *p, int rank) {
    uint32_t at;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(sm100::smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}

} // namespace detail
} // namespace opworks
