#pragma once

// What the tree attention kernels share: the arguments, the span of a
// sequence, the tree mask, cluster helpers (ops/tree_attention.cuh has the
// operator).

#include <algorithm>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <mutex>
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

// Lets `kernel` have `bytes` of dynamic shared memory and clusters above 8 CTAs on
// the current device, and returns the largest cluster that it may be launched
// with: 16, or the portable 8 where no part of the device has room for 16 such
// CTAs. Asked once per kernel and device.
template <typename... P> inline int allow_shared_bytes(void (*kernel)(P...), int threads, int bytes) {
    struct Known {
        const void *kernel;
        int device, cluster;
    };
    static std::mutex mu;
    static std::vector<Known> all;
    static thread_local std::vector<Known> mine; // no lock once a thread knows
    const void *id = reinterpret_cast<const void *>(kernel);
    const int device = device_facts().device;
    for (const Known &k : mine)
        if (k.kernel == id && k.device == device)
            return k.cluster;
    const std::lock_guard<std::mutex> lock(mu);
    for (const Known &k : all)
        if (k.kernel == id && k.device == device) {
            mine.push_back(k);
            return k.cluster;
        }
    OPWORKS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    OPWORKS_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 16, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError(); // no more than an answer to the question
        clusters = 0;
    }
    const Known k{id, device, clusters > 0 ? 16 : 8};
    all.push_back(k);
    mine.push_back(k);
    return k.cluster;
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

// The sequence with the `order`-th most work (the longest context, equal ones by
// index), so that CTAs that wait for a place come longest first: what is left
// over at the end is short. Every thread of the block calls it; `room` is shared
// memory for batch + 1 ints, batch <= the block's threads.
__device__ __forceinline__ int sequence_by_work(const TreeBatch &t, int order, int *room) {
    const int tid = threadIdx.x;
    if (tid < t.batch) {
        const int n = t.row_start[tid + 1] - t.row_start[tid];
        room[1 + tid] = n > 0 ? t.ctx_lens[tid] : -1;
    }
    __syncthreads();
    if (tid < t.batch) {
        const int mine = room[1 + tid];
        int before = 0;
        for (int i = 0; i < t.batch; ++i)
            before += room[1 + i] > mine || (room[1 + i] == mine && i < tid) ? 1 : 0;
        if (before == order)
            room[0] = tid;
    }
    __syncthreads();
    const int b = room[0];
    sm100::fence_proxy_async_smem(); // `room` may lie where bulk copies go next
    __syncthreads();
    return b;
}

// Bit i: node `node` (row `row` of the mask) sees the key j0 + i, i < 32, where
// keys below 0 are context and there are none from `limit` (>= 0) on.
__device__ __forceinline__ uint32_t tree_sees32(const TreeBatch &t, int row, int node, int j0, int limit) {
    uint32_t bits = ~0u;
    if (j0 <= -32)
        return bits;
    if (t.mask == nullptr) {
        limit = min(limit, node + 1);
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
    return left >= 32 ? bits : left <= 0 ? 0u : bits & ((1u << left) - 1u);
}

constexpr float kLazy = 4.f;  // log2 units a score may pass the reference maximum by
constexpr float kLift = 10.f; // P is scaled by 2^kLift: at most 2^14
constexpr float kNone = -1e30f; // reference of a row that has seen nothing yet
// A reference above this is so coarse that a weight may come out too large for
// fp16: from there on weights are cut off.
constexpr float kWary = 0x1p20f;
// How far below the largest score `top` the reference lies: by `lift`, but at
// least by two units in its last place, so that the weight of that score, however
// the difference is rounded, is not below one.
__device__ __forceinline__ float reference_lift(float lift, float top) { return fmaxf(lift, fabsf(top) * 0x1p-22f); }
// V scales below this are not told apart from it (fp16 loses their low bits);
// lower, and l in their units would leave fp32's range. The same for the
// magnitudes of single fp32 V rows.
constexpr float kMinVLog = -80.f, kMinVTop = 0x1p-80f;
constexpr int kMinVKey = -60;
constexpr float kLowV = 0x1p-12f; // V scales this far below their power of two get a new one

// fp16 pair (a, b) as one register, a in the low half
__device__ __forceinline__ uint32_t half2_rn(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 half2_floats(uint32_t h) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// Two pairs of fp16 from the four codes of a word: (0, 1) and (2, 3). Exact.
template <KvFormat kFmt> __device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (kFmt == KvFormat::kInt8) {
        // byte + 128 in the low bits of fp16 1024 .. 1279, minus 1152
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t bias = 0x64806480u; // fp16 1152, twice
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&bias));
        const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), *reinterpret_cast<const __half2 *>(&bias));
        lo = *reinterpret_cast<const uint32_t *>(&x);
        hi = *reinterpret_cast<const uint32_t *>(&y);
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) <= 3.4028235e38f ? x : 0.f; }

// The power of two next above magnitude `top` (bits of it) as an exponent
// field, held where its inverse and its products with 2^10 are normal too (up to
// `most`: 254 where its inverse times 2^8 or more is all that is wanted).
__device__ __forceinline__ uint32_t exponent_above(uint32_t top_bits, uint32_t most = 240u) {
    return min(max((top_bits >> 23) + 1u, 16u), most);
}
__device__ __forceinline__ float pow2_field(uint32_t ex) { return __uint_as_float(ex << 23); }

// e4m3 NaN codes (never written by ops::kv_quant_write) replaced by zero: a
// masked row may hold them, and zero times NaN is NaN.
__device__ __forceinline__ uint32_t clear_e4m3_nan(uint32_t w) {
    return w & ~__vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
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
