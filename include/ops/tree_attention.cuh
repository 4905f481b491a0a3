#pragma once

// ops::tree_attention — attention of several new tokens per sequence over the
// paged KV cache (fp32 pools, or the 8-bit pool of ops/kv_quant.cuh). No
// reference counterpart (the reference decodes one token per step).
//
// The new tokens of sequence b are nodes 0 .. n - 1 (rows row_start[b] ..
// row_start[b + 1] of q and out); their K/V rows are in the cache already, at
// positions ctx + node with ctx = ctx_lens[b]. Node i attends to the context,
// positions 0 .. ctx - 1, and to the nodes j whose bit is set in its mask row
// (mask[row][j / 32] bit j % 32), or to the nodes j <= i where no mask is
// given (a chain of tokens; n = 1 is a plain decode step):
//   o = sum_j softmax_j(scale q . k_j) v_j
// A node that sees nothing gets zeros. Scores, softmax statistics and sums are
// fp32. A masked key has no influence, whatever its row holds.

#include <cstdint>
#include <cuda_bf16.h>

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

// Keys and rows of a sequence, held inside the table and the row count.
struct TreeSpan {
    int row0, n, ctx, keys;
    __device__ TreeSpan(const TreeBatch &t, int b) {
        row0 = max(0, t.row_start[b]);
        n = max(0, min(min(t.row_start[b + 1], t.rows) - row0, t.max_rows));
        ctx = max(0, t.ctx_lens[b]);
        const int64_t all = min(static_cast<int64_t>(ctx) + n, static_cast<int64_t>(t.table_stride) * kKvPage);
        keys = static_cast<int>(all);
    }
};

__device__ __forceinline__ bool tree_sees(const TreeBatch &t, int row, int i, int j) {
    if (t.mask == nullptr)
        return j <= i;
    return (t.mask[static_cast<int64_t>(row) * t.mask_words + (j >> 5)] >> (j & 31)) & 1u;
}

constexpr int kTreeThreads = 128;

// One CTA per (row, query head); its warps take the keys in turn and are
// merged at the end.
template <typename T, int D, KvFormat kFmt>
static __global__ void __launch_bounds__(kTreeThreads)
    tree_attention_kernel(const T *__restrict__ q, T *__restrict__ out, TreeArgs a) {
    constexpr int kE = D / 32, kWarps = kTreeThreads / 32;
    __shared__ float om[kWarps][D], mm[kWarps], ll[kWarps];
    const int i = blockIdx.x, hq = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const TreeSpan s(a.t, b);
    if (i >= s.n)
        return;
    const int row = s.row0 + i, h = hq / (a.qh / a.kvh);
    float qr[kE], o[kE] = {}, m = kNegInf, l = 0.f;
    for (int e = 0; e < kE; ++e)
        qr[e] = static_cast<float>(q[row * a.q_stride + hq * D + lane * kE + e]) * a.scale_log2;
    for (int t = warp; t < s.keys; t += kWarps) {
        if (t >= s.ctx && !tree_sees(a.t, row, i, t - s.ctx))
            continue;
        const int64_t rec = static_cast<int64_t>(a.t.block_table[static_cast<int64_t>(b) * a.t.table_stride + t / kKvPage]) * a.kvh + h;
        const int slot = t % kKvPage;
        float kk[kE], vv[kE];
        if constexpr (kFmt == KvFormat::kF32) {
            const int64_t at = (rec * kKvPage + slot) * D + lane * kE;
            for (int e = 0; e < kE; ++e) {
                kk[e] = static_cast<const float *>(a.k)[at + e];
                vv[e] = static_cast<const float *>(a.v)[at + e];
            }
        } else {
            using R = KvRecord<D>;
            const uint8_t *p = static_cast<const uint8_t *>(a.k) + rec * R::kBytes;
            const float ks = *reinterpret_cast<const float *>(p + R::kKScale + 4 * slot);
            const float vs = *reinterpret_cast<const float *>(p + R::kVScale + 4 * slot);
            for (int e = 0; e < kE; ++e) {
                float x[4];
                kv_decode4<kFmt>(p[slot * D + lane * kE + e], ks, x);
                kk[e] = x[0];
                kv_decode4<kFmt>(p[R::kCodes + slot * D + lane * kE + e], vs, x);
                vv[e] = x[0];
            }
        }
        float x = 0.f;
        for (int e = 0; e < kE; ++e)
            x = fmaf(qr[e], kk[e], x);
        for (int off = 16; off; off >>= 1)
            x += __shfl_xor_sync(kFullWarpMask, x, off);
        const float m1 = fmaxf(m, x);
        const float c = m == kNegInf ? 0.f : exp2f(m - m1), p = exp2f(x - m1);
        m = m1;
        l = l * c + p;
        for (int e = 0; e < kE; ++e)
            o[e] = o[e] * c + p * vv[e];
    }
    for (int e = 0; e < kE; ++e)
        om[warp][lane * kE + e] = o[e];
    if (lane == 0)
        mm[warp] = m, ll[warp] = l;
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kTreeThreads) {
        float top = kNegInf, L = 0.f, O = 0.f;
        for (int w = 0; w < kWarps; ++w)
            top = fmaxf(top, mm[w]);
        for (int w = 0; w < kWarps; ++w) {
            const float f = mm[w] == kNegInf ? 0.f : exp2f(mm[w] - top);
            L += f * ll[w];
            O += f * om[w][d];
        }
        out[row * a.out_stride + hq * D + d] = static_cast<T>(L > 0.f || L != L ? O / L : 0.f);
    }
}

inline void validate_tree(const TreeBatch &t, const void *q, const void *out, int64_t q_stride, int64_t out_stride,
                          int elem, int q_heads, int kv_heads, int head_dim, const void *k, const void *v) {
    require(t.batch >= 0 && t.batch <= 65535, "tree attention: batch must be 0 to 65535");
    require(t.rows >= 0 && t.max_rows >= 0 && t.max_rows <= t.rows, "tree attention: 0 <= max_rows <= rows");
    require(t.max_ctx >= 0 && t.table_stride > 0, "tree attention: max_ctx must be nonnegative, table_stride positive");
    require(kv_heads > 0 && kv_heads <= 4096 && q_heads > 0 && q_heads <= 65535 && q_heads % kv_heads == 0,
            "tree attention: query heads must be a multiple of the kv heads");
    require(head_dim == 64 || head_dim == 128, "tree attention: head_dim must be 64 or 128");
    if (t.batch == 0 || t.max_rows == 0)
        return;
    require(q && out && k && v && t.block_table && t.ctx_lens && t.row_start, "tree attention: null pointer");
    require(t.mask == nullptr || static_cast<int64_t>(t.mask_words) * 32 >= t.max_rows,
            "tree attention: the mask rows are shorter than the trees");
    const int64_t width = static_cast<int64_t>(q_heads) * head_dim;
    require(q_stride >= width && out_stride >= width, "tree attention: rows overlap (stride below heads * head_dim)");
    require(aligned16(q) && aligned16(out) && aligned16(k) && aligned16(v) && (q_stride * elem) % 16 == 0 &&
                (out_stride * elem) % 16 == 0,
            "tree attention: q, out and pools must be 16-byte aligned, and the row strides too");
}

template <typename T, int D, KvFormat kFmt>
inline void tree_attention_launch(const T *q, T *out, const TreeArgs &a, cudaStream_t stream) {
    launch_ex(tree_attention_kernel<T, D, kFmt>, dim3(a.t.max_rows, a.qh, a.t.batch), dim3(kTreeThreads), 0, stream, q,
              out, a);
}

template <typename T>
inline void tree_attention_any(const T *q, int64_t q_stride, KvFormat format, const void *k, const void *v,
                               const TreeBatch &t, int q_heads, int kv_heads, int head_dim, float scale, T *out,
                               int64_t out_stride, cudaStream_t stream) {
    validate_tree(t, q, out, q_stride, out_stride, sizeof(T), q_heads, kv_heads, head_dim, k, v);
    if (t.batch == 0 || t.max_rows == 0)
        return;
    const TreeArgs a{t, k, v, q_heads, kv_heads, scale * kLog2e, q_stride, out_stride};
    switch (format) {
    case KvFormat::kF32:
        head_dim == 64 ? tree_attention_launch<T, 64, KvFormat::kF32>(q, out, a, stream)
                       : tree_attention_launch<T, 128, KvFormat::kF32>(q, out, a, stream);
        break;
    case KvFormat::kInt8:
        head_dim == 64 ? tree_attention_launch<T, 64, KvFormat::kInt8>(q, out, a, stream)
                       : tree_attention_launch<T, 128, KvFormat::kInt8>(q, out, a, stream);
        break;
    case KvFormat::kE4M3:
        head_dim == 64 ? tree_attention_launch<T, 64, KvFormat::kE4M3>(q, out, a, stream)
                       : tree_attention_launch<T, 128, KvFormat::kE4M3>(q, out, a, stream);
        break;
    default: throw std::invalid_argument("tree attention: unknown cache format");
    }
}

} // namespace detail

namespace ops {

// Over fp32 pools [blocks][kv_heads][16][head_dim]. q row r, head h at r *
// q_stride + h * head_dim; T fp32 or bf16; out in the same form and type.
template <typename T>
inline void tree_attention(const T *q, int64_t q_stride, const float *kpool, const float *vpool, const TreeBatch &t,
                           int q_heads, int kv_heads, int head_dim, float scale, T *out, int64_t out_stride,
                           cudaStream_t stream = nullptr) {
    detail::tree_attention_any(q, q_stride, KvFormat::kF32, kpool, vpool, t, q_heads, kv_heads, head_dim, scale, out,
                               out_stride, stream);
}

// Over the 8-bit pool [blocks][kv_heads][record] of ops/kv_quant.cuh.
template <typename T>
inline void tree_attention_q8(const T *q, int64_t q_stride, const uint8_t *pool, KvFormat format, const TreeBatch &t,
                              int q_heads, int kv_heads, int head_dim, float scale, T *out, int64_t out_stride,
                              cudaStream_t stream = nullptr) {
    detail::require(format == KvFormat::kInt8 || format == KvFormat::kE4M3,
                    "tree attention: format must be int8 (1) or e4m3 (2)");
    detail::tree_attention_any(q, q_stride, format, pool, pool, t, q_heads, kv_heads, head_dim, scale, out, out_stride,
                               stream);
}

} // namespace ops
} // namespace opworks
