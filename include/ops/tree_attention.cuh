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
// fp32. A masked key has no influence, whatever its row holds; an infinity or a
// NaN in a K or V row that a node does see makes the node's whole output NaN,
// and so does one in its query row.
//
// K and V values may lie anywhere in fp32's range. Those of the context share a
// power of two, 16 keys (rows kernel; of V 32 dims) or 8 to 32 (tiles), and are
// held to 2^-22 of the largest of them at least; those of nodes have their own.
// V rows that one node sees may differ 2^100-fold.

#include "tree_attention_common.cuh"
#include "tree_attention_rows.cuh"
#include "tree_attention_tiles.cuh"

namespace opworks {
namespace detail {

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
    constexpr int kTile = TreeRowsGeo<T, D, kFmt, 1>::kRows;
    const int64_t rows = static_cast<int64_t>(a.t.max_rows) * (a.qh / a.kvh), tiles = (rows + kTile - 1) / kTile;
    // The rows kernel's time grows with the rows, that of 128-row tiles does not. 8 (32)
    // sequences of 4096 (2048) tokens with equal trees, 8 kv heads, us with rows / tiles:
    //   fp32 rows, fp32, D 64     24 rows  54 / 79 (89 / 147)     32   88 / 80 (167 / 149)
    //   fp32 rows, fp32, D 128    16 rows 102 / 127 (193 / 242)   24  180 / 126 (374 / 243)
    //   bf16 rows, fp32, D 64     48 rows  56 / 67 (86 / 126)     64   88 / 68 (162 / 130)
    //   bf16 rows, fp32, D 128    32 rows  97 / 127 (177 / 247)   48  159 / 129 (339 / 251)
    //   fp32 rows, int8, D 64     48 rows  53 / 59 (82 / 112)     64   71 / 60 (120 / 113)
    //   fp32 rows, e4m3, D 64     48 rows  49 / 60 (74 / 114)     64   62 / 61 (109 / 117)   80   62 / 62 (144 / 120)
    //   bf16 rows, int8, D 64     48 rows  44 / 41 (49 / 76)      64   61 / 42 (94 / 77)
    //   bf16 rows, int8, D 128    32 rows  54 / 53 (80 / 102)     48   75 / 55 (140 / 105)
    // Where trees differ it is the mean that tells: one sequence of 64 rows among 32 of
    // 2000 tokens and 4 rows, fp32 rows: fp32 92 / 138, int8 51 / 100; one of 2048 rows:
    // 545 / 404, 373 / 323. (fp32 rows of 128 dims over 8-bit pools have no tiles.)
    constexpr bool kBf16 = std::is_same_v<T, __nv_bfloat16>, kWide = kFmt == KvFormat::kF32;
    constexpr bool kHasTiles = kBf16 || kWide || D == 64;
    constexpr int kFrom = kBf16 ? (D == 64 ? 48 : 32) : kWide ? (D == 64 ? 24 : 16) : 60; // rows of a kv head
    const bool many = static_cast<int64_t>(a.t.rows) * (a.qh / a.kvh) > static_cast<int64_t>(kFrom) * a.t.batch;
    if constexpr (kHasTiles) {
        if (many) {
            // two row tiles to a CTA where shared memory holds both
            constexpr int kPair = D == 64 || (!kWide && kBf16) ? 2 : 1;
            if (rows <= 128 || kPair == 1)
                tree_tiles_launch<T, D, kFmt, 1>(q, out, a, stream);
            else
                tree_tiles_launch<T, D, kFmt, kPair>(q, out, a, stream);
            return;
        }
    }
    if (tiles == 1) {
        tree_rows_launch<T, D, kFmt, 1>(q, out, a, stream);
    } else if (D == 128 || tiles == 2) {
        tree_rows_launch<T, D, kFmt, 2>(q, out, a, stream);
    } else { // more tiles to a CTA: K and V are widened once for all of them
        tree_rows_launch<T, D, kFmt, D == 64 ? 3 : 2>(q, out, a, stream);
    }
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
