#pragma once

// ops::tree_attention_q4 — attention of several new tokens per sequence
// (ops/tree_attention.cuh has the definition of the operator: rows, contexts,
// masks, and what a masked key may hold) over the 4-bit pool of ops/kv4.cuh. No
// reference counterpart.
//
// What is held there is an fp16 number, so K and V enter the tensor cores' fp16
// products exactly, with no units and no factors behind them (the rows kernel takes
// K's codes, and multiplies the sum over a group's dims by the scale in fp32). A query row is scaled by a power of two, to a
// largest magnitude of 2^14 to 2^15, and is one fp16 term where it comes in bf16
// (exact down to 2^-29 of the largest), two where it comes in fp32 (22 bits).
//
// The softmax weights of fp32 rows have 22 bits, two terms. Those of bf16 rows are one fp16 number
// of 11 bits, while their sum takes them as they are: rows come out 1e-4 to 3e-4 off before they
// are rounded to bf16 (1.7e-3), in the 2-norm. A second term, up to 4 rows a head in the column
// that is empty there, takes as long as fp32 rows do: 12 sequences of 32,000 tokens, 8 x 128, 102
// us for 88, and the error goes from 1.67e-3 to 1.66e-3.

#include "tree_attention.cuh"
#include "kv4.cuh"
#include "tree_attention_q4_rows.cuh"
#include "tree_attention_q4_tiles.cuh"

namespace opworks {
namespace detail {

template <typename T, int D> inline void q4_call(const T *q, T *out, const TreeArgs &a, cudaStream_t stream) {
    // The rows kernel's time grows with the rows, that of 128-row tiles does not. 8 (32)
    // sequences of 4096 (2048) tokens with up to n rows of a kv head, 0.8 n on average, 8 kv
    // heads, us with rows / tiles:
    //   fp32 rows, D 64     n = 32  25 / 40 (38 / 61)   48  40 / 41 (61 / 63)   64  40 / 41 (65 / 64)   80  58 / 42 (89 / 65)
    //   bf16 rows, D 64     n = 32  19 / 31 (28 / 48)   48  29 / 32 (45 / 49)   64  29 / 31 (47 / 50)   80  43 / 32 (65 / 51)
    //   bf16 rows, D 128    n = 32  29 / 41 (45 / 63)   48  47 / 42 (72 / 64)   64  47 / 43 (76 / 65)   80  68 / 44 (102 / 66)
    // It is the mean that tells, in batches of like rows. (fp32 rows of 128 dims have no tiles.)
    constexpr bool kHasTiles = D == 64 || std::is_same_v<T, __nv_bfloat16>;
    constexpr int kFrom = D == 128 ? 32 : 53; // rows of a kv head
    const bool many = static_cast<int64_t>(a.t.rows) * (a.qh / a.kvh) > static_cast<int64_t>(kFrom) * a.t.batch;
    if constexpr (kHasTiles)
        if (many) {
            q4_tiles_call<T, D>(q, out, a, stream);
            return;
        }
    q4_rows_call<T, D>(q, out, a, stream);
}

} // namespace detail

namespace ops {

// Over the 4-bit pool [blocks][kv_heads][record] of ops/kv4.cuh. q row r, head h at
// r * q_stride + h * head_dim; T fp32 or bf16; out in the same form and type.
template <typename T>
inline void tree_attention_q4(const T *q, int64_t q_stride, const uint8_t *pool, const TreeBatch &t, int q_heads, int kv_heads,
                              int head_dim, float scale, T *out, int64_t out_stride, cudaStream_t stream = nullptr) {
    using namespace detail;
    validate_tree(t, q, out, q_stride, out_stride, sizeof(T), q_heads, kv_heads, head_dim, pool, pool);
    require(static_cast<int64_t>(t.max_rows) * (q_heads / kv_heads) <= 0x7fffffff, "tree attention: too many rows for one call");
    if (t.batch == 0 || t.max_rows == 0)
        return;
    const TreeArgs a{t, pool, nullptr, q_heads, kv_heads, scale * kLog2e, q_stride, out_stride};
    head_dim == 64 ? q4_call<T, 64>(q, out, a, stream) : q4_call<T, 128>(q, out, a, stream);
}

} // namespace ops
} // namespace opworks
