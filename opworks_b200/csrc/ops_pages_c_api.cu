// libopworks_ops.so, third part: pages and slots, norm and rotation of heads, the
// 4-bit paged KV cache and attention and commit over it. Same conventions as
// ops_c_api.cu.

#include "opworks_ops.h"
#include "ops/kv4.cuh"
#include "ops/pages.cuh"
#include "ops/qk_norm_rope.cuh"
#include "ops/tree_attention_q4.cuh"
#include "ops/tree_commit.cuh"
#include "ops_guard.h"

using opworks_ops::guarded;

namespace {

cudaStream_t as_stream(void *s) { return static_cast<cudaStream_t>(s); }

// f(tag) with the row type that `type` names: 0 fp32, 1 bf16.
template <typename F> void with_type(int type, F &&f) {
    switch (type) {
    case 0: f(static_cast<float *>(nullptr)); break;
    case 1: f(static_cast<__nv_bfloat16 *>(nullptr)); break;
    default: throw std::invalid_argument("type must be fp32 (0) or bf16 (1)");
    }
}

template <typename T> T *as(void *p, T *) { return static_cast<T *>(p); }
template <typename T> const T *as(const void *p, T *) { return static_cast<const T *>(p); }

} // namespace

extern "C" {

int opw_page_take(const int32_t *lens, const int32_t *row_start, int batch, int rows, int32_t *block_table,
                  int table_stride, const int32_t *free_blocks, const int32_t *free_count, int32_t *positions,
                  int64_t *slots, int32_t *free_left, int32_t *status, void *stream) {
    return guarded([&] {
        opworks::ops::page_take({lens, row_start, batch, rows, block_table, table_stride, free_blocks, free_count, positions,
                                 slots, free_left, status},
                                as_stream(stream));
    });
}

int opw_page_give(const int32_t *old_lens, const int32_t *new_lens, int batch, const int32_t *block_table,
                  int table_stride, int32_t *free_blocks, int capacity, const int32_t *free_count, int32_t *free_left,
                  int32_t *status, void *stream) {
    return guarded([&] {
        opworks::ops::page_give({old_lens, new_lens, batch, block_table, table_stride, free_blocks, capacity, free_count,
                                 free_left, status},
                                as_stream(stream));
    });
}

int opw_qk_norm_rope(const void *q, int64_t q_stride, const void *k, int64_t k_stride, int type, const float *q_weight,
                     const float *k_weight, float eps, const int32_t *positions, const float *inv_freq, int rot_dim,
                     int rows, int q_heads, int kv_heads, int head_dim, void *q_out, int64_t q_out_stride, void *k_out,
                     int64_t k_out_stride, void *stream) {
    return guarded([&] {
        with_type(type, [&](auto *t) {
            using T = std::remove_pointer_t<decltype(t)>;
            opworks::ops::qk_norm_rope(opworks::QkNormRope<T>{as(q, t), q_stride, as(k, t), k_stride, q_weight, k_weight, eps,
                                                              positions, inv_freq, rot_dim, rows, q_heads, kv_heads, head_dim,
                                                              as(q_out, t), q_out_stride, as(k_out, t), k_out_stride},
                                       as_stream(stream));
        });
    });
}

int opw_kv4_record_bytes(int head_dim) {
    int r = -1;
    guarded([&] { r = opworks::ops::kv4_record_bytes(head_dim); });
    return r;
}

int opw_kv4_write(const void *k, int64_t k_stride, const void *v, int64_t v_stride, int type, uint8_t *pool, int blocks,
                  const int64_t *slots, int rows, int num_kv_heads, int head_dim, void *stream) {
    return guarded([&] {
        with_type(type, [&](auto *t) {
            opworks::ops::kv4_write(as(k, t), k_stride, as(v, t), v_stride, pool, blocks, slots, rows, num_kv_heads, head_dim,
                                    as_stream(stream));
        });
    });
}

int opw_kv4_read(const uint8_t *pool, int blocks, const int64_t *slots, int rows, int num_kv_heads, int head_dim, void *k,
                 int64_t k_stride, void *v, int64_t v_stride, int type, void *stream) {
    return guarded([&] {
        with_type(type, [&](auto *t) {
            opworks::ops::kv4_read(pool, blocks, slots, rows, num_kv_heads, head_dim, as(k, t), k_stride, as(v, t), v_stride,
                                   as_stream(stream));
        });
    });
}

int opw_tree_attention_q4(const void *q, int type, int64_t q_stride, const uint8_t *pool, const int32_t *block_table,
                          int table_stride, const int32_t *ctx_lens, const int32_t *row_start, const uint32_t *mask,
                          int mask_words, int batch, int rows, int max_rows, int max_ctx, int num_q_heads,
                          int num_kv_heads, int head_dim, float scale, void *out, int64_t out_stride, void *stream) {
    return guarded([&] {
        const opworks::TreeBatch b{block_table, table_stride, ctx_lens, row_start, mask, mask_words, batch, rows, max_rows, max_ctx};
        with_type(type, [&](auto *t) {
            opworks::ops::tree_attention_q4(as(q, t), q_stride, pool, b, num_q_heads, num_kv_heads, head_dim, scale, as(out, t),
                                            out_stride, as_stream(stream));
        });
    });
}

int opw_tree_commit_q4(const int32_t *draft, const int32_t *target, const int32_t *parent, const int32_t *row_start,
                       const int32_t *ctx_lens, int batch, int max_rows, uint8_t *pool, int64_t layer_stride, int layers,
                       const int32_t *block_table, int table_stride, int num_kv_heads, int head_dim, int32_t *path,
                       int32_t *count, int32_t *next, int32_t *new_lens, void *stream) {
    return guarded([&] {
        const opworks::TreeVerify t{draft, target, parent, row_start, ctx_lens, batch, max_rows, path, count, next, new_lens};
        opworks::ops::tree_commit_q4(t, pool, layer_stride, layers, block_table, table_stride, num_kv_heads, head_dim,
                                     as_stream(stream));
    });
}

} // extern "C"
