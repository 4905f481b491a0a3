// libopworks_ops.so, second part: the 8-bit paged KV cache and the drafted-
// token step (attention and commit) over paged caches. Same conventions as
// ops_c_api.cu.

#include "opworks_ops.h"
#include "ops/kv_quant.cuh"
#include "ops/tree_attention.cuh"
#include "ops/tree_commit.cuh"
#include "ops_guard.h"

using opworks_ops::guarded;

namespace {

using opworks::KvFormat;
using opworks::TreeBatch;
using opworks::TreeVerify;

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

int opw_kv_quant_record_bytes(int head_dim) {
    int r = -1;
    guarded([&] { r = opworks::ops::kv_quant_record_bytes(head_dim); });
    return r;
}

int opw_kv_quant_write(const void *k, const void *v, int type, int64_t row_stride, uint8_t *pool, int format,
                       const int32_t *block_table, int table_stride, const int32_t *first_pos,
                       const int32_t *row_start, int batch, int rows, int num_kv_heads, int head_dim, void *stream) {
    return guarded([&] {
        with_type(type, [&](auto *t) {
            opworks::ops::kv_quant_write(as(k, t), as(v, t), row_stride, pool, static_cast<KvFormat>(format),
                                         block_table, table_stride, first_pos, row_start, batch, rows, num_kv_heads,
                                         head_dim, as_stream(stream));
        });
    });
}

int opw_kv_quant_read(const uint8_t *pool, int format, const int32_t *block_table, int table_stride,
                      const int32_t *first_pos, const int32_t *row_start, int batch, int rows, int num_kv_heads,
                      int head_dim, void *k, void *v, int type, int64_t row_stride, void *stream) {
    return guarded([&] {
        with_type(type, [&](auto *t) {
            opworks::ops::kv_quant_read(pool, static_cast<KvFormat>(format), block_table, table_stride, first_pos,
                                        row_start, batch, rows, num_kv_heads, head_dim, as(k, t), as(v, t), row_stride,
                                        as_stream(stream));
        });
    });
}

int opw_tree_attention(const void *q, int type, int64_t q_stride, const float *kpool, const float *vpool,
                       const int32_t *block_table, int table_stride, const int32_t *ctx_lens, const int32_t *row_start,
                       const uint32_t *mask, int mask_words, int batch, int rows, int max_rows, int max_ctx,
                       int num_q_heads, int num_kv_heads, int head_dim, float scale, void *out, int64_t out_stride,
                       void *stream) {
    return guarded([&] {
        const TreeBatch b{block_table, table_stride, ctx_lens, row_start, mask, mask_words, batch, rows, max_rows, max_ctx};
        with_type(type, [&](auto *t) {
            opworks::ops::tree_attention(as(q, t), q_stride, kpool, vpool, b, num_q_heads, num_kv_heads, head_dim,
                                         scale, as(out, t), out_stride, as_stream(stream));
        });
    });
}

int opw_tree_attention_q8(const void *q, int type, int64_t q_stride, const uint8_t *pool, int format,
                          const int32_t *block_table, int table_stride, const int32_t *ctx_lens,
                          const int32_t *row_start, const uint32_t *mask, int mask_words, int batch, int rows,
                          int max_rows, int max_ctx, int num_q_heads, int num_kv_heads, int head_dim, float scale,
                          void *out, int64_t out_stride, void *stream) {
    return guarded([&] {
        const TreeBatch b{block_table, table_stride, ctx_lens, row_start, mask, mask_words, batch, rows, max_rows, max_ctx};
        with_type(type, [&](auto *t) {
            opworks::ops::tree_attention_q8(as(q, t), q_stride, pool, static_cast<KvFormat>(format), b, num_q_heads,
                                            num_kv_heads, head_dim, scale, as(out, t), out_stride, as_stream(stream));
        });
    });
}

int opw_tree_commit(const int32_t *draft, const int32_t *target, const int32_t *parent, const int32_t *row_start,
                    const int32_t *ctx_lens, int batch, int max_rows, float *kpool, float *vpool, int64_t layer_stride,
                    int layers, const int32_t *block_table, int table_stride, int num_kv_heads, int head_dim,
                    int32_t *path, int32_t *count, int32_t *next, int32_t *new_lens, void *stream) {
    return guarded([&] {
        const TreeVerify t{draft, target, parent, row_start, ctx_lens, batch, max_rows, path, count, next, new_lens};
        opworks::ops::tree_commit(t, kpool, vpool, layer_stride, layers, block_table, table_stride, num_kv_heads,
                                  head_dim, as_stream(stream));
    });
}

int opw_tree_commit_q8(const int32_t *draft, const int32_t *target, const int32_t *parent, const int32_t *row_start,
                       const int32_t *ctx_lens, int batch, int max_rows, uint8_t *pool, int64_t layer_stride,
                       int layers, const int32_t *block_table, int table_stride, int num_kv_heads, int head_dim,
                       int32_t *path, int32_t *count, int32_t *next, int32_t *new_lens, void *stream) {
    return guarded([&] {
        const TreeVerify t{draft, target, parent, row_start, ctx_lens, batch, max_rows, path, count, next, new_lens};
        opworks::ops::tree_commit_q8(t, pool, layer_stride, layers, block_table, table_stride, num_kv_heads, head_dim,
                                     as_stream(stream));
    });
}

} // extern "C"
