/* C ABI over the OpWorks-B200 operator layer (libopworks_ops.so).
 *
 * OpWorks exposes its operators to foreign callers through one-function
 * `extern "C" void solve(...)` adapters (tests/integration/*.cu: vector_add,
 * relu, reduction, softmax, layer_normalization, matrix_multiplication) that
 * run one op on device pointers and synchronise. This library exports the
 * same capability for every operator on the Llama hot path, one named symbol
 * per op, so a ctypes / cgo / JNI caller can bind them all from one .so.
 *
 * Conventions: every pointer is a DEVICE pointer unless stated otherwise;
 * `stream` is a cudaStream_t (NULL = legacy default stream); calls are
 * asynchronous unless they say otherwise. Functions return 0 on success and
 * -1 when the C++ API rejected the arguments (std::invalid_argument); the
 * message is then available from opw_ops_last_error() (thread-local). CUDA
 * runtime failures abort the process, as in OpWorks (OPWORKS_CUDA_CHECK).
 */
#ifndef OPWORKS_OPS_H
#define OPWORKS_OPS_H

#include <stddef.h>
#include <stdint.h>

/* Only the C ABI is exported; the libraries are built with hidden default
 * visibility so two of them (or the reference's library) can share a process. */
#ifndef OPW_API
#define OPW_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* Thread-local message of the last failed call. */
OPW_API const char *opw_ops_last_error(void);
/* Waits for `stream`; returns 0, or -1 if the device error word is set (a
 * bounded device-side wait ran out), clearing it. */
OPW_API int opw_ops_sync(void *stream);
/* The number of the graph capture that `stream` takes part in, 0 where it takes
 * part in none: what a caller keeps between calls belongs to one capture. */
OPW_API int opw_ops_capture_id(void *stream, int64_t *id);

/* ops::map with fixed functors (include/ops/elementwise.cuh:63-77;
 * tests/integration/vector_add.cu, relu.cu). */
OPW_API int opw_map_add(const float *a, const float *b, float *out, int n, void *stream);
OPW_API int opw_map_relu(const float *in, float *out, int n, void *stream);
OPW_API int opw_map_scale(const float *in, float *out, int n, float factor, void *stream);

/* ops::reduce<Sum|Max> (include/ops/reduction.cuh:34-67;
 * tests/integration/reduction.cu). kind: 0 = sum, 1 = max, 2 = product.
 * workspace may be NULL with workspace_size 0 to use stream-ordered scratch. */
OPW_API int opw_reduction_workspace_size(int n);
OPW_API int opw_reduce(int kind, const float *in, float *out, int n, float *workspace, int workspace_size, void *stream);

/* Allocation-free reduction: no reference counterpart (an extension of this
 * library). Same kinds and result as opw_reduce, with the workspace taken
 * from a static device buffer of 1025 floats (4100 bytes, the largest
 * workspace any n needs) instead of a caller buffer or a stream-ordered
 * allocation; a request that would need more is rejected with an error.
 * Each call clears the buffer's arrival counter before its kernel.
 * - The buffer is shared by every call on a device: calls that may overlap
 *   (different streams, host threads or graph branches without an ordering
 *   between them) race on it and must be serialised by the caller.
 * - The first call on each device looks the buffer's address up and must not
 *   run inside a stream capture; later calls may be captured. */
OPW_API int opw_reduce_static(int kind, const float *in, float *out, int n, void *stream);

/* ops::softmax / ops::layer_norm (softmax.cuh:36-43, layer_norm.cuh:38-47). */
OPW_API int opw_softmax(const float *in, float *out, int rows, int cols, void *stream);
OPW_API int opw_layer_norm(const float *in, float *out, const float *gamma, const float *beta, int rows, int cols, float eps,
                   void *stream);

/* ops::mat_mul (matmul.cuh:78-91): C(MxK) = epi(A(MxN) @ B(NxK)).
 * epilogue: 0 = pass-through, 1 = relu, 2 = scale by `param`. */
OPW_API int opw_mat_mul(const float *A, const float *B, float *C, int M, int N, int K, int epilogue, float param,
                void *stream);

/* MatmulBuilder + ops::matmul_launcher (builders/matmul.cuh:9-57): bias may
 * be NULL; activation 0 none, 1 relu, 2 gelu. */
OPW_API int opw_matmul_builder(const float *A, const float *B, float *C, int M, int N, int K, int transpose_a,
                       int transpose_b, const float *bias, int activation, void *stream);

/* RowwiseBuilder + ops::rowwise_launcher (builders/rowwise.cuh:11-63):
 * op 0 softmax, 1 layer_norm (param, beta), 2 rms_norm (param). */
OPW_API int opw_rowwise_builder(int op, const float *in, float *out, const float *param, const float *beta, int rows,
                        int cols, float eps, void *stream);

/* Model operators (include/ops/*.cuh of OpWorks, same argument order). */
OPW_API int opw_rms_norm(const float *x, const float *weight, float *out, int rows, int cols, float eps, void *stream);
OPW_API int opw_linear_f32(const float *X, const float *W, float *Y, int rows, int in_features, int out_features,
                   void *stream);
OPW_API int opw_linear_bf16(const float *X, const uint16_t *W_bf16, float *Y, int rows, int in_features, int out_features,
                    void *stream);
OPW_API int opw_linear_mma_bf16(const float *X, const uint16_t *W_bf16, float *Y, int rows, int in_features,
                        int out_features, void *stream);
OPW_API int opw_embedding_f32(const float *table, const int32_t *ids, float *out, int n, int hidden, void *stream);
OPW_API int opw_embedding_bf16(const uint16_t *table, const int32_t *ids, float *out, int n, int hidden, void *stream);
OPW_API int opw_rope(float *x, const float *inv_freq, int rows, int heads, int head_dim, int pos_start, void *stream);
OPW_API int opw_split_heads(const float *in, float *out, int rows, int heads, int head_dim, int out_row_stride,
                    int out_row_offset, void *stream);
OPW_API int opw_merge_heads(const float *in, float *out, int rows, int heads, int head_dim, int in_row_stride,
                    int in_row_offset, void *stream);
OPW_API int opw_causal_scale(float *scores, int rows, int cols, float scale, void *stream);
OPW_API int opw_swiglu(const float *gate, const float *up, float *out, int64_t n, void *stream);
OPW_API int opw_add(const float *a, const float *b, float *out, int64_t n, void *stream);
OPW_API int opw_argmax(const float *x, int n, int32_t *out, void *stream);
OPW_API int opw_attention_decode(const float *q, const float *kcache, const float *vcache, float *out, int num_q_heads,
                         int kv_rep, int head_dim, int len, int max_seq, void *stream);
OPW_API int opw_attention_prefill_chunked(const float *q_heads, const float *kcache, const float *vcache, float *out, int T,
                                  int S, int q_offset, int num_q_heads, int kv_rep, int head_dim, int cap,
                                  void *stream);

/* Fused greedy / top-p sampler of the Llama runtime (ops/llama_kernels.cuh),
 * the device form of OpWorks' host sampler examples/llama/generate.py:83-109:
 * one token per row of logits [rows, vocab]; temperature[r] <= 0 selects the
 * first argmax, otherwise top-p with uniform[r] (device arrays). */
OPW_API int opw_sample(const float *logits, int rows, int vocab, const float *temperature, const float *top_p,
               const double *uniform, int32_t *out, void *stream);

/* Batched decode attention over a paged fp32 KV cache (the Llama runtime's
 * kernel): q [B][qh*64], pools [blocks][kvh][16][64], block_table
 * [B][table_stride], lens[B] (device int32); out [B][qh*64] fp32. Scratch for
 * the split-KV partials comes from stream-ordered allocation. */
OPW_API int opw_paged_attention_decode(const float *q, const float *kpool, const float *vpool,
                                       const int32_t *block_table, int table_stride, const int32_t *lens, int B,
                                       int max_len, int num_q_heads, int num_kv_heads, float *out, void *stream);
/* Causal GQA prefill attention of query rows [0, T) of sequence b (absolute
 * positions q_offset + t) over a paged fp32 KV pool [num_blocks][kvh][16][64]
 * with block_table[b * table_stride + page]; q and out are [T][num_q_heads *
 * 64] fp32; head_dim 64, scale 1/8. tensor_cores = 1: TF32 tcgen05 flash
 * attention (include/ops/attention_prefill_tc.cuh); 0: the fp32 SIMT kernel.
 * Extension of this library (no reference counterpart; the reference's
 * prefill attention is ops::attention_prefill_chunked over contiguous K/V). */
OPW_API int opw_paged_attention_prefill(const float *q, const float *kpool, const float *vpool, const int32_t *block_table,
                                        int table_stride, int num_blocks, int b, int T, int q_offset, int num_q_heads,
                                        int num_kv_heads, float *out, int tensor_cores, void *stream);
/* out[split][M][N] (fp32 partials) = W[N][K] (bf16) . (Xhi + Xlo)[M][K]^T with
 * the runtime's two-term bf16 activation GEMM; splits = 0 picks the runtime's
 * split-K plan. Returns the split count used, or -1. */
OPW_API int opw_gemm_bf16x2(const uint16_t *W, const uint16_t *x_hi, const uint16_t *x_lo, float *out, int N, int K,
                            int M, int splits, void *stream);
/* out[M][N] (fp32) = W[N][K] (bf16) . (Xhi + Xlo)[M][K]^T by the two-SM
 * (tcgen05 cta_group::2) GEMM of the runtime's prefill projections: pairs of
 * CTAs compute 256 x 256 tiles (include/ops/gemm_sm100_pair.cuh). K must be a
 * multiple of 8. Extension of this library (no reference counterpart). */
OPW_API int opw_gemm_bf16x2_pair(const uint16_t *W, const uint16_t *x_hi, const uint16_t *x_lo, float *out, int N,
                                 int K, int M, void *stream);
/* The same two GEMMs with every 16-bit word read as fp16 instead of bf16 (the
 * format the runtime's fast path uses for float32 packs: 11 significant bits
 * at 2 bytes). The pair entry points accept x_lo == NULL: one activation term,
 * one MMA per K step. Extensions of this library (no reference counterpart). */
OPW_API int opw_gemm_f16x2(const uint16_t *W, const uint16_t *x_hi, const uint16_t *x_lo, float *out, int N, int K,
                           int M, int splits, void *stream);
OPW_API int opw_gemm_f16x2_pair(const uint16_t *W, const uint16_t *x_hi, const uint16_t *x_lo, float *out, int N,
                                int K, int M, void *stream);

/* ---- 8-bit paged KV cache (include/ops/kv_quant.cuh). Extensions of this
 * library (no reference counterpart).
 *
 * Pages of 16 tokens and block tables as in the fp32 pools; the pool holds one
 * record of 32 * head_dim + 128 bytes per (block, kv head): K codes
 * [16][head_dim], V codes [16][head_dim], K scales f32[16], V scales f32[16].
 * format: 1 = int8, 2 = e4m3; a row is code * scale with scale = max|x| / 127
 * (448), rounded to nearest even; a row with an infinity or a NaN has scale
 * NaN and codes 0. type of plain rows: 0 = fp32, 1 = bf16. head_dim 64 or 128.
 * Rows are ragged: sequence b owns rows [row_start[b], row_start[b + 1])
 * (device int32, batch + 1 of them, row_start[batch] == rows), at positions
 * first_pos[b] + 0, 1, ...; K and V of row r, head h lie at r * row_stride + h
 * * head_dim elements. Plain rows and the pool are 16-byte aligned, row_stride
 * too. Rows of positions outside the block table's row are left out. */
OPW_API int opw_kv_quant_record_bytes(int head_dim); /* -1: not a supported head_dim */
OPW_API int opw_kv_quant_write(const void *k, const void *v, int type, int64_t row_stride, uint8_t *pool, int format,
                               const int32_t *block_table, int table_stride, const int32_t *first_pos,
                               const int32_t *row_start, int batch, int rows, int num_kv_heads, int head_dim,
                               void *stream);
OPW_API int opw_kv_quant_read(const uint8_t *pool, int format, const int32_t *block_table, int table_stride,
                              const int32_t *first_pos, const int32_t *row_start, int batch, int rows,
                              int num_kv_heads, int head_dim, void *k, void *v, int type, int64_t row_stride,
                              void *stream);

/* ---- Several new tokens per sequence over a paged cache
 * (include/ops/tree_attention.cuh, include/ops/tree_commit.cuh). Extensions of
 * this library.
 *
 * The new (drafted) tokens of sequence b are nodes 0 .. n - 1 = rows
 * [row_start[b], row_start[b + 1]) of q and out; their K/V rows are already in
 * the cache at positions ctx_lens[b] + node. Node i attends to the context and
 * to the nodes j with bit j % 32 of mask[row][j / 32] set; mask NULL: to the
 * nodes j <= i (one row per sequence is a plain decode step). A node that sees
 * nothing gets zeros; a masked key has no influence whatever it holds.
 * max_rows: the most rows of one sequence (at most 32 * mask_words with a
 * mask); max_ctx: an upper bound of ctx_lens, which plans the launch only.
 * type: q and out fp32 (0) or bf16 (1); scores are scale * q . k; any number
 * of query heads per kv head; q_stride and out_stride in elements. q, out and
 * the pools are 16-byte aligned, and the row strides multiples of 16 bytes. */
OPW_API int opw_tree_attention(const void *q, int type, int64_t q_stride, const float *kpool, const float *vpool,
                               const int32_t *block_table, int table_stride, const int32_t *ctx_lens,
                               const int32_t *row_start, const uint32_t *mask, int mask_words, int batch, int rows,
                               int max_rows, int max_ctx, int num_q_heads, int num_kv_heads, int head_dim, float scale,
                               void *out, int64_t out_stride, void *stream);
OPW_API int opw_tree_attention_q8(const void *q, int type, int64_t q_stride, const uint8_t *pool, int format,
                                  const int32_t *block_table, int table_stride, const int32_t *ctx_lens,
                                  const int32_t *row_start, const uint32_t *mask, int mask_words, int batch, int rows,
                                  int max_rows, int max_ctx, int num_q_heads, int num_kv_heads, int head_dim,
                                  float scale, void *out, int64_t out_stride, void *stream);
/* Verifies drafted trees and keeps the accepted paths. draft[row]: the node's
 * token; target[row]: the token that the model chose after the node;
 * parent[row]: the node it follows (below it; -1 for node 0, the root, which is
 * always accepted). From a node the walk goes on to its child whose draft is
 * the node's target (the first of several). Writes path[row] (the accepted
 * nodes of each sequence in order, then -1), count[b], next[b] (the target of
 * the last accepted node; -1 for an empty tree) and new_lens[b] = ctx_lens[b] +
 * count[b] (not in place), and moves cache row ctx + path[i] to ctx + i in all
 * `layers` pools, layer_stride elements apart (floats; bytes in the _q8 form).
 * At most 2048 nodes per sequence. */
OPW_API int opw_tree_commit(const int32_t *draft, const int32_t *target, const int32_t *parent,
                            const int32_t *row_start, const int32_t *ctx_lens, int batch, int max_rows, float *kpool,
                            float *vpool, int64_t layer_stride, int layers, const int32_t *block_table,
                            int table_stride, int num_kv_heads, int head_dim, int32_t *path, int32_t *count,
                            int32_t *next, int32_t *new_lens, void *stream);
OPW_API int opw_tree_commit_q8(const int32_t *draft, const int32_t *target, const int32_t *parent,
                               const int32_t *row_start, const int32_t *ctx_lens, int batch, int max_rows,
                               uint8_t *pool, int64_t layer_stride, int layers, const int32_t *block_table,
                               int table_stride, int num_kv_heads, int head_dim, int32_t *path, int32_t *count,
                               int32_t *next, int32_t *new_lens, void *stream);

/* ---- Block tables and slot maps built on the GPU (include/ops/pages.cuh).
 * Extensions of this library.
 *
 * Sequence b holds lens[b] tokens in the first ceil(lens[b] / 16) pages of its
 * table row and gets rows [row_start[b], row_start[b + 1]) (device int32, batch +
 * 1 of them). free_blocks is a stack of free_count[0] block ids, taken from its
 * end, sequence by sequence. Writes the new ids into the table, position lens[b] +
 * i and slot 16 * block + position % 16 of every row (rows past the last
 * sequence's: position 0, slot -1) and what is left of the stack (free_left may be
 * free_count). free_blocks NULL: the table is complete; positions and slots only.
 * status[0]: 0; the pages missing; or -1 where a length is below zero, a sequence
 * longer than its table row, or a row past `rows`. Unless it is 0 nothing is taken
 * and every slot is -1. */
OPW_API int opw_page_take(const int32_t *lens, const int32_t *row_start, int batch, int rows, int32_t *block_table,
                          int table_stride, const int32_t *free_blocks, const int32_t *free_count, int32_t *positions,
                          int64_t *slots, int32_t *free_left, int32_t *status, void *stream);
/* The other way round: pages ceil(new / 16) .. ceil(old / 16) - 1 of each sequence
 * go onto the stack (room for `capacity` ids), in order; new >= old gives none.
 * status[0]: 0, or -1 (a length below zero or past the table row, a stack without
 * room), and then nothing is given. */
OPW_API int opw_page_give(const int32_t *old_lens, const int32_t *new_lens, int batch, const int32_t *block_table,
                          int table_stride, int32_t *free_blocks, int capacity, const int32_t *free_count,
                          int32_t *free_left, int32_t *status, void *stream);

/* ---- Norms of queries and keys for each head, and their rotation, in one pass
 * (include/ops/qk_norm_rope.cuh). Extension of this library.
 *
 * Head h of row r lies at r * stride + h * head_dim (head_dim 32, 64, 128 or 256),
 * type 0 fp32 or 1 bf16; x / sqrt(mean(x^2) + eps) * weight (fp32 [head_dim]; NULL:
 * that side is not normalised), then the pairs (i, i + rot_dim / 2) are turned by
 * positions[r] * inv_freq[i] (rot_dim a multiple of 16 up to head_dim; 0: no
 * rotation). The outputs may be the inputs. Rows are 16-byte aligned, strides too. */
OPW_API int opw_qk_norm_rope(const void *q, int64_t q_stride, const void *k, int64_t k_stride, int type,
                             const float *q_weight, const float *k_weight, float eps, const int32_t *positions,
                             const float *inv_freq, int rot_dim, int rows, int q_heads, int kv_heads, int head_dim,
                             void *q_out, int64_t q_out_stride, void *k_out, int64_t k_out_stride, void *stream);

/* ---- 4-bit paged KV cache (include/ops/kv4.cuh). Extensions of this library.
 *
 * One record of 18 * head_dim bytes per (block, kv head), G = head_dim / 32 groups
 * of 32 dims: K codes [G][16 tokens][16 bytes], V codes the same, K scales fp16
 * [G][16], V scales fp16 [G][16]; byte i of a group's 16 holds dims 2 i (low half)
 * and 2 i + 1. A value is (code - 8) * scale; scale = max|x| / 7 of the group,
 * rounded to 5 significant bits, code = 8 + x / scale rounded to nearest even, 1 to
 * 15. A group with a value above 55,552 (whose scale would be above 7,936), an
 * infinity or a NaN has scale NaN and codes 8. Row r of K and V goes to (comes
 * from) slot slots[r] = 16 * block + place of a pool of `blocks` blocks; rows with a
 * slot outside of it are left out. No two rows written have the same slot. type,
 * alignment and head_dim as in the 8-bit cache; K and V have a stride each. */
OPW_API int opw_kv4_record_bytes(int head_dim); /* -1: not a supported head_dim */
OPW_API int opw_kv4_write(const void *k, int64_t k_stride, const void *v, int64_t v_stride, int type, uint8_t *pool,
                          int blocks, const int64_t *slots, int rows, int num_kv_heads, int head_dim, void *stream);
OPW_API int opw_kv4_read(const uint8_t *pool, int blocks, const int64_t *slots, int rows, int num_kv_heads,
                         int head_dim, void *k, int64_t k_stride, void *v, int64_t v_stride, int type, void *stream);
/* opw_tree_attention and opw_tree_commit over the 4-bit pool (layer_stride in bytes).
 * Softmax weights: 22 bits where q is fp32, 11 where it is bf16 (their sum takes them
 * unrounded), which puts rows 1e-4 to 3e-4 off before they are rounded to bf16. A table
 * row that ends before ctx_lens + its rows ends the sequence there. */
OPW_API int opw_tree_attention_q4(const void *q, int type, int64_t q_stride, const uint8_t *pool,
                                  const int32_t *block_table, int table_stride, const int32_t *ctx_lens,
                                  const int32_t *row_start, const uint32_t *mask, int mask_words, int batch, int rows,
                                  int max_rows, int max_ctx, int num_q_heads, int num_kv_heads, int head_dim,
                                  float scale, void *out, int64_t out_stride, void *stream);
OPW_API int opw_tree_commit_q4(const int32_t *draft, const int32_t *target, const int32_t *parent,
                               const int32_t *row_start, const int32_t *ctx_lens, int batch, int max_rows,
                               uint8_t *pool, int64_t layer_stride, int layers, const int32_t *block_table,
                               int table_stride, int num_kv_heads, int head_dim, int32_t *path, int32_t *count,
                               int32_t *next, int32_t *new_lens, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* OPWORKS_OPS_H */
