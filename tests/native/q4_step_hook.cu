// Test-only hook (not part of the product; built into tests/native/ by
// oracle/build_ref.py): steps of taking pages, norm and rotation, store, attention
// and commit, reading back and giving back over one 4-bit cache (head size 64),
// with or without programmatic launches.

#include <exception>

#include "ops/kv4.cuh"
#include "ops/pages.cuh"
#include "ops/qk_norm_rope.cuh"
#include "ops/tree_attention_q4.cuh"
#include "ops/tree_commit.cuh"

using namespace opworks;

// Step s of rows qkv + s * rows * (qh + 2 kvh) * 64, normalised and rotated in place; out + s rows qh 64; back + 2 s rows kvh
// 64 (K, then V); lens [steps + 1][batch], of which the first is given.
extern "C" __attribute__((visibility("default"))) int q4_step_run(int programmatic, int steps, float *qkv, const float *weight, const float *inv_freq, uint8_t *pool,
                             int blocks, int *table, int stride, int *free_blocks, int *free_count, const int *start, const int *ends, int batch, int rows,
                             int most, int max_ctx, int qh, int kvh, const int *draft, const int *target, const int *parent, int *path, int *count, int *next,
                             int *lens, int *full, int *positions, int64_t *slots, int *status, float *out, float *back, void *stream) {
    try {
        const PdlScope scope(programmatic != 0);
        const auto st = static_cast<cudaStream_t>(stream);
        const int64_t wide = (qh + 2 * kvh) * 64, row = kvh * 64;
        for (int s = 0; s < steps; ++s) {
            float *q = qkv + s * rows * wide, *k = q + qh * 64, *v = k + row, *b = back + 2 * s * rows * row;
            const int *ctx = lens + s * batch;
            ops::page_take({ctx, start, batch, rows, table, stride, free_blocks, free_count, positions, slots, free_count, status + s}, st);
            ops::qk_norm_rope(QkNormRope<float>{q, wide, k, wide, weight, weight, 1e-5f, positions, inv_freq, 64, rows, qh, kvh, 64, q, wide, k, wide}, st);
            ops::kv4_write(k, wide, v, wide, pool, blocks, slots, rows, kvh, 64, st);
            const TreeBatch t{table, stride, ctx, start, nullptr, 0, batch, rows, most, max_ctx};
            ops::tree_attention_q4(q, wide, pool, t, qh, kvh, 64, 0.125f, out + static_cast<int64_t>(s) * rows * qh * 64, static_cast<int64_t>(qh) * 64, st);
            const TreeVerify c{draft, target, parent, start, ctx, batch, most, path + s * rows, count + s * batch, next + s * batch, lens + (s + 1) * batch};
            ops::tree_commit_q4(c, pool, 0, 1, table, stride, kvh, 64, st);
            ops::kv4_read(pool, blocks, slots, rows, kvh, 64, b, row, b + rows * row, row, st);
            // ends[b]: what the step's rows reached to, of which the commit keeps less
            ops::page_give({ends + s * batch, lens + (s + 1) * batch, batch, table, stride, free_blocks, blocks, free_count, free_count, full + s}, st);
        }
        return 0;
    } catch (const std::exception &) {
        return -1;
    }
}
