// Test-only hook (not part of the product; built into tests/native/ by
// oracle/build_ref.py): steps of write, attend, commit and read back over one
// 8-bit cache (int8, head size 64), with or without programmatic launches.

#include <exception>

#include "ops/kv_quant.cuh"
#include "ops/tree_attention_common.cuh"
#include "ops/tree_attention_rows.cuh"
#include "ops/tree_commit.cuh"

using namespace opworks;

// Step s writes rows k + s * rows * kvh * 64 (and v) of every sequence after its context, attends to them with q into
// out + s * rows * qh * 64, commits the trees, and reads the rows back into back + 2 s rows kvh 64 (K, then V).
extern "C" __attribute__((visibility("default"))) int tree_step_run(int programmatic, int steps, const float *q, const float *k, const float *v, uint8_t *pool,
                             const int *table, int stride, const int *ctx, const int *start, int batch, int rows, int most,
                             int max_ctx, int qh, int kvh, const int *draft, const int *target, const int *parent, int *path,
                             int *count, int *next, int *lens, float *out, float *back, void *stream) {
    try {
        const PdlScope scope(programmatic != 0);
        const auto st = static_cast<cudaStream_t>(stream);
        const int64_t row = kvh * 64;
        for (int s = 0; s < steps; ++s) {
            ops::kv_quant_write(k + s * rows * row, v + s * rows * row, row, pool, KvFormat::kInt8, table, stride, ctx, start,
                                batch, rows, kvh, 64, st);
            const TreeBatch t{table, stride, ctx, start, nullptr, 0, batch, rows, most, max_ctx};
            const detail::TreeArgs a{t, pool, pool, qh, kvh, 0.125f * detail::kLog2e, qh * 64, qh * 64};
            detail::tree_rows_launch<float, 64, KvFormat::kInt8, 1>(q, out + static_cast<int64_t>(s) * rows * qh * 64, a, st);
            const TreeVerify c{draft, target, parent, start, ctx, batch, most, path + s * rows, count + s * batch,
                               next + s * batch, lens + s * batch};
            ops::tree_commit_q8(c, pool, 0, 1, table, stride, kvh, 64, st);
            float *b = back + 2 * static_cast<int64_t>(s) * rows * row;
            ops::kv_quant_read(pool, KvFormat::kInt8, table, stride, ctx, start, batch, rows, kvh, 64, b, b + rows * row, row, st);
        }
        return 0;
    } catch (const std::exception &) {
        return -1;
    }
}
