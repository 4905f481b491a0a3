#pragma once

// An 8-bit form of the paged KV cache: rows quantised as they are written
// (ops::kv_quant_write) and read back (ops::kv_quant_read). No reference
// counterpart; the reference's cache is fp32 (include/runtime/kv_cache.cuh).
//
// Format. A row x of one token and kv head (D values of K, or of V) is held as
// 8-bit codes c and one fp32 scale s, x ~ c s:
//   a = max |x_i|,  s = a * fl(1 / Q),  c_i = round(x_i / s)
// Q = 127 for int8 (nearest integer, ties to even), 448 for e4m3 (nearest e4m3
// value). a = 0 (or so small that s is 0) gives s = 0 and c = 0. A row that
// holds an infinity or a NaN gets s = NaN and c = 0, so codes are always
// finite, and the row reads back as NaN in every place.
//
// Layout. Pages of 16 tokens like the fp32 pools', and one record per (block,
// kv head) of 32 D + 128 bytes:
//   K codes [16][D] | V codes [16][D] | K scales f32[16] | V scales f32[16]
// so the attention fetches a page of a head (K, V and both scales) with one
// bulk copy: 2,176 bytes at D = 64 against 8,192 in the fp32 pools.
//
// Both directions are bound by HBM; a row takes the memory it must and nothing is
// staged. Measured (kernel time, one B200; copy rate 6.45 TB/s): writing 32,768
// rows of 8 heads x 64 fp32 as int8 28.1 us, 5.0 TB/s (instructions: 57 % of the
// issue slots); reading 51,000 rows of 8 x 128 as bf16 55.4 us, 6.1 TB/s; the 32
// rows of a decode step 2.8 us, launch included.
//
// Rows are ragged: row r belongs to the sequence b with row_start[b] <= r <
// row_start[b + 1] and to position first_pos[b] + r - row_start[b].

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "../core/cuda_utils.cuh"

namespace opworks {

enum class KvFormat : int { kF32 = 0, kInt8 = 1, kE4M3 = 2 };

namespace detail {

constexpr int kKvPage = 16; // tokens per page

// Byte offsets inside a record.
template <int D> struct KvRecord {
    static constexpr int kCodes = kKvPage * D; // of K, and again of V
    static constexpr int kKScale = 2 * kCodes;
    static constexpr int kVScale = kKScale + 4 * kKvPage;
    static constexpr int kBytes = kVScale + 4 * kKvPage;
};

// The sequence that row `row` belongs to: the last one that starts at or
// before it (empty sequences start where the next one does). Whole warps, one
// row per warp: 32 starts per load instead of a chain of dependent loads.
__device__ __forceinline__ int sequence_of_row(const int *row_start, int batch, int row, int lane) {
    int n = 0;
    for (int base = 0; base < batch; base += 32) {
        const int i = base + lane;
        n += __popc(__ballot_sync(kFullWarpMask, i < batch && row_start[i] <= row));
    }
    return n - 1;
}

struct KvRowsArgs {
    const int *table;
    int table_stride;
    const int *first_pos;
    const int *row_start;
    int batch, rows, kvh;
};

// Block and slot of a row in the pool; false where the row belongs to no
// sequence or lies outside its row of the block table.
__device__ __forceinline__ bool kv_row_place(const KvRowsArgs &a, int row, int lane, int64_t &block, int &slot) {
    const int b = sequence_of_row(a.row_start, a.batch, row, lane);
    if (b < 0)
        return false;
    const int64_t pos = static_cast<int64_t>(a.first_pos[b]) + row - a.row_start[b];
    if (row >= a.row_start[b + 1] || pos < 0 || pos >= static_cast<int64_t>(a.table_stride) * kKvPage)
        return false;
    block = a.table[static_cast<int64_t>(b) * a.table_stride + pos / kKvPage];
    slot = static_cast<int>(pos % kKvPage);
    return true;
}

// 16 bytes of a row: 4 fp32 or 8 bf16 values.
template <typename T> struct KvVec;
template <> struct KvVec<float> {
    static constexpr int kN = 4;
    __device__ static void unpack(uint4 w, float (&x)[4]) {
        x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y);
        x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
    }
    __device__ static uint4 pack(const float (&x)[4]) {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
};
template <> struct KvVec<__nv_bfloat16> {
    static constexpr int kN = 8;
    __device__ static void unpack(uint4 w, float (&x)[8]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(u[i] << 16);
            x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
    __device__ static uint4 pack(const float (&x)[8]) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            u[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
};

constexpr float kInt8Top = 127.f, kE4M3Top = 448.f;

// The largest magnitude of three, NaN if one is.
__device__ __forceinline__ float max_abs_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four codes of x / s, the first in the low byte; inv is about 1 / s (NaN: do
// not use it). The quotients are those of an IEEE division: x * inv is within
// 2^-22 of them, so it gives the same code unless a rounding boundary lies that
// close, and then the division is made (a few elements in ten thousand).
template <KvFormat kFmt> __device__ __forceinline__ uint32_t kv_encode4(const float *x, float s, float inv) {
    const float2 i2 = make_float2(inv, inv);
    const float2 y0 = __fmul2_rn(make_float2(x[0], x[1]), i2), y1 = __fmul2_rn(make_float2(x[2], x[3]), i2);
    if constexpr (kFmt == KvFormat::kInt8) {
        constexpr float kRound = 12582912.f; // 1.5 2^23: the sum's low byte is the nearest integer
        const float2 up = make_float2(kRound, kRound), down = make_float2(-kRound, -kRound);
        const float2 t0 = __fadd2_rn(y0, up), t1 = __fadd2_rn(y1, up);
        const float2 r0 = __fadd2_rn(t0, down), r1 = __fadd2_rn(t1, down);
        const float2 d0 = __fadd2_rn(y0, make_float2(-r0.x, -r0.y)), d1 = __fadd2_rn(y1, make_float2(-r1.x, -r1.y));
        uint32_t c[4] = {__float_as_uint(t0.x), __float_as_uint(t0.y), __float_as_uint(t1.x), __float_as_uint(t1.y)};
        if (!(max_abs_nan(max_abs_nan(d0.x, d0.y, d1.x), d1.y, d1.y) < 0.4999f))
#pragma unroll
            for (int i = 0; i < 4; ++i)
                c[i] = static_cast<uint32_t>(max(-127, min(127, __float2int_rn(x[i] / s))));
        return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    } else {
        const auto four = [&](float a, float b, float c, float d) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
            return lo | (hi << 16);
        };
        constexpr float kLess = 1.f - 0x1p-21f, kMore = 1.f + 0x1p-21f;
        const float2 less = make_float2(kLess, kLess), more = make_float2(kMore, kMore);
        const float2 l0 = __fmul2_rn(y0, less), l1 = __fmul2_rn(y1, less), m0 = __fmul2_rn(y0, more), m1 = __fmul2_rn(y1, more);
        const uint32_t lo = four(l0.x, l0.y, l1.x, l1.y), hi = four(m0.x, m0.y, m1.x, m1.y);
        return lo == hi && inv == inv ? lo : four(x[0] / s, x[1] / s, x[2] / s, x[3] / s);
    }
}

template <KvFormat kFmt> __device__ __forceinline__ void kv_decode4(uint32_t w, float s, float *x) {
    if constexpr (kFmt == KvFormat::kInt8) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i))) * s;
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * i)), __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            x[2 * i] = f.x * s;
            x[2 * i + 1] = f.y * s;
        }
    }
}

constexpr int kKvThreads = 256;
// 16-byte pieces that a lane has in flight. Writing: 8 take as long for prompts
// and 3.6 us for 3.0 in a decode step; reading: 4 take 60.4 us for 55.1 (16
// prefixes of 4096 tokens, 128 dims, bf16), as the second half of a row then
// comes long after the first.
constexpr int kKvWritePasses = 4, kKvReadPasses = 8;

// A warp takes one row and kKvWritePasses x (32 / lanes per item) of its 2 x kvh
// items (K and V of each head). An item's D values lie on D / kN lanes, which
// find the maximum together.
template <typename T, int D, KvFormat kFmt>
static __global__ void __launch_bounds__(kKvThreads)
    kv_quant_write_kernel(const T *__restrict__ k, const T *__restrict__ v, int64_t stride, uint8_t *__restrict__ pool,
                          KvRowsArgs a) {
    using V = KvVec<T>;
    using R = KvRecord<D>;
    constexpr int kLanes = D / V::kN, kItems = 32 / kLanes;
    const int lane = threadIdx.x & 31;
    const int row = static_cast<int>(blockIdx.x) * (kKvThreads / 32) + static_cast<int>(threadIdx.x >> 5);
    pdl_wait();
    if (row >= a.rows)
        return;
    const int item0 = static_cast<int>(blockIdx.y) * kKvWritePasses * kItems + lane / kLanes;
    const int d0 = (lane % kLanes) * V::kN;
    uint4 raw[kKvWritePasses];
#pragma unroll
    for (int p = 0; p < kKvWritePasses; ++p) {
        const int item = item0 + p * kItems;
        raw[p] = make_uint4(0, 0, 0, 0);
        if (item < 2 * a.kvh)
            raw[p] = __ldcs(reinterpret_cast<const uint4 *>((item & 1 ? v : k) + row * stride + (item >> 1) * D + d0));
    }
    int64_t block;
    int slot;
    if (!kv_row_place(a, row, lane, block, slot))
        return;
    uint8_t *recs = pool + block * a.kvh * R::kBytes;
#pragma unroll
    for (int p = 0; p < kKvWritePasses; ++p) {
        const int item = item0 + p * kItems;
        float x[V::kN];
        V::unpack(raw[p], x);
        float top = max_abs_nan(x[0], x[1], x[2]); // NaN and infinity show
#pragma unroll
        for (int i = 3; i < V::kN; i += 2)
            top = max_abs_nan(top, x[i], x[i + 1 < V::kN ? i + 1 : i]);
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) {
            const float other = __shfl_xor_sync(kFullWarpMask, top, off);
            top = max_abs_nan(top, other, other);
        }
        if (item >= 2 * a.kvh)
            continue;
        constexpr float kInv = 1.f / (kFmt == KvFormat::kInt8 ? kInt8Top : kE4M3Top);
        const float s = top < __uint_as_float(0x7f800000u) ? top * kInv : __uint_as_float(0x7fc00000u);
        uint32_t codes[V::kN / 4] = {};
        if (s > 0.f) {
            const float inv = s > 0x1p-120f && s < 0x1p+120f ? rcp_approx(s) : __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int i = 0; i < V::kN / 4; ++i)
                codes[i] = kv_encode4<kFmt>(x + 4 * i, s, inv);
        }
        uint8_t *rec = recs + (item >> 1) * R::kBytes;
        uint8_t *dst = rec + (item & 1) * R::kCodes + slot * D + d0;
        if constexpr (V::kN == 4)
            *reinterpret_cast<uint32_t *>(dst) = codes[0];
        else
            *reinterpret_cast<uint2 *>(dst) = make_uint2(codes[0], codes[V::kN / 4 - 1]);
        if (lane % kLanes == 0)
            *reinterpret_cast<float *>(rec + (item & 1 ? R::kVScale : R::kKScale) + 4 * slot) = s;
    }
}

// The same shape the other way round: codes times scale, one 16-byte store of
// the output type per lane and pass.
template <typename T, int D, KvFormat kFmt>
static __global__ void __launch_bounds__(kKvThreads)
    kv_quant_read_kernel(const uint8_t *__restrict__ pool, T *__restrict__ k, T *__restrict__ v, int64_t stride,
                         KvRowsArgs a) {
    using V = KvVec<T>;
    using R = KvRecord<D>;
    constexpr int kLanes = D / V::kN, kItems = 32 / kLanes;
    const int lane = threadIdx.x & 31;
    const int row = static_cast<int>(blockIdx.x) * (kKvThreads / 32) + static_cast<int>(threadIdx.x >> 5);
    pdl_wait();
    if (row >= a.rows)
        return;
    const int item0 = static_cast<int>(blockIdx.y) * kKvReadPasses * kItems + lane / kLanes;
    const int d0 = (lane % kLanes) * V::kN;
    int64_t block;
    int slot;
    if (!kv_row_place(a, row, lane, block, slot))
        return;
    uint2 codes[kKvReadPasses];
    float scale[kKvReadPasses];
#pragma unroll
    for (int p = 0; p < kKvReadPasses; ++p) {
        const int item = item0 + p * kItems;
        codes[p] = make_uint2(0, 0);
        scale[p] = 0.f;
        if (item < 2 * a.kvh) {
            const uint8_t *rec = pool + (block * a.kvh + (item >> 1)) * R::kBytes;
            const uint8_t *src = rec + (item & 1) * R::kCodes + slot * D + d0;
            if constexpr (V::kN == 4)
                codes[p].x = *reinterpret_cast<const uint32_t *>(src);
            else
                codes[p] = *reinterpret_cast<const uint2 *>(src);
            scale[p] = *reinterpret_cast<const float *>(rec + (item & 1 ? R::kVScale : R::kKScale) + 4 * slot);
        }
    }
#pragma unroll
    for (int p = 0; p < kKvReadPasses; ++p) {
        const int item = item0 + p * kItems;
        if (item >= 2 * a.kvh)
            continue;
        float x[V::kN];
        kv_decode4<kFmt>(codes[p].x, scale[p], x);
        if constexpr (V::kN == 8)
            kv_decode4<kFmt>(codes[p].y, scale[p], x + 4);
        __stcs(reinterpret_cast<uint4 *>((item & 1 ? v : k) + row * stride + (item >> 1) * D + d0), V::pack(x));
    }
}

inline bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

inline void validate_kv_rows(const KvRowsArgs &a, int head_dim) {
    require(a.batch >= 0 && a.rows >= 0, "kv cache rows: batch and rows must be nonnegative");
    require(a.kvh > 0 && a.kvh <= 4096, "kv cache rows: 1 to 4096 kv heads are supported");
    require(head_dim == 64 || head_dim == 128, "kv cache rows: head_dim must be 64 or 128");
    require(a.table_stride > 0, "kv cache rows: table_stride must be positive");
}

template <typename T>
inline void validate_kv_io(const void *k, const void *v, int64_t stride, const void *pool, const KvRowsArgs &a,
                           int head_dim) {
    require(k && v && pool && a.table && a.first_pos && a.row_start, "kv cache rows: null pointer");
    require(stride >= static_cast<int64_t>(a.kvh) * head_dim, "kv cache rows: rows overlap (stride below kvh * head_dim)");
    require(aligned16(k) && aligned16(v) && aligned16(pool) && (stride * static_cast<int64_t>(sizeof(T))) % 16 == 0,
            "kv cache rows: rows and pool must be 16-byte aligned");
}

// A warp per row and kPasses x (32 / lanes per item) of its items.
template <typename T, int D, int kPasses> inline dim3 kv_row_grid(int rows, int kvh) {
    constexpr int kPer = kPasses * 32 / (D / KvVec<T>::kN), kWarps = kKvThreads / 32;
    return dim3(static_cast<unsigned>(rows / kWarps + (rows % kWarps != 0)), static_cast<unsigned>((2 * kvh + kPer - 1) / kPer));
}

// f(std::integral_constant-like tags) for the two formats and head sizes.
template <typename F> inline void kv_dispatch(KvFormat fmt, int head_dim, F &&f) {
    require(fmt == KvFormat::kInt8 || fmt == KvFormat::kE4M3, "kv cache rows: format must be int8 (1) or e4m3 (2)");
    if (fmt == KvFormat::kInt8)
        head_dim == 64 ? f.template operator()<64, KvFormat::kInt8>() : f.template operator()<128, KvFormat::kInt8>();
    else
        head_dim == 64 ? f.template operator()<64, KvFormat::kE4M3>() : f.template operator()<128, KvFormat::kE4M3>();
}

template <typename T> struct KvWriteCall {
    const T *k, *v;
    int64_t stride;
    uint8_t *pool;
    KvRowsArgs a;
    cudaStream_t stream;
    template <int D, KvFormat kFmt> void operator()() const {
        launch_ex(kv_quant_write_kernel<T, D, kFmt>, kv_row_grid<T, D, kKvWritePasses>(a.rows, a.kvh), dim3(kKvThreads), 0, stream, k, v,
                  stride, pool, a);
    }
};

template <typename T> struct KvReadCall {
    const uint8_t *pool;
    T *k, *v;
    int64_t stride;
    KvRowsArgs a;
    cudaStream_t stream;
    template <int D, KvFormat kFmt> void operator()() const {
        launch_ex(kv_quant_read_kernel<T, D, kFmt>, kv_row_grid<T, D, kKvReadPasses>(a.rows, a.kvh), dim3(kKvThreads), 0, stream, pool,
                  k, v, stride, a);
    }
};

} // namespace detail

namespace ops {

// Bytes of one (block, kv head) record of the 8-bit pool.
inline int kv_quant_record_bytes(int head_dim) {
    detail::require(head_dim == 64 || head_dim == 128, "kv cache rows: head_dim must be 64 or 128");
    return 2 * detail::kKvPage * head_dim + 8 * detail::kKvPage;
}

// Quantises rows [0, rows) of K and V (row r, head h at r * stride + h *
// head_dim; T fp32 or bf16) into the pages of their sequences.
template <typename T>
inline void kv_quant_write(const T *k, const T *v, int64_t stride, uint8_t *pool, KvFormat format,
                           const int *block_table, int table_stride, const int *first_pos, const int *row_start,
                           int batch, int rows, int kv_heads, int head_dim, cudaStream_t stream = nullptr) {
    const detail::KvRowsArgs a{block_table, table_stride, first_pos, row_start, batch, rows, kv_heads};
    detail::validate_kv_rows(a, head_dim);
    if (batch == 0 || rows == 0)
        return;
    detail::validate_kv_io<T>(k, v, stride, pool, a, head_dim);
    detail::kv_dispatch(format, head_dim, detail::KvWriteCall<T>{k, v, stride, pool, a, stream});
}

// Reads the same rows back: code * scale in fp32, rounded once to T.
template <typename T>
inline void kv_quant_read(const uint8_t *pool, KvFormat format, const int *block_table, int table_stride,
                          const int *first_pos, const int *row_start, int batch, int rows, int kv_heads, int head_dim,
                          T *k, T *v, int64_t stride, cudaStream_t stream = nullptr) {
    const detail::KvRowsArgs a{block_table, table_stride, first_pos, row_start, batch, rows, kv_heads};
    detail::validate_kv_rows(a, head_dim);
    if (batch == 0 || rows == 0)
        return;
    detail::validate_kv_io<T>(k, v, stride, pool, a, head_dim);
    detail::kv_dispatch(format, head_dim, detail::KvReadCall<T>{pool, k, v, stride, a, stream});
}

} // namespace ops
} // namespace opworks
