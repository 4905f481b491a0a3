#pragma once

// A 4-bit form of the paged KV cache: rows stored where a slot map says
// (ops::kv4_write) and fetched again (ops::kv4_read). No reference counterpart;
// the reference's cache is fp32 (include/runtime/kv_cache.cuh).
//
// Format. A row of one token and kv head (D values of K, or of V) is held in
// groups of 32 dims, as 4-bit codes c of -7 .. 7 and one scale s a group:
//   s = max |x_i| / 7 rounded to an fp16 number of 5 significant bits
//   c_i = round(x_i / s), ties to even; x_i ~ c_i s, off by at most s / 2
// (below 2^-20 fp16 has fewer bits: s is a multiple of 2^-24, and c is held at
// 7). c s has at most 8 significant bits, so what is held is an fp16 number and
// a bf16 number: attention multiplies codes and scales out for the tensor cores
// with nothing lost, and reading back as bf16 is exact. 5 bits and not all of
// fp16's make a scale 3.1 % wider or narrower at most. s goes up to 7,936, so the largest value
// is 55,552; a group with a larger one (its s would round above), an infinity or
// a NaN gets s = NaN and reads back as NaN in every place. s = 0: all zeros.
//
// Layout. Pages of 16 tokens, a record of 576 G bytes per (block, kv head), G =
// D / 32 (1,152 bytes at D = 64; 8,192 in the fp32 pools, 2,176 in 8 bits):
//   K codes [G][16 tokens][16 bytes] | V codes the same |
//   K scales fp16 [G][16] | V scales fp16 [G][16]
// Byte i of a group's 16 holds c + 8 of dims 2 i (low half) and 2 i + 1, so that
// 8 tokens of a group are one 8 x 8 matrix of 16-bit elements, which ldmatrix
// hands out as K's fragments and, transposed, as V's.
//
// The slot of a row is 16 * block + place in the page; rows with a slot below
// zero or past the pool are left out (padded batches).
//
// Both directions are bound by HBM. Measured (kernel time, one B200; copy rate 6.46
// TB/s): writing 26,000 rows of 8 heads x 128 in bf16 26.8 us, 5.4 TB/s, in fp32 (L2
// holds part of them) 34.4 us; reading them back as bf16 27.7 us, 5.2 TB/s, as fp32 43.8
// us, 5.8 TB/s; the 32 rows of a decode step about 2 us each way, launch included.

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../core/cuda_utils.cuh"
#include "kv_quant.cuh"

namespace opworks {
namespace detail {

constexpr int kKv4Group = 32; // dims that share a scale

// Byte offsets inside a record.
template <int D> struct Kv4Record {
    static constexpr int kGroups = D / kKv4Group;
    static constexpr int kCodes = kGroups * kKvPage * 16; // of K, and again of V
    static constexpr int kKScale = 2 * kCodes;
    static constexpr int kVScale = kKScale + 2 * kGroups * kKvPage;
    static constexpr int kBytes = kVScale + 2 * kGroups * kKvPage;
};

constexpr uint32_t kKv4MaxScale = 0x45f80000u; // fp32 bits of 7,936

// The scale of a group whose largest magnitude is `top` (NaN or infinity: one of them is).
__device__ __forceinline__ float kv4_scale(float top) {
    const float t = top * (1.f / 7.f);
    if (t < 0x1p-20f)
        return __half2float(__float2half_rn(t));
    const uint32_t u = __float_as_uint(t), s = (u + 0x3ffffu + ((u >> 19) & 1u)) & ~0x7ffffu;
    return __uint_as_float(s <= kKv4MaxScale && top <= 3.4028235e38f ? s : 0x7fc00000u);
}

// Eight codes + 8 of x / s, the first in the lowest bits; inv = 1 / s, rounded to
// nearest. The quotients are correctly rounded (Markstein, IBM J. Res. Dev. 34, 1990:
// from such a reciprocal y, q = x y, then q + (x - q s) y is): a code is that of an
// IEEE division, ties included, which half-way numbers of bf16 rows often are. Sums
// of codes times powers of 16 are exact in fp32, four codes to a sum.
__device__ __forceinline__ uint32_t kv4_encode8(const float (&x)[8], float s, float inv) {
    constexpr float kRound = 12582912.f, kBias = kRound + 0x8888; // 1.5 2^23: what is added to it is rounded to an integer
    const float2 y = make_float2(inv, inv), less = make_float2(-s, -s), up = make_float2(kRound, kRound), down = make_float2(-kRound, -kRound);
    float2 r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = make_float2(x[2 * i], x[2 * i + 1]), q = __fmul2_rn(v, y);
        r[i] = __fadd2_rn(__fadd2_rn(__ffma2_rn(__ffma2_rn(q, less, v), y, q), up), down);
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 e = __ffma2_rn(r[2 * i + 1], make_float2(256.f, 256.f), r[2 * i]);
        w[i] = __float_as_uint(fmaf(e.y, 16.f, e.x + kBias));
    }
    return __byte_perm(w[0], w[1], 0x5410);
}

// The same for scales near or below the smallest normal numbers, and none (0, NaN).
__device__ __forceinline__ uint32_t kv4_encode8_small(const float (&x)[8], float s) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i)
        w = (w << 4) | static_cast<uint32_t>(s > 0.f ? 8 + max(-7, min(7, __float2int_rn(x[i] / s))) : 8);
    return w;
}

// (w & kMask) | kOr in one instruction; written out in C it takes two.
template <uint32_t kMask, uint32_t kOr> __device__ __forceinline__ uint32_t kv4_pick(uint32_t w) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(w), "n"(kMask), "n"(kOr));
    return d;
}
__device__ __forceinline__ __half2 kv4_half2(uint32_t u) { return *reinterpret_cast<const __half2 *>(&u); }
__device__ __forceinline__ uint32_t kv4_bits(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// Four pairs of codes from the eight of a word, as fp16 numbers: (0, 4), (1, 5), (2,
// 6), (3, 7). A code + 8 goes into the low bits of fp16 1024 .. 1039 (or, 16-fold, 1024
// .. 1264), from which 1032 (72) is taken away: the way of Kim et al., "Who Says Elephants
// Can't Run", 2022, from integers to floating point, with this format's offsets.
__device__ __forceinline__ void kv4_integers(uint32_t w, __half2 (&h)[4]) {
    const uint32_t hi = w >> 8;
    const auto low = [](uint32_t u) { return __hsub2(kv4_half2(kv4_pick<0x000f000fu, 0x64006400u>(u)), kv4_half2(0x64086408u)); };
    const auto high = [](uint32_t u) { // 1 / 16, -72
        return __hfma2(kv4_half2(kv4_pick<0x00f000f0u, 0x64006400u>(u)), kv4_half2(0x2c002c00u), kv4_half2(0xd480d480u));
    };
    h[0] = low(w), h[1] = high(w), h[2] = low(hi), h[3] = high(hi);
}

// The same times the pair `scale`. Exact.
__device__ __forceinline__ void kv4_widen(uint32_t w, __half2 scale, uint32_t (&h)[4]) {
    __half2 c[4];
    kv4_integers(w, c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        h[i] = kv4_bits(__hmul2(c[i], scale));
}

struct Kv4Rows {
    const int64_t *slots;
    int rows, kvh;
    int64_t places; // 16 * blocks of the pool
};

constexpr int kKv4Threads = 256;
// Times 8 groups of K and of V that a warp has in flight. Writing, more cost registers
// and so warps (26,000 rows of 8 x 128, bf16: 26.8 us with 1, 35.8 with 2, 57.8 with 4);
// reading, less leaves too few loads (31.9, 27.7, 27.8).
constexpr int kKv4WritePasses = 1, kKv4ReadPasses = 2;

// A lane's eight values of a row.
template <typename T> __device__ __forceinline__ void kv4_load8(const T *p, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8 / KvVec<T>::kN; ++i) {
        float y[KvVec<T>::kN];
        KvVec<T>::unpack(__ldcs(reinterpret_cast<const uint4 *>(p) + i), y);
#pragma unroll
        for (int j = 0; j < KvVec<T>::kN; ++j)
            x[i * KvVec<T>::kN + j] = y[j];
    }
}
// A warp takes one row and 8 * kKv4WritePasses of its kvh * G groups, K and V of each:
// four lanes a group, eight dims a lane.
template <typename T, int D>
static __global__ void __launch_bounds__(kKv4Threads)
    kv4_write_kernel(const T *__restrict__ k, int64_t k_stride, const T *__restrict__ v, int64_t v_stride,
                     uint8_t *__restrict__ pool, Kv4Rows a) {
    using R = Kv4Record<D>;
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kKv4Threads / 32) + (threadIdx.x >> 5);
    pdl_wait();
    if (row >= a.rows)
        return;
    const int groups = a.kvh * R::kGroups, group0 = static_cast<int>(blockIdx.y) * kKv4WritePasses * 8 + lane / 4;
    float x[2 * kKv4WritePasses][8] = {};
#pragma unroll
    for (int p = 0; p < kKv4WritePasses; ++p) {
        const int at = group0 + 8 * p;
        if (at < groups) {
            kv4_load8(k + row * k_stride + at * kKv4Group + lane % 4 * 8, x[2 * p]);
            kv4_load8(v + row * v_stride + at * kKv4Group + lane % 4 * 8, x[2 * p + 1]);
        }
    }
    const int64_t place = a.slots[row];
    if (place < 0 || place >= a.places)
        return;
    const int slot = static_cast<int>(place % kKvPage);
    uint8_t *recs = pool + place / kKvPage * a.kvh * R::kBytes;
#pragma unroll
    for (int p = 0; p < 2 * kKv4WritePasses; ++p) {
        const float(&y)[8] = x[p];
        float top = max_abs_nan(max_abs_nan(max_abs_nan(y[0], y[1], y[2]), y[3], y[4]), max_abs_nan(y[5], y[6], y[7]), 0.f);
#pragma unroll
        for (int off = 1; off < 4; off <<= 1)
            top = max_abs_nan(top, __shfl_xor_sync(kFullWarpMask, top, off), 0.f);
        const int at = group0 + 8 * (p / 2);
        if (at >= groups)
            continue;
        const float s = kv4_scale(top);
        const uint32_t w = s >= 0x1p-20f ? kv4_encode8(y, s, __frcp_rn(s)) : kv4_encode8_small(y, s);
        uint8_t *rec = recs + at / R::kGroups * R::kBytes;
        const int g = at % R::kGroups;
        *reinterpret_cast<uint32_t *>(rec + (p & 1 ? R::kCodes : 0) + (g * kKvPage + slot) * 16 + lane % 4 * 4) = w;
        if (lane % 4 == 0)
            *reinterpret_cast<__half *>(rec + (p & 1 ? R::kVScale : R::kKScale) + (g * kKvPage + slot) * 2) = __float2half_rn(s);
    }
}

// The other way round, 16 bytes of the output a lane: 4 (fp32) or 8 lanes' worth of a
// group's 32 dims, so that a warp's store is one run of 512 bytes.
template <typename T, int D>
static __global__ void __launch_bounds__(kKv4Threads)
    kv4_read_kernel(const uint8_t *__restrict__ pool, T *__restrict__ k, int64_t k_stride, T *__restrict__ v, int64_t v_stride,
                    Kv4Rows a) {
    using R = Kv4Record<D>;
    constexpr int kN = KvVec<T>::kN, kLanes = kKv4Group / kN, kPer = 32 / kLanes, kPasses = kKv4ReadPasses * 8 / kPer;
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (kKv4Threads / 32) + (threadIdx.x >> 5);
    pdl_wait();
    if (row >= a.rows)
        return;
    const int64_t place = a.slots[row];
    if (place < 0 || place >= a.places)
        return;
    const int slot = static_cast<int>(place % kKvPage);
    const uint8_t *recs = pool + place / kKvPage * a.kvh * R::kBytes;
    const int groups = a.kvh * R::kGroups, group0 = static_cast<int>(blockIdx.y) * kKv4ReadPasses * 8 + lane / kLanes, part = lane % kLanes;
    uint32_t w[2 * kPasses];
    __half s[2 * kPasses];
#pragma unroll
    for (int p = 0; p < 2 * kPasses; ++p) {
        const int at = min(group0 + kPer * (p / 2), groups - 1), g = at % R::kGroups;
        const uint8_t *rec = recs + at / R::kGroups * R::kBytes;
        const uint8_t *codes = rec + (p & 1 ? R::kCodes : 0) + (g * kKvPage + slot) * 16;
        if constexpr (kN == 8)
            w[p] = reinterpret_cast<const uint32_t *>(codes)[part];
        else
            w[p] = reinterpret_cast<const uint16_t *>(codes)[part];
        s[p] = *reinterpret_cast<const __half *>(rec + (p & 1 ? R::kVScale : R::kKScale) + (g * kKvPage + slot) * 2);
    }
#pragma unroll
    for (int p = 0; p < 2 * kPasses; ++p) {
        const int at = group0 + kPer * (p / 2);
        if (at >= groups)
            continue;
        uint32_t h[4];
        kv4_widen(w[p], __half2half2(s[p]), h); // codes (0, 4), (1, 5), (2, 6), (3, 7)
        float x[kN];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(kv4_half2(h[i]));
            x[i] = f.x;
            if constexpr (kN == 8)
                x[i + 4] = f.y;
        }
        T *dst = (p & 1 ? v + row * v_stride : k + row * k_stride) + at * kKv4Group + part * kN;
        __stcs(reinterpret_cast<uint4 *>(dst), KvVec<T>::pack(x));
    }
}

template <typename T>
inline void validate_kv4(const void *k, int64_t k_stride, const void *v, int64_t v_stride, const void *pool, int blocks,
                         const Kv4Rows &a, int head_dim) {
    require(a.rows >= 0 && blocks >= 0, "4-bit cache rows: rows and blocks must be nonnegative");
    require(a.kvh > 0 && a.kvh <= 4096, "4-bit cache rows: 1 to 4096 kv heads are supported");
    require(head_dim == 64 || head_dim == 128, "4-bit cache rows: head_dim must be 64 or 128");
    if (a.rows == 0)
        return;
    require(k && v && pool && a.slots, "4-bit cache rows: null pointer");
    const int64_t width = static_cast<int64_t>(a.kvh) * head_dim, elem = static_cast<int64_t>(sizeof(T));
    require(k_stride >= width && v_stride >= width, "4-bit cache rows: rows overlap (stride below kvh * head_dim)");
    require(aligned16(k) && aligned16(v) && aligned16(pool) && k_stride * elem % 16 == 0 && v_stride * elem % 16 == 0,
            "4-bit cache rows: rows and pool must be 16-byte aligned");
}

template <int D, int kPasses> inline dim3 kv4_grid(int rows, int kvh) {
    constexpr int kWarps = kKv4Threads / 32, kPer = 8 * kPasses;
    const int groups = kvh * Kv4Record<D>::kGroups;
    return dim3(static_cast<unsigned>(rows / kWarps + (rows % kWarps != 0)), static_cast<unsigned>((groups + kPer - 1) / kPer));
}

} // namespace detail

namespace ops {

// Bytes of one (block, kv head) record of the 4-bit pool.
inline int kv4_record_bytes(int head_dim) {
    detail::require(head_dim == 64 || head_dim == 128, "4-bit cache rows: head_dim must be 64 or 128");
    return 18 * head_dim;
}

// Stores rows [0, rows) of K and V (row r, head h at r * stride + h * head_dim; T
// fp32 or bf16) at their slots of a pool of `blocks` blocks. No two rows have the
// same slot.
template <typename T>
inline void kv4_write(const T *k, int64_t k_stride, const T *v, int64_t v_stride, uint8_t *pool, int blocks,
                      const int64_t *slots, int rows, int kv_heads, int head_dim, cudaStream_t stream = nullptr) {
    const detail::Kv4Rows a{slots, rows, kv_heads, static_cast<int64_t>(blocks) * detail::kKvPage};
    detail::validate_kv4<T>(k, k_stride, v, v_stride, pool, blocks, a, head_dim);
    if (rows == 0)
        return;
    if (head_dim == 64)
        launch_ex(detail::kv4_write_kernel<T, 64>, detail::kv4_grid<64, detail::kKv4WritePasses>(rows, kv_heads), dim3(detail::kKv4Threads), 0, stream, k,
                  k_stride, v, v_stride, pool, a);
    else
        launch_ex(detail::kv4_write_kernel<T, 128>, detail::kv4_grid<128, detail::kKv4WritePasses>(rows, kv_heads), dim3(detail::kKv4Threads), 0, stream, k,
                  k_stride, v, v_stride, pool, a);
}

// Fetches the rows at the slots; a row without a slot is left as it was.
template <typename T>
inline void kv4_read(const uint8_t *pool, int blocks, const int64_t *slots, int rows, int kv_heads, int head_dim, T *k,
                     int64_t k_stride, T *v, int64_t v_stride, cudaStream_t stream = nullptr) {
    const detail::Kv4Rows a{slots, rows, kv_heads, static_cast<int64_t>(blocks) * detail::kKvPage};
    detail::validate_kv4<T>(k, k_stride, v, v_stride, pool, blocks, a, head_dim);
    if (rows == 0)
        return;
    if (head_dim == 64)
        launch_ex(detail::kv4_read_kernel<T, 64>, detail::kv4_grid<64, detail::kKv4ReadPasses>(rows, kv_heads), dim3(detail::kKv4Threads), 0, stream, pool, k,
                  k_stride, v, v_stride, a);
    else
        launch_ex(detail::kv4_read_kernel<T, 128>, detail::kv4_grid<128, detail::kKv4ReadPasses>(rows, kv_heads), dim3(detail::kKv4Threads), 0, stream, pool, k,
                  k_stride, v, v_stride, a);
}

} // namespace ops
} // namespace opworks
