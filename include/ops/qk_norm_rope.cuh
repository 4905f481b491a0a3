#pragma once

// ops::qk_norm_rope — queries and keys of a step: the root-mean-square norm of
// each head, and the rotation by the row's position, in one pass. The reference
// has a row norm (include/ops/rms_norm.cuh) and a rotation of rows at positions
// one after another (include/ops/rope.cuh), and no norm of heads.
//
// For head x of D values, weight w (none: the head is not normalised), position p:
//   y_i = x_i / sqrt(mean(x^2) + eps) * w_i
//   pairs (i, i + rot / 2) of the first rot values: a cos - b sin, b cos + a sin
//   with the angle p * inv_freq[i]
// and the values from rot on as they are. Norms, angles and rotation are fp32 with
// one rounding to the output's type at the end; the angle is reduced to an eighth
// of a turn in 64 bits, so that far positions keep their bits (fp32 products of
// position 100,000 are off by 0.004 rad).
//
// What bounds it is HBM and the issue of instructions together: each value is read and
// written once, 16 bytes a lane, a head on D / 32 (fp32) or D / 16 (bf16) lanes. A lane has the same pairs
// in every head, so a warp computes cos and sin of its row once, each lane some of
// them, and keeps them in registers; no warp waits for another one. 32 warps an SM
// (64 registers, weights in shared memory) hide the loads better than loads further
// ahead do (two rounds ahead: 61.6 us for 57.9; weights in registers, 20 warps: 73.5).
// Measured: 16,384 rows of 40 heads x 128, bf16: 57.9 us, 5.8 TB/s of what is read and
// written (copy rate 6.46; DRAM itself moves 5.0, L2 holds the rest; issue slots 71 % busy);
// 32 rows, fp32: 2.6 us, launch included.

#include <algorithm>
#include <cstdint>
#include <cuda_bf16.h>

#include "../core/cuda_utils.cuh"
#include "kv_quant.cuh"

namespace opworks {

// Queries and keys of `rows` rows: head h of row r at r * stride + h * head_dim.
// The outputs may be the inputs (same strides); else nothing overlaps.
template <typename T> struct QkNormRope {
    const T *q;
    int64_t q_stride;
    const T *k;
    int64_t k_stride;
    const float *q_weight, *k_weight; // [head_dim], null: no norm
    float eps;
    const int *positions;  // [rows]
    const float *inv_freq; // [rot_dim / 2]
    int rot_dim;
    int rows, q_heads, kv_heads, head_dim;
    T *q_out;
    int64_t q_out_stride;
    T *k_out;
    int64_t k_out_stride;
};

namespace detail {

constexpr int kNormRopeThreads = 128;

// cos and sin of position * frequency.
__device__ __forceinline__ void turn(int position, float frequency, float &c, float &s) {
    constexpr double kTurns = 0.15915494309189533577; // 1 / (2 pi)
    const double turns = static_cast<double>(position) * static_cast<double>(frequency) * kTurns;
    const double eighths = rint(turns * 4.0);
    float sn, cs;
    sincospif(static_cast<float>((turns - eighths * 0.25) * 2.0), &sn, &cs);
    const int quarter = static_cast<int>(static_cast<long long>(eighths) & 3);
    s = quarter == 0 ? sn : quarter == 1 ? cs : quarter == 2 ? -sn : -cs;
    c = quarter == 0 ? cs : quarter == 1 ? -sn : quarter == 2 ? -cs : sn;
}

// A warp takes one of `parts` equal parts of a row's heads, 32 / kLanes at a time.
template <typename T, int D>
static __global__ void __launch_bounds__(kNormRopeThreads, 8) qk_norm_rope_kernel(QkNormRope<T> a, int parts) {
    using V = KvVec<T>;
    constexpr int kN = V::kN, kLanes = D / (2 * kN), kPer = 32 / kLanes; // heads of a warp at a time
    const int lane = threadIdx.x & 31, j = lane % kLanes, sub = lane / kLanes;
    const int64_t task = static_cast<int64_t>(blockIdx.x) * (kNormRopeThreads / 32) + (threadIdx.x >> 5);
    const int64_t row = task / parts;
    const int heads = a.q_heads + a.kv_heads, half = a.rot_dim / 2;
    const int rounds = ((heads + kPer - 1) / kPer + parts - 1) / parts; // of a part
    pdl_trigger();
    pdl_wait();
    const int first = static_cast<int>(task - row * parts) * rounds * kPer;
    // the lane's two vectors of a head: a pair of rotated ones, or two of the rest
    const bool turned = j * kN < half;
    const int at0 = turned ? j * kN : a.rot_dim + (j - half / kN) * 2 * kN;
    const int at1 = turned ? half + j * kN : at0 + kN;
    uint4 r0{}, r1{}; // of the next round
    const auto load = [&](int round) {
        const int h = first + round * kPer + sub;
        if (row < a.rows && round < rounds && h < heads) {
            const T *src = h < a.q_heads ? a.q + row * a.q_stride + h * D : a.k + row * a.k_stride + (h - a.q_heads) * D;
            r0 = *reinterpret_cast<const uint4 *>(src + at0), r1 = *reinterpret_cast<const uint4 *>(src + at1);
        }
    };
    load(0);
    __shared__ __align__(16) float weights[2][D];
    for (int i = threadIdx.x; i < D; i += kNormRopeThreads) {
        weights[0][i] = a.q_weight != nullptr ? __ldg(a.q_weight + i) : 1.f;
        weights[1][i] = a.k_weight != nullptr ? __ldg(a.k_weight + i) : 1.f;
    }
    __syncthreads();
    if (row >= a.rows)
        return;
    // cos and sin of the lane's pairs: the lanes that have the same ones share the work
    float c[kN], s[kN];
    if (half > 0) {
        constexpr int kEach = kN > kPer ? kN / kPer : 1;
        const int position = a.positions[row];
        float mc[kEach], ms[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            mc[i] = 1.f, ms[i] = 0.f;
            if (turned && sub * kEach + i < kN)
                turn(position, __ldg(a.inv_freq + at0 + sub * kEach + i), mc[i], ms[i]);
        }
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            c[i] = __shfl_sync(kFullWarpMask, mc[i % kEach], i / kEach * kLanes + j);
            s[i] = __shfl_sync(kFullWarpMask, ms[i % kEach], i / kEach * kLanes + j);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i)
            c[i] = 1.f, s[i] = 0.f;
    }
    for (int round = 0; round < rounds; ++round) {
        const int h = first + round * kPer + sub;
        float x[kN], y[kN];
        V::unpack(r0, x), V::unpack(r1, y);
        load(round + 1);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < kN; ++i)
            sum += x[i] * x[i] + y[i] * y[i];
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1)
            sum += __shfl_xor_sync(kFullWarpMask, sum, off);
        const bool key = h >= a.q_heads;
        if ((key ? a.k_weight : a.q_weight) != nullptr) {
            const float inv = rsqrtf(sum / D + a.eps);
#pragma unroll
            for (int i = 0; i < kN; i += 4) {
                const float4 w0 = *reinterpret_cast<const float4 *>(&weights[key][at0 + i]), w1 = *reinterpret_cast<const float4 *>(&weights[key][at1 + i]);
                x[i] = x[i] * inv * w0.x, x[i + 1] = x[i + 1] * inv * w0.y, x[i + 2] = x[i + 2] * inv * w0.z, x[i + 3] = x[i + 3] * inv * w0.w;
                y[i] = y[i] * inv * w1.x, y[i + 1] = y[i + 1] * inv * w1.y, y[i + 2] = y[i + 2] * inv * w1.z, y[i + 3] = y[i + 3] * inv * w1.w;
            }
        }
#pragma unroll
        for (int i = 0; i < kN; ++i) { // (the rest as it is: zero times an infinity would be NaN)
            const float u = x[i], v = y[i];
            x[i] = turned ? u * c[i] - v * s[i] : u;
            y[i] = turned ? v * c[i] + u * s[i] : v;
        }
        if (h < heads) {
            T *dst = h < a.q_heads ? a.q_out + row * a.q_out_stride + h * D : a.k_out + row * a.k_out_stride + (h - a.q_heads) * D;
            *reinterpret_cast<uint4 *>(dst + at0) = V::pack(x);
            *reinterpret_cast<uint4 *>(dst + at1) = V::pack(y);
        }
    }
}

template <typename T, int D> inline void qk_norm_rope_launch(const QkNormRope<T> &a, cudaStream_t stream) {
    constexpr int kPer = 32 / (D / (2 * KvVec<T>::kN)), kWarps = kNormRopeThreads / 32;
    // few rows: parts of a row's heads, as long as that brings warps to SMs that have fewer than 16
    const int pieces = (a.q_heads + a.kv_heads + kPer - 1) / kPer;
    const int64_t want = 16LL * device_facts().sm_count / a.rows;
    const int parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(pieces, want)));
    const int64_t blocks = (static_cast<int64_t>(a.rows) * parts + kWarps - 1) / kWarps;
    launch_ex(qk_norm_rope_kernel<T, D>, dim3(static_cast<unsigned>(blocks)), dim3(kNormRopeThreads), 0, stream, a, parts);
}

} // namespace detail

namespace ops {

template <typename T> inline void qk_norm_rope(const QkNormRope<T> &a, cudaStream_t stream = nullptr) {
    const int D = a.head_dim;
    detail::require(a.rows >= 0, "qk_norm_rope: rows must be nonnegative");
    detail::require(a.q_heads >= 0 && a.kv_heads >= 0 && a.q_heads <= 65535 && a.kv_heads <= 65535,
                    "qk_norm_rope: 0 to 65535 heads of each kind");
    detail::require(D == 32 || D == 64 || D == 128 || D == 256, "qk_norm_rope: head_dim must be 32, 64, 128 or 256");
    detail::require(a.rot_dim >= 0 && a.rot_dim <= D && a.rot_dim % 16 == 0,
                    "qk_norm_rope: rot_dim must be a multiple of 16 up to head_dim");
    detail::require((a.q_weight == nullptr && a.k_weight == nullptr) || a.eps > 0.f, "qk_norm_rope: eps must be positive");
    if (a.rows == 0 || a.q_heads + a.kv_heads == 0)
        return;
    detail::require(a.rot_dim == 0 || (a.positions && a.inv_freq), "qk_norm_rope: null pointer");
    constexpr int64_t kElem = sizeof(T);
    const auto check = [&](const void *p, int64_t stride, int heads) {
        if (heads == 0)
            return;
        detail::require(p != nullptr, "qk_norm_rope: null pointer");
        detail::require(stride >= static_cast<int64_t>(heads) * D, "qk_norm_rope: rows overlap (stride below heads * head_dim)");
        detail::require(detail::aligned16(p) && stride * kElem % 16 == 0, "qk_norm_rope: rows must be 16-byte aligned");
    };
    check(a.q, a.q_stride, a.q_heads), check(a.q_out, a.q_out_stride, a.q_heads);
    check(a.k, a.k_stride, a.kv_heads), check(a.k_out, a.k_out_stride, a.kv_heads);
    switch (D) {
    case 32: detail::qk_norm_rope_launch<T, 32>(a, stream); break;
    case 64: detail::qk_norm_rope_launch<T, 64>(a, stream); break;
    case 128: detail::qk_norm_rope_launch<T, 128>(a, stream); break;
    default: detail::qk_norm_rope_launch<T, 256>(a, stream); break;
    }
}

} // namespace ops
} // namespace opworks
