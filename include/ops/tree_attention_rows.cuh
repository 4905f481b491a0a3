#pragma once

// Tree attention, kernel for few query rows per KV head (ops/tree_attention.cuh
// has the definition of the operator).
//
// Bound: HBM, as for any decode attention, so every byte of a page is fetched
// once and everything else has to fit under that stream.
//
// Split. CTA = (split of the keys, row group, kv head, sequence). The query
// rows of a KV head (row = node * rep + head in group) share its pages; a group
// is kMT tensor-core tiles of rows. The splits of one (group, head, sequence)
// form a thread-block cluster and are joined through distributed shared memory
// in rank order: one launch, no workspace, the same bits every time.
//
// Warps are independent until the end: warp w takes pages w, w + kWarps, ... of
// the split through its own ring of bulk copies (an 8-bit page of a head is one
// copy), with its own softmax state.
//
// Products on mma.sync: with few rows a tcgen05 tile of 128 would be mostly
// empty, and fragments go from shared memory to registers directly, so 8-bit
// codes are widened to fp16 (exactly) on the way and no widened tile is
// written anywhere. Layout: S = Q K^T has the rows of Q along M = 16, so the
// accumulator of S is the A operand of O = P V. fp32 rows are two terms hi + lo
// (22 bits): a tile holds 8 rows, hi in its upper half and lo in its lower, so
// one product gives both and a lane adds its own two accumulators. bf16 rows
// fit in one term: 16 rows to a tile. K and V: 8-bit codes are exact in fp16,
// their scales are applied to S and folded into P; fp32 pools are two tf32
// terms. Contraction indices and output columns are permuted so that a lane's
// fragments are contiguous bytes of a row (see the index comments below).
//
// Softmax: one pass, running maximum in log2 units. The maximum is a reference
// only: it is raised when a score passes it by kLazy, so most pages rescale
// nothing. P is held as 2^kLift times its value, so that fp16 keeps 22 bits of
// two terms down to 2^-28 of the largest weight.

#include <cuda_fp16.h>

#include "tree_attention_common.cuh"

namespace opworks::detail {

constexpr float kLazy = 4.f;  // log2 units a score may pass the reference maximum by
constexpr float kLift = 10.f; // P is scaled by 2^kLift: at most 2^14

template <typename T, int D, KvFormat kFmt, int kMT> struct TreeRowsGeo {
    static constexpr bool kTwo = std::is_same_v<T, float>; // two terms of Q and P
    static constexpr int kRPL = kTwo ? 1 : 2;              // rows of a tile that a lane holds scores of
    static constexpr int kTileRows = 8 * kRPL;
    static constexpr int kRows = kMT * kTileRows;
    static constexpr bool kWide = kFmt == KvFormat::kF32;
    static constexpr int kPageBytes = kWide ? 2 * kKvPage * D * 4 : KvRecord<D>::kBytes;
    static constexpr int kWarps = kWide ? 4 : 8;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kStages = kWide ? 3 : 4;
    static constexpr int kRing = kWarps * kStages * kPageBytes;
    static constexpr int kPitch = D + 4; // floats per row of a warp's partial result
    static constexpr int kMerge = kWarps * kRows * kPitch * 4;
    static constexpr int kBuf = (kRing > kMerge ? kRing : kMerge);
    static constexpr int kBytes = kBuf + 8 * kWarps * kStages + 4 * (2 * kWarps + 2) * kRows;
    static constexpr int kQRegs = kWide ? D / 8 : D / 16; // k steps
};

// d += a (16 x 16 fp16) b (16 x 8 fp16)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d += a (16 x 8 tf32) b (8 x 8 tf32)
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x as two tf32 terms: rounded to the nearest (by magnitude), and the rest,
// whose last bit the tensor cores drop: 2^-24 of x. Truncation instead left
// 2^-21, all of it towards zero, which showed in the results.
__device__ __forceinline__ uint32_t tf32_hi(float x) { return (__float_as_uint(x) + 0x1000u) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf32_lo(float x) { return __float_as_uint(x - __uint_as_float(tf32_hi(x))); }

// fp16 pair (a, b) as one register, a in the low half
__device__ __forceinline__ uint32_t half2_rn(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 half2_floats(uint32_t h) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// Two pairs of fp16 from the four codes of a word: (0, 1) and (2, 3). Exact.
template <KvFormat kFmt> __device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (kFmt == KvFormat::kInt8) {
        // byte + 128 in the low bits of fp16 1024 .. 1279, minus 1152
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t bias = 0x64806480u; // fp16 1152, twice
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&bias));
        const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), *reinterpret_cast<const __half2 *>(&bias));
        lo = *reinterpret_cast<const uint32_t *>(&x);
        hi = *reinterpret_cast<const uint32_t *>(&y);
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

__device__ __forceinline__ float finite_or_zero(float x) { return fabsf(x) <= 3.4028235e38f ? x : 0.f; }

// e4m3 NaN codes (never written by ops::kv_quant_write) replaced by zero: a
// masked row may hold them, and zero times NaN is NaN.
__device__ __forceinline__ uint32_t clear_e4m3_nan(uint32_t w) {
    return w & ~__vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu);
}

template <typename T, int D, KvFormat kFmt, int kMT>
static __global__ void __launch_bounds__(TreeRowsGeo<T, D, kFmt, kMT>::kThreads)
    tree_rows_kernel(const T *__restrict__ q, T *__restrict__ out, TreeArgs a, int groups, int splits, int *err) {
    using G = TreeRowsGeo<T, D, kFmt, kMT>;
    using R = KvRecord<D>;
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + G::kBuf);
    float *stat = reinterpret_cast<float *>(bars + G::kWarps * G::kStages); // m [warps][rows], l [warps][rows]
    float *joined = stat + 2 * G::kWarps * G::kRows;                          // m [rows], l [rows] of the CTA

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % splits, unit = blockIdx.x / splits;
    const int group = unit % groups, h = unit / groups, b = blockIdx.y;
    const int rep = a.qh / a.kvh;

    uint64_t *bar = bars + warp * G::kStages;
    if (lane == 0) {
        for (int s = 0; s < G::kStages; ++s)
            sm100::mbar_init(&bar[s], 1);
        sm100::fence_mbarrier_init();
    }
    __syncwarp();
    pdl_trigger();
    pdl_wait();

    const TreeSpan span(a.t, b);
    const int row_base = group * G::kRows, rows = span.n * rep; // query rows of this (sequence, head)
    int keys = span.keys;
    if (a.t.mask == nullptr) // a chain: nothing after the group's last node is seen
        keys = min(keys, span.ctx + (min(row_base + G::kRows, rows) + rep - 1) / rep);
    const int pages = row_base < rows ? (keys + kKvPage - 1) / kKvPage : 0;
    const int per = (pages + splits - 1) / splits;
    const int p0 = min(pages, rank * per), p1 = min(pages, p0 + per);
    const int mine = p1 - p0 > warp ? (p1 - p0 - warp + G::kWarps - 1) / G::kWarps : 0; // pages of this warp
    uint8_t *ring = smem + warp * G::kStages * G::kPageBytes;

    const int *table = a.t.block_table + static_cast<int64_t>(b) * a.t.table_stride;
    int ids = 0; // block ids of 32 pages of this warp, one per lane
    const auto refill = [&](int base) {
        const int i = base + lane;
        ids = i < mine ? table[p0 + warp + i * G::kWarps] : 0;
    };
    const auto issue = [&](int i) { // page i of this warp into its stage
        const int blk = __shfl_sync(kFullWarpMask, ids, i & 31);
        if (lane == 0) {
            const int s = i % G::kStages;
            uint8_t *dst = ring + s * G::kPageBytes;
            const int64_t rec = static_cast<int64_t>(blk) * a.kvh + h;
            sm100::mbar_arrive_expect_tx(&bar[s], G::kPageBytes);
            if constexpr (G::kWide) {
                constexpr int kHalf = kKvPage * D * 4;
                sm100::bulk_load(dst, static_cast<const uint8_t *>(a.k) + rec * kHalf, kHalf, &bar[s]);
                sm100::bulk_load(dst + kHalf, static_cast<const uint8_t *>(a.v) + rec * kHalf, kHalf, &bar[s]);
            } else {
                sm100::bulk_load(dst, static_cast<const uint8_t *>(a.k) + rec * R::kBytes, R::kBytes, &bar[s]);
            }
        }
    };
    refill(0);
    for (int i = 0; i < min(mine, G::kStages); ++i)
        issue(i);

    // Q fragments. fp16: k step s = 4c + i of 16 dims, lane t holds dims 64c +
    // 16t + 4i + {0, 1} (k = 2t, 2t + 1) and + {2, 3} (k = 2t + 8, 2t + 9).
    // tf32: k step 2c + e of 8 dims, dims 16c + 4t + 2e (k = t), + 1 (k = t + 4).
    uint32_t qf[kMT][G::kQRegs][4];
    float row_scale[kMT][G::kRPL];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
        float x[G::kRPL][D / 4];
#pragma unroll
        for (int rr = 0; rr < G::kRPL; ++rr) {
            const int r = row_base + mt * G::kTileRows + rr * 8 + g;
            const bool live = r < rows;
            const T *src = q + static_cast<int64_t>(span.row0 + (live ? r / rep : 0)) * a.q_stride +
                           static_cast<int64_t>(h * rep + (live ? r % rep : 0)) * D;
            if constexpr (G::kWide && !G::kTwo) { // 4 bf16 values at a time
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    const uint2 w = live ? *reinterpret_cast<const uint2 *>(src + 16 * c + 4 * t) : make_uint2(0, 0);
                    x[rr][4 * c] = __uint_as_float(w.x << 16), x[rr][4 * c + 1] = __uint_as_float(w.x & 0xffff0000u);
                    x[rr][4 * c + 2] = __uint_as_float(w.y << 16), x[rr][4 * c + 3] = __uint_as_float(w.y & 0xffff0000u);
                }
            } else {
                constexpr int kN = KvVec<T>::kN, kRun = G::kWide ? 4 : 16; // kRun: contiguous dims of a lane
#pragma unroll
                for (int v = 0; v < D / 4 / kN; ++v) {
                    float y[kN] = {};
                    if (live)
                        KvVec<T>::unpack(*reinterpret_cast<const uint4 *>(src + v * kN / kRun * 4 * kRun + kRun * t + v * kN % kRun), y);
#pragma unroll
                    for (int e = 0; e < kN; ++e)
                        x[rr][v * kN + e] = y[e];
                }
            }
        }
#pragma unroll
        for (int rr = 0; rr < G::kRPL; ++rr) {
            row_scale[mt][rr] = a.scale_log2;
            if constexpr (!G::kWide) {
                // a power of two brings the row's largest magnitude to 2^10 ..
                // 2^11, so that fp16 holds the row to 2^-22 of it in two terms
                // (and a bf16 row exactly in one)
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < D / 4; ++e)
                    top = fmaxf(top, fabsf(x[rr][e]));
                top = fmaxf(top, __shfl_xor_sync(kFullWarpMask, top, 1));
                top = fmaxf(top, __shfl_xor_sync(kFullWarpMask, top, 2));
                const int ex = top > 0.f ? static_cast<int>(__float_as_uint(top) >> 23) - 127 : 0; // floor(log2)
                const int up = max(-100, min(100, 10 - ex));
                const float f = __uint_as_float(static_cast<uint32_t>(127 + up) << 23);
                row_scale[mt][rr] *= __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
#pragma unroll
                for (int e = 0; e < D / 4; ++e)
                    x[rr][e] *= f;
            }
        }
        if constexpr (G::kWide) {
#pragma unroll
            for (int s = 0; s < G::kQRegs; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float hi = x[0][2 * s + e];
                    qf[mt][s][2 * e] = G::kTwo ? tf32_hi(hi) : __float_as_uint(hi);
                    qf[mt][s][2 * e + 1] = G::kTwo ? tf32_lo(hi) : __float_as_uint(x[G::kRPL - 1][2 * s + e]);
                }
        } else {
#pragma unroll
            for (int s = 0; s < G::kQRegs; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float u = x[0][4 * s + 2 * e], v = x[0][4 * s + 2 * e + 1];
                    const uint32_t hi = half2_rn(u, v);
                    qf[mt][s][2 * e] = hi;
                    if constexpr (G::kTwo) {
                        const float2 f = half2_floats(hi);
                        qf[mt][s][2 * e + 1] = half2_rn(u - f.x, v - f.y);
                    } else {
                        qf[mt][s][2 * e + 1] = half2_rn(x[1][4 * s + 2 * e], x[1][4 * s + 2 * e + 1]);
                    }
                }
        }
    }

    float o[kMT][D / 8][4] = {};
    float m[kMT][G::kRPL], l[kMT][G::kRPL];
    float vtop = 0.f, vinv = 0.f; // power of two above every V scale so far, and 1 / it
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int rr = 0; rr < G::kRPL; ++rr)
            m[mt][rr] = -1e30f, l[mt][rr] = 0.f;

    bool ok = true;
    int done = 0;
    for (; done < mine; ++done) {
        const int s = done % G::kStages;
        if (!sm100::mbar_wait_warp(&bar[s], static_cast<uint32_t>(done / G::kStages) & 1u)) {
            ok = false;
            break;
        }
        const uint8_t *page = ring + s * G::kPageBytes;
        const int key0 = (p0 + warp + done * G::kWarps) * kKvPage;
        const bool edge = key0 + kKvPage > span.ctx; // holds nodes, or places after the last key

        // S. Score column g of n tile j is key 8j + 4 (g & 1) + g / 2, so that
        // lane t's columns 2t + col are keys 8j + 4 col + t.
        float sc[kMT][2][4] = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int krow = 8 * j + 4 * (g & 1) + (g >> 1);
            if constexpr (G::kWide) {
                const float4 *src = reinterpret_cast<const float4 *>(page + krow * D * 4) + t;
#pragma unroll
                for (int c = 0; c < D / 16; ++c) {
                    const float4 w = src[4 * c];
                    const float y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int mt = 0; mt < kMT; ++mt) {
                            mma_tf32(sc[mt][j], qf[mt][2 * c + e], tf32_hi(y[2 * e]), tf32_hi(y[2 * e + 1]));
                            mma_tf32(sc[mt][j], qf[mt][2 * c + e], tf32_lo(y[2 * e]), tf32_lo(y[2 * e + 1]));
                        }
                }
            } else {
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {
                    const uint4 w4 = *reinterpret_cast<const uint4 *>(page + krow * D + 64 * c + 16 * t);
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t b0, b1;
                        codes_to_half<kFmt>(w[i], b0, b1);
#pragma unroll
                        for (int mt = 0; mt < kMT; ++mt)
                            mma_f16(sc[mt][j], qf[mt][4 * c + i], b0, b1);
                    }
                }
            }
        }
        // scores in log2 units, masked ones -inf; V factors
        float kscale[4], vfac[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            kscale[i] = G::kWide ? 1.f : *reinterpret_cast<const float *>(page + R::kKScale + 16 * i + 4 * t);
            vfac[i] = G::kWide ? 1.f : *reinterpret_cast<const float *>(page + R::kVScale + 16 * i + 4 * t);
        }
        float x[kMT][G::kRPL][4];
        bool raise = false;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int rr = 0; rr < G::kRPL; ++rr) {
                uint32_t seen = 0xffffu;
                if (edge) {
                    const int r = row_base + mt * G::kTileRows + rr * 8 + g;
                    seen = r < rows ? tree_sees16(a.t, span.row0 + r / rep, r / rep, key0 - span.ctx, keys - span.ctx) : 0u;
                }
                float top = kNegInf;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float *c = sc[mt][i >> 1];
                    float v = G::kTwo ? c[i & 1] + c[2 + (i & 1)] : c[2 * rr + (i & 1)];
                    v *= row_scale[mt][rr] * kscale[i];
                    if (edge && !((seen >> (4 * i + t)) & 1u))
                        v = kNegInf;
                    x[mt][rr][i] = v;
                    top = fmaxf(top, v);
                }
                raise |= top > m[mt][rr] + kLazy;
            }
        if constexpr (!G::kWide) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (edge && (key0 + 4 * i + t >= keys))
                    vfac[i] = 0.f;
                raise |= vfac[i] > vtop && vfac[i] < 3e38f;
            }
        }
        if (__any_sync(kFullWarpMask, raise)) {
            float vfix = 1.f;
            if constexpr (!G::kWide) {
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    top = vfac[i] < 3e38f ? fmaxf(top, vfac[i]) : top;
                top = fmaxf(top, __shfl_xor_sync(kFullWarpMask, top, 1));
                top = fmaxf(top, __shfl_xor_sync(kFullWarpMask, top, 2));
                if (top > vtop) { // the same in every lane of the warp
                    // next power of two, held where its inverse is a normal number too
                    const uint32_t ex = min(max((__float_as_uint(top) >> 23) + 1u, 4u), 250u);
                    vfix = vtop * __uint_as_float((254u - ex) << 23);
                    vtop = __uint_as_float(ex << 23);
                    vinv = __uint_as_float((254u - ex) << 23);
                }
            }
#pragma unroll
            for (int mt = 0; mt < kMT; ++mt) {
                float fix[G::kRPL];
#pragma unroll
                for (int rr = 0; rr < G::kRPL; ++rr) {
                    float top = fmaxf(fmaxf(x[mt][rr][0], x[mt][rr][1]), fmaxf(x[mt][rr][2], x[mt][rr][3]));
                    top = fmaxf(top, __shfl_xor_sync(kFullWarpMask, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(kFullWarpMask, top, 2));
                    const float up = fmaxf(m[mt][rr], top);
                    fix[rr] = exp2_approx(m[mt][rr] - up);
                    m[mt][rr] = up;
                    l[mt][rr] *= fix[rr];
                    fix[rr] *= vfix;
                }
#pragma unroll
                for (int n = 0; n < D / 8; ++n) {
                    o[mt][n][0] *= fix[0];
                    o[mt][n][1] *= fix[0];
                    o[mt][n][2] *= fix[G::kRPL - 1];
                    o[mt][n][3] *= fix[G::kRPL - 1];
                }
            }
        }
        // A V row with an infinity or a NaN must not reach the rows that do not
        // see it (zero times either is NaN). Only nodes are seen by some rows
        // and not by others, so on edge pages such values count as zero below
        // and the rows that do see them turn NaN here.
        uint32_t bad = 0;
        if (G::kWide && edge) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bool odd = false;
                const float4 *v = reinterpret_cast<const float4 *>(page + kKvPage * D * 4 + (4 * i + t) * D * 4) + g;
#pragma unroll
                for (int c = 0; c < D / 32; ++c)
                    odd |= !(finite_or_zero(v[8 * c].x) == v[8 * c].x && finite_or_zero(v[8 * c].y) == v[8 * c].y &&
                             finite_or_zero(v[8 * c].z) == v[8 * c].z && finite_or_zero(v[8 * c].w) == v[8 * c].w);
                bad |= ((__ballot_sync(kFullWarpMask, odd) >> t) & 0x11111111u) != 0u ? 1u << i : 0u;
            }
        }
        // P as A fragments; l sums the weights before they are rounded
        uint32_t pf[kMT][G::kWide ? 2 : 1][4];
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
            float p[G::kRPL][4];
#pragma unroll
            for (int rr = 0; rr < G::kRPL; ++rr)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[rr][i] = exp2_approx(x[mt][rr][i] - m[mt][rr] + kLift);
                    l[mt][rr] += p[rr][i];
                    if (G::kWide && edge && (bad >> i & 1u) && x[mt][rr][i] != kNegInf)
                        l[mt][rr] = __uint_as_float(0x7fc00000u);
                    if constexpr (!G::kWide) {
                        const float w = p[rr][i] * (vfac[i] * vinv);
                        p[rr][i] = x[mt][rr][i] == kNegInf ? 0.f : w;
                    }
                }
            if constexpr (G::kWide) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float v = p[0][2 * j + e];
                        if constexpr (G::kTwo) {
                            pf[mt][j][2 * e] = tf32_hi(v);
                            pf[mt][j][2 * e + 1] = tf32_lo(v);
                        } else {
                            pf[mt][j][2 * e] = tf32_rna(v);
                            pf[mt][j][2 * e + 1] = tf32_rna(p[G::kRPL - 1][2 * j + e]);
                        }
                    }
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t hi = half2_rn(p[0][2 * j], p[0][2 * j + 1]);
                    pf[mt][0][2 * j] = hi;
                    if constexpr (G::kTwo) {
                        const float2 f = half2_floats(hi);
                        pf[mt][0][2 * j + 1] = half2_rn(p[0][2 * j] - f.x, p[0][2 * j + 1] - f.y);
                    } else {
                        pf[mt][0][2 * j + 1] = half2_rn(p[G::kRPL - 1][2 * j], p[G::kRPL - 1][2 * j + 1]);
                    }
                }
            }
        }
        // O += P V. 8-bit: column g of n tile n is dim (D / 8) g + n. fp32:
        // column g of n tile 4c + e is dim 32c + 4g + e.
        if constexpr (G::kWide) {
            const uint8_t *v = page + kKvPage * D * 4;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    float4 u = *reinterpret_cast<const float4 *>(v + (8 * j + t) * D * 4 + 128 * c + 16 * g);
                    float4 w = *reinterpret_cast<const float4 *>(v + (8 * j + 4 + t) * D * 4 + 128 * c + 16 * g);
                    float ue[4] = {u.x, u.y, u.z, u.w}, we[4] = {w.x, w.y, w.z, w.w};
                    if (edge)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            ue[e] = finite_or_zero(ue[e]);
                            we[e] = finite_or_zero(we[e]);
                        }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int mt = 0; mt < kMT; ++mt) {
                            if constexpr (G::kTwo) {
                                mma_tf32(o[mt][4 * c + e], pf[mt][j], tf32_hi(ue[e]), tf32_hi(we[e]));
                                mma_tf32(o[mt][4 * c + e], pf[mt][j], tf32_lo(ue[e]), tf32_lo(we[e]));
                            } else {
                                mma_tf32(o[mt][4 * c + e], pf[mt][j], tf32_rna(ue[e]), tf32_rna(we[e]));
                            }
                        }
                }
        } else {
            constexpr int kWords = D / 32;
            uint32_t w[4][kWords];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t *src = page + R::kCodes + (4 * i + t) * D + (D / 8) * g;
                if constexpr (kWords == 2) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(src);
                    w[i][0] = u.x, w[i][1] = u.y;
                } else {
                    const uint4 u = *reinterpret_cast<const uint4 *>(src);
                    w[i][0] = u.x, w[i][1] = u.y, w[i][kWords - 2] = u.z, w[i][kWords - 1] = u.w;
                }
                if (kFmt == KvFormat::kE4M3 && edge)
#pragma unroll
                    for (int c = 0; c < kWords; ++c)
                        w[i][c] = clear_e4m3_nan(w[i][c]);
            }
#pragma unroll
            for (int c = 0; c < kWords; ++c) {
                uint32_t b0[4], b1[4]; // keys (t, 4 + t) and (8 + t, 12 + t) of dims 4c .. 4c + 3
                codes_to_half<kFmt>(__byte_perm(w[0][c], w[1][c], 0x5140), b0[0], b0[1]);
                codes_to_half<kFmt>(__byte_perm(w[0][c], w[1][c], 0x7362), b0[2], b0[3]);
                codes_to_half<kFmt>(__byte_perm(w[2][c], w[3][c], 0x5140), b1[0], b1[1]);
                codes_to_half<kFmt>(__byte_perm(w[2][c], w[3][c], 0x7362), b1[2], b1[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int mt = 0; mt < kMT; ++mt)
                        mma_f16(o[mt][4 * c + e], pf[mt][0], b0[e], b1[e]);
            }
        }
        __syncwarp(); // every lane has read the stage
        const int next = done + G::kStages;
        if ((next & 31) == 0 && next < mine)
            refill(next);
        if (next < mine)
            issue(next);
    }
    // a wait that ran out: the copies still in flight must land before the ring is used again
    if (!ok)
        for (int i = done; i < min(mine, done + G::kStages); ++i)
            sm100::mbar_wait(&bar[i % G::kStages], static_cast<uint32_t>(i / G::kStages) & 1u);
    if (!__syncthreads_and(ok) && tid == 0)
        atomicExch(err, 7);

    // the warps' results over the ring, joined in warp order
    float *part = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int rr = 0; rr < G::kRPL; ++rr) {
            const int r = mt * G::kTileRows + rr * 8 + g;
            float sum = l[mt][rr];
            sum += __shfl_xor_sync(kFullWarpMask, sum, 1);
            sum += __shfl_xor_sync(kFullWarpMask, sum, 2);
            float *dst = part + (warp * G::kRows + r) * G::kPitch;
            const float unit_v = G::kWide ? 1.f : vtop;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int col = 0; col < 2; ++col) {
                    const float v = G::kTwo ? o[mt][n][col] + o[mt][n][2 + col] : o[mt][n][2 * rr + col];
                    const int d = G::kWide ? 32 * (n / 4) + 4 * (2 * t + col) + n % 4 : (D / 8) * (2 * t + col) + n;
                    dst[d] = v * unit_v;
                }
            if (t == 0) {
                stat[warp * G::kRows + r] = m[mt][rr];
                stat[(G::kWarps + warp) * G::kRows + r] = sum;
            }
        }
    __syncthreads();
    const int live = min(G::kRows, rows - row_base); // may be negative
    for (int i = tid; i < G::kRows * D; i += G::kThreads) {
        const int r = i / D, d = i % D;
        if (r >= live)
            break;
        float top = -1e30f, L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < G::kWarps; ++w)
            top = fmaxf(top, stat[w * G::kRows + r]);
#pragma unroll
        for (int w = 0; w < G::kWarps; ++w) {
            const float f = exp2_approx(stat[w * G::kRows + r] - top);
            L += f * stat[(G::kWarps + w) * G::kRows + r];
            O += f * part[(w * G::kRows + r) * G::kPitch + d];
        }
        if (splits == 1) {
            const int row = row_base + r;
            out[static_cast<int64_t>(span.row0 + row / rep) * a.out_stride + static_cast<int64_t>(h * rep + row % rep) * D + d] =
                static_cast<T>(L == 0.f ? 0.f : O / L);
        } else {
            part[r * G::kPitch + d] = O; // warp 0's place: read by this thread alone
            if (d == 0) {
                joined[r] = top;
                joined[G::kRows + r] = L;
            }
        }
    }
    if (splits == 1)
        return;
    __syncthreads();
    cluster_sync_all();
    for (int i = rank * G::kThreads + tid; i < G::kRows * D; i += splits * G::kThreads) {
        const int r = i / D, d = i % D;
        if (r >= live)
            break;
        float top = -1e30f, L = 0.f, O = 0.f;
        for (int c = 0; c < splits; ++c)
            top = fmaxf(top, peer_load(&joined[r], c));
        for (int c = 0; c < splits; ++c) {
            const float f = exp2_approx(peer_load(&joined[r], c) - top);
            L += f * peer_load(&joined[G::kRows + r], c);
            O += f * peer_load(&part[r * G::kPitch + d], c);
        }
        const int row = row_base + r;
        out[static_cast<int64_t>(span.row0 + row / rep) * a.out_stride + static_cast<int64_t>(h * rep + row % rep) * D + d] =
            static_cast<T>(L == 0.f ? 0.f : O / L);
    }
    __syncthreads();
    cluster_sync_all(); // peers read this CTA's shared memory until here
}

template <typename T, int D, KvFormat kFmt, int kMT>
inline void tree_rows_launch(const T *q, T *out, const TreeArgs &a, cudaStream_t stream) {
    using G = TreeRowsGeo<T, D, kFmt, kMT>;
    const auto kernel = tree_rows_kernel<T, D, kFmt, kMT>;
    allow_shared_bytes(kernel, G::kBytes);
    const int64_t rows = static_cast<int64_t>(a.t.max_rows) * (a.qh / a.kvh);
    const int64_t groups = (rows + G::kRows - 1) / G::kRows;
    const int64_t units = groups * a.kvh;
    const int64_t pages = (static_cast<int64_t>(a.t.max_ctx) + a.t.max_rows + kKvPage - 1) / kKvPage;
    // splits until two CTAs per SM are filled, while each warp still has two pages
    int splits = 1;
    while (splits < 8 && units * a.t.batch * splits * 2 <= 2 * device_facts().sm_count &&
           pages >= static_cast<int64_t>(splits) * 2 * G::kWarps * 2)
        splits *= 2;
    require(units * splits <= 0x7fffffff, "tree attention: too many rows for one call");
    launch_ex_cluster(kernel, dim3(static_cast<unsigned>(units * splits), a.t.batch), dim3(splits), dim3(G::kThreads),
                      G::kBytes, stream, q, out, a, static_cast<int>(groups), splits, sm100::device_error_word());
}

} // namespace opworks::detail
