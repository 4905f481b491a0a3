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
// Warps are independent until the end: chunks of keys (two 8-bit pages or one
// fp32 page) go round the warps of the cluster, and a warp takes its own through
// its own ring of bulk copies (an 8-bit page of a head is one copy), with its own
// softmax state.
//
// Products on mma.sync: with few rows a tcgen05 tile of 128 would be mostly
// empty, and fragments go from shared memory to registers directly, so 8-bit
// codes are widened to fp16 (exactly) on the way and no widened tile is
// written anywhere. Layout: S = Q K^T has the rows of Q along M = 16, so the
// accumulator of S is the A operand of O = P V. fp32 rows are two fp16 terms hi
// + lo (22 bits): a tile holds 8 rows, hi in its upper half and lo in its
// lower, so one product gives both and a lane adds its own two accumulators.
// bf16 rows fit in one term: 16 rows to a tile. K and V: 8-bit codes are exact
// in fp16, their scales are applied to S and folded into P; fp32 pools are two
// fp16 terms too, after a power of two that a page shares (for V, 32 dims of it):
// kept from page to page while it brings their largest to 2^-3 to 2^14, so that
// the terms hold 2^-22 of that at least. tf32 terms took as many
// conversions and twice the tensor time. Contraction indices and output columns
// are permuted so that a lane's fragments are contiguous bytes of a row (see
// the index comments below).
//
// Softmax: one pass, running maximum in log2 units. The maximum is a reference
// only: it is raised when a score passes it by kLazy, so most chunks rescale
// nothing. P is held as 2^kLift times its value, so that fp16 keeps 22 bits of
// two terms down to 2^-28 of the largest weight. The V scales of 8-bit pools
// are folded into P, and a power of two above them into the reference.
//
// Chunks that hold nodes: every K and V row has a power of two of its own there,
// and the reference of a query row counts those V rows only that it sees, so a
// row that is masked takes no bits from the others, whatever its size.
//
// The tensor cores cut an accumulator off at every step, so the O of fp32 rows is
// summed outside of them, a page's product at a time: two packed additions for
// each, 3 to 4 % of a decode step's time (10 % at D = 128), and errors over 12,000
// keys of 5e-7 to 8e-7 relative to 64 bits (fp32 sums in torch 7e-7 to 2e-6) where
// they were 1.5e-6 to 5.8e-6.
//
// Measured (kernel time): a decode step of 32 sequences of 1090 to 2180 tokens, 32
// query and 8 kv heads of 64, int8: 19.7 us, 2.9 TB/s; 4 chains of 5 rows over up
// to 8192 tokens, fp32 pools: 48.5 us, 2.2 TB/s; one row over 511 tokens: 7.0 us.
// What bounds it is instruction latency: over 200 instructions per 8-bit page and
// tile (over 900 per fp32 page and three tiles), 7 cycles each at the 16 (8) warps
// per SM that registers leave room for.

#include "tree_attention_common.cuh"

namespace opworks::detail {

template <typename T, int D, KvFormat kFmt, int kMT> struct TreeRowsGeo {
    static constexpr bool kTwo = std::is_same_v<T, float>; // two terms of Q and P
    static constexpr int kRPL = kTwo ? 1 : 2;              // rows of a tile that a lane holds scores of
    static constexpr int kTileRows = 8 * kRPL;
    static constexpr int kRows = kMT * kTileRows;
    static constexpr bool kWide = kFmt == KvFormat::kF32;
    static constexpr int kPageBytes = kWide ? 2 * kKvPage * D * 4 : KvRecord<D>::kBytes;
    static constexpr int kChunk = kWide ? 1 : 2; // pages
    static constexpr int kChunkBytes = kChunk * kPageBytes;
    static constexpr int kWarps = kWide ? (D == 128 ? 6 : 4) : kMT == 1 ? 8 : 4;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kStages = kWide && D == 128 ? 2 : 3; // chunks
    static constexpr int kRing = kWarps * kStages * kChunkBytes;
    static constexpr int kPitch = D + 4; // floats per row of a warp's partial result
    static constexpr int kMerge = kWarps * kRows * kPitch * 4;
    static constexpr int kBuf = kRing > kMerge ? kRing : kMerge;
    static constexpr int kBytes = kBuf + 8 * kWarps * kStages + 4 * (2 * kWarps + 2) * kRows;
    static constexpr int kSteps = D / 16; // k steps of Q K^T
    // resident CTAs: what shared memory and about (48 D / 64 kMT + 70) registers a thread leave
    static constexpr int kCtas = kWide ? (D == 64 ? 2 : 1) : kMT == 1 ? (D == 64 ? 2 : 1) : kMT == 2 && D == 64 ? 2 : 1;
};

// d += a (16 x 16 fp16) b (16 x 8 fp16)
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d += s, rounded: the tensor cores cut a sum off at every step, which over thousands
// of keys would cost fp32 rows bits
__device__ __forceinline__ void add4(float (&d)[4], const float (&s)[4]) {
    const float2 a = __fadd2_rn(make_float2(d[0], d[1]), make_float2(s[0], s[1])), b = __fadd2_rn(make_float2(d[2], d[3]), make_float2(s[2], s[3]));
    d[0] = a.x, d[1] = a.y, d[2] = b.x, d[3] = b.y;
}
// int8 codes as K operands: fp16 subnormals (c + 128) 2^-24, exact too. The
// offset is taken off by the accumulators' start, -128 sum q: two instructions
// a pair fewer than codes_to_half. (Not for V: its sums of many keys cancel,
// so the offset would cost the result's last bits.)
template <KvFormat kFmt> __device__ __forceinline__ void k_codes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if constexpr (kFmt == KvFormat::kInt8) {
        const uint32_t u = w ^ 0x80808080u;
        lo = __byte_perm(u, 0u, 0x4140);
        hi = __byte_perm(u, 0u, 0x4342);
    } else {
        codes_to_half<kFmt>(w, lo, hi);
    }
}

// x f and y f as two fp16 terms each, both rounded to nearest: 2^-24 is lost (a
// first term cut off instead: 2^-22, which showed in the results). `top` keeps
// the largest magnitude of the first terms, NaN and infinity included.
__device__ __forceinline__ void split_half2(float x, float y, float f, uint32_t &hi, uint32_t &lo, __half2 &top) {
    const float2 u = __fmul2_rn(make_float2(x, y), make_float2(f, f));
    hi = half2_rn(u.x, u.y);
    const float2 h = half2_floats(hi), r = __fadd2_rn(u, make_float2(-h.x, -h.y));
    lo = half2_rn(r.x, r.y);
    top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __half2 *>(&hi)));
}
// Whether a lane's magnitudes `top` are over 2^14, infinite or NaN, or all the warp's
// are below 2^-3 (two terms have 2^-22 of them left). The same in every lane.
__device__ __forceinline__ bool half2_out_of_range(__half2 top) {
    const float a = __low2float(top), b = __high2float(top);
    return __any_sync(kFullWarpMask, !(a <= 16384.f && b <= 16384.f)) || !__any_sync(kFullWarpMask, a >= 0.125f || b >= 0.125f);
}

template <typename T, int D, KvFormat kFmt, int kMT>
static __global__ void __launch_bounds__(TreeRowsGeo<T, D, kFmt, kMT>::kThreads, TreeRowsGeo<T, D, kFmt, kMT>::kCtas)
    tree_rows_kernel(const T *__restrict__ q, T *__restrict__ out, TreeArgs a, int groups, int splits, int first_wave, int *err) {
    using G = TreeRowsGeo<T, D, kFmt, kMT>;
    using R = KvRecord<D>;
    constexpr int kC = G::kChunk;
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + G::kBuf);
    float *stat = reinterpret_cast<float *>(bars + G::kWarps * G::kStages); // m [warps][rows], l [warps][rows]
    float *joined = stat + 2 * G::kWarps * G::kRows;                          // m [rows], l [rows] of the CTA

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int rank = blockIdx.x % splits, unit = blockIdx.x / splits;
    const int group = unit % groups, h = unit / groups;
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
    // Sequences longest first as far as every CTA gets an SM to itself, then
    // shortest first: the SMs that hold two CTAs hold a long and a short one (32
    // sequences of 1090 to 2180 tokens: 19.5 -> 18.9 us).
    int b = blockIdx.y;
    if (first_wave > 0)
        b = sequence_by_work(a.t, b < first_wave ? b : a.t.batch - 1 - (b - first_wave), reinterpret_cast<int *>(smem));

    // The chunks of a sequence go round the cluster's warps, so that a warp knows
    // its pages before it knows the sequence's length: chunk i of a warp is
    // first + i * step. Lane c of a chunk's first kC lanes copies its page c, and
    // a lane holds the block id of one page of the next 32 / kC chunks.
    const int first = rank * G::kWarps + warp, step = splits * G::kWarps;
    const int *table = a.t.block_table + static_cast<int64_t>(b) * a.t.table_stride;
    int ids = 0;
    const auto refill = [&](int base) {
        const int64_t page = (first + static_cast<int64_t>(base + lane / kC) * step) * kC + lane % kC;
        ids = page < a.t.table_stride ? table[page] : -1;
    };
    refill(0);

    const TreeSpan span(a.t, b);
    const int row_base = group * G::kRows, rows = span.n * rep; // query rows of this (sequence, head)
    int keys = span.keys;
    if (a.t.mask == nullptr) // a chain: nothing after the group's last node is seen
        keys = min(keys, span.ctx + (min(row_base + G::kRows, rows) + rep - 1) / rep);
    const int pages = row_base < rows ? (keys + kKvPage - 1) / kKvPage : 0;
    const int chunks = (pages + kC - 1) / kC;
    const int mine = chunks > first ? (chunks - first + step - 1) / step : 0; // chunks of this warp
    uint8_t *ring = smem + warp * G::kStages * G::kChunkBytes;

    const auto issue = [&](int i, int s) { // chunk i of this warp into stage s
        const int blk = __shfl_sync(kFullWarpMask, ids, (i * kC + lane % kC) & 31);
        const int n = min(kC, pages - (first + i * step) * kC);
        if (lane == 0)
            sm100::mbar_arrive_expect_tx(&bar[s], static_cast<uint32_t>(n * G::kPageBytes));
        __syncwarp();
        if (lane < n) {
            uint8_t *dst = ring + s * G::kChunkBytes + lane * G::kPageBytes;
            const int64_t rec = static_cast<int64_t>(blk) * a.kvh + h;
            if constexpr (G::kWide) {
                constexpr int kHalf = kKvPage * D * 4;
                sm100::bulk_load(dst, static_cast<const uint8_t *>(a.k) + rec * kHalf, kHalf, &bar[s]);
                sm100::bulk_load(dst + kHalf, static_cast<const uint8_t *>(a.v) + rec * kHalf, kHalf, &bar[s]);
            } else {
                sm100::bulk_load(dst, static_cast<const uint8_t *>(a.k) + rec * R::kBytes, R::kBytes, &bar[s]);
            }
        }
    };
    for (int i = 0; i < min(mine, G::kStages); ++i)
        issue(i, i);

    // Q fragments: k step s = 4c + i of 16 dims; lane t holds dims 64c + 16t +
    // 4i + {0, 1} (k = 2t, 2t + 1) and + {2, 3} (k = 2t + 8, 2t + 9). A negative
    // scale turns their sign, so that row_scale is not below zero.
    uint32_t qf[kMT][G::kSteps][4];
    float row_scale[kMT][G::kRPL], start[kMT][2];
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt) {
        float x[G::kRPL][D / 4];
#pragma unroll
        for (int rr = 0; rr < G::kRPL; ++rr) {
            const int r = row_base + mt * G::kTileRows + rr * 8 + g;
            const bool live = r < rows;
            const T *src = q + static_cast<int64_t>(span.row0 + (live ? r / rep : 0)) * a.q_stride +
                           static_cast<int64_t>(h * rep + (live ? r % rep : 0)) * D + 16 * t;
            constexpr int kN = KvVec<T>::kN;
#pragma unroll
            for (int v = 0; v < D / 4 / kN; ++v) {
                float y[kN] = {};
                if (live)
                    KvVec<T>::unpack(*reinterpret_cast<const uint4 *>(src + v * kN / 16 * 64 + v * kN % 16), y);
#pragma unroll
                for (int e = 0; e < kN; ++e)
                    x[rr][v * kN + e] = y[e];
            }
            // a power of two brings the row's largest magnitude to 2^9 .. 2^10,
            // so that fp16 holds the row to 2^-22 of it in two terms (and a
            // bf16 row exactly in one)
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < D / 4; ++e)
                top = max(top, __float_as_uint(x[rr][e]) & 0x7fffffffu);
            top = max(top, __shfl_xor_sync(kFullWarpMask, top, 1));
            top = max(top, __shfl_xor_sync(kFullWarpMask, top, 2));
            const uint32_t ex = exponent_above(top);
            const float f = copysignf(pow2_field(254u - ex + 10u), a.scale_log2);
            row_scale[mt][rr] = fabsf(a.scale_log2) * pow2_field(ex - 10u) * (kFmt == KvFormat::kInt8 ? 16777216.f : 1.f);
            if (top >= 0x7f800000u) // an infinity would be a score like others, or none
                row_scale[mt][rr] = __uint_as_float(0x7fc00000u);
#pragma unroll
            for (int e = 0; e < D / 4; ++e)
                x[rr][e] *= f;
        }
        float sum[2] = {0.f, 0.f}; // of rows g and g + 8 of the tile
#pragma unroll
        for (int s = 0; s < G::kSteps; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float u = x[0][4 * s + 2 * e], v = x[0][4 * s + 2 * e + 1];
                const uint32_t hi = half2_rn(u, v);
                const float2 f = half2_floats(hi);
                const uint32_t lo = G::kTwo ? half2_rn(u - f.x, v - f.y)
                                            : half2_rn(x[G::kRPL - 1][4 * s + 2 * e], x[G::kRPL - 1][4 * s + 2 * e + 1]);
                qf[mt][s][2 * e] = hi;
                qf[mt][s][2 * e + 1] = lo;
                sum[0] += f.x + f.y;
                sum[1] += half2_floats(lo).x + half2_floats(lo).y;
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            start[mt][i] = 0.f;
            if constexpr (kFmt == KvFormat::kInt8) {
                sum[i] += __shfl_xor_sync(kFullWarpMask, sum[i], 1);
                sum[i] += __shfl_xor_sync(kFullWarpMask, sum[i], 2);
                start[mt][i] = sum[i] * (-128.f / 16777216.f);
            }
        }
    }

    float o[kMT][D / 8][4] = {};
    // m: the reference that weights are relative to, 2^(x - m)
    float m[kMT][G::kRPL], l[kMT][G::kRPL];
    // 8-bit: a power of two next above the V scales of late and its log2, which goes
    // into m. fp32: the powers of two that K and V (32 dims each) of the last chunk were
    // multiplied by (0: not chosen yet)
    float vtop = kMinVTop, vlog = kMinVLog, kmul = 0.f, vmul[D / 32] = {};
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int rr = 0; rr < G::kRPL; ++rr)
            m[mt][rr] = kNone, l[mt][rr] = 0.f;
    bool wary = false; // the warp has met large scores
    const auto rescale = [&](int mt, const float (&fix)[G::kRPL]) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
            o[mt][n][0] *= fix[0];
            o[mt][n][1] *= fix[0];
            o[mt][n][2] *= fix[G::kRPL - 1];
            o[mt][n][3] *= fix[G::kRPL - 1];
        }
    };
    // fp32: columns 32 c .. of O go over to V times `next`
    const auto resize = [&](int c, float next) {
        const float up = vmul[c] == 0.f ? 1.f : next * pow2_field(254u - (__float_as_uint(vmul[c]) >> 23));
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[mt][4 * c + e][i] *= up;
        vmul[c] = next;
    };
    // one factor for all of O: the largest rows'. Returns it.
    const auto one_vmul = [&] {
        float least = 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
            least = vmul[c] == 0.f || (least != 0.f && least < vmul[c]) ? least : vmul[c];
        least = least == 0.f ? 1.f : least;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
            if (vmul[c] != least)
                resize(c, least);
        return least;
    };
    const auto poison = [&] { // a row that every node sees holds an infinity or a NaN
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int rr = 0; rr < G::kRPL; ++rr)
                l[mt][rr] = __uint_as_float(0x7fc00000u);
    };

    // One chunk. Edge chunks hold nodes, or places after the last key; chunks of
    // large scores are taken in the same way.
    // Score column g of n tile j of a page is key 8j + 4 (g & 1) + g / 2, so that
    // lane t's columns 2t + col are keys 8j + 4 col + t: value i = 2j + col of a
    // lane is key 4i + t.
    // False: not taken, for its scores are large (m is raised; see kWary).
    const auto take = [&](const uint8_t *chunk, int key0, auto edge_tag) -> bool {
        constexpr bool kEdge = decltype(edge_tag)::value;
        float sc[kMT][2 * kC][4];
        float kfac[4 * kC], vfac[4 * kC]; // factors of a lane's scores and weights
        float vlogs[kEdge ? 4 * kC : 1];  // log2 of the weights' factors, or a little more
        float vkey[kEdge ? 4 : 1];        // fp32: what V rows are multiplied by
        uint32_t bad = 0;                 // bit i: fp32 row i of the lane holds an infinity or a NaN
        float x[kMT][G::kRPL][4 * kC];
        const auto zero_scores = [&] {
#pragma unroll
            for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
                for (int j = 0; j < 2 * kC; ++j) {
                    sc[mt][j][0] = sc[mt][j][1] = start[mt][0];
                    sc[mt][j][2] = sc[mt][j][3] = start[mt][1];
                }
        };
        // fp32: a value of a key that is there and finite, else zero
        const auto sane = [&](float v, int key) { return key0 + key < keys ? finite_or_zero(v) : 0.f; };
        // fp32: largest magnitude (bits) among the K or V rows of the chunk
        const auto top_of = [&](const uint8_t *part) {
            uint32_t top = 0;
#pragma unroll 8
            for (int i = lane; i < kKvPage * D / 4; i += 32) {
                const float4 w = reinterpret_cast<const float4 *>(part)[i];
                const float y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    top = max(top, __float_as_uint(kEdge ? sane(y[e], i / (D / 4)) : y[e]) & 0x7fffffffu);
            }
            return __reduce_max_sync(kFullWarpMask, top);
        };

        if constexpr (G::kWide) {
            float kkey[2] = {kmul, kmul}; // what the lane's two K rows are multiplied by
            if constexpr (kEdge) {
                // Rows that are not finite, and each row's largest magnitude: a row that a
                // node does not see takes no bits from the others. Lanes t, t + 4, .. hold
                // a row's eighths.
                const int unit = static_cast<int>(__float_as_uint(one_vmul()) >> 23) - 127;
                uint32_t kex[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        const float4 *src = reinterpret_cast<const float4 *>(chunk + (part * kKvPage + 4 * i + t) * D * 4) + g;
                        bool odd = false;
                        uint32_t top = 0;
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            const float4 w = src[8 * c];
                            const float y[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                odd |= !(fabsf(y[e]) <= 3.4028235e38f);
                                top = max(top, __float_as_uint(sane(y[e], 4 * i + t)) & 0x7fffffffu);
                            }
                        }
                        bad |= ((__ballot_sync(kFullWarpMask, odd) >> t) & 0x11111111u) != 0u ? 1u << i : 0u;
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1)
                            top = max(top, __shfl_xor_sync(kFullWarpMask, top, off));
                        const uint32_t ex = exponent_above(top, 254u);
                        if (part == 0) {
                            kex[i] = ex;
                            kfac[i] = pow2_field(ex - 8u);
                        } else {
                            const int log = max(static_cast<int>(ex) - 127, kMinVKey) - 8; // to 2^7 .. 2^8
                            vkey[i] = pow2_field(static_cast<uint32_t>(127 - log));
                            vlogs[i] = static_cast<float>(max(-126, min(126, log + unit)));
                            vfac[i] = pow2_field(static_cast<uint32_t>(127 + static_cast<int>(vlogs[i])));
                        }
                    }
#pragma unroll
                for (int j = 0; j < 2; ++j) { // K row 8j + 4 (g & 1) + (g >> 1) is row 4i + t of lane g >> 1, i = 2j + (g & 1)
                    const uint32_t ex0 = __shfl_sync(kFullWarpMask, kex[2 * j], g >> 1), ex1 = __shfl_sync(kFullWarpMask, kex[2 * j + 1], g >> 1);
                    kkey[j] = pow2_field(254u - (g & 1 ? ex1 : ex0) + 8u);
                }
            }
            bool anew = !kEdge && kmul == 0.f; // (edge chunks: each row has its own factor)
            zero_scores();
#pragma unroll 1
            for (int attempt = 0;; ++attempt) { // again after a new kmul
                if (anew) {
                    const uint32_t top = top_of(chunk);
                    if (top >= 0x7f800000u) {
                        poison();
                        break;
                    }
                    if (attempt > 0 && top == 0u)
                        break;
                    kkey[0] = kkey[1] = kmul = pow2_field(254u - exponent_above(top, 254u) + 8u); // to 2^7 .. 2^8
                }
                zero_scores();
                float small[kMT][2][4] = {}; // the small products: an accumulator is cut off at every step, to its size
                __half2 seen_top = __float2half2_rn(0.f);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int krow = 8 * j + 4 * (g & 1) + (g >> 1);
                    const uint8_t *src = chunk + krow * D * 4 + 64 * t;
#pragma unroll
                    for (int st = 0; st < G::kSteps; ++st) {
                        const float4 w = *reinterpret_cast<const float4 *>(src + st / 4 * 256 + st % 4 * 16);
                        float y[4] = {w.x, w.y, w.z, w.w};
                        if (kEdge)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                y[e] = sane(y[e], krow);
                        uint32_t h0, h1, l0, l1;
                        split_half2(y[0], y[1], kkey[j], h0, l0, seen_top);
                        split_half2(y[2], y[3], kkey[j], h1, l1, seen_top);
#pragma unroll
                        for (int mt = 0; mt < kMT; ++mt) {
                            mma_f16(sc[mt][j], qf[mt][st], h0, h1);
                            mma_f16(small[mt][j], qf[mt][st], l0, l1);
                        }
                    }
                }
#pragma unroll
                for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
                    for (int n = 0; n < 8; ++n)
                        sc[mt][n / 4][n % 4] += small[mt][n / 4][n % 4];
                anew = !kEdge && attempt < 2 && half2_out_of_range(seen_top);
                if (!anew)
                    break;
            }
        } else {
            zero_scores();
#pragma unroll
            for (int j = 0; j < 2 * kC; ++j) {
                const uint8_t *src = chunk + j / 2 * G::kPageBytes + (8 * (j % 2) + 4 * (g & 1) + (g >> 1)) * D + 16 * t;
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {
                    const uint4 w4 = *reinterpret_cast<const uint4 *>(src + 64 * c);
                    const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t b0, b1;
                        k_codes_to_half<kFmt>(w[i], b0, b1);
#pragma unroll
                        for (int mt = 0; mt < kMT; ++mt)
                            mma_f16(sc[mt][j], qf[mt][4 * c + i], b0, b1);
                    }
                }
            }
        }
        // factors of the scores, and the largest V scale of the lane
        float vscale = 0.f;
#pragma unroll
        for (int i = 0; i < 4 * kC; ++i) {
            if constexpr (G::kWide && kEdge) {
                // set above
            } else if constexpr (G::kWide) {
                kfac[i] = vfac[i] = 1.f; // K's is the page's, see kunit
            } else {
                const uint8_t *page = chunk + i / 4 * G::kPageBytes + 16 * (i % 4) + 4 * t;
                kfac[i] = *reinterpret_cast<const float *>(page + R::kKScale);
                vfac[i] = *reinterpret_cast<const float *>(page + R::kVScale);
                if constexpr (kEdge) { // (places after the last key have none)
                    const float nan = __uint_as_float(0x7fc00000u);
                    kfac[i] = fabsf(kfac[i]) <= 3.4028235e38f ? kfac[i] : nan;
                    vfac[i] = fabsf(vfac[i]) <= 3.4028235e38f ? vfac[i] : nan;
                    const uint32_t ex = exponent_above(__float_as_uint(key0 + 4 * i + t < keys ? finite_or_zero(vfac[i]) : 0.f), 253u);
                    vlogs[i] = fmaxf(static_cast<float>(static_cast<int>(ex) - 127), kMinVLog);
                } else {
                    vscale = fmaxf(vscale, vfac[i]);
                }
            }
        }
        const float kunit = G::kWide && !kEdge ? pow2_field(254u - (__float_as_uint(kmul) >> 23)) : 1.f;
        // Scores: less their row's scale; of edge chunks in log2 units, masked ones -inf,
        // and the V factors of the keys that a row sees enter its own reference
        bool raise = vscale > vtop;
        if (!kEdge && !G::kWide) // V far below the chunks before: its own size again
            raise |= vtop > kMinVTop && !__any_sync(kFullWarpMask, vscale >= vtop * kLowV);
        const float slack = G::kWide || kEdge ? kLazy + kLift : kLazy + kLift - vlog;
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
            for (int rr = 0; rr < G::kRPL; ++rr) {
#pragma unroll
                for (int i = 0; i < 4 * kC; ++i) {
                    const float *c = sc[mt][i >> 1], s = G::kTwo ? c[i & 1] + c[2 + (i & 1)] : c[2 * rr + (i & 1)];
                    x[mt][rr][i] = G::kWide ? s : s * kfac[i];
                }
                const float scale = row_scale[mt][rr] * kunit;
                float top = kNegInf;
                if constexpr (kEdge) {
                    const int r = row_base + mt * G::kTileRows + rr * 8 + g;
                    uint32_t seen = 0;
                    if (r < rows)
                        seen = tree_sees32(a.t, span.row0 + r / rep, r / rep, key0 - span.ctx, keys - span.ctx);
#pragma unroll
                    for (int i = 0; i < 4 * kC; ++i) {
                        float y = G::kWide ? x[mt][rr][i] * scale * kfac[i] : x[mt][rr][i] * scale;
                        if (G::kWide && (bad >> i & 1u))
                            y = __uint_as_float(0x7fc00000u);
                        if (!(seen >> (4 * i + t) & 1u))
                            y = kNegInf;
                        x[mt][rr][i] = y;
                        top = fmaxf(top, y + vlogs[i]);
                    }
                    raise |= top > m[mt][rr] + slack;
                } else {
#pragma unroll
                    for (int i = 0; i < 4 * kC; ++i)
                        top = fmaxf(top, x[mt][rr][i]);
                    raise |= top * scale > m[mt][rr] + slack;
                }
            }
        if (__any_sync(kFullWarpMask, raise)) {
            if (!kEdge && !G::kWide) {
                const uint32_t top = __reduce_max_sync(kFullWarpMask, __float_as_uint(vscale)); // not below zero
                if (top >= 0x7f800000u) {
                    poison();
                } else if (__uint_as_float(top) > vtop || __uint_as_float(top) < vtop * kLowV) {
                    vtop = fmaxf(pow2_field(exponent_above(top, 253u)), kMinVTop);
                    vlog = static_cast<float>(static_cast<int>(__float_as_uint(vtop) >> 23) - 127);
                }
            }
#pragma unroll
            for (int mt = 0; mt < kMT; ++mt) {
                float fix[G::kRPL];
#pragma unroll
                for (int rr = 0; rr < G::kRPL; ++rr) {
                    float up = kNegInf;
#pragma unroll
                    for (int i = 0; i < 4 * kC; ++i)
                        up = fmaxf(up, kEdge ? x[mt][rr][i] + vlogs[kEdge ? i : 0] : x[mt][rr][i]);
                    up = fmaxf(up, __shfl_xor_sync(kFullWarpMask, up, 1));
                    up = fmaxf(up, __shfl_xor_sync(kFullWarpMask, up, 2));
                    if (!kEdge)
                        up = up * (row_scale[mt][rr] * kunit) + (G::kWide ? 0.f : vlog);
                    up = fmaxf(m[mt][rr], up - reference_lift(kLift, up));
                    wary |= fabsf(up) > kWary && up > kNone;
                    fix[rr] = exp2_approx(m[mt][rr] - up);
                    m[mt][rr] = up;
                    l[mt][rr] *= fix[rr];
                }
                rescale(mt, fix);
            }
            wary = __any_sync(kFullWarpMask, wary);
            if (!kEdge && wary)
                return false;
        }
        // P as A fragments; l sums the weights before they are rounded
        uint32_t pf[kMT][kC][4];
#pragma unroll
        for (int mt = 0; mt < kMT; ++mt) {
            float p[G::kRPL][4 * kC];
#pragma unroll
            for (int rr = 0; rr < G::kRPL; ++rr) {
                const float scale = row_scale[mt][rr] * kunit;
#pragma unroll
                for (int i = 0; i < 4 * kC; ++i) {
                    float e = kEdge ? x[mt][rr][i] - m[mt][rr] : fmaf(x[mt][rr][i], scale, -m[mt][rr]);
                    if (kEdge) { // (a NaN stays)
                        const float cap = kLift + kLazy + 1.f - vlogs[kEdge ? i : 0];
                        e = e > cap ? cap : e;
                    }
                    const float w = exp2_approx(e);
                    const bool masked = kEdge && x[mt][rr][i] == kNegInf; // no weight, whatever the row's scales
                    l[mt][rr] += w;
                    p[rr][i] = (G::kWide && !kEdge) || masked ? w : w * vfac[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 2 * kC; ++i) {
                const uint32_t hi = half2_rn(p[0][2 * i], p[0][2 * i + 1]);
                pf[mt][i >> 1][2 * (i & 1)] = hi;
                if constexpr (G::kTwo) {
                    const float2 f = half2_floats(hi);
                    pf[mt][i >> 1][2 * (i & 1) + 1] = half2_rn(p[0][2 * i] - f.x, p[0][2 * i + 1] - f.y);
                } else {
                    pf[mt][i >> 1][2 * (i & 1) + 1] = half2_rn(p[G::kRPL - 1][2 * i], p[G::kRPL - 1][2 * i + 1]);
                }
            }
        }
        // O += P V. 8-bit: column g of n tile n is dim (D / 8) g + n. fp32:
        // column g of n tile 4c + e is dim 32c + 4g + e.
        if constexpr (G::kWide) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t hi[4][2], lo[4][2]; // of dims 32c + 4g + e, keys (t, 4 + t) and (8 + t, 12 + t)
                bool anew = !kEdge && vmul[c] == 0.f;
#pragma unroll 1
                for (int attempt = 0;; ++attempt) {
                    float y[4][4]; // value i's key, dim e
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 w = *reinterpret_cast<const float4 *>(chunk + (kKvPage + 4 * i + t) * D * 4 + 128 * c + 16 * g);
                        y[i][0] = w.x, y[i][1] = w.y, y[i][2] = w.z, y[i][3] = w.w;
                        if (kEdge)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                y[i][e] = sane(y[i][e], 4 * i + t) * vkey[kEdge ? i : 0];
                    }
                    if (anew) {
                        uint32_t top = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                top = max(top, __float_as_uint(y[i][e]) & 0x7fffffffu);
                        top = __reduce_max_sync(kFullWarpMask, top);
                        if (top >= 0x7f800000u) {
                            poison();
                            top = 0u;
                        }
                        if (attempt > 0 && top == 0u)
                            break;
                        // to 2^7 .. 2^8; what is summed already must not leave fp32's range
                        float next = pow2_field(254u - max(exponent_above(top, 254u), static_cast<uint32_t>(127 + kMinVKey)) + 8u);
                        if (next > vmul[c] && vmul[c] != 0.f) {
                            uint32_t most = 0;
#pragma unroll
                            for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
                                for (int n = 4 * c; n < 4 * c + 4; ++n)
#pragma unroll
                                    for (int i = 0; i < 4; ++i)
                                        most = max(most, __float_as_uint(o[mt][n][i]) & 0x7fffffffu);
                            most = __reduce_max_sync(kFullWarpMask, most) >> 23;
                            const uint32_t room = most < 227u ? min(227u - most, 100u) : 0u; // to 2^100
                            next = fminf(next, vmul[c] * pow2_field(127u + room));
                        }
                        resize(c, next);
                    }
                    const float vmul_here = kEdge ? 1.f : vmul[c];
                    __half2 seen_top = __float2half2_rn(0.f);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            if constexpr (G::kTwo) {
                                split_half2(y[2 * j][e], y[2 * j + 1][e], vmul_here, hi[e][j], lo[e][j], seen_top);
                            } else {
                                hi[e][j] = half2_rn(y[2 * j][e] * vmul_here, y[2 * j + 1][e] * vmul_here);
                                seen_top = __hmax2_nan(seen_top, __habs2(*reinterpret_cast<const __half2 *>(&hi[e][j])));
                            }
                        }
                    anew = !kEdge && attempt < 2 && half2_out_of_range(seen_top);
                    if (!anew)
                        break;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int mt = 0; mt < kMT; ++mt) {
                        float sum[4] = {};
                        if constexpr (G::kTwo)
                            mma_f16(sum, pf[mt][0], lo[e][0], lo[e][1]);
                        mma_f16(sum, pf[mt][0], hi[e][0], hi[e][1]);
                        add4(o[mt][4 * c + e], sum);
                    }
            }
        } else {
#pragma unroll
            for (int pg = 0; pg < kC; ++pg) {
                constexpr int kWords = D / 32;
                uint32_t w[4][kWords];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint8_t *src = chunk + pg * G::kPageBytes + R::kCodes + (4 * i + t) * D + (D / 8) * g;
                    if constexpr (kWords == 2) {
                        const uint2 u = *reinterpret_cast<const uint2 *>(src);
                        w[i][0] = u.x, w[i][1] = u.y;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4 *>(src);
                        w[i][0] = u.x, w[i][1] = u.y, w[i][kWords - 2] = u.z, w[i][kWords - 1] = u.w;
                    }
                    if (kFmt == KvFormat::kE4M3 && kEdge)
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
                            if constexpr (G::kTwo) {
                                float sum[4] = {};
                                mma_f16(sum, pf[mt][pg], b0[e], b1[e]);
                                add4(o[mt][4 * c + e], sum);
                            } else {
                                mma_f16(o[mt][4 * c + e], pf[mt][pg], b0[e], b1[e]);
                            }
                }
            }
        }
        return true;
    };

    bool ok = true;
    int done = 0, stage = 0;
    uint32_t parity = 0;
    for (; done < mine; ++done) {
        if (!sm100::mbar_wait_warp(&bar[stage], parity)) {
            ok = false;
            break;
        }
        const uint8_t *chunk = ring + stage * G::kChunkBytes;
        const int key0 = (first + done * step) * kC * kKvPage;
        if (key0 + kC * kKvPage > span.ctx || wary || !take(chunk, key0, std::false_type{}))
            take(chunk, key0, std::true_type{});
        __syncwarp(); // every lane has read the stage
        const int next = done + G::kStages;
        if (next < mine) {
            if (next % (32 / kC) == 0)
                refill(next);
            issue(next, stage);
        }
        if (++stage == G::kStages) {
            stage = 0;
            parity ^= 1u;
        }
    }
    // a wait that ran out: the copies still in flight must land before the ring is used again
    if (!ok)
        for (int i = done; i < min(mine, done + G::kStages); ++i)
            sm100::mbar_wait(&bar[i % G::kStages], static_cast<uint32_t>(i / G::kStages) & 1u);
    if (!__syncthreads_and(ok) && tid == 0)
        atomicExch(err, 7);

    // the warps' results over the ring, joined in warp order
    float *part = reinterpret_cast<float *>(smem);
    // fp32: V's unit goes into m and l, for O times it may leave fp32's range
    float vunit = 1.f, unit_log = 0.f;
    if constexpr (G::kWide) {
        vunit = one_vmul();
        unit_log = static_cast<float>(static_cast<int>(__float_as_uint(vunit) >> 23) - 127);
    }
#pragma unroll
    for (int mt = 0; mt < kMT; ++mt)
#pragma unroll
        for (int rr = 0; rr < G::kRPL; ++rr) {
            const int r = mt * G::kTileRows + rr * 8 + g;
            float sum = l[mt][rr];
            sum += __shfl_xor_sync(kFullWarpMask, sum, 1);
            sum += __shfl_xor_sync(kFullWarpMask, sum, 2);
            float *dst = part + (warp * G::kRows + r) * G::kPitch;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int col = 0; col < 2; ++col) {
                    const float v = G::kTwo ? o[mt][n][col] + o[mt][n][2 + col] : o[mt][n][2 * rr + col];
                    const int d = G::kWide ? 32 * (n / 4) + 4 * (2 * t + col) + n % 4 : (D / 8) * (2 * t + col) + n;
                    dst[d] = v;
                }
            if (t == 0) {
                stat[warp * G::kRows + r] = m[mt][rr] - unit_log;
                stat[(G::kWarps + warp) * G::kRows + r] = sum * vunit;
            }
        }
    __syncthreads();
    const int live = min(G::kRows, rows - row_base); // may be negative
    for (int i = tid; i < G::kRows * D; i += G::kThreads) {
        const int r = i / D, d = i % D;
        if (r >= live)
            break;
        float top = kNone, L = 0.f, O = 0.f;
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
        float top = kNone, L = 0.f, O = 0.f;
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
    const int most = allow_shared_bytes(kernel, G::kThreads, G::kBytes);
    const int64_t rows = static_cast<int64_t>(a.t.max_rows) * (a.qh / a.kvh);
    const int64_t groups = (rows + G::kRows - 1) / G::kRows;
    const int64_t units = groups * a.kvh;
    const int64_t pages = (static_cast<int64_t>(a.t.max_ctx) + a.t.max_rows + kKvPage - 1) / kKvPage;
    // As many splits as all CTAs still run at once and warps have a chunk: a CTA
    // has about 5 us of latencies to pay for (lengths, table, first copies,
    // joining), so a second wave costs more than it evens out (32 sequences of
    // 2180 tokens, 8 kv heads: 19.3 us with 1 split, 25.6 with 2, 33.7 with 4).
    // 16 CTAs to a cluster only where each warp has much to do.
    const int64_t slots = static_cast<int64_t>(G::kCtas) * device_facts().sm_count;
    const int64_t per_warp = pages / (G::kWarps * G::kChunk), all = units * a.t.batch;
    const int64_t room = slots / all;
    const int64_t cap = room >= 16 && per_warp >= 64 ? most : std::min<int64_t>(8, 2 * per_warp);
    const int splits = static_cast<int>(std::max<int64_t>(1, std::min(cap, room)));
    require(units * splits <= 0x7fffffff, "tree attention: too many rows for one call");
    const int64_t per_sequence = units * splits, sms = device_facts().sm_count;
    const bool sort = a.t.batch > 1 && a.t.batch < G::kThreads && per_sequence * a.t.batch > sms;
    const int first_wave = sort ? static_cast<int>((sms + per_sequence - 1) / per_sequence) : 0;
    launch_ex_cluster(kernel, dim3(static_cast<unsigned>(units * splits), a.t.batch), dim3(splits), dim3(G::kThreads),
                      G::kBytes, stream, q, out, a, static_cast<int>(groups), splits, first_wave, sm100::device_error_word());
}

} // namespace opworks::detail
