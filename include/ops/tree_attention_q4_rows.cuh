#pragma once

// Attention over the 4-bit cache, kernel for few query rows per KV head
// (ops/tree_attention_q4.cuh has the definition): mma.sync, K and V widened in
// registers.
//
// The keys of a step (32: two pages) are the M side of the scores, the dims that of
// the output, and the rows of a KV head (row = node * rep + head in group) the N
// side of both, 8 columns a tile: so few rows waste little, and a lane holds the
// scores of few rows and many keys. Every warp of the CTA has the same rows and
// takes every n-th step; the steps of a sequence go round the warps of a cluster,
// and what they have is joined at the end through shared memory, in rank order.
//
// A page record comes with 16-byte asynchronous copies into a ring that only this
// warp uses, so nothing in the loop waits for another warp. ldmatrix hands out its
// codes as fragments, four codes to a 16-bit element: of K eight dims of a key (the
// four k slots of two products, in an order that Q follows), of V, transposed, four
// dims of two keys each. Widening them is most of what the loop does. K's stay
// integers, two operations a pair of codes, and their scale multiplies the sum over
// the group's dims; V's are multiplied out, since a scale is a key's there, which
// the product sums over.
//
// fp32 rows are two fp16 terms, and so are their weights. Up to 4 rows have two
// columns each, which are the two terms (bf16 rows: one is empty); above that fp32 rows take a product for each term, in one
// accumulator. The tensor cores cut an accumulator off at every step, so fp32 rows
// add up O outside of them, rounded, once a step.
//
// What bounds it is instructions (issue slots 67 % busy over long contexts): per 32 keys
// of 64 dims about 490 a warp, of which widening is 176, products 16, scales and softmax
// 90, copies and the rest of the loop the others. Per warp 600 more come before and after
// (lengths, queries, joining). Measured (kernel time, one B200): 32 sequences of up to
// 2180 tokens, one token each, 8 x 64 fp32, 4 rows a head 13.2 us (with nothing to attend
// to 5; floor 4.8); 12 of up to 32,000 tokens, 8 x 128 bf16 86 us, 3.9 TB/s (floor 52).
// Rows on the M side of the products, 16 to a tile, took 20.6 and 135.8 us.

#include <type_traits>

#include "tree_attention_common.cuh"
#include "tree_attention_rows.cuh"
#include "kv4.cuh"

namespace opworks::detail {

// The tensor cores cut a sum off at every product of 16 keys, by less than a unit in its last
// place. bf16 rows of more than 4 a head are summed there, and over V of one sign they came out
// smaller by 2^-23.6 a product (160 sequences of 1,000,000 tokens: by 3.0e-4 over the 62,500 keys
// of a warp here, by 2.5e-3 over the 500,000 of a stream of the tiles; rounding to bf16 is 1.3e-3
// in the mean). So the sum of kQ4SumKeys (4e-5), of kQ4SumTiles tiles (8e-5), is put by: added,
// rounded, to one in local memory, which only a reference that is raised touches else. A kernel of
// its own does that, where the context may be so long: the code alone costs 0 to 4 % (2048 rows
// behind 40,000 tokens, D 128: 2.16 ms without, 2.20 with; 8 rows a head of 64 sequences of 2,000:
// 46.4 us, 47.7). Sums of one step added up outside, as fp32 rows have them, cost 4 to 8 % at every
// length, and tiles of 128 dims have no room for them; more splits by the bound of the context are
// paid by every short sequence (a bound of 131,072: 2.5 to 4 times as long).
constexpr int kQ4SumKeys = 8192, kQ4SumTiles = 128;

// kNT: tiles of 8 columns; 0: one tile with two columns a row.
template <typename T, int D, int kNT> struct Q4RowsGeo {
    static constexpr bool kWide = std::is_same_v<T, float>, kPair = kNT == 0;
    static constexpr int kTiles = kPair ? 1 : kNT;
    static constexpr int kGroups = D / kKv4Group;
    static constexpr float kLift = kWide ? 6.f : 0.f; // see kQ4Top
    static constexpr int kRows = kPair ? 4 : 8 * kNT;
    static constexpr int kRPL = kPair ? 1 : 2 * kNT;         // rows that a lane has scores of
    static constexpr int kSets = kWide && !kPair ? 2 : 1;    // products of a k step
    static constexpr bool kQShared = kSets * kTiles * D > 256; // queries in shared memory, not in registers
    // 8 warps, as long as two CTAs of them fit on an SM; else 4 (16 rows, 32 sequences of 2180
    // tokens: fp32 27.7 us with 8, 25.7 with 4; bf16, D 128 33.2, 31.2; bf16, D 64 23.1, 26.9)
    static constexpr int kWarps = kNT <= 1 || (kNT == 2 && D == 64 && !kWide) ? 8 : 4, kThreads = 32 * kWarps;
    // a step: 64 keys where registers and shared memory have room, since what is done once a
    // step is a third of the instructions of 32
    static constexpr int kPairs = D == 64 && kNT <= 1 ? 2 : 1; // of pages
    static constexpr int kStepPages = 2 * kPairs, kStepKeys = kStepPages * kKvPage;
    static constexpr int kStages = kPairs == 2 ? 2 : 3;
    static constexpr bool kInCore = !kWide && !kPair;           // O is summed by the tensor cores,
    static constexpr int kPeriod = kQ4SumKeys / kStepKeys;      // and put by after so many steps of a warp
    static constexpr int kFar = 8 * kGroups * kTiles;           // floats of O that a lane has
    static constexpr int kPageBytes = Kv4Record<D>::kBytes, kStage = kStepPages * kPageBytes;
    static constexpr int kQBytes = kSets * kTiles * kGroups * 2 * 32 * 8 + 128; // fragments; a factor a row
    static constexpr int kRing = kStages * kStage; // of a warp
    static constexpr int kPitch = D + 4; // floats of a row of partial sums
    // O of the warps, then of the CTA; m and l of the warps, then of the CTA
    static constexpr int kJoin = 4 * ((kWarps + 1) * kRows * kPitch + 2 * (kWarps + 1) * kRows);
    static constexpr int kLoop = kQBytes + kWarps * kRing;
    static constexpr int kBytes = kLoop > kJoin ? kLoop : kJoin;
};

// Weights are 2^(x - reference). Scores may pass a row's reference by kQ4Top log2
// units before it is raised, to kLift below the largest: fp16 keeps steps of 2^-24, so
// 2^-25 of the largest weight is what a bf16 row's may be off by, 2^-31 an fp32 row's.
// (Raised to 8 below it, prompts did so for some row of a warp in every few tiles.)
constexpr float kQ4Top = 15.f;
constexpr float kQ4None = -3.4028235e38f; // reference of a row that has seen nothing yet
constexpr uint32_t kQ4BadScale = 0x7000u; // fp16 8,192: above every scale that is written; junk, infinity, NaN

__device__ __forceinline__ void q4_copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void q4_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void q4_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

template <bool kTrans> __device__ __forceinline__ void q4_ldmatrix(uint32_t at, uint32_t (&r)[4]) {
    if constexpr (kTrans)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(at)
                     : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(at)
                     : "memory");
}
// An 8 x 8 matrix of 16-bit elements, two of a row to a lane, turned round.
__device__ __forceinline__ uint32_t q4_transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// x, y as an fp16 pair, and what that leaves of them
__device__ __forceinline__ uint32_t q4_term(float &x, float &y) {
    const uint32_t h = half2_rn(x, y);
    const float2 f = half2_floats(h);
    x -= f.x, y -= f.y;
    return h;
}
// both terms of x, and of y, as pairs
__device__ __forceinline__ void q4_terms(float x, float y, uint32_t &px, uint32_t &py) {
    const uint32_t hi = q4_term(x, y), lo = half2_rn(x, y);
    px = __byte_perm(hi, lo, 0x5410), py = __byte_perm(hi, lo, 0x7632);
}

__device__ __forceinline__ float4 peer_load4(const float *p, int rank) {
    uint32_t at;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(sm100::smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

__device__ __forceinline__ void q4_store4(float *p, const float (&x)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void q4_store4(__nv_bfloat16 *p, const float (&x)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// The scale of a query row (a power of two that brings its largest magnitude `top`
// to 2^14 .. 2^15, held where its inverse is a normal number) and what scores are
// multiplied by. NaN where the row holds one, or an infinity, or the scale is one. The latter is held to 2^86,
// where scores stay finite; what differs at all differs by far more than a weight can
// tell, then.
__device__ __forceinline__ float q4_row_scale(float top, float scale_log2, float &factor) {
    const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -106), 127);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 - e) << 23), down = __uint_as_float(static_cast<uint32_t>(127 + e - 14) << 23);
    factor = fminf(fmaxf(scale_log2 * down, -0x1p86f), 0x1p86f);
    if (!(top <= 3.4028235e38f) || scale_log2 != scale_log2)
        factor = __uint_as_float(0x7fc00000u);
    return up;
}

// The span of the sequence that CTAs with z = `order` take: the one with the
// order-th most work (the longest context, equal ones by index) up to `descending`,
// from there on the one with the least first. So CTAs come longest first, or, where
// all run at once and each SM gets some of the first and of the second kind, long ones
// share an SM with short ones. Every thread of the block calls it; `room` is shared
// memory for 4 ints and one more a sequence.
__device__ __forceinline__ TreeSpan q4_span_by_work(const TreeBatch &t, int order, int descending, int *room) {
    const int tid = threadIdx.x;
    if (order >= descending)
        order = t.batch - 1 - (order - descending);
    for (int b = tid; b < t.batch; b += blockDim.x) {
        const TreeSpan s(t, b);
        room[4 + b] = s.n > 0 ? s.ctx : -1;
    }
    __syncthreads();
    for (int b0 = 0; b0 < t.batch; b0 += blockDim.x / 8) { // eight threads a sequence
        const int b = b0 + tid / 8, work = b < t.batch ? room[4 + b] : 0;
        int before = 0;
        if (b < t.batch)
            for (int i = tid % 8; i < t.batch; i += 8)
                before += room[4 + i] > work || (room[4 + i] == work && i < b) ? 1 : 0;
#pragma unroll
        for (int off = 1; off < 8; off <<= 1)
            before += __shfl_xor_sync(kFullWarpMask, before, off);
        if (b < t.batch && before == order && tid % 8 == 0)
            room[0] = b;
    }
    __syncthreads();
    const TreeSpan s(t, room[0]);
    __syncthreads(); // `room` may lie where copies go next
    return s;
}

// kPutBy: a warp may have more than kPeriod steps, and sums are put by.
template <typename T, int D, int kNT, bool kPutBy>
static __global__ void __launch_bounds__(Q4RowsGeo<T, D, kNT>::kThreads, kNT <= 1 ? 2 : 1)
    q4_rows_kernel(const T *__restrict__ q, T *__restrict__ out, TreeArgs a, int rep, int splits, int descending) {
    using G = Q4RowsGeo<T, D, kNT>;
    using R = Kv4Record<D>;
    constexpr bool kPair = G::kPair;
    extern __shared__ __align__(128) uint8_t q4_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    constexpr int threads = G::kThreads, warps = G::kWarps;
    const int h = blockIdx.y;
    int rank = blockIdx.x, group = 0; // groups of rows side by side, the CTAs of a cluster each
    if (gridDim.x != splits)
        group = rank / splits, rank -= group * splits;
    pdl_trigger();
    pdl_wait();
    const TreeSpan span = descending > 0 ? q4_span_by_work(a.t, blockIdx.z, descending, reinterpret_cast<int *>(q4_smem)) : TreeSpan(a.t, blockIdx.z);
    const int b = span.b, row_base = group * G::kRows, rows = span.n * rep;
    if (row_base >= rows)
        return; // the whole cluster
    int keys = span.keys;
    if (a.t.mask == nullptr) // a chain: nothing after the tile's last node is seen
        keys = min(keys, span.ctx + (min(row_base + G::kRows, rows) + rep - 1) / rep);
    const int steps = (keys + G::kStepKeys - 1) / G::kStepKeys;
    const int first = rank * warps + warp, stride = splits * warps;
    const int mine = steps > first ? (steps - first + stride - 1) / stride : 0;

    const auto node_of = [&](int r) { return span.n == 1 ? 0 : r / rep; };

    // ---- copies
    const int *table = a.t.block_table + static_cast<int64_t>(b) * a.t.table_stride;
    const int pages = (keys + kKvPage - 1) / kKvPage;
    uint8_t *ring = q4_smem + G::kQBytes + warp * G::kRing;
    int ids = 0; // a lane has the block of one page of the next steps
    const auto fetch = [&](int i, int to) {
        constexpr int kAhead = 32 / G::kStepPages; // steps whose pages are looked up at once
        if (i < mine) {
            if (i % kAhead == 0) {
                const int s = i + lane / G::kStepPages, page = (first + s * stride) * G::kStepPages + lane % G::kStepPages;
                ids = s < mine && page < pages ? max(0, table[page]) : 0; // after the last page: block 0, and masked
            }
            const uint32_t dst = sm100::smem_u32(ring + to * G::kStage);
#pragma unroll
            for (int pg = 0; pg < G::kStepPages; ++pg) {
                const int64_t id = __shfl_sync(kFullWarpMask, ids, i % kAhead * G::kStepPages + pg);
                const uint8_t *src = static_cast<const uint8_t *>(a.k) + (id * a.kvh + h) * R::kBytes;
#pragma unroll
                for (int c = 0; c < G::kPageBytes; c += 512)
                    if (c + lane * 16 < G::kPageBytes)
                        q4_copy16(dst + pg * G::kPageBytes + c + lane * 16, src + c + lane * 16);
            }
        }
        q4_copy_commit();
    };
#pragma unroll
    for (int i = 0; i < G::kStages - 1; ++i)
        fetch(i, i);

    // ---- queries, as fragments: column g of a tile, k slots 2t, 2t + 1 and 2t + 8, 2t + 9 of product u: dims 8t + 2u, + 4
    // and 8t + 2u + 1, + 5 of the group. Every warp wants the same ones: the tiles are shared out, and handed round through
    // shared memory.
    constexpr int kInRegs = G::kQShared ? 1 : G::kGroups; // (not used where they stay in shared memory)
    uint32_t qf[G::kSets][G::kTiles][kInRegs][2][2];
    uint2 *q_shared = reinterpret_cast<uint2 *>(q4_smem); // [set][tile][group][u][lane]
    float *factors = reinterpret_cast<float *>(q4_smem + G::kQBytes - 4 * G::kRows); // of the scores of each row
    float factor[G::kRPL];
#pragma unroll 1
    for (int nt = warp; nt < G::kTiles; nt += warps) {
        const int r = row_base + (kPair ? g / 2 : nt * 8 + g), node = node_of(r);
        float x[G::kGroups][8];
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < G::kGroups; ++c) {
            if (r < rows) {
                const T *src = q + static_cast<int64_t>(span.row0 + node) * a.q_stride + static_cast<int64_t>(h * rep + r - node * rep) * D + 32 * c + 8 * t;
#pragma unroll
                for (int i = 0; i < 8 / KvVec<T>::kN; ++i) {
                    float y[KvVec<T>::kN];
                    KvVec<T>::unpack(*reinterpret_cast<const uint4 *>(src + i * KvVec<T>::kN), y);
#pragma unroll
                    for (int j = 0; j < KvVec<T>::kN; ++j)
                        x[c][i * KvVec<T>::kN + j] = y[j];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[c][i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < 8; i += 2)
                top = max_abs_nan(top, x[c][i], x[c][i + 1]);
        }
        top = max_abs_nan(top, __shfl_xor_sync(kFullWarpMask, top, 1), 0.f);
        top = max_abs_nan(top, __shfl_xor_sync(kFullWarpMask, top, 2), 0.f);
        float mine_f;
        const float up = q4_row_scale(top, a.scale_log2, mine_f);
        if (t == 0)
            factors[kPair ? g / 2 : nt * 8 + g] = mine_f; // (pairs: the same number twice)
#pragma unroll
        for (int c = 0; c < G::kGroups; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t f[2][2]; // [term][slots]
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float v0 = x[c][2 * u + i] * up, v1 = x[c][2 * u + i + 4] * up;
                    f[0][i] = q4_term(v0, v1);
                    f[1][i] = half2_rn(v0, v1);
                    if constexpr (kPair)
                        f[0][i] = g & 1 ? f[1][i] : f[0][i];
                }
#pragma unroll
                for (int set = 0; set < G::kSets; ++set)
                    q_shared[(((set * G::kTiles + nt) * G::kGroups + c) * 2 + u) * 32 + lane] = make_uint2(f[set][0], f[set][1]);
            }
    }
    __syncthreads();
#pragma unroll
    for (int rr = 0; rr < G::kRPL; ++rr)
        factor[rr] = factors[kPair ? t : rr / 2 * 8 + 2 * t + rr % 2];
    if constexpr (!G::kQShared)
#pragma unroll
        for (int set = 0; set < G::kSets; ++set)
#pragma unroll
            for (int nt = 0; nt < G::kTiles; ++nt)
#pragma unroll
                for (int c = 0; c < G::kGroups; ++c)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint2 f = q_shared[(((set * G::kTiles + nt) * G::kGroups + c) * 2 + u) * 32 + lane];
                        qf[set][nt][c][u][0] = f.x, qf[set][nt][c][u][1] = f.y;
                    }
    float o[G::kGroups][2][G::kTiles][kPair ? 2 : 4] = {}; // dims 32 c + 4 g + 2 i and + 1 of the lane's rows
    float m[G::kRPL], l[G::kRPL];
#pragma unroll
    for (int rr = 0; rr < G::kRPL; ++rr)
        m[rr] = kQ4None, l[rr] = 0.f;

    [[maybe_unused]] float far_room[kPutBy ? G::kFar : 1]; // what has been put by, in the order of o
    [[maybe_unused]] float *far = far_room;
    if constexpr (kPutBy)
        asm volatile("" : "+l"(far)); // (stays in local memory)

    const uint32_t ring_at = sm100::smem_u32(ring) + (lane / 16) * G::kPageBytes + lane % 16 * 16; // both pages' rows of a group
    int at = 0;
    int i = 0;
    for (int end = 0; i < mine;) {
        end = kPutBy ? min(mine, end + G::kPeriod) : mine;
        for (; i < end; ++i) {
            q4_copy_wait<G::kStages - 2>();
            __syncwarp(); // all lanes' copies are there; all have done with the stage that is filled next
            fetch(i + G::kStages - 1, at == 0 ? G::kStages - 1 : at - 1);
            const uint8_t *stage = ring + at * G::kStage;
            const uint32_t stage_at = ring_at + at * G::kStage;
            at = at + 1 == G::kStages ? 0 : at + 1;
            const int key0 = (first + i * stride) * G::kStepKeys;
            const bool edge = key0 + G::kStepKeys > span.ctx;

            // ---- scores: of key 16 p + 8 e + g at place 2 p + e
            float x[G::kRPL][2 * G::kStepPages] = {};
#pragma unroll
            for (int pp = 0; pp < G::kPairs; ++pp)
#pragma unroll
                for (int c = 0; c < G::kGroups; ++c) {
                    uint32_t w[4], k[4][4];
                    q4_ldmatrix<false>(stage_at + pp * 2 * G::kPageBytes + c * 256, w);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        __half2 codes[4];
                        kv4_integers(w[j], codes);
#pragma unroll
                        for (int n = 0; n < 4; ++n)
                            k[j][n] = kv4_bits(codes[n]);
                    }
                    float sum[2][G::kTiles][4];
#pragma unroll
                    for (int p = 0; p < 2; ++p)
#pragma unroll
                        for (int nt = 0; nt < G::kTiles; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                sum[p][nt][e] = 0.f;
#pragma unroll
                    for (int set = G::kSets - 1; set >= 0; --set)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int nt = 0; nt < G::kTiles; ++nt) {
                                uint32_t b0, b1;
                                if constexpr (G::kQShared) {
                                    const uint2 f = q_shared[(((set * G::kTiles + nt) * G::kGroups + c) * 2 + u) * 32 + lane];
                                    b0 = f.x, b1 = f.y;
                                } else {
                                    b0 = qf[set][nt][G::kQShared ? 0 : c][u][0], b1 = qf[set][nt][G::kQShared ? 0 : c][u][1];
                                }
#pragma unroll
                                for (int p = 0; p < 2; ++p) {
                                    const uint32_t f[4] = {k[2 * p][2 * u], k[2 * p + 1][2 * u], k[2 * p][2 * u + 1], k[2 * p + 1][2 * u + 1]};
                                    mma_f16(sum[p][nt], f, b0, b1);
                                }
                            }
#pragma unroll
                    for (int p = 0; p < 2; ++p)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float s = __half2float(
                                *reinterpret_cast<const __half *>(stage + (2 * pp + p) * G::kPageBytes + R::kKScale + (c * kKvPage + e * 8 + g) * 2));
#pragma unroll
                            for (int rr = 0; rr < G::kRPL; ++rr)
                                x[rr][4 * pp + 2 * p + e] += s * (kPair ? sum[p][0][2 * e] + sum[p][0][2 * e + 1] : sum[p][rr / 2][2 * e + rr % 2]);
                        }
                }
#pragma unroll
            for (int rr = 0; rr < G::kRPL; ++rr)
#pragma unroll
                for (int n = 0; n < 2 * G::kStepPages; ++n)
                    x[rr][n] *= factor[rr];
            if (edge) {
                uint32_t bad = 0; // keys whose V is no number: a row that sees one gets NaN, the others nothing of it
#pragma unroll
                for (int n = 0; n < 2 * G::kStepPages; ++n)
#pragma unroll
                    for (int c = 0; c < G::kGroups; ++c) {
                        const uint32_t v = *reinterpret_cast<const uint16_t *>(stage + n / 2 * G::kPageBytes + R::kVScale + (c * kKvPage + n % 2 * 8 + g) * 2);
                        bad |= ((v & 0x7fffu) >= kQ4BadScale ? 1u : 0u) << n;
                    }
#pragma unroll
                for (int rr = 0; rr < G::kRPL; ++rr) {
                    const int r = row_base + (kPair ? t : rr / 2 * 8 + 2 * t + rr % 2);
#pragma unroll
                    for (int pp = 0; pp < G::kPairs; ++pp) {
                        uint32_t seen = 0;
                        if (r < rows)
                            seen = tree_sees32(a.t, span.row0 + node_of(r), node_of(r), key0 + 32 * pp - span.ctx, keys - span.ctx);
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            if (bad >> (4 * pp + n) & 1u)
                                x[rr][4 * pp + n] = __uint_as_float(0x7fc00000u);
                            if (!(seen >> (n * 8 + g) & 1u))
                                x[rr][4 * pp + n] = kNegInf;
                        }
                    }
                }
            }

            // ---- weights
            bool raise = false;
            float top[G::kRPL];
#pragma unroll
            for (int rr = 0; rr < G::kRPL; ++rr) {
                top[rr] = x[rr][0];
#pragma unroll
                for (int n = 1; n < 2 * G::kStepPages; ++n)
                    top[rr] = fmaxf(top[rr], x[rr][n]);
                raise |= top[rr] - m[rr] > kQ4Top;
            }
            if (__any_sync(kFullWarpMask, raise)) {
#pragma unroll
                for (int rr = 0; rr < G::kRPL; ++rr) {
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1)
                        top[rr] = fmaxf(top[rr], __shfl_xor_sync(kFullWarpMask, top[rr], off));
                    if (top[rr] - m[rr] > kQ4Top) {
                        // below scores that are large a lift would be lost in the rounding, or grow by it
                        const float up = fabsf(top[rr]) < 0x1p20f ? top[rr] - G::kLift : top[rr];
                        const float fix = exp2_approx(m[rr] - up);
                        m[rr] = up;
                        l[rr] *= fix;
                        if constexpr (kPutBy)
                            if (end > G::kPeriod)
#pragma unroll 1
                                for (int n = rr / 2 * 4 + rr % 2; n < G::kFar; n += 4 * G::kTiles)
                                    far[n] *= fix, far[n + 2] *= fix;
#pragma unroll
                        for (int c = 0; c < G::kGroups; ++c)
#pragma unroll
                            for (int n = 0; n < 2; ++n) {
                                if constexpr (kPair) {
                                    for (float &y : o[c][n][0])
                                        y *= fix;
                                } else {
                                    o[c][n][rr / 2][rr % 2] *= fix, o[c][n][rr / 2][2 + rr % 2] *= fix;
                                }
                            }
                    }
                }
            }
            uint32_t pf[G::kSets][G::kTiles][G::kStepPages][2]; // of page p: keys 2t, 2t + 1, and 8 more, of column g
#pragma unroll
            for (int n = 0; n < 2 * G::kStepPages; ++n) {
                if constexpr (kPair) {
                    if (n % 2)
                        continue;
                    const float p0 = exp2_approx(x[0][n] - m[0]), p1 = exp2_approx(x[0][n + 1] - m[0]);
                    l[0] += p0 + p1;
                    uint32_t t0, t1;
                    if constexpr (G::kWide)
                        q4_terms(p0, p1, t0, t1);
                    else
                        t0 = half2_rn(p0, 0.f), t1 = half2_rn(p1, 0.f);
                    pf[0][0][n / 2][0] = q4_transposed(t0), pf[0][0][n / 2][1] = q4_transposed(t1);
                } else {
#pragma unroll
                    for (int nt = 0; nt < G::kTiles; ++nt) {
                        float p0 = exp2_approx(x[2 * nt][n] - m[2 * nt]), p1 = exp2_approx(x[2 * nt + 1][n] - m[2 * nt + 1]);
                        l[2 * nt] += p0, l[2 * nt + 1] += p1;
                        if constexpr (G::kSets == 2) {
                            pf[0][nt][n / 2][n % 2] = q4_transposed(q4_term(p0, p1));
                            pf[1][nt][n / 2][n % 2] = q4_transposed(half2_rn(p0, p1));
                        } else {
                            pf[0][nt][n / 2][n % 2] = q4_transposed(half2_rn(p0, p1));
                        }
                    }
                }
            }

            // ---- output
#pragma unroll
            for (int c = 0; c < G::kGroups; ++c) {
                uint32_t v[2 * G::kStepPages][4];
#pragma unroll
                for (int pp = 0; pp < G::kPairs; ++pp) {
                    uint32_t w[4];
                    q4_ldmatrix<true>(stage_at + pp * 2 * G::kPageBytes + R::kCodes + c * 256, w);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t s = *reinterpret_cast<const uint32_t *>(stage + (2 * pp + j / 2) * G::kPageBytes + R::kVScale +
                                                                         (c * kKvPage + j % 2 * 8 + 2 * t) * 2);
                        if (edge) // (times a weight of zero it would be NaN)
                            s &= ((s & 0x7fffu) >= kQ4BadScale ? 0u : 0xffffu) | ((s >> 16 & 0x7fffu) >= kQ4BadScale ? 0u : 0xffff0000u);
                        kv4_widen(w[j], kv4_half2(s), v[4 * pp + j]);
                    }
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float sum[G::kTiles][4] = {};
#pragma unroll
                    for (int set = G::kSets - 1; set >= 0; --set)
#pragma unroll
                        for (int p = 0; p < G::kStepPages; ++p) {
                            const uint32_t f[4] = {v[2 * p][2 * n], v[2 * p][2 * n + 1], v[2 * p + 1][2 * n], v[2 * p + 1][2 * n + 1]};
#pragma unroll
                            for (int nt = 0; nt < G::kTiles; ++nt) {
                                if constexpr (G::kWide || kPair)
                                    mma_f16(sum[nt], f, pf[set][nt][p][0], pf[set][nt][p][1]);
                                else
                                    mma_f16(o[c][n][nt], f, pf[set][nt][p][0], pf[set][nt][p][1]);
                            }
                        }
                    if constexpr (kPair) { // (the second column of bf16 rows is zero)
                        o[c][n][0][0] += G::kWide ? sum[0][0] + sum[0][1] : sum[0][0];
                        o[c][n][0][1] += G::kWide ? sum[0][2] + sum[0][3] : sum[0][2];
                    } else if constexpr (G::kWide) {
#pragma unroll
                        for (int nt = 0; nt < G::kTiles; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                o[c][n][nt][e] += sum[nt][e];
                    }
                }
            }
        }
        if constexpr (kPutBy)
            if (mine > G::kPeriod)
#pragma unroll
                for (int n = 0; n < G::kFar; ++n) {
                    float &y = o[n / (8 * G::kTiles)][n / (4 * G::kTiles) % 2][n / 4 % G::kTiles][n % 4];
                    if (end > G::kPeriod)
                        y += far[n];
                    if (end < mine)
                        far[n] = y, y = 0.f;
                }
    }
    q4_copy_wait<0>();

    // ---- joining: the warps, then the cluster
    __syncthreads(); // the rings are done with
    float *part = reinterpret_cast<float *>(q4_smem), *joined = part + warps * G::kRows * G::kPitch;
    float *stat = joined + G::kRows * G::kPitch, *joined_stat = stat + 2 * warps * G::kRows; // m, l by warp; of the CTA
#pragma unroll
    for (int rr = 0; rr < G::kRPL; ++rr) {
        const int r = kPair ? t : rr / 2 * 8 + 2 * t + rr % 2;
        float any = 0.f;
#pragma unroll
        for (int c = 0; c < G::kGroups; ++c) {
            float y[4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                if constexpr (kPair) {
                    y[2 * n] = o[c][n][0][0], y[2 * n + 1] = o[c][n][0][1];
                } else {
                    y[2 * n] = o[c][n][rr / 2][rr % 2], y[2 * n + 1] = o[c][n][rr / 2][2 + rr % 2];
                }
            }
            any = max_abs_nan(max_abs_nan(any, y[0], y[1]), y[2], y[3]);
            q4_store4(part + (warp * G::kRows + r) * G::kPitch + 32 * c + 4 * g, y);
        }
        // a V row that is no number, in a group of some dims, makes the whole output none
        l[rr] = any == any ? l[rr] : any;
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
            l[rr] += __shfl_xor_sync(kFullWarpMask, l[rr], off);
        if (g == 0) {
            stat[warp * G::kRows + r] = m[rr];
            stat[(warps + warp) * G::kRows + r] = l[rr];
        }
    }
    __syncthreads();
    const int live = min(G::kRows, rows - row_base);
    const auto put = [&](int r, int d, float L, const float (&y)[4]) {
        const int row = row_base + r, node = node_of(row);
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const float z[4] = {L == 0.f ? 0.f : y[0] * inv, L == 0.f ? 0.f : y[1] * inv, L == 0.f ? 0.f : y[2] * inv, L == 0.f ? 0.f : y[3] * inv};
        q4_store4(out + static_cast<int64_t>(span.row0 + node) * a.out_stride + static_cast<int64_t>(h * rep + row - node * rep) * D + d, z);
    };
    for (int i = tid; i < live * (D / 4); i += threads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float M = kQ4None, L = 0.f, y[4] = {};
        for (int w = 0; w < warps; ++w)
            M = fmaxf(M, stat[w * G::kRows + r]);
        for (int w = 0; w < warps; ++w) {
            const float f = exp2_approx(stat[w * G::kRows + r] - M);
            const float4 p = *reinterpret_cast<const float4 *>(part + (w * G::kRows + r) * G::kPitch + d);
            L += f * stat[(warps + w) * G::kRows + r];
            y[0] += f * p.x, y[1] += f * p.y, y[2] += f * p.z, y[3] += f * p.w;
        }
        if (splits == 1) {
            put(r, d, L, y);
        } else {
            *reinterpret_cast<float4 *>(joined + r * G::kPitch + d) = make_float4(y[0], y[1], y[2], y[3]);
            if (d == 0)
                joined_stat[r] = M, joined_stat[G::kRows + r] = L;
        }
    }
    if (splits == 1)
        return;
    __syncthreads();
    cluster_sync_all();
    for (int i = rank * threads + tid; i < live * (D / 4); i += splits * threads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float M = kQ4None, L = 0.f, y[4] = {};
        for (int c = 0; c < splits; ++c)
            M = fmaxf(M, peer_load(&joined_stat[r], c));
        for (int c = 0; c < splits; ++c) {
            const float f = exp2_approx(peer_load(&joined_stat[r], c) - M);
            const float4 p = peer_load4(joined + r * G::kPitch + d, c);
            L += f * peer_load(&joined_stat[G::kRows + r], c);
            y[0] += f * p.x, y[1] += f * p.y, y[2] += f * p.z, y[3] += f * p.w;
        }
        put(r, d, L, y);
    }
    cluster_sync_all(); // peers read this CTA's shared memory until here
}

// CTAs of a kernel that run at once on the current device. Asked once.
template <typename... P> inline int q4_slots(void (*kernel)(P...), int threads, int bytes) {
    struct Known {
        const void *kernel;
        int device, slots;
    };
    static thread_local std::vector<Known> mine;
    const int device = device_facts().device;
    for (const Known &k : mine)
        if (k.kernel == reinterpret_cast<const void *>(kernel) && k.device == device)
            return k.slots;
    int per_sm = 0;
    OPWORKS_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, bytes));
    mine.push_back({reinterpret_cast<const void *>(kernel), device, std::max(1, per_sm) * device_facts().sm_count});
    return mine.back().slots;
}

template <typename T, int D, int kNT> inline void q4_rows_launch(const T *q, T *out, const TreeArgs &a, cudaStream_t stream) {
    using G = Q4RowsGeo<T, D, kNT>;
    auto kernel = q4_rows_kernel<T, D, kNT, false>;
    const int most = allow_shared_bytes(kernel, G::kThreads, G::kBytes);
    const int64_t slots = q4_slots(kernel, G::kThreads, G::kBytes), sms = device_facts().sm_count;
    const int64_t rows = static_cast<int64_t>(a.t.max_rows) * (a.qh / a.kvh);
    const int64_t groups = (rows + G::kRows - 1) / G::kRows, all = groups * a.kvh * a.t.batch;
    const int64_t keys = static_cast<int64_t>(a.t.max_ctx) + a.t.max_rows, steps = (keys + G::kStepKeys - 1) / G::kStepKeys;
    // A cluster costs 2 us and more (32 sequences x 8 heads with nothing to do: 5.3 us, 7 with
    // clusters of two), so keys are split only where there are SMs to spare or each warp has 16
    // steps and more; then into up to a third more CTAs than run at once, since sequences differ
    // in length, while each warp keeps one or two steps. By powers of two, which fill the device's
    // groups of SMs: 12 x 8 of 32,000 tokens, 296 CTAs at once: 113 us with 2 splits, 109 with 3,
    // 87 with 4, 91 with 5; 16 x 8 of 4,000: 16.1 with 1, 14.5 with 2, 20.9 with 3; 4 x 8 of
    // 32,000: 48 with 4 and 12, 41 with 8.
    const int64_t cap = std::min<int64_t>(most, 2 * steps / (3 * G::kWarps));
    int64_t splits = 1;
    if (all < sms || steps >= 16 * G::kWarps)
        while (2 * splits <= cap && 2 * splits * all * 3 <= slots * 4)
            splits *= 2;
    require(groups * splits <= 0x7fffffff, "tree attention: too many rows for one call");
    if constexpr (G::kInCore)
        if (steps > G::kPeriod * G::kWarps * splits) {
            kernel = q4_rows_kernel<T, D, kNT, true>;
            allow_shared_bytes(kernel, G::kThreads, G::kBytes);
        }
    // sequences in the order of their length, where SMs have more than one CTA (their list is short
    // beside the rings)
    const int64_t per_sequence = groups * splits * a.kvh, total = per_sequence * a.t.batch;
    int descending = 0;
    if (a.t.batch > 1 && a.t.batch <= 1024 && total > sms)
        descending = total <= slots ? static_cast<int>(std::min<int64_t>(a.t.batch, (sms + per_sequence - 1) / per_sequence)) : a.t.batch;
    launch_ex_cluster(kernel, dim3(static_cast<unsigned>(groups * splits), a.kvh, a.t.batch), dim3(static_cast<unsigned>(splits)), dim3(G::kThreads), G::kBytes, stream,
                      q, out, a, a.qh / a.kvh, static_cast<int>(splits), descending);
}

template <typename T, int D> inline void q4_rows_call(const T *q, T *out, const TreeArgs &a, cudaStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.t.max_rows) * (a.qh / a.kvh);
    if (rows <= 4)
        q4_rows_launch<T, D, 0>(q, out, a, stream);
    else if (rows <= 8)
        q4_rows_launch<T, D, 1>(q, out, a, stream);
    else if constexpr (D == 128 && std::is_same_v<T, float>) // (four tiles do not fit into registers)
        q4_rows_launch<T, D, 2>(q, out, a, stream);
    else if (rows <= 16)
        q4_rows_launch<T, D, 2>(q, out, a, stream);
    else
        q4_rows_launch<T, D, 4>(q, out, a, stream);
}

} // namespace opworks::detail
