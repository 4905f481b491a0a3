#pragma once

// Attention over the 4-bit cache, kernel for many query rows per KV head
// (ops/tree_attention_q4.cuh has the definition): tcgen05 tiles of 128 rows x 128
// keys, fp16 operands that hold what the cache holds exactly.
//
// Two streams per CTA: while the softmax of one stream's tile runs, the products of
// the other's do. With more than 128 query rows (row = node * rep + head in group)
// the streams are two row tiles over the same keys; with at most 128 they are the
// even and the odd key tiles of one row tile, joined at the end. Each stream has S
// (128 columns) and O (D columns) in tensor memory and a warpgroup that owns a row
// per thread.
//
//   warps 0-7    softmax of stream 0, 1: S from tensor memory, weights P back over
//                it as fp16 (the A operand of P V)
//   warps 8-14   widen pages, from global memory through registers to fp16 tiles in
//                shared memory (128-byte swizzle; K as it lies is K-major, V as it
//                lies is MN-major), a page of K or of V at a time
//   warp 15      tensor memory, and one thread that issues all products
//
// A word of eight codes widens to the pairs (0, 4), (1, 5), (2, 6), (3, 7) and is
// stored so: Q's dims lie in the same order, and O's columns are put right when
// they leave.
//
// Weights are 2^(score - reference). A row's reference is raised only when a weight
// would pass 2^15 (rare: it is set to give the largest score 1, or 2^6 in fp32): then
// O and the tile's weights so far are multiplied down in place. So scores are looked
// at once.
//
// What bounds it is the chain of a tile: scores, softmax, weights, sum, each waiting for
// the one before: 5,300 cycles for 256 rows x 128 keys, of which the products are 2,048
// and the exponentials as much, side by side (tensor pipe 37 % busy, exponentials 38 %).
// Measured (kernel time, one B200): 3 prompts' pieces of up to 2048 rows x 32 heads behind
// up to 2100 tokens, 8 x 128 bf16: 326 us, 0.69 PFLOP/s; 8 trees of up to 26 nodes x 32
// heads over up to 4099 tokens, 8 x 64 fp32: 41 us.
//
// fp32 rows have two fp16 terms of Q and P. The tensor cores cut an accumulator off
// at every step, so for them O is the sum over one tile and is added, rounded, to a
// sum of its own in tensor memory, where two streams leave room for that at D = 64 only (at
// D = 128 one stream would, with half the overlap; fp32 rows go to the kernel for few rows there).

#include "detail/sm100.cuh"
#include "tree_attention_q4_rows.cuh"
#include "tree_attention_tiles.cuh"

namespace opworks::detail {

template <typename T, int D, int kM> struct Q4TilesGeo {
    static constexpr bool kWide = std::is_same_v<T, float>;
    static_assert(!kWide || D == 64, "two streams leave no room in tensor memory for the sums of fp32 rows of 128 dims");
    static constexpr int kTerms = kWide ? 2 : 1;             // of Q and P
    static constexpr float kLift = kWide ? 6.f : 0.f;         // see kQ4Top
    static constexpr int kSlabs = D / 64, kSlab = kTileKeys * 128; // 64 dims of 128 rows: 128 bytes each
    static constexpr int kTileBytes = kSlabs * kSlab;        // a K or V tile
    static constexpr int kStages = 2;
    static constexpr int kQBytes = kTerms * kSlabs * kM * kSlab;
    static constexpr int kRows = kM * 128;
    static constexpr int kPitch = D + 4;
    static constexpr int kJoin = 256 * kPitch * 4; // partial results of both streams
    static constexpr int kTiles = kQBytes + 2 * kStages * kTileBytes;
    static constexpr int kBuf = kTiles > kJoin ? kTiles : kJoin;
    // row factors; m and l of 2 x 128 rows; joined m and l; keys whose V is no number (4 tiles); barriers
    static constexpr int kBytes = kBuf + 4 * 256 + 8 * 256 + 8 * 256 + 4 * 16 + 256;
    static constexpr int kPages = kTileKeys / kKvPage, kItems = 2 * kPages; // of a tile: K's pages, then V's
    static constexpr int kLoads = D / 64;                     // pieces of 16 bytes a lane and page
    static constexpr int kPeriod = kQ4SumTiles;               // steps of a stream after which the sum of bf16 rows is put by
};

constexpr float kQ4Wary = 0x1p20f; // scores from here on are so coarse that they are rounded before the reference is taken off

__device__ __forceinline__ float q4_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// True in one lane of a warp that runs together.
__device__ __forceinline__ bool q4_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// The stored weights of 32 keys (a chunk's columns: 16 of each term) times the factor that their
// sum takes: in fp32, and split again. fp16 has few bits of a factor below 2^-14, or none (32
// keys could so vanish from the output and stay in the sum), and lo corrects hi only as they were
// split.
template <int kTerms> __device__ __forceinline__ void q4_lower_weights(uint32_t at, float fix) {
    uint32_t o[kTerms][16];
#pragma unroll
    for (int t = 0; t < kTerms; ++t)
        sm100::tmem_ld_32x16(at + 16u * t, o[t]);
    sm100::tmem_wait_ld();
#pragma unroll
    for (int t = 0; t < kTerms; ++t)
        sm100::tmem_reg_fence(o[t]);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        float2 p = half2_floats(o[0][k]);
        if constexpr (kTerms == 2) {
            const float2 rest = half2_floats(o[1][k]);
            p.x += rest.x, p.y += rest.y;
        }
        p.x *= fix, p.y *= fix;
        o[0][k] = q4_term(p.x, p.y);
        if constexpr (kTerms == 2)
            o[1][k] = half2_rn(p.x, p.y);
    }
#pragma unroll
    for (int t = 0; t < kTerms; ++t)
        tile_tmem_st16(at + 16u * t, o[t]);
}
// The same as a call, for bf16 rows: inlined into the four chunks of a tile it costs prompts 10 %
// (3 x 2048 rows, D 128: 363 us, 326 so), though it hardly ever runs. (fp32 rows, D 64: 409 us
// inlined, 433 with a call.)
__device__ __noinline__ void q4_lower_weights_apart(uint32_t at, float fix) { q4_lower_weights<1>(at, fix); }

// Adds a row's O (sets, the first time) to what has been put by of it, in local memory; and that,
// times the factor of a reference that is raised. Calls, since they hardly ever run.
template <int D> __device__ __noinline__ void q4_put_by(uint32_t ot, float *far, bool first) {
#pragma unroll 1
    for (int d = 0; d < D; d += 16) {
        uint32_t o[16];
        sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(d), o);
        sm100::tmem_wait_ld();
        sm100::tmem_reg_fence(o);
#pragma unroll
        for (int k = 0; k < 16; ++k)
            far[d + k] = first ? __uint_as_float(o[k]) : far[d + k] + __uint_as_float(o[k]);
    }
}
template <int D> __device__ __noinline__ void q4_lower_far(float *far, float fix) {
#pragma unroll 4
    for (int d = 0; d < D; ++d)
        far[d] *= fix;
}

// kPutBy: a stream may have more than kPeriod steps, and sums are put by.
template <typename T, int D, int kM, bool kPutBy>
static __global__ void __launch_bounds__(kTileThreads, 1)
    q4_tiles_kernel(const T *__restrict__ q, T *__restrict__ out, TreeArgs a, int rep, int splits, bool sorted, int *err) {
    using G = Q4TilesGeo<T, D, kM>;
    using R = Kv4Record<D>;
    extern __shared__ __align__(1024) uint8_t tile_smem[];
    uint8_t *smem = tile_smem;
    if ((sm100::smem_u32(smem) & 1023u) != 0) { // never taken: no static shared memory. The whole grid returns.
        if (threadIdx.x == 0)
            atomicExch(err, 5);
        return;
    }
    uint8_t *qs = smem, *ks = qs + G::kQBytes, *vs = ks + G::kStages * G::kTileBytes;
    float *row_fac = reinterpret_cast<float *>(smem + G::kBuf); // [256]
    float *stat = row_fac + 256;                                // m [256], l [256]
    float *joined = stat + 512;                                 // m [256], l [256] of the CTA
    uint16_t *v_bad = reinterpret_cast<uint16_t *>(joined + 512); // [4][8]: a bit a key of tile i % 4
    uint64_t *bars = reinterpret_cast<uint64_t *>(v_bad + 32);
    uint64_t *k_full = bars, *v_full = k_full + 4, *v_empty = v_full + 4; // [4]: tile i's at i % 4
    // [stream][4]: step e's at e % 4. S is there; so its K has been read, and all products before it are done
    uint64_t *s_ready = v_empty + 4, *p_ready = s_ready + 8; // p_ready: [stream][half of the keys]
    uint64_t *half_done = p_ready + 4; // [stream]: step e's products on the first half of the keys are done
    uint64_t *drain = half_done + 2, *q_full = drain + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(q_full + 1);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.y;
    const int row_groups = static_cast<int>(gridDim.x) / splits;
    const int rank = blockIdx.x % splits;
    // later rows of a chain see more keys: they come first
    const int group = row_groups - 1 - static_cast<int>(blockIdx.x) / splits;
    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            sm100::mbar_init(&k_full[i], G::kPages);
            sm100::mbar_init(&v_full[i], G::kPages);
            sm100::mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            for (int n = 0; n < 4; ++n)
                sm100::mbar_init(&s_ready[4 * i + n], 1);
            sm100::mbar_init(&p_ready[2 * i], 4); // warps
            sm100::mbar_init(&p_ready[2 * i + 1], 4);
            sm100::mbar_init(&half_done[i], 1);
        }
        sm100::mbar_init(drain, 1);
        sm100::mbar_init(q_full, 8);
        sm100::fence_mbarrier_init();
    }
    if (warp == 15) {
        sm100::tmem_alloc(tmem_slot, 512);
        sm100::tmem_relinquish();
    }
    pdl_trigger();
    sm100::tc_fence_before();
    __syncthreads();
    sm100::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    const TreeSpan span = sorted ? q4_span_by_work(a.t, blockIdx.z, a.t.batch, reinterpret_cast<int *>(row_fac)) : TreeSpan(a.t, blockIdx.z);
    const int b = span.b, row_base = group * G::kRows, rows = span.n * rep;
    int keys = span.keys;
    if (a.t.mask == nullptr) // a chain: nothing after the group's last node is seen
        keys = min(keys, span.ctx + (min(row_base + G::kRows, rows) + rep - 1) / rep);
    const int all_tiles = row_base < rows ? (keys + kTileKeys - 1) / kTileKeys : 0;
    // tiles go round the cluster: this CTA's tile i is rank + i * splits
    const int tiles = all_tiles > rank ? (all_tiles - rank + splits - 1) / splits : 0;
    const auto key_of = [&](int i) { return (rank + i * splits) * kTileKeys; };
    // Tile i's barriers are those at i % 4, in phase i / 4, whatever the number of
    // stages: no waiter is as much as four tiles behind, so a parity is enough.
    const auto phase_of = [](int i) { return static_cast<uint32_t>(i >> 2) & 1u; };
    const auto edge_of = [&](int i) { return key_of(i) + kTileKeys > span.ctx; }; // holds nodes, or places after the last key
    bool ok = true;

    if (warp >= 8 && warp < 15) {
        // ---- widening warps. The items of all tiles in one row: K's pages of tile 0, V's
        // of tile 0, K's of tile 1, ..; warp w takes items w, w + 7, ... So whatever an item
        // waits for depends on items before it only. Two are in flight.
        const int *table = a.t.block_table + static_cast<int64_t>(b) * a.t.table_stride;
        const int pages = (keys + kKvPage - 1) / kKvPage, items = tiles * G::kItems;
        struct Item {
            uint4 r[G::kLoads];
            uint16_t scale[G::kLoads];
        };
        const int token = lane % 16, first_group = lane / 16; // groups first_group + 2 j
        int ids = 0; // the blocks of the warp's next 32 items; 0 past the pages: read, and masked
        const auto fetch = [&](int item, Item &it) {
            const int step = (item - (warp - 8)) / kWidenWarps % 32;
            if (step == 0) {
                const int mine = item + lane * kWidenWarps, page = key_of(mine / G::kItems) / kKvPage + mine % G::kPages;
                ids = mine < items && page < pages ? max(0, table[page]) : 0;
            }
            const int64_t rec = __shfl_sync(kFullWarpMask, ids, step);
            const uint8_t *src = static_cast<const uint8_t *>(a.k) + (rec * a.kvh + h) * R::kBytes;
            const bool v = item / G::kPages % 2;
#pragma unroll
            for (int j = 0; j < G::kLoads; ++j) {
                const int g = first_group + 2 * j;
                it.r[j] = __ldg(reinterpret_cast<const uint4 *>(src + (v ? R::kCodes : 0) + (g * kKvPage + token) * 16));
                it.scale[j] = __ldg(reinterpret_cast<const uint16_t *>(src + (v ? R::kVScale : R::kKScale) + (g * kKvPage + token) * 2));
            }
        };
        const auto widen = [&](int item, const Item &it) -> bool {
            const int i = item / G::kItems, page = item % G::kPages, stage = i % G::kStages;
            const bool v = item / G::kPages % 2;
            const int before = i - G::kStages; // the tile that has the stage until its products are done
            if (before >= 0) {
                const int e = kM == 1 ? before >> 1 : before; // its step, in the last stream that reads its K
                uint64_t *bar = v ? &v_empty[before & 3] : &s_ready[(kM == 2 ? 4 : (before & 1) * 4) + (e & 3)];
                if (!sm100::mbar_wait_warp(bar, phase_of(v ? before : e)))
                    return false;
            }
            uint8_t *tile = (v ? vs : ks) + stage * G::kTileBytes;
            const int row = page * kKvPage + token;
            bool bad = false;
#pragma unroll
            for (int j = 0; j < G::kLoads; ++j) {
                uint32_t s = it.scale[j];
                if (v && (s & 0x7fffu) >= kQ4BadScale) {
                    bad = true;
                    if (edge_of(i)) // (times a weight of zero it would be NaN)
                        s = 0;
                }
                const __half2 scale = kv4_half2(s | s << 16);
                const uint32_t w[4] = {it.r[j].x, it.r[j].y, it.r[j].z, it.r[j].w};
                const int g = first_group + 2 * j;
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    uint32_t x[4];
                    kv4_widen(w[n], scale, x);
                    *reinterpret_cast<uint4 *>(tile + g / 2 * G::kSlab + swizzled(row, g % 2 * 4 + n)) = make_uint4(x[0], x[1], x[2], x[3]);
                }
            }
            if (v) {
                const uint32_t bits = __ballot_sync(kFullWarpMask, bad);
                if (lane == 0)
                    v_bad[(i & 3) * 8 + page] = static_cast<uint16_t>(bits | bits >> 16);
            }
            sm100::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0)
                sm100::mbar_arrive(&(v ? v_full : k_full)[i & 3]);
            return true;
        };
        Item even, odd;
        int item = warp - 8;
        if (items > 0) {
            fetch(item, even);
            fetch(item + kWidenWarps, odd);
        }
        for (; item < items; item += 2 * kWidenWarps) {
            if (!widen(item, even)) {
                ok = false;
                break;
            }
            fetch(item + 2 * kWidenWarps, even);
            if (item + kWidenWarps < items && !widen(item + kWidenWarps, odd)) {
                ok = false;
                break;
            }
            fetch(item + 3 * kWidenWarps, odd);
        }
    } else if (warp == 15) {
        // ---- all products. The warp runs together, so that what addresses them is
        // uniform, and one lane issues.
        if (tiles > 0) {
            const uint32_t tm = __shfl_sync(kFullWarpMask, tmem, 0);
            constexpr uint32_t idesc_s = sm100::idesc_make(sm100::kFmtF16, 128, kTileKeys);
            constexpr uint32_t idesc_o = sm100::idesc_make(sm100::kFmtF16, 128, D) | (1u << 16); // B MN-major
            // descriptors move by additions to their address field (16-byte units)
            const uint64_t qd = sm100::sdesc_k128(sm100::smem_u32(qs)), kd = sm100::sdesc_k128(sm100::smem_u32(ks));
            const uint64_t vd = sdesc_mn128_16b(sm100::smem_u32(vs), G::kSlab);
            const auto scores = [&](int stream, int i) {
                const uint64_t q0 = qd + static_cast<uint32_t>((kM == 2 ? stream : 0) * (G::kSlab >> 4));
                const uint64_t k0 = kd + static_cast<uint32_t>((i % G::kStages) * (G::kTileBytes >> 4));
                const uint32_t d = tm + static_cast<uint32_t>(stream * kTileKeys);
                if (q4_elect())
#pragma unroll
                    for (int term = G::kTerms - 1; term >= 0; --term) // small products first
#pragma unroll
                        for (int s = 0; s < G::kSlabs; ++s)
#pragma unroll
                            for (int st = 0; st < 4; ++st) // 16 dims: 32 bytes
                                sm100::umma_bf16(d, q0 + static_cast<uint32_t>(((term * G::kSlabs + s) * kM * G::kSlab + 32 * st) >> 4),
                                                 k0 + static_cast<uint32_t>((s * G::kSlab + 32 * st) >> 4), idesc_s,
                                                 term < G::kTerms - 1 || s + st > 0 ? 1u : 0u);
                __syncwarp();
            };
            // the weights of one half of the keys times V: products on the first half begin while the
            // other half's weights are made
            const auto weigh = [&](int stream, int i, int half, uint32_t acc) {
                const uint64_t v0 = vd + static_cast<uint32_t>((i % G::kStages) * (G::kTileBytes >> 4));
                const uint32_t d = tm + 256u + static_cast<uint32_t>(stream * D), p0 = tm + static_cast<uint32_t>(stream * kTileKeys);
                if (q4_elect())
#pragma unroll
                    for (int term = G::kTerms - 1; term >= 0; --term)
#pragma unroll
                        for (int n = 0; n < kTileKeys / 32; ++n) { // chunk of 32 keys: 16 columns of each term
                            const int st = half * (kTileKeys / 32) + n;
                            umma_16_ts(d, p0 + static_cast<uint32_t>(st / 2 * 32 + term * 16 + st % 2 * 8),
                                       v0 + static_cast<uint32_t>((st * 2048) >> 4), idesc_o,
                                       term < G::kTerms - 1 || n > 0 ? 1u : acc);
                        }
                __syncwarp();
            };
            const auto commit = [&](uint64_t *bar) {
                if (q4_elect())
                    sm100::umma_commit(bar);
                __syncwarp();
            };
            const auto k_ready = [&](int i) {
                ok = sm100::mbar_wait_warp(&k_full[i & 3], phase_of(i));
                sm100::tc_fence_after();
                return ok;
            };
            const auto tile_of = [&](int stream, int e) { return tile_at<2, kM>(stream, e, tiles); };
            ok = sm100::mbar_wait_warp(q_full, 0);
            for (int s = 0; ok && s < 2; ++s)
                if (tile_of(s, 0) < tiles && (kM == 2 && s == 1 ? true : k_ready(tile_of(s, 0)))) {
                    scores(s, tile_of(s, 0));
                    commit(&s_ready[4 * s]);
                }
            for (int e = 0; ok && tile_of(0, e) < tiles; ++e)
                for (int s = 0; ok && s < 2; ++s) {
                    const int i = tile_of(s, e), next = tile_of(s, e + 1);
                    if (i >= tiles)
                        break;
                    for (int half = 0; ok && half < 2; ++half) {
                        if (!sm100::mbar_wait_warp(&p_ready[2 * s + half], static_cast<uint32_t>(e) & 1u) ||
                            (half == 0 && !sm100::mbar_wait_warp(&v_full[i & 3], phase_of(i)))) {
                            ok = false;
                            break;
                        }
                        sm100::tc_fence_after();
                        weigh(s, i, half, half == 1 || (!G::kWide && (kPutBy ? e % G::kPeriod != 0 : e > 0)));
                        if (half == 0)
                            commit(&half_done[s]);
                    }
                    if (!ok)
                        break;
                    if (kM == 1 || s == 1)
                        commit(&v_empty[i & 3]);
                    if (next < tiles && (kM == 2 && s == 1 ? true : k_ready(next))) {
                        scores(s, next);
                        commit(&s_ready[4 * s + ((e + 1) & 3)]);
                    }
                }
            // every product is done before tensor memory and the tiles are used for anything else
            commit(drain);
            if (!sm100::mbar_wait_warp(drain, 0))
                ok = false;
        }
    } else {
        // ---- softmax warps. First Q: 8 dims a lane, scaled to 2^14 .. 2^15 and split into
        // terms. The sign of the scale goes with it, so that larger products are larger scores.
        constexpr int kLanes = D / 8, kPer = 32 / kLanes, kAll = G::kRows / (8 * kPer); // rows of a warp at a time; times
        constexpr int kBatch = kAll < 16 / (8 / KvVec<T>::kN) ? kAll : 16 / (8 / KvVec<T>::kN); // in flight
        static_assert(G::kRows % (8 * kPer * kBatch) == 0, "rows of the tiles");
#pragma unroll 1
        for (int r0 = warp * kPer; r0 < G::kRows; r0 += 8 * kPer * kBatch) {
            constexpr int kVecs = 8 / KvVec<T>::kN;
            uint4 raw[kBatch][kVecs];
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const int row = row_base + r0 + 8 * kPer * n + lane / kLanes, node = row / rep;
#pragma unroll
                for (int k = 0; k < kVecs; ++k)
                    raw[n][k] = make_uint4(0, 0, 0, 0);
                if (row < rows) {
                    const T *src = q + static_cast<int64_t>(span.row0 + node) * a.q_stride + static_cast<int64_t>(h * rep + row - node * rep) * D + lane % kLanes * 8;
#pragma unroll
                    for (int k = 0; k < kVecs; ++k)
                        raw[n][k] = __ldg(reinterpret_cast<const uint4 *>(src) + k);
                }
            }
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const int r = r0 + 8 * kPer * n + lane / kLanes;
                float x[8];
#pragma unroll
                for (int k = 0; k < kVecs; ++k) {
                    float y[KvVec<T>::kN];
                    KvVec<T>::unpack(raw[n][k], y);
#pragma unroll
                    for (int e = 0; e < KvVec<T>::kN; ++e)
                        x[k * KvVec<T>::kN + e] = y[e];
                }
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    top = max_abs_nan(top, x[e], x[e + 1]);
#pragma unroll
                for (int off = 1; off < kLanes; off <<= 1)
                    top = max_abs_nan(top, __shfl_xor_sync(kFullWarpMask, top, off), 0.f);
                float factor;
                const float up = copysignf(q4_row_scale(top, fabsf(a.scale_log2), factor), a.scale_log2);
                const int dim = lane % kLanes * 8;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) { // pairs (k, k + 4), as K's
                    float u = x[k] * up, v = x[k + 4] * up;
                    hi[k] = q4_term(u, v);
                    lo[k] = half2_rn(u, v);
                }
                uint8_t *dst = qs + (dim / 64 * kM + r / 128) * G::kSlab + swizzled(r % 128, dim % 64 / 8);
                *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (G::kWide)
                    *reinterpret_cast<uint4 *>(dst + G::kSlabs * kM * G::kSlab) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                if (lane % kLanes == 0)
                    row_fac[r] = factor;
            }
        }
        sm100::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0)
            sm100::mbar_arrive(q_full);
        if (!sm100::mbar_wait_warp(q_full, 0)) // row_fac of other warps' rows
            ok = false;

        const int stream = warp / 4, r = (warp % 4) * 32 + lane; // row of the tile
        const int row = row_base + (kM == 2 ? stream * 128 : 0) + r;
        const int node = row / rep;
        const bool live = row < rows;
        const int first_node = (row - lane) / rep; // of the warp's rows
        const float rs = row_fac[kM == 2 ? stream * 128 + r : r];
        const float2 rs2 = make_float2(rs, rs);
        const uint32_t quarter = static_cast<uint32_t>((warp % 4) * 32) << 16;
        const uint32_t st = tmem + quarter + static_cast<uint32_t>(stream * kTileKeys);
        const uint32_t ot = tmem + quarter + 256u + static_cast<uint32_t>(stream * D);
        constexpr uint32_t kLong = 128; // columns from O to the sum of fp32 rows
        float m = kQ4None, l = 0.f;
        [[maybe_unused]] float far[kPutBy ? D : 1]; // what has been put by of O
        bool wary = false; // the same in a warp
        int e = 0; // steps done
        for (; ok; ++e) {
            const int i = tile_at<2, kM>(stream, e, tiles);
            if (i >= tiles)
                break;
            const int key0 = key_of(i);
            if (!sm100::mbar_wait_warp(&s_ready[4 * stream + (e & 3)], phase_of(e))) {
                ok = false;
                break;
            }
            sm100::tc_fence_after();
            bool edge = edge_of(i);
            if (edge && !sm100::mbar_wait_warp(&v_full[i & 3], phase_of(i))) { // v_bad
                ok = false;
                break;
            }
            if (edge && a.t.mask == nullptr) { // a chain, whose rows of this warp see all of the tile
                const uint4 odd = *reinterpret_cast<const uint4 *>(v_bad + (i & 3) * 8);
                edge = key0 + kTileKeys > min(keys, span.ctx + first_node + 1) || (odd.x | odd.y | odd.z | odd.w) != 0;
            }
            const auto ask = [&](int c, uint32_t (&x)[2][16]) {
                sm100::tmem_ld_32x16(st + static_cast<uint32_t>(32 * c), x[0]);
                sm100::tmem_ld_32x16(st + static_cast<uint32_t>(32 * c + 16), x[1]);
            };
            const auto await = [&](uint32_t (&x)[2][16]) {
                sm100::tmem_wait_ld();
                sm100::tmem_reg_fence(x[0]);
                sm100::tmem_reg_fence(x[1]);
            };
            if constexpr (kPutBy)
                if (e > 0 && e % G::kPeriod == 0) // (this tile's S is there, so the products before it are done)
                    q4_put_by<D>(ot, far, e == G::kPeriod);
            uint32_t xa[2][16], xb[2][16];
            ask(0, xa);
            ask(1, xb);
            // fp32 rows: O of the tile before to the long sum (this tile's S is there, so the products before it are done)
            if (G::kWide && e > 0) {
                await(xa);
                await(xb);
#pragma unroll 1
                for (int d = 0; d < D; d += 16) {
                    uint32_t o[16], x[16];
                    sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(d), o);
                    if (e > 1)
                        sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(d) + kLong, x);
                    sm100::tmem_wait_ld();
                    sm100::tmem_reg_fence(o);
                    if (e > 1) {
                        sm100::tmem_reg_fence(x);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            o[k] = __float_as_uint(__uint_as_float(o[k]) + __uint_as_float(x[k]));
                    }
                    tile_tmem_st16(ot + static_cast<uint32_t>(d) + kLong, o);
                }
                tile_tmem_wait_st();
                ask(0, xa);
                ask(1, xb);
            }
            // What the row has so far, times fix: O, its long sum, and the weights of this tile's
            // first c chunks. From the third chunk on the first half's are in O, or soon will be.
            const auto rescale = [&](float fix, int c) {
                const bool second = c >= 2;
                if (second) {
                    if (!sm100::mbar_wait_warp(&half_done[stream], static_cast<uint32_t>(e) & 1u))
                        ok = false;
                    sm100::tc_fence_after();
                }
                const auto scale = [&](uint32_t at) {
#pragma unroll 1
                    for (int d = 0; d < D; d += 16) {
                        uint32_t o[16];
                        sm100::tmem_ld_32x16(at + static_cast<uint32_t>(d), o);
                        sm100::tmem_wait_ld();
                        sm100::tmem_reg_fence(o);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            o[k] = __float_as_uint(__uint_as_float(o[k]) * fix);
                        tile_tmem_st16(at + static_cast<uint32_t>(d), o);
                    }
                };
                if (second || (!G::kWide && (kPutBy ? e % G::kPeriod != 0 : e > 0)))
                    scale(ot);
                if constexpr (kPutBy)
                    if (e >= G::kPeriod)
                        q4_lower_far<D>(far, fix);
                if (G::kWide && e > 0)
                    scale(ot + kLong);
                tile_tmem_wait_st(); // the chunks' weights are stored before they are read
#pragma unroll 1
                for (int n = second ? 2 : 0; n < c; ++n) {
                    if constexpr (G::kWide)
                        q4_lower_weights<G::kTerms>(st + static_cast<uint32_t>(32 * n), fix);
                    else
                        q4_lower_weights_apart(st + static_cast<uint32_t>(32 * n), fix);
                }
                tile_tmem_wait_st();
            };
            // 32 scores, in place: less the reference, in log2 units. True where one is so far above it
            // that it has to be raised.
            const auto scored = [&](uint32_t (&x)[2][16]) {
                const float2 m2 = make_float2(-m, -m);
                float top[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
                for (int n = 0; n < 16; ++n) {
                    uint32_t &u = x[n / 8][2 * n % 16], &v = x[n / 8][2 * n % 16 + 1];
                    const float2 y = __ffma2_rn(make_float2(__uint_as_float(u), __uint_as_float(v)), rs2, m2);
                    top[n % 4] = q4_max3(top[n % 4], y.x, y.y);
                    u = __float_as_uint(y.x), v = __float_as_uint(y.y);
                }
                return q4_max3(q4_max3(top[0], top[1], top[2]), top[3], kNegInf) > kQ4Top;
            };
            // The same for chunk c with masks, a reference that is raised, and scores so large that
            // they are rounded before it is taken off. From tensor memory again.
            const auto careful = [&](int c, uint32_t (&x)[2][16], uint32_t seen, uint32_t odd) {
                ask(c, x);
                await(x);
                float top = kNegInf;
#pragma unroll
                for (int n = 0; n < 32; ++n) {
                    float y = __uint_as_float(x[n / 16][n % 16]) * rs;
                    y = !(seen >> n & 1u) ? kNegInf : odd >> n & 1u ? __uint_as_float(0x7fc00000u) : y;
                    top = fmaxf(top, y);
                    x[n / 16][n % 16] = __float_as_uint(y);
                }
                const bool up = top - m > kQ4Top;
                if (__any_sync(kFullWarpMask, up)) {
                    const float to = !up ? m : fabsf(top) < kQ4Wary ? top - G::kLift : top, fix = exp2_approx(m - to);
                    rescale(fix, c);
                    l *= fix;
                    m = to;
                    wary = wary || __any_sync(kFullWarpMask, fabsf(m) >= kQ4Wary && m != kQ4None);
                }
#pragma unroll
                for (int n = 0; n < 32; ++n)
                    x[n / 16][n % 16] = __float_as_uint(__uint_as_float(x[n / 16][n % 16]) - m);
            };
            // Chunk c of 32 keys, scored in y (high: one is too high), the next one's scores on their way
            // to `next`: weights of the one beside scores of the other.
            bool high;
            const auto chunk = [&](int c, uint32_t (&y)[2][16], uint32_t (&next)[2][16]) {
                uint32_t seen = ~0u, odd = 0u; // keys that the row sees (rows past the last one: any); whose V is no number
                if (edge) {
                    if (live)
                        seen = tree_sees32(a.t, span.row0 + node, node, key0 + 32 * c - span.ctx, keys - span.ctx);
                    odd = *reinterpret_cast<const uint32_t *>(v_bad + (i & 3) * 8 + 2 * c);
                    high = high || seen != ~0u || odd != 0u;
                }
                if (__any_sync(kFullWarpMask, high || wary)) {
                    await(next);
                    careful(c, y, seen, odd);
                }
                if (c < 3) {
                    await(next);
                    high = scored(next);
                }
                float2 sum[4] = {};
#pragma unroll
                for (int part = 0; part < 2; ++part) { // 16 keys, a step of the product
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        float2 p = make_float2(exp2_approx(__uint_as_float(y[part][2 * n])), exp2_approx(__uint_as_float(y[part][2 * n + 1])));
                        sum[n % 4] = __fadd2_rn(sum[n % 4], p);
                        if constexpr (G::kWide) {
                            hi[n] = q4_term(p.x, p.y);
                            lo[n] = half2_rn(p.x, p.y);
                        } else {
                            hi[n] = half2_rn(p.x, p.y);
                        }
                    }
                    tile_tmem_st8(st + static_cast<uint32_t>(32 * c + 8 * part), hi);
                    if constexpr (G::kWide)
                        tile_tmem_st8(st + static_cast<uint32_t>(32 * c + 16 + 8 * part), lo);
                }
                if (c < 2)
                    ask(c + 2, y);
                const float2 all = __fadd2_rn(__fadd2_rn(sum[0], sum[1]), __fadd2_rn(sum[2], sum[3]));
                l += all.x + all.y;
            };
            await(xa); // (both)
            high = scored(xa);
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                chunk(c, xa, xb);
                chunk(c + 1, xb, xa);
                tile_tmem_wait_st();
                sm100::tc_fence_before();
                __syncwarp();
                if (lane == 0)
                    sm100::mbar_arrive(&p_ready[2 * stream + c / 2]);
            }
        }
        // ---- the stream's O, m and l
        const bool any = ok && e > 0;
        if (any && !sm100::mbar_wait_warp(drain, 0)) // all products: O is there, and the tiles are free
            ok = false;
        sm100::tc_fence_after();
        const bool direct = kM == 2 && splits == 1;
        // where nothing is joined a row goes out as it is; else to shared memory, once all products are done
        if (!direct)
            asm volatile("bar.sync 1, 256;" ::: "memory"); // both streams have waited for that
        const auto load = [&](int c, uint32_t (&o)[16]) {
            __syncwarp();
            if (any) { // the same in a warp
                sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(c), o);
                sm100::tmem_wait_ld();
                sm100::tmem_reg_fence(o);
                if (G::kWide && e > 1) {
                    uint32_t x[16];
                    sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(c) + kLong, x);
                    sm100::tmem_wait_ld();
                    sm100::tmem_reg_fence(x);
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        o[k] = __float_as_uint(__uint_as_float(o[k]) + __uint_as_float(x[k]));
                }
                if constexpr (kPutBy)
                    if (e > G::kPeriod)
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            o[k] = __float_as_uint(__uint_as_float(o[k]) + far[c + k]);
            } else {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    o[k] = 0;
            }
        };
        // Rows leave through shared memory, which is free now: finished, and written out 16 bytes a
        // lane along the row, or as they are, to be joined.
        const float inv = l == 0.f ? 0.f : 1.f / l;
        constexpr int kOutPitch = D * static_cast<int>(sizeof(T)) + 16; // bytes
        uint8_t *done = smem + (stream * 128 + r) * kOutPitch;
        float *part = reinterpret_cast<float *>(smem) + (stream * 128 + r) * G::kPitch;
        float odd = 0.f;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            load(c, o);
#pragma unroll
            for (int k = 0; k < 16; k += 8) { // columns 0, 2, 4, 6, 1, 3, 5, 7 are dims 0 .. 7
                float y[8];
#pragma unroll
                for (int n = 0; n < 8; ++n)
                    y[n] = __uint_as_float(o[k + n % 4 * 2 + n / 4]);
#pragma unroll
                for (int n = 0; n < 8; n += 2)
                    odd = max_abs_nan(odd, y[n], y[n + 1]);
                if (direct) {
#pragma unroll
                    for (int n = 0; n < 8; n += KvVec<T>::kN) {
                        float z[KvVec<T>::kN];
#pragma unroll
                        for (int j = 0; j < KvVec<T>::kN; ++j)
                            z[j] = l == 0.f ? 0.f : y[n + j] * inv;
                        *reinterpret_cast<uint4 *>(done + (c + k + n) * sizeof(T)) = KvVec<T>::pack(z);
                    }
                } else {
                    *reinterpret_cast<float4 *>(part + c + k) = make_float4(y[0], y[1], y[2], y[3]);
                    *reinterpret_cast<float4 *>(part + c + k + 4) = make_float4(y[4], y[5], y[6], y[7]);
                }
            }
        }
        // a V row that is no number, in a group of some dims, makes the whole output none
        l = odd == odd ? l : odd;
        if (direct) {
            if (odd != odd)
                for (int c = 0; c < D; ++c)
                    reinterpret_cast<T *>(done)[c] = static_cast<T>(odd);
            __syncwarp();
            const uint64_t dst = reinterpret_cast<uint64_t>(out + static_cast<int64_t>(span.row0 + node) * a.out_stride +
                                                            static_cast<int64_t>(h * rep + row - node * rep) * D);
            constexpr int kChunks = D * static_cast<int>(sizeof(T)) / 16; // of a row: 8 or 16
            const int live_rows = min(32, rows - (row - lane));
#pragma unroll 4
            for (int n = 0; n < kChunks; ++n) {
                const int at = n * (32 / kChunks) + lane / kChunks; // of the warp's rows
                const uint64_t to = __shfl_sync(kFullWarpMask, dst, at);
                if (at < live_rows)
                    reinterpret_cast<uint4 *>(to)[lane % kChunks] =
                        *reinterpret_cast<const uint4 *>(smem + (stream * 128 + r - lane + at) * kOutPitch + lane % kChunks * 16);
            }
        }
        stat[stream * 128 + r] = m;
        stat[256 + stream * 128 + r] = l;
    }
    if (!ok)
        atomicExch(err, 7);
    sm100::tc_fence_before();
    __syncthreads();
    if (warp == 15) {
        sm100::tc_fence_after();
        sm100::tmem_dealloc(tmem, 512);
    }
    if (kM == 2 && splits == 1)
        return;
    // ---- join: the two streams of a row tile, then the cluster's CTAs
    float *part = reinterpret_cast<float *>(smem);
    const int live_rows = max(0, min(G::kRows, rows - row_base));
    const auto put = [&](int r, int d, float L, const float (&y)[4]) {
        const int row = row_base + r, node = row / rep;
        const float inv = 1.f / L;
        const float z[4] = {L == 0.f ? 0.f : y[0] * inv, L == 0.f ? 0.f : y[1] * inv, L == 0.f ? 0.f : y[2] * inv, L == 0.f ? 0.f : y[3] * inv};
        q4_store4(out + static_cast<int64_t>(span.row0 + node) * a.out_stride + static_cast<int64_t>(h * rep + row - node * rep) * D + d, z);
    };
    if (kM == 1) {
        for (int i = tid; i < live_rows * (D / 4); i += kTileThreads) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            const float m0 = stat[r], m1 = stat[128 + r], top = fmaxf(m0, m1);
            const float f0 = exp2_approx(m0 - top), f1 = exp2_approx(m1 - top);
            const float4 p0 = *reinterpret_cast<const float4 *>(part + r * G::kPitch + d);
            const float4 p1 = *reinterpret_cast<const float4 *>(part + (128 + r) * G::kPitch + d);
            const float y[4] = {f0 * p0.x + f1 * p1.x, f0 * p0.y + f1 * p1.y, f0 * p0.z + f1 * p1.z, f0 * p0.w + f1 * p1.w};
            const float L = f0 * stat[256 + r] + f1 * stat[384 + r];
            if (splits == 1) {
                put(r, d, L, y);
            } else {
                q4_store4(part + r * G::kPitch + d, y); // read by this thread alone
                if (d == 0) {
                    joined[r] = top;
                    joined[256 + r] = L;
                }
            }
        }
    } else {
        for (int r = tid; r < 256; r += kTileThreads) {
            joined[r] = stat[r];
            joined[256 + r] = stat[256 + r];
        }
    }
    if (splits == 1)
        return;
    __syncthreads();
    cluster_sync_all();
    for (int i = rank * kTileThreads + tid; i < live_rows * (D / 4); i += splits * kTileThreads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float top = kQ4None, L = 0.f, y[4] = {};
        for (int c = 0; c < splits; ++c)
            top = fmaxf(top, peer_load(&joined[r], c));
        for (int c = 0; c < splits; ++c) {
            const float f = exp2_approx(peer_load(&joined[r], c) - top);
            const float4 p = peer_load4(part + r * G::kPitch + d, c);
            L += f * peer_load(&joined[256 + r], c);
            y[0] += f * p.x, y[1] += f * p.y, y[2] += f * p.z, y[3] += f * p.w;
        }
        put(r, d, L, y);
    }
    __syncthreads();
    cluster_sync_all(); // peers read this CTA's shared memory until here
}

// Clusters of `size` CTAs that run at once on the current device. Asked once.
template <typename... P> inline int q4_clusters(void (*kernel)(P...), int threads, int bytes, int size) {
    struct Known {
        const void *kernel;
        int device, size, clusters;
    };
    static thread_local std::vector<Known> mine;
    const int device = device_facts().device;
    for (const Known &k : mine)
        if (k.kernel == reinterpret_cast<const void *>(kernel) && k.device == device && k.size == size)
            return k.clusters;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(size), attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(size));
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError(); // no more than an answer to the question
        clusters = 0;
    }
    mine.push_back({reinterpret_cast<const void *>(kernel), device, size, clusters});
    return clusters;
}

template <typename T, int D, int kM> inline void q4_tiles_launch(const T *q, T *out, const TreeArgs &a, cudaStream_t stream) {
    using G = Q4TilesGeo<T, D, kM>;
    static_assert(G::kBytes <= 232448, "shared memory");
    auto kernel = q4_tiles_kernel<T, D, kM, false>;
    allow_shared_bytes(kernel, kTileThreads, G::kBytes);
    const int64_t rows = static_cast<int64_t>(a.t.max_rows) * (a.qh / a.kvh);
    const int64_t groups = (rows + G::kRows - 1) / G::kRows, all = groups * a.kvh * a.t.batch;
    const int64_t tiles = (static_cast<int64_t>(a.t.max_ctx) + a.t.max_rows + kTileKeys - 1) / kTileKeys;
    // splits (powers of two) while all clusters still run at once and each CTA has four tiles
    int splits = 1;
    while (2 * splits <= 8 && 8 * splits <= tiles && all <= q4_clusters(kernel, kTileThreads, G::kBytes, 2 * splits))
        splits *= 2;
    require(groups * splits <= 0x7fffffff, "tree attention: too many rows for one call");
    if constexpr (!G::kWide)
        if (tiles > static_cast<int64_t>(G::kPeriod) * (kM == 1 ? 2 : 1) * splits) {
            kernel = q4_tiles_kernel<T, D, kM, true>;
            allow_shared_bytes(kernel, kTileThreads, G::kBytes);
        }
    // more CTAs than places: sequences in the order of their length (the list of them lies over row_fac, stat and joined)
    const bool sorted = a.t.batch > 1 && a.t.batch <= kTileThreads && all * splits > device_facts().sm_count;
    launch_ex_cluster(kernel, dim3(static_cast<unsigned>(groups * splits), a.kvh, a.t.batch), dim3(splits), dim3(kTileThreads), G::kBytes,
                      stream, q, out, a, a.qh / a.kvh, splits, sorted, sm100::device_error_word());
}

template <typename T, int D> inline void q4_tiles_call(const T *q, T *out, const TreeArgs &a, cudaStream_t stream) {
    if (static_cast<int64_t>(a.t.max_rows) * (a.qh / a.kvh) <= 128)
        q4_tiles_launch<T, D, 1>(q, out, a, stream);
    else
        q4_tiles_launch<T, D, 2>(q, out, a, stream);
}

} // namespace opworks::detail
