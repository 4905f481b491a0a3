#pragma once

// Tree attention, kernel for many query rows per KV head (ops/tree_attention.cuh
// has the definition of the operator): tcgen05 tiles of 128 rows x 128 keys.
//
// The floor is the tensor cores' time, nearly level with the exponential unit's.
// What bounds it now is the chain of a tile: scores, softmax, weights, sum, each
// waiting for the one before (6,400 cycles for 256 rows x 128 keys, of which the
// products are 2,048). Measured: 32 sequences of 4096 to 8192 tokens with up to 64
// nodes of 32 heads (8 kv heads, D = 128, int8, bf16 rows): 344 us, 0.50 PFLOP/s.
//
// Two streams per CTA keep both busy: while the softmax of one stream's tile
// runs, the products of the other's do. With more than 128 query rows (row =
// node * rep + head in group) the streams are two row tiles over the same keys;
// with at most 128 they are the even and the odd key tiles of one row tile,
// joined at the end. (fp32 rows of 128 dims: one stream, all key tiles; see
// kSplitO.) Each stream has S (128 columns) and O (D columns) in tensor
// memory and a warpgroup that owns a row per thread.
//
//   warps 0-7    softmax of stream 0, 1: S from tensor memory, weights P back
//                over it as fp16 (the A operand of P V), O rescaled in place
//                when the reference maximum is raised (rare, see kLazy)
//   warps 8-14   widen pages from global memory, through registers, to fp16
//                tiles in shared memory (128-byte swizzle; K as it lies is
//                K-major, V as it lies is MN-major), one item of keys per warp,
//                its next item already on its way
//   warp 15      tensor memory, and one thread that issues all products
//
// Precision as in the rows kernel: fp32 queries and weights are two fp16 terms
// (a product each), bf16 rows one. The tensor cores cut an accumulator off at
// every step, so fp32 rows are summed in periods (see kPeriod): relative to 64
// bits 5.6e-7 (D = 64) and 7.4e-7 (D = 128) over 600 to 4000 keys, fp32 pools, where
// fp32 sums in torch are 7.6e-7 to 1.5e-6 off; with one accumulator all along 1.5e-6
// over 1300 keys and 1.4e-5 over 15,000 in one CTA.
// K's 8-bit codes are one exact term, and the softmax multiplies a score by its
// key's scale, four to a shared-memory broadcast (20 us of the case above; codes and
// scale rounded to one term left weights of scores near -60 off by 1e-2 and more).
// V's codes are widened with their scale, and fp32 rows as they are (one term for
// bf16 queries over 8-bit pools, 11 bits of V being more than the output has;
// else two: hi hi + hi lo + lo hi), but for a power of two that the keys of an
// item share, which the softmax adds to the exponent (see kUnlike).
//
// Splits of the keys form a cluster and are joined through distributed shared
// memory in rank order.

#include "detail/sm100.cuh"
#include "tree_attention_common.cuh"

namespace opworks::detail {

constexpr int kTileKeys = 128;
constexpr int kTileThreads = 512; // 8 softmax warps, 7 widening, 1 tensor: 4 on each scheduler, 128 registers a thread
constexpr int kWidenWarps = 7;
// Weights are 2^(x - m), with the log2 of the key's V unit in x, so that they are
// what O takes up: the first visible tile's largest gets 2^kTileLift, and m is
// raised when one would pass 2^kTileTop, so scores are looked at once, with no
// pass for a maximum. l sums them over their V units.
constexpr float kTileLift = 8.f, kTileTop = 14.f;
// The keys of an item share a unit unless some of its nodes' rows are 2^kUnlike
// smaller than its largest: then each has its own, for a row that a node does not
// see takes no bits from those that it sees. V units are 2^-60 at least (exponent
// field kMinVField - 1): lower, and l would leave fp32's range beside large rows.
constexpr uint32_t kUnlike = 12, kMinVField = 68;

template <typename T, int D, KvFormat kFmt, int kM> struct TreeTilesGeo {
    static constexpr bool kWide = kFmt == KvFormat::kF32;
    static constexpr int kQT = std::is_same_v<T, float> ? 2 : 1; // terms of Q and P
    static constexpr int kKT = kWide ? 2 : 1;                    // terms of K: 8-bit codes are exact
    static constexpr int kVT = kWide || kQT == 2 ? 2 : 1;        // terms of V
    static constexpr int kSlabs = D / 64;                        // 64 dims: 128 bytes of fp16
    static constexpr int kSlab = kTileKeys * 128;                // bytes
    static constexpr int kQBytes = kQT * kSlabs * kM * kSlab;
    static constexpr int kKBytes = kKT * kSlabs * kSlab, kVBytes = kVT * kSlabs * kSlab; // of a tile
    static constexpr int kStages = kVT == 2 && D == 128 ? 1 : 2;
    // An accumulator is cut off at every step, to its size. So for fp32 rows O is summed
    // over one or two tiles only and then added, rounded, to a sum of its own (kLong, in
    // columns from O's); at D = 128, with one stream, tensor memory has room for another
    // accumulator for its small products (widening is what takes the time there, so that
    // little is lost).
    static constexpr bool kSplitO = kQT == 2 && D == 128;
    static constexpr int kPeriod = kQT == 1 ? 1 << 30 : kSplitO ? 2 : 1; // tiles
    static constexpr int kLong = kSplitO ? -128 : 128;
    static constexpr int kStreams = kSplitO ? 1 : 2;
    static constexpr int kKvBytes = kStages * (kKBytes + kVBytes);
    static constexpr int kRowBytes = D * (kWide ? 4 : 1);
    // an item: 4 KB of K or of V, but at most 32 keys: a tile has at least as many
    // items as there are widening warps, so that no warp passes over a whole tile
    static constexpr int kItemKeys = 4096 / kRowBytes < 32 ? 4096 / kRowBytes : 32;
    static constexpr int kItems = kTileKeys / kItemKeys; // of K, and again of V
    static constexpr int kLoads = kItemKeys * kRowBytes / 512; // of 16 bytes a lane
    static constexpr int kItemPages = (kItemKeys + kKvPage - 1) / kKvPage;
    static constexpr int kRows = kM * 128;
    static constexpr int kPitch = D + 4;
    static constexpr int kJoin = 256 * kPitch * 4; // partial results of both streams
    static constexpr int kTiles = kQBytes + kKvBytes;
    static constexpr int kBuf = kTiles > kJoin ? kTiles : kJoin;
    // factors of K's keys (4 tiles), V's units as log2 and turned round (stages), the rows that
    // are not finite, and the items whose keys have a unit each; row factors; m and l of 2 x 128
    // rows; joined m and l; barriers
    static constexpr int kFactors = 4 * ((4 + 2 * kStages) * kTileKeys + (4 + kStages) * 16) + (4 + kStages) * 16;
    static constexpr int kBytes = kBuf + kFactors + 4 * 256 + 8 * 256 + 8 * 256 + 256;
};

// Step e of a stream: tile e (two row tiles, or one stream), or tile 2 e + stream
// (even and odd key tiles); from `tiles` on there is none.
template <int kStreams, int kM> __device__ __forceinline__ int tile_at(int stream, int e, int tiles) {
    return kStreams == 1 ? (stream == 0 ? e : tiles) : kM == 2 ? e : 2 * e + stream;
}

// K-major tile rows of 128 bytes: the byte of 16-byte chunk c of row r.
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// MN-major 16-bit operand in the 128-byte swizzle: atoms of 8 keys x 64 dims
// (8 rows of 128 bytes), `lbo` bytes from one 64 dims to the next, 1024 from 8
// keys to the next.
__device__ __forceinline__ uint64_t sdesc_mn128_16b(uint32_t smem_addr, uint32_t lbo) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
    d |= static_cast<uint64_t>(1024u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}

// D[tmem] (+)= A[tmem] B[smem]^T, 16-bit operands.
__device__ __forceinline__ void umma_16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
                 "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}

__device__ __forceinline__ void tile_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tile_tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tile_tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T, int D, KvFormat kFmt, int kM>
static __global__ void __launch_bounds__(kTileThreads, 1)
    tree_tiles_kernel(const T *__restrict__ q, T *__restrict__ out, TreeArgs a, int groups, int splits, bool sorted, int *err) {
    using G = TreeTilesGeo<T, D, kFmt, kM>;
    using R = KvRecord<D>;
    extern __shared__ __align__(1024) uint8_t tile_smem[];
    uint8_t *smem = tile_smem;
    if ((sm100::smem_u32(smem) & 1023u) != 0) { // never taken: no static shared memory. The whole grid returns.
        if (threadIdx.x == 0)
            atomicExch(err, 5);
        return;
    }
    uint8_t *qs = smem, *ks = qs + G::kQBytes, *vs = ks + G::kStages * G::kKBytes;
    // K's are read until the weights are done, longer than the K tile: tile i's lie in place i % 4
    float *k_unit = reinterpret_cast<float *>(smem + G::kBuf);         // [4][128]: of each key
    float *v_log = k_unit + 4 * kTileKeys;                              // [stages][128]: log2 of V's unit
    float *v_inv = v_log + G::kStages * kTileKeys;                      // [stages][128]: 2^-v_log
    uint32_t *k_odd = reinterpret_cast<uint32_t *>(v_inv + G::kStages * kTileKeys); // [4][16]: bit per key of the item
    uint32_t *v_odd = k_odd + 4 * 16;                                   // [stages][16]
    uint8_t *k_each = reinterpret_cast<uint8_t *>(v_odd + G::kStages * 16), *v_each = k_each + 4 * 16; // [4][16], [stages][16]
    float *row_fac = reinterpret_cast<float *>(v_each + G::kStages * 16); // [256]
    float *stat = row_fac + 256;                                    // m [256], l [256]
    float *joined = stat + 512;                                     // m [256], l [256] of the CTA
    uint64_t *bars = reinterpret_cast<uint64_t *>(joined + 512);
    uint64_t *k_full = bars, *v_full = k_full + 4, *v_empty = v_full + 4; // [4]: tile i's at i % 4
    // [stream][4]: step e's at e % 4. S is there; so the K tile is free (for two row
    // tiles: with the second stream's), and all products before it are done
    uint64_t *s_ready = v_empty + 4, *p_ready = s_ready + 8; // p_ready: [stream]
    uint64_t *drain = p_ready + 2, *q_full = drain + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(q_full + 1);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x % splits, unit = blockIdx.x / splits;
    const int group = unit % groups, h = unit / groups;
    const int rep = a.qh / a.kvh;
    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            sm100::mbar_init(&k_full[i], G::kItems);
            sm100::mbar_init(&v_full[i], G::kItems);
            sm100::mbar_init(&v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            for (int n = 0; n < 4; ++n)
                sm100::mbar_init(&s_ready[4 * i + n], 2); // the products, and the thread that issued them
            sm100::mbar_init(&p_ready[i], 4); // warps: 128 threads arriving on one barrier take 600 cycles
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
    const int b = sorted ? sequence_by_work(a.t, blockIdx.y, reinterpret_cast<int *>(stat)) : blockIdx.y;

    const TreeSpan span(a.t, b);
    const int row_base = group * G::kRows, rows = span.n * rep;
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
    bool ok = true;

    if (warp >= 8 && warp < 15) {
        // ---- widening warps. The items of all tiles in one row: K of tile 0, V
        // of tile 0, K of tile 1, ..; warp w takes items w, w + 7, ... So whatever
        // an item waits for depends on items before it only. Two are in flight.
        const int *table = a.t.block_table + static_cast<int64_t>(b) * a.t.table_stride;
        const int pages = (keys + kKvPage - 1) / kKvPage, items = tiles * 2 * G::kItems;
        struct Item {
            uint4 r[G::kLoads];
            float scale; // 8-bit: of key `lane`
        };
        // load j of a lane. fp32: rows one after another. 8-bit: 8 rows by 64 bytes,
        // so that the eight lanes of a store phase are two rows, one even and one
        // odd, and the swizzle keeps them on different banks.
        constexpr int kRowLanes = G::kWide ? G::kRowBytes / 16 : 4, kRowsPerLoad = 32 / kRowLanes;
        constexpr int kHalves = G::kWide ? 1 : G::kSlabs; // loads side by side in a row
        const int lrow = lane / kRowLanes, lbyte = (lane % kRowLanes) * 16;
        const auto item_key = [&](int item) { return key_of(item / (2 * G::kItems)) + item % G::kItems * G::kItemKeys; };
        // A lane holds the block id of one page of the warp's next 32 or 16 items.
        // Past the pages it is 0: what is read there is valid memory and takes no
        // part (its keys come after the last one). A load that depended on the
        // page being there would be followed by a select, and that waits for it.
        constexpr int kIdItems = 32 / G::kItemPages;
        int ids = 0;
        const auto look_up = [&](int item) {
            const int mine = item + lane / G::kItemPages * kWidenWarps;
            const int page = item_key(mine) / kKvPage + lane % G::kItemPages;
            ids = mine < items && page < pages ? table[page] : 0;
        };
        const auto fetch = [&](int item, Item &it) {
            const bool v = item / G::kItems % 2;
            const int key0 = item_key(item);
            const int step = (item - (warp - 8)) / kWidenWarps % kIdItems; // which of the items looked up
            if (step == 0)
                look_up(item);
            const int id = __shfl_sync(kFullWarpMask, ids, step * G::kItemPages + (lane & (G::kItemPages - 1)));
            constexpr int kLoads = G::kLoads / G::kItemPages; // of a page
#pragma unroll
            for (int pg = 0; pg < G::kItemPages; ++pg) {
                const int64_t rec = __shfl_sync(kFullWarpMask, id, pg);
                const uint8_t *src;
                if constexpr (G::kWide)
                    src = static_cast<const uint8_t *>(v ? a.v : a.k) + ((rec * a.kvh + h) * kKvPage + key0 % kKvPage) * G::kRowBytes;
                else
                    src = static_cast<const uint8_t *>(a.k) + (rec * a.kvh + h) * R::kBytes + (v ? R::kCodes : 0);
                src += lrow * G::kRowBytes + lbyte;
#pragma unroll
                for (int j = 0; j < kLoads; ++j)
                    it.r[pg * kLoads + j] = __ldg(reinterpret_cast<const uint4 *>(src + j / kHalves * kRowsPerLoad * G::kRowBytes + j % kHalves * 64));
            }
            if constexpr (!G::kWide) { // an item is 32 keys
                const int64_t rec = __shfl_sync(kFullWarpMask, id, lane / kKvPage);
                it.scale = __ldg(reinterpret_cast<const float *>(static_cast<const uint8_t *>(a.k) + (rec * a.kvh + h) * R::kBytes +
                                                                 (v ? R::kVScale : R::kKScale)) + lane % kKvPage);
            }
        };
        // terms of two values into 4 bytes of the tile(s)
        const auto terms = [&](float x, float y, uint32_t &hi, uint32_t &lo) {
            if constexpr (G::kVT == 2) {
                hi = half2_rn(x, y);
                const float2 h = half2_floats(hi), r = __fadd2_rn(make_float2(x, y), make_float2(-h.x, -h.y));
                lo = half2_rn(r.x, r.y);
            } else {
                hi = half2_rn(x, y);
            }
        };
        // Widens an item into its tile. Values come to 2^10 at most, times a power
        // of two that the item's keys share.
        const auto widen = [&](int item, const Item &it) -> bool {
            const int i = item / (2 * G::kItems), part = item % G::kItems, stage = i % G::kStages;
            const bool v = item / G::kItems % 2;
            const int row0 = part * G::kItemKeys, key0 = item_key(item), left = keys - key0;
            const bool edge = key0 + G::kItemKeys > span.ctx;
            const int before = i - G::kStages; // the tile that has the stage until its products are done
            if (before >= 0) {
                constexpr bool kAlternate = kM == 1 && G::kStreams == 2;
                const int e = kAlternate ? before >> 1 : before; // its step, in the last stream that reads its K
                uint64_t *bar = v ? &v_empty[before & 3] : &s_ready[(kM == 2 ? 4 : kAlternate ? (before & 1) * 4 : 0) + (e & 3)];
                if (!sm100::mbar_wait_warp(bar, phase_of(v ? before : e)))
                    return false;
            }
            uint8_t *tile = v ? vs + stage * G::kVBytes : ks + stage * G::kKBytes;
            // Rows that hold an infinity or a NaN: where all nodes see them (no
            // edge) the unit says so; else they are zeros here and marked.
            uint32_t odd = 0;
            bool each = false; // the item's keys have a unit each, not one for all
            float unit;
            const auto put_unit = [&](int row, float unit) { // of the tile's key `row`; NaN stays NaN
                if (v) {
                    const int field = static_cast<int>(__float_as_uint(unit) >> 23);
                    v_log[stage * kTileKeys + row] = unit == unit ? static_cast<float>(field - 127) : unit;
                    v_inv[stage * kTileKeys + row] = pow2_field(254 - field);
                } else {
                    k_unit[(i & 3) * kTileKeys + row] = unit;
                }
            };
            if constexpr (G::kWide) {
                float most = 0.f; // largest magnitude, NaN if a value is
                float y[G::kLoads][4];
#pragma unroll
                for (int j = 0; j < G::kLoads; ++j) {
                    y[j][0] = __uint_as_float(it.r[j].x), y[j][1] = __uint_as_float(it.r[j].y);
                    y[j][2] = __uint_as_float(it.r[j].z), y[j][3] = __uint_as_float(it.r[j].w);
                    if (edge) {
                        bool bad = false;
                        const bool there = j * kRowsPerLoad + lrow < left;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float z = there ? finite_or_zero(y[j][e]) : 0.f;
                            bad |= there && !(z == y[j][e]);
                            y[j][e] = z;
                        }
                        const uint32_t some = __ballot_sync(kFullWarpMask, bad);
#pragma unroll
                        for (int n = 0; n < kRowsPerLoad; ++n)
                            if (some >> (n * kRowLanes) & (kRowLanes == 32 ? 0xffffffffu : (1u << (kRowLanes & 31)) - 1u))
                                odd |= 1u << (j * kRowsPerLoad + n);
                    }
                    most = max_abs_nan(max_abs_nan(most, y[j][0], y[j][1]), y[j][2], y[j][3]);
                }
                const uint32_t bits = __reduce_max_sync(kFullWarpMask, __float_as_uint(most));
                const uint32_t ex = max(exponent_above(bits, 254u), v ? kMinVField + 9u : 0u);
                const float f = pow2_field(254u - ex + 10u);
                unit = bits < 0x7f800000u ? pow2_field(ex - 10u) : __uint_as_float(0x7fc00000u);
                if (edge) { // a row that some nodes do not see takes no bits from the others
                    const float low = pow2_field(max(ex, kUnlike + 1u) - kUnlike);
                    const auto top = [&](int j) { return max_abs_nan(max_abs_nan(y[j][0], y[j][1], y[j][2]), y[j][3], y[j][3]); };
                    float least = low;
#pragma unroll
                    for (int j = 0; j < G::kLoads; ++j)
                        least = fminf(least, j * kRowsPerLoad + lrow < left ? top(j) : low);
                    if (__any_sync(kFullWarpMask, least < low)) // (four values of a row that are all small)
#pragma unroll 1
                        for (int n = 0; n < G::kItemKeys; ++n) {
                            float t = 0.f;
#pragma unroll
                            for (int j = 0; j < G::kLoads; ++j)
                                t = j * kRowsPerLoad + lrow == n ? top(j) : t;
                            const uint32_t all = __reduce_max_sync(kFullWarpMask, __float_as_uint(t));
                            each |= all > 0u && all < __float_as_uint(low);
                        }
                    if (each) // rows to the item's size, for their units to make up for
#pragma unroll
                        for (int j = 0; j < G::kLoads; ++j) {
                            float t = top(j);
#pragma unroll
                            for (int off = 1; off < kRowLanes; off <<= 1)
                                t = fmaxf(t, __shfl_xor_sync(kFullWarpMask, t, off));
                            const uint32_t own = max(exponent_above(__float_as_uint(t), 254u), v ? kMinVField + 9u : 0u);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                y[j][e] = y[j][e] * pow2_field(254u - own + 10u) * pow2_field(ex - 10u);
                            if (lbyte == 0)
                                put_unit(row0 + j * kRowsPerLoad + lrow, pow2_field(own - 10u));
                        }
                }
#pragma unroll
                for (int j = 0; j < G::kLoads; ++j) {
                    uint32_t h0, h1, l0, l1;
                    const float2 a = __fmul2_rn(make_float2(y[j][0], y[j][1]), make_float2(f, f)), b = __fmul2_rn(make_float2(y[j][2], y[j][3]), make_float2(f, f));
                    terms(a.x, a.y, h0, l0);
                    terms(b.x, b.y, h1, l1);
                    const int row = row0 + j * kRowsPerLoad + lrow, dim = lbyte / 4; // 4 dims: 8 bytes of fp16
                    uint8_t *dst = tile + dim / 64 * G::kSlab + swizzled(row, dim % 64 / 8) + dim % 8 * 2;
                    *reinterpret_cast<uint2 *>(dst) = make_uint2(h0, h1);
                    *reinterpret_cast<uint2 *>(dst + G::kSlabs * G::kSlab) = make_uint2(l0, l1);
                }
            } else {
                float scale = lane < left ? it.scale : 0.f;
                const bool bad = !(fabsf(scale) <= 3.4028235e38f);
                odd = __ballot_sync(kFullWarpMask, bad);
                if (!v) { // the codes as they are; the softmax has a key's scale as the factor of its scores
                    unit = bad ? edge ? 0.f : __uint_as_float(0x7fc00000u) : scale;
#pragma unroll
                    for (int j = 0; j < G::kLoads; ++j) {
                        const uint32_t w[4] = {it.r[j].x, it.r[j].y, it.r[j].z, it.r[j].w};
                        const int r = row0 + j / kHalves * kRowsPerLoad + lrow, c = lbyte / 8;
                        uint32_t h[8];
#pragma unroll
                        for (int n = 0; n < 4; ++n)
                            codes_to_half<kFmt>(kFmt == KvFormat::kE4M3 && edge ? clear_e4m3_nan(w[n]) : w[n], h[2 * n], h[2 * n + 1]);
                        uint8_t *slab = tile + j % kHalves * G::kSlab;
                        *reinterpret_cast<uint4 *>(slab + swizzled(r, c)) = make_uint4(h[0], h[1], h[2], h[3]);
                        *reinterpret_cast<uint4 *>(slab + swizzled(r, c + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
                    }
                } else {
                    const uint32_t own = bad ? 0u : __float_as_uint(scale);
                    uint32_t ex = exponent_above(__reduce_max_sync(kFullWarpMask, own), 254u);
                    if (edge) // a row that some nodes do not see takes no bits from the others
                        each = !__all_sync(kFullWarpMask, own == 0u || exponent_above(own, 254u) + kUnlike >= ex);
                    ex = max(each ? exponent_above(own, 254u) : ex, kMinVField);
                    scale = bad ? 0.f : scale * pow2_field(254u - ex + 1u); // at most 2
#pragma unroll
                    for (int j = 0; j < G::kLoads; ++j) {
                        const uint32_t w[4] = {it.r[j].x, it.r[j].y, it.r[j].z, it.r[j].w};
                        const int r = j / kHalves * kRowsPerLoad + lrow, c = lbyte / 8;
                        const float f = __shfl_sync(kFullWarpMask, scale, r);
                        const float2 f2 = make_float2(f, f);
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            float2 x, y;
                            if constexpr (kFmt == KvFormat::kInt8) {
                                // byte + 128 in the low bits of fp32 2^23 .. 2^23 + 255
                                const uint32_t u = w[n] ^ 0x80808080u;
                                const float2 bias = make_float2(-8388736.f, -8388736.f);
                                x = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441))), bias);
                                y = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)), __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443))), bias);
                            } else {
                                uint32_t h0, h1;
                                codes_to_half<kFmt>(edge ? clear_e4m3_nan(w[n]) : w[n], h0, h1);
                                x = half2_floats(h0), y = half2_floats(h1);
                            }
                            x = __fmul2_rn(x, f2), y = __fmul2_rn(y, f2);
                            terms(x.x, x.y, hi[2 * n], lo[2 * n]);
                            terms(y.x, y.y, hi[2 * n + 1], lo[2 * n + 1]);
                        }
                        uint8_t *slab = tile + j % kHalves * G::kSlab, *d0 = slab + swizzled(row0 + r, c), *d1 = slab + swizzled(row0 + r, c + 1);
                        *reinterpret_cast<uint4 *>(d0) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4 *>(d1) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
                        if constexpr (G::kVT == 2) {
                            *reinterpret_cast<uint4 *>(d0 + G::kSlabs * G::kSlab) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                            *reinterpret_cast<uint4 *>(d1 + G::kSlabs * G::kSlab) = make_uint4(lo[4], lo[5], lo[6], lo[7]);
                        }
                    }
                    unit = odd && !edge ? __uint_as_float(0x7fc00000u) : pow2_field(ex - 1u);
                }
            }
            if (lane < G::kItemKeys && !(G::kWide && each))
                put_unit(row0 + lane, unit);
            if (lane == 0) {
                const int at = (v ? stage : i & 3) * 16 + part;
                (v ? v_odd : k_odd)[at] = odd;
                (v ? v_each : k_each)[at] = each;
            }
            sm100::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0)
                sm100::mbar_arrive(&(v ? v_full : k_full)[i & 3]);
            return true;
        };
        Item even, odd;
        int item = warp - 8;
        fetch(item, even);
        fetch(item + kWidenWarps, odd);
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
        // uniform, and one lane issues: a product every 64 cycles leaves no room
        // for moving each operand out of a thread's registers.
        if (tiles > 0) {
            const bool leader = lane == 0;
            const uint32_t tm = __shfl_sync(kFullWarpMask, tmem, 0);
            using Zero = std::integral_constant<int, 0>;
            using One = std::integral_constant<int, 1>;
            constexpr uint32_t idesc_s = sm100::idesc_make(sm100::kFmtF16, 128, kTileKeys);
            constexpr uint32_t idesc_o = sm100::idesc_make(sm100::kFmtF16, 128, D) | (1u << 16); // B MN-major
            // descriptors move by additions to their address field (16-byte units)
            const uint64_t qd = sm100::sdesc_k128(sm100::smem_u32(qs)), kd = sm100::sdesc_k128(sm100::smem_u32(ks));
            const uint64_t vd = sdesc_mn128_16b(sm100::smem_u32(vs), G::kSlab);
            const auto scores = [&](int stream, int i) {
                const uint64_t q0 = qd + static_cast<uint32_t>((kM == 2 ? stream : 0) * (G::kSlab >> 4));
                const uint64_t k0 = kd + static_cast<uint32_t>((i % G::kStages) * (G::kKBytes >> 4));
                const uint32_t d = tm + static_cast<uint32_t>(stream * kTileKeys);
                const auto product = [&](auto qt, auto kt, uint32_t acc) {
#pragma unroll
                    for (int s = 0; s < G::kSlabs; ++s)
#pragma unroll
                        for (int st = 0; st < 4; ++st) // 16 dims: 32 bytes
                            sm100::umma_bf16(d, q0 + static_cast<uint32_t>(((decltype(qt)::value * G::kSlabs + s) * kM * G::kSlab + 32 * st) >> 4),
                                             k0 + static_cast<uint32_t>(((decltype(kt)::value * G::kSlabs + s) * G::kSlab + 32 * st) >> 4),
                                             idesc_s, s + st > 0 ? 1u : acc);
                };
                // small products first: the accumulator is cut off at every step, to its size at the time
                if (leader) {
                    if constexpr (G::kKT == 2)
                        product(Zero{}, One{}, 0);
                    if constexpr (G::kQT == 2)
                        product(One{}, Zero{}, G::kKT == 2);
                    product(Zero{}, Zero{}, G::kKT == 2 || G::kQT == 2);
                }
                __syncwarp();
            };
            const auto weigh = [&](int stream, int i, uint32_t acc) {
                const uint64_t v0 = vd + static_cast<uint32_t>((i % G::kStages) * (G::kVBytes >> 4));
                const uint32_t d = tm + 256u + static_cast<uint32_t>(stream * D), p0 = tm + static_cast<uint32_t>(stream * kTileKeys);
                const auto product = [&](auto pt, auto vt, uint32_t d, uint32_t first) {
#pragma unroll
                    for (int st = 0; st < kTileKeys / 16; ++st) // chunk of 32 keys: 16 columns of each term
                        umma_16_ts(d, p0 + static_cast<uint32_t>(st / 2 * 32 + decltype(pt)::value * 16 + st % 2 * 8),
                                   v0 + static_cast<uint32_t>((decltype(vt)::value * G::kSlabs * G::kSlab + st * 2048) >> 4),
                                   idesc_o, st > 0 ? 1u : first);
                };
                if (leader) {
                    // small products first, where they begin a sum
                    if constexpr (G::kQT == 2) {
                        const uint32_t small = G::kSplitO ? tm + 384u + static_cast<uint32_t>(stream * D) : d;
                        product(Zero{}, One{}, small, acc);
                        product(One{}, Zero{}, small, 1);
                    }
                    product(Zero{}, Zero{}, d, G::kQT == 2 && !G::kSplitO ? 1u : acc);
                }
                __syncwarp();
            };
            const auto commit = [&](uint64_t *bar) {
                if (leader)
                    sm100::umma_commit(bar);
                __syncwarp();
            };
            const auto k_ready = [&](int i) {
                ok = sm100::mbar_wait_warp(&k_full[i & 3], phase_of(i));
                sm100::tc_fence_after();
                return ok;
            };
            // the thread's own arrival passes on what it has seen: the K units
            const auto s_issued = [&](int stream, int e) {
                uint64_t *bar = &s_ready[4 * stream + (e & 3)];
                commit(bar);
                if (leader)
                    sm100::mbar_arrive(bar);
            };
            const auto tile_of = [&](int stream, int e) { return tile_at<G::kStreams, kM>(stream, e, tiles); };
            ok = sm100::mbar_wait_warp(q_full, 0);
            for (int s = 0; ok && s < 2; ++s)
                if (tile_of(s, 0) < tiles && (kM == 2 && s == 1 ? true : k_ready(tile_of(s, 0)))) {
                    scores(s, tile_of(s, 0));
                    s_issued(s, 0);
                }
            for (int e = 0; ok && tile_of(0, e) < tiles; ++e)
                for (int s = 0; ok && s < 2; ++s) {
                    const int i = tile_of(s, e), next = tile_of(s, e + 1);
                    if (i >= tiles)
                        break;
                    if (!sm100::mbar_wait_warp(&p_ready[s], static_cast<uint32_t>(e) & 1u) ||
                        !sm100::mbar_wait_warp(&v_full[i & 3], phase_of(i))) {
                        ok = false;
                        break;
                    }
                    sm100::tc_fence_after();
                    weigh(s, i, e % G::kPeriod != 0);
                    if (kM == 1 || s == 1)
                        commit(&v_empty[i & 3]);
                    if (next < tiles && (kM == 2 && s == 1 ? true : k_ready(next))) {
                        scores(s, next);
                        s_issued(s, e + 1);
                    }
                }
            // every product is done before tensor memory and the tiles are used for anything else
            commit(drain);
            if (!sm100::mbar_wait_warp(drain, 0))
                ok = false;
        }
    } else {
        // ---- softmax warps. First Q: a warp per row, scaled to 2^9 .. 2^10 and split into terms
        constexpr int kE = D / 32; // values per lane
        constexpr int kBatch = 8; // rows whose loads are in flight together
#pragma unroll 1
        for (int r0 = warp; r0 < G::kRows; r0 += 8 * kBatch) {
            float x[kBatch][kE];
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const int row = row_base + r0 + 8 * n;
                const T *src = q + static_cast<int64_t>(span.row0 + row / rep) * a.q_stride + static_cast<int64_t>(h * rep + row % rep) * D + kE * lane;
#pragma unroll
                for (int e = 0; e < kE; ++e)
                    x[n][e] = row < rows ? static_cast<float>(src[e]) : 0.f;
            }
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const int r = r0 + 8 * n;
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < kE; ++e)
                    top = max(top, __float_as_uint(x[n][e]) & 0x7fffffffu);
                top = __reduce_max_sync(kFullWarpMask, top);
                const uint32_t ex = exponent_above(top);
                const float f = copysignf(pow2_field(254u - ex + 10u), a.scale_log2);
                const int dim = kE * lane;
                uint8_t *dst = qs + (dim / 64 * kM + r / 128) * G::kSlab + swizzled(r % 128, dim % 64 / 8) + dim % 8 * 2;
#pragma unroll
                for (int e = 0; e < kE; e += 2) {
                    const float u = x[n][e] * f, v = x[n][e + 1] * f;
                    const uint32_t hi = half2_rn(u, v);
                    *reinterpret_cast<uint32_t *>(dst + 2 * e) = hi;
                    if constexpr (G::kQT == 2) {
                        const float2 w = half2_floats(hi);
                        *reinterpret_cast<uint32_t *>(dst + G::kSlabs * kM * G::kSlab + 2 * e) = half2_rn(u - w.x, v - w.y);
                    }
                }
                if (lane == 0)
                    row_fac[r] = top < 0x7f800000u ? fabsf(a.scale_log2) * pow2_field(ex - 10u) : __uint_as_float(0x7fc00000u);
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
        const float rs = row_fac[kM == 2 ? stream * 128 + r : r];
        const uint32_t quarter = static_cast<uint32_t>((warp % 4) * 32) << 16;
        const uint32_t st = tmem + quarter + static_cast<uint32_t>(stream * kTileKeys);
        const uint32_t ot = tmem + quarter + 256u + static_cast<uint32_t>(stream * D);
        float m = kNone, l = 0.f;
        constexpr int kGroup = G::kItemKeys, kGroups = 32 / kGroup; // keys that share their units; such groups in a chunk
        int e = 0; // steps done
        for (; ok; ++e) {
            const int i = tile_at<G::kStreams, kM>(stream, e, tiles);
            if (i >= tiles)
                break;
            const int stage = i % G::kStages, key0 = key_of(i);
            if (!sm100::mbar_wait_warp(&s_ready[4 * stream + (e & 3)], phase_of(e))) {
                ok = false;
                break;
            }
            sm100::tc_fence_after();
            const float *ku = k_unit + (i & 3) * kTileKeys, *vl = v_log + stage * kTileKeys, *vi = v_inv + stage * kTileKeys;
            const bool edge = key0 + kTileKeys > span.ctx; // holds nodes, or places after the last key
            const auto seen_of = [&](int c) {
                return live ? tree_sees32(a.t, span.row0 + node, node, key0 + 32 * c - span.ctx, keys - span.ctx) : 0u;
            };
            // 32 scores of the row, from tensor memory: asked for, and there
            const auto ask = [&](int c, uint32_t (&x)[2][16]) {
                sm100::tmem_ld_32x16(st + static_cast<uint32_t>(32 * c), x[0]);
                sm100::tmem_ld_32x16(st + static_cast<uint32_t>(32 * c + 16), x[1]);
            };
            const auto await = [&](uint32_t (&x)[2][16]) {
                sm100::tmem_wait_ld();
                sm100::tmem_reg_fence(x[0]);
                sm100::tmem_reg_fence(x[1]);
            };
            // a chunk's keys that the row sees, and those that are not finite
            const auto odd_of = [&](int c) {
                uint32_t bits = 0;
#pragma unroll
                for (int n = 0; n < kGroups; ++n)
                    bits |= (k_odd[(i & 3) * 16 + kGroups * c + n] | v_odd[stage * 16 + kGroups * c + n]) << (n * kGroup & 31);
                return bits;
            };
            // what two scores of chunk c are multiplied by: 8-bit keys have a factor each, four to
            // a broadcast; the keys of a group of fp32 rows share theirs
            const auto factors = [&](int c, int n, auto each_tag) {
                if constexpr (G::kWide && !decltype(each_tag)::value) {
                    const float f = rs * ku[32 * c + n / kGroup * kGroup];
                    return make_float2(f, f);
                } else {
                    const float4 f = *reinterpret_cast<const float4 *>(ku + 32 * c + n / 4 * 4);
                    return __fmul2_rn(n % 4 == 0 ? make_float2(f.x, f.y) : make_float2(f.z, f.w), make_float2(rs, rs));
                }
            };
            // log2 of the V units of two keys of chunk c, less m
            const auto bases = [&](int c, int n, float m, auto each_tag) {
                if constexpr (decltype(each_tag)::value) {
                    const float2 log = *reinterpret_cast<const float2 *>(vl + 32 * c + n);
                    return make_float2(log.x - m, log.y - m);
                } else {
                    const float base = vl[32 * c + n / kGroup * kGroup] - m;
                    return make_float2(base, base);
                }
            };
            // two scores of a chunk in log2 units less `m`; masked ones -inf (edge tiles)
            const auto scored = [&](const uint32_t (&x)[2][16], int n, float2 f, float2 m2, uint32_t seen, uint32_t odd, auto edge_tag) {
                float2 y = __ffma2_rn(make_float2(__uint_as_float(x[n / 16][n % 16]), __uint_as_float(x[n / 16][n % 16 + 1])), f, m2);
                if constexpr (decltype(edge_tag)::value) {
                    const float bad = __uint_as_float(0x7fc00000u);
                    y.x = !(seen >> n & 1u) ? kNegInf : odd >> n & 1u ? bad : y.x;
                    y.y = !(seen >> (n + 1) & 1u) ? kNegInf : odd >> (n + 1) & 1u ? bad : y.y;
                }
                return y;
            };
            // a period's end: O to the long sum (this tile's S is there, so the products
            // before it are done; the next ones start O anew)
            if (G::kQT == 2 && e > 0 && e % G::kPeriod == 0) {
#pragma unroll 1
                for (int d = 0; d < D; d += 16) {
                    uint32_t o[16], x[16];
                    sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(d), o);
                    if (G::kSplitO)
                        sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(d + 128), x);
                    sm100::tmem_wait_ld();
                    sm100::tmem_reg_fence(o);
                    if constexpr (G::kSplitO) {
                        sm100::tmem_reg_fence(x);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            o[k] = __float_as_uint(__uint_as_float(o[k]) + __uint_as_float(x[k]));
                    }
                    if (e > G::kPeriod) {
                        sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(d + G::kLong), x);
                        sm100::tmem_wait_ld();
                        sm100::tmem_reg_fence(x);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            o[k] = __float_as_uint(__uint_as_float(o[k]) + __uint_as_float(x[k]));
                    }
                    tile_tmem_st16(ot + static_cast<uint32_t>(d + G::kLong), o);
                }
                tile_tmem_wait_st();
            }
            uint32_t xa[2][16], xb[2][16];
            ask(0, xa);
            if (!sm100::mbar_wait_warp(&v_full[i & 3], phase_of(i))) {
                await(xa);
                ok = false;
                break;
            }
            // O, where there is one, times fix; the weights of this tile's first `c` chunks too
            const auto rescale = [&](float fix, int c) {
                if (e > 0) {
                    // (this tile's S is there, so the products before it are done)
#pragma unroll 1
                    for (int n = 0; n < (G::kSplitO ? 2 * D : D) + (G::kQT == 2 && e >= G::kPeriod ? D : 0); n += 16) {
                        // the small products' columns lie 128 on
                        const int d = n < D ? n : G::kSplitO && n < 2 * D ? n - D + 128 : n % D + G::kLong;
                        uint32_t o[16];
                        sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(d), o);
                        sm100::tmem_wait_ld();
                        sm100::tmem_reg_fence(o);
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            o[k] = __float_as_uint(__uint_as_float(o[k]) * fix);
                        tile_tmem_st16(ot + static_cast<uint32_t>(d), o);
                    }
                }
                tile_tmem_wait_st(); // chunks' weights are stored before they are read
                const __half2 half_fix = __float2half2_rn(fix);
#pragma unroll 1
                for (int d = 0; d < 32 * c; d += 16) {
                    uint32_t o[16];
                    sm100::tmem_ld_32x16(st + static_cast<uint32_t>(d), o);
                    sm100::tmem_wait_ld();
                    sm100::tmem_reg_fence(o);
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const __half2 p = __hmul2(*reinterpret_cast<const __half2 *>(&o[k]), half_fix);
                        o[k] = *reinterpret_cast<const uint32_t *>(&p);
                    }
                    tile_tmem_st16(st + static_cast<uint32_t>(d), o);
                }
                tile_tmem_wait_st();
            };
            const auto tile = [&](auto edge_tag, auto each_tag) {
                constexpr bool kEdge = decltype(edge_tag)::value, kEach = decltype(each_tag)::value;
                // The first reference: the largest score of the first tile of which the row sees
                // anything. It has to come from the scores: against m's first value every
                // score is the same number. (Rows past the last one have scores of the context
                // too, zeros, and would raise theirs many times over.)
                if (__any_sync(kFullWarpMask, m == kNone && (live || !kEdge))) {
                    float top = kNegInf;
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        ask(c, xb);
                        await(xb);
                        const uint32_t seen = kEdge ? seen_of(c) : 0u;
#pragma unroll
                        for (int n = 0; n < 32; n += 2) {
                            const float2 y = scored(xb, n, factors(c, n, each_tag), bases(c, n, 0.f, each_tag), seen, 0u, edge_tag);
                            top = fmaxf(top, fmaxf(y.x, y.y));
                        }
                    }
                    if (m == kNone)
                        m = fmaxf(m, top - reference_lift(kTileLift, top));
                }
                // one chunk of 32 keys, whose scores are in x, the next one's on their way to `next`
                const auto chunk = [&](int c, uint32_t (&x)[2][16], uint32_t (&next)[2][16]) {
                    await(x);
                    if (c < 3)
                        ask(c + 1, next);
                    const uint32_t seen = kEdge ? seen_of(c) : 0u, odd = kEdge ? odd_of(c) : 0u;
                    // Scores and weights at once, for weights up to 2^kTileTop fit in
                    // fp16 but for a rare chunk: one with a larger one raises the
                    // reference and is done again (its scores are still there). From a
                    // reference far below, each time brings the rest to 2^-19 of it; scores
                    // of 2^28 and more are rounded by more than kTileTop, so that what is
                    // too large in the end is cut off.
#pragma unroll 1
                    for (int raises = 0;; ++raises) {
                        float top[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
                        for (int n = 0; n < 32; n += 2) {
                            const float2 y = scored(x, n, factors(c, n, each_tag), bases(c, n, m, each_tag), seen, odd, edge_tag);
                            top[n / 2 % 4] = fmaxf(top[n / 2 % 4], fmaxf(y.x, y.y));
                            x[n / 16][n % 16] = __float_as_uint(y.x);
                            x[n / 16][n % 16 + 1] = __float_as_uint(y.y);
                        }
#pragma unroll
                        for (int n = 0; n < 32; ++n)
                            x[n / 16][n % 16] = __float_as_uint(exp2_approx(__uint_as_float(x[n / 16][n % 16])));
                        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                        if (!__any_sync(kFullWarpMask, most > kTileTop))
                            break;
                        if (raises == 6) {
                            const float cap = exp2_approx(kTileTop);
#pragma unroll
                            for (int n = 0; n < 32; ++n) { // (a NaN stays)
                                const float p = __uint_as_float(x[n / 16][n % 16]);
                                x[n / 16][n % 16] = __float_as_uint(p > cap ? cap : p);
                            }
                            break;
                        }
                        const float less = fmaxf(0.f, ceilf(most - reference_lift(kTileLift, 2.f * fmaxf(fabsf(most), fabsf(m))))), fix = exp2_approx(-less);
                        if (c < 3)
                            await(next);
                        rescale(fix, c);
                        l *= fix;
                        m += less;
                        ask(c, x);
                        await(x);
                    }
                    float2 sum[kGroups];
#pragma unroll
                    for (int n = 0; n < kGroups; ++n)
                        sum[n] = make_float2(0.f, 0.f);
#pragma unroll
                    for (int part = 0; part < 2; ++part) { // 16 keys, a step of the product
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int n = 0; n < 8; ++n) {
                            const int k = (16 * part + 2 * n) / kGroup;
                            const float2 p = make_float2(__uint_as_float(x[part][2 * n]), __uint_as_float(x[part][2 * n + 1]));
                            if constexpr (kEach)
                                sum[0] = __ffma2_rn(p, *reinterpret_cast<const float2 *>(vi + 32 * c + 16 * part + 2 * n), sum[0]);
                            else
                                sum[k] = __fadd2_rn(sum[k], p);
                            hi[n] = half2_rn(p.x, p.y);
                            if constexpr (G::kQT == 2) {
                                const float2 w = half2_floats(hi[n]);
                                const float2 r = __fadd2_rn(p, make_float2(-w.x, -w.y));
                                lo[n] = half2_rn(r.x, r.y);
                            }
                        }
                        tile_tmem_st8(st + static_cast<uint32_t>(32 * c + 8 * part), hi);
                        if constexpr (G::kQT == 2)
                            tile_tmem_st8(st + static_cast<uint32_t>(32 * c + 16 + 8 * part), lo);
                    }
#pragma unroll
                    for (int n = 0; n < (kEach ? 1 : kGroups); ++n) // from weights in units of V to l
                        l = fmaf(sum[n].x + sum[n].y, kEach ? 1.f : vi[32 * c + n * kGroup], l);
                };
#pragma unroll 1
                for (int c = 0; c < 4; c += 2) {
                    chunk(c, xa, xb);
                    chunk(c + 1, xb, xa);
                }
            };
            // whether an item of the tile has a unit for each key (edge tiles)
            const auto any_each = [&] {
                const uint4 k = *reinterpret_cast<const uint4 *>(k_each + (i & 3) * 16), v = *reinterpret_cast<const uint4 *>(v_each + stage * 16);
                const uint32_t none = G::kItems < 16 ? 0u : ~0u; // what lies after the items is not theirs
                return ((k.x | v.x) | (G::kItems >= 8 ? k.y | v.y : 0u) | ((k.z | v.z | k.w | v.w) & none)) != 0u;
            };
            if (!edge)
                tile(std::false_type{}, std::false_type{});
            else if (!any_each())
                tile(std::true_type{}, std::false_type{});
            else
                tile(std::true_type{}, std::true_type{});
            tile_tmem_wait_st();
            sm100::tc_fence_before();
            __syncwarp();
            if (lane == 0)
                sm100::mbar_arrive(&p_ready[stream]);
        }
        // the stream's O, m and l
        const bool any = ok && e > 0;
        if (any && !sm100::mbar_wait_warp(drain, 0)) // all products: O is there, and the tiles are free
            ok = false;
        sm100::tc_fence_after();
        const bool direct = kM == 2 && splits == 1;
        // where nothing is joined a row goes out as it is; else to shared memory, once all products are done
        if (!direct)
            asm volatile("bar.sync 1, 256;" ::: "memory"); // both streams have waited for that
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T *dst = out + static_cast<int64_t>(span.row0 + node) * a.out_stride + static_cast<int64_t>(h * rep + row % rep) * D;
        float *part = reinterpret_cast<float *>(smem) + (stream * 128 + r) * G::kPitch;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            __syncwarp();
            if (any) { // the same in a warp
                sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(c), o);
                sm100::tmem_wait_ld();
                sm100::tmem_reg_fence(o);
                const auto plus = [&](int from) {
                    uint32_t x[16];
                    sm100::tmem_ld_32x16(ot + static_cast<uint32_t>(c + from), x);
                    sm100::tmem_wait_ld();
                    sm100::tmem_reg_fence(x);
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        o[k] = __float_as_uint(__uint_as_float(o[k]) + __uint_as_float(x[k]));
                };
                if (G::kSplitO)
                    plus(128);
                if (G::kQT == 2 && e > G::kPeriod)
                    plus(G::kLong);
            } else {
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    o[k] = 0;
            }
            if (direct) {
                if (live)
#pragma unroll
                    for (int k = 0; k < 16; k += KvVec<T>::kN) {
                        float y[KvVec<T>::kN];
#pragma unroll
                        for (int n = 0; n < KvVec<T>::kN; ++n)
                            y[n] = l == 0.f ? 0.f : __uint_as_float(o[k + n]) * inv;
                        *reinterpret_cast<uint4 *>(dst + c + k) = KvVec<T>::pack(y);
                    }
            } else {
#pragma unroll
                for (int k = 0; k < 16; k += 4)
                    *reinterpret_cast<float4 *>(part + c + k) =
                        make_float4(__uint_as_float(o[k]), __uint_as_float(o[k + 1]), __uint_as_float(o[k + 2]), __uint_as_float(o[k + 3]));
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
    // join: the two streams of a row tile, then the cluster's CTAs
    float *part = reinterpret_cast<float *>(smem);
    const int rows_here = min(G::kRows, rows - row_base); // may be negative
    const auto put = [&](int r, int d, float O, float L) {
        const int row = row_base + r;
        out[static_cast<int64_t>(span.row0 + row / rep) * a.out_stride + static_cast<int64_t>(h * rep + row % rep) * D + d] =
            static_cast<T>(L == 0.f ? 0.f : O / L);
    };
    if (kM == 1) {
        for (int i = tid; i < 128 * D; i += kTileThreads) {
            const int r = i / D, d = i % D;
            if (r >= rows_here)
                break;
            const float m0 = stat[r], m1 = stat[128 + r], top = fmaxf(m0, m1);
            const float f0 = exp2_approx(m0 - top), f1 = exp2_approx(m1 - top);
            const float O = f0 * part[r * G::kPitch + d] + f1 * part[(128 + r) * G::kPitch + d];
            const float L = f0 * stat[256 + r] + f1 * stat[384 + r];
            if (splits == 1) {
                put(r, d, O, L);
            } else {
                part[r * G::kPitch + d] = O; // read by this thread alone
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
    for (int i = rank * kTileThreads + tid; i < G::kRows * D; i += splits * kTileThreads) {
        const int r = i / D, d = i % D;
        if (r >= rows_here)
            break;
        float top = kNone, L = 0.f, O = 0.f;
        for (int c = 0; c < splits; ++c)
            top = fmaxf(top, peer_load(&joined[r], c));
        for (int c = 0; c < splits; ++c) {
            const float f = exp2_approx(peer_load(&joined[r], c) - top);
            L += f * peer_load(&joined[256 + r], c);
            O += f * peer_load(&part[r * G::kPitch + d], c);
        }
        put(r, d, O, L);
    }
    __syncthreads();
    cluster_sync_all(); // peers read this CTA's shared memory until here
}

template <typename T, int D, KvFormat kFmt, int kM>
inline void tree_tiles_launch(const T *q, T *out, const TreeArgs &a, cudaStream_t stream) {
    using G = TreeTilesGeo<T, D, kFmt, kM>;
    static_assert(G::kItems <= 16 && 2 * G::kItems >= kWidenWarps && G::kBytes <= 232448, "shared memory");
    const auto kernel = tree_tiles_kernel<T, D, kFmt, kM>;
    allow_shared_bytes(kernel, kTileThreads, G::kBytes);
    const int64_t rows = static_cast<int64_t>(a.t.max_rows) * (a.qh / a.kvh);
    const int64_t groups = (rows + G::kRows - 1) / G::kRows, units = groups * a.kvh;
    const int64_t tiles = (static_cast<int64_t>(a.t.max_ctx) + a.t.max_rows + kTileKeys - 1) / kTileKeys;
    // as many splits as all CTAs still run at once and each has four tiles
    const int64_t all = units * a.t.batch;
    const int splits = static_cast<int>(std::max<int64_t>(1, std::min(std::min<int64_t>(8, tiles / 4), device_facts().sm_count / all)));
    require(units * splits <= 0x7fffffff, "tree attention: too many rows for one call");
    // more CTAs than places: sequences in the order of their length
    const bool sorted = a.t.batch > 1 && a.t.batch <= kTileThreads - 1 && units * splits * a.t.batch > device_facts().sm_count;
    launch_ex_cluster(kernel, dim3(static_cast<unsigned>(units * splits), a.t.batch), dim3(splits), dim3(kTileThreads),
                      G::kBytes, stream, q, out, a, static_cast<int>(groups), splits, sorted, sm100::device_error_word());
}

} // namespace opworks::detail
