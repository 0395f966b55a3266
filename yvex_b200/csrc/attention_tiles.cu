// Attention of many rows per (request, kv head) over the paged cache - drafted trees, chunks of prompts - on tcgen05.
//
// Keys and values come page by page by TMA, straight from where they lie (boxes of as many rows as a page's size allows, up to the 128
// keys of a block), scores and the output's sums live in tensor memory, and a thread of the softmax warps owns a row, so its
// maximum and sum need no shuffles. S = Q K^T reads both operands from shared memory; the weights P go back to tensor memory, rounded once to
// the cache's type, and are the A operand of O += P V, whose B is the V tile as it lies (N-major). P has columns of its own, so the buffer of S is
// free as soon as its row is in registers and the next S is computed during the softmax (with P over S a block's chain S, softmax, PV
// was 3960 cycles for two streams, of which the tensor cores worked 2048). Two streams of softmax warps, each with scores and
// sums of its own, take turns with the tensor cores: with more than 128 rows they are two tiles of rows over the same keys (each block
// of keys is read once for 256 rows); with up to 128 they are the even and the odd blocks of one tile's keys, joined when the item
// ends. 256 columns of a head leave room for one stream (O alone takes 256 of the 512 columns of tensor memory).
//
// The running maximum is only followed when it grows by more than kSlack powers of two: rescaling O means reading and writing it back, and a
// weight of up to 2^kSlack costs no precision in f32 sums. f16 weights are lifted by 2^10, so that those down to 2^-24 of the
// maximum keep all their bits and smaller ones are off by at most 2^-35 of it, and follow the maximum sooner.
//
// A block of 128 keys for two tiles takes 2900 to 3000 cycles, of which the tensor cores work 2048 and the exponentials (16 a cycle and SM) as much, an
// item 17 K besides; counted, both units are busy 58 to 61 % of an SM's active cycles. What is left is that S and PV stand behind one another
// in the tensor cores' queue and that there is one buffer of S for two streams. 16 trees of 32 to 64 nodes over 100 to 32768 keys (32 query heads,
// 8 kv heads, 128 dims, 1.02 GB of cache): 405 K cycles from the first CTA to the last, 349 K of them active on an SM; 256 us after a rest and 299 in a
// row, where the power cap holds the clock at 1470 MHz (307 with three sets of inputs). Chunks of two prompts (573 GFLOP): 898 K cycles, 827 K active;
// 522 us after a rest, 579 in a row at 1700 MHz (591 with three sets: 0.97 PFLOP/s). 168 registers at launch, 172 bytes of them spilled (64 and 128 dims).
#include <cuda.h>
#include <cudaTypedefs.h>

#include "paged_work.cuh"
#include "tcgen05.cuh"

namespace yb {

template <int D> struct TilePlan {
    static constexpr int kStreams = D == 256 ? 1 : 2, kRows = 128 * kStreams, kKeys = D == 256 ? 64 : 128;
    static constexpr int kStages = D == 64 ? 4 : 2;
    static constexpr uint32_t kQBytes = 128 * D * 2, kTileBytes = kKeys * D * 2;      // Q of a stream, K or V of a block
    static constexpr int kSoftmaxWarps = 4 * kStreams, kThreads = 32 * (kSoftmaxWarps + 4);
    // registers per thread: the softmax warps hold a row of scores, the last warpgroup (copies, products) hands theirs over
    static constexpr int kLaunched = 65536 / kThreads > 255 ? 248 : 65536 / kThreads & ~7, kSoftmaxRegs = kStreams == 2 ? 208 : kLaunched, kControlRegs = kStreams == 2 ? 80 : kLaunched;
    static_assert(kSoftmaxWarps * kSoftmaxRegs + 4 * kControlRegs <= kLaunched * (kThreads / 32), "an increase would wait forever");
    // columns of tensor memory: the buffers of S (64 dims: one a stream; 128: one that the streams use in turn; 256: two that the stream
    // uses in turn), then P and O of each stream
    static constexpr uint32_t kSBuffers = D == 128 ? 1 : 2, kPCol = kSBuffers * kKeys, kOCol = kPCol + kStreams * kKeys / 2;
    static_assert(kOCol + kStreams * D <= 512, "tensor memory has 512 columns");
    static constexpr uint32_t kBadRing = 8, kStaging = 2048;                            // bytes of output rows that a warp turns at a time
};
constexpr uint32_t kTilesTmem = 512;

template <int D> struct TileSmem {
    using Plan = TilePlan<D>;
    uint4 staging[Plan::kSoftmaxWarps][Plan::kStaging / 16];
    uint64_t q_full, q_free, k_full[Plan::kStages], k_empty[Plan::kStages], v_full[Plan::kStages], v_empty[Plan::kStages];
    uint64_t s_full[2], s_free[2], p_full[2], o_done[2], v_clean[Plan::kStages], all, looked, noted, drain[2];
    PagedScratch<Plan::kThreads> scan;
    float ml[2][2][128];
    unsigned long long odd_mask;                 // the item's fresh tokens with values that are not finite: as bits, and the first of them
    int odd_first;
    uint32_t bad_keys[Plan::kBadRing];
    uint32_t tmem_base;
    int abort;
};

// q: rows of Q as {head_dim, query heads, tokens}, boxes of 64 values x a group x 128 / group tokens
struct TileMaps { CUtensorMap k, v, q; };

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(sm100::smem_u32(dst)), "l"(map), "r"(sm100::smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

// two sums or products in one instruction each
__device__ __forceinline__ float2 fma2(float2 a, float b, float c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void add2(float2 &a, float2 b) {
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a.x), "+f"(a.y) : "f"(b.x), "f"(b.y));
}
template <class T> struct PairOf { using type = __half2; };
template <> struct PairOf<__nv_bfloat16> { using type = __nv_bfloat162; };
template <class T> __device__ __forceinline__ typename PairOf<T>::type pair_of(uint32_t w) { return *reinterpret_cast<typename PairOf<T>::type *>(&w); }
// 16 bytes global -> shared that complete with the thread's group of copies; zeros where `live` is false
__device__ __forceinline__ void copy16(void *dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sm100::smem_u32(dst)), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <class T, int D>
__global__ void __launch_bounds__(TilePlan<D>::kThreads, 1) paged_tiles_kernel(const __grid_constant__ TileMaps maps, const PagedParams p, const int box_keys, const int q_tokens) {
    using namespace sm100;
    using Plan = TilePlan<D>;
    constexpr int BK = Plan::kKeys, NS = Plan::kStreams, kStages = Plan::kStages, kHalves = D / 64;
    constexpr uint32_t kTileBytes = Plan::kTileBytes, kQBytes = Plan::kQBytes;
    constexpr bool kHalfType = std::is_same<T, __half>::value;
    constexpr float kLift = kHalfType ? 10.0f : 0.0f, kSlack = kHalfType ? 4.0f : 8.0f;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    if (smem_u32(smem_raw) & 1023u) {                           // uniform: nothing has been set up yet
        pdl_wait();
        if (threadIdx.x == 0) { raise(p.status, YVEX_B200_STATUS_TIMEOUT); p.share[blockIdx.x].rows = 0; }
        return;
    }
    uint8_t *q_tiles = smem_raw, *k_tiles = q_tiles + NS * kQBytes, *v_tiles = k_tiles + kStages * kTileBytes;
    TileSmem<D> *sm = reinterpret_cast<TileSmem<D> *>(v_tiles + kStages * kTileBytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        mbar_init(&sm->q_full, 1);
        mbar_init(&sm->q_free, 1);
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sm->k_full[i], 1); mbar_init(&sm->k_empty[i], 1);
            mbar_init(&sm->v_full[i], 1); mbar_init(&sm->v_empty[i], 2); mbar_init(&sm->v_clean[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm->s_full[i], 1); mbar_init(&sm->s_free[i], 4); mbar_init(&sm->p_full[i], 4); mbar_init(&sm->o_done[i], 1);
            mbar_init(&sm->drain[i], 1);
        }
        mbar_init(&sm->all, Plan::kSoftmaxWarps);
        mbar_init(&sm->looked, 1);
        mbar_init(&sm->noted, Plan::kSoftmaxWarps);
        sm->abort = 0;
        fence_barrier_init();
    }
    if (warp == 0) tmem_alloc(&sm->tmem_base, kTilesTmem);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm->tmem_base;
    volatile int *abort = &sm->abort;
    pdl_trigger();
    pdl_wait();
    const PagedStart start = paged_start<Plan::kThreads, Plan::kRows, BK, kTilesCost>(p, &sm->scan);
    // An item of more rows than a stream has is two tiles over the same keys, otherwise the streams take turns with the blocks of keys.
    using Walk = PagedWalk<Plan::kRows, BK, kTilesCost>;
    // ..., and the keys before this one are seen by every row.
    auto safe_keys = [&](const Walk &w) { return (int)w.q.n.cached + (p.tree ? 0 : (int)(w.tile * Plan::kRows / p.group) + 1); };
    auto rows_of = [](const Walk &w) { return min(w.q.rows - w.tile * Plan::kRows, (uint32_t)Plan::kRows); };
    Walk w;

    // Q of an item into shared memory, K-major with the 128-byte swizzle. Where a tile's 128 rows are whole tokens (q_tokens of them) it is
    // a box per 64 dims; the rows behind the item's last one are then some other rows, whose results go nowhere.
    auto load_q = [&]() {                                       // by one lane
        const uint32_t tiles = NS == 2 && rows_of(w) > 128u ? 2u : 1u;
        mbar_expect_tx(&sm->q_full, tiles * kQBytes);
        for (uint32_t t = 0; t < tiles; ++t)
            for (int h = 0; h < kHalves; ++h)
                tma_load_3d(q_tiles + t * kQBytes + h * 16384, &maps.q, 64 * h, (int)(w.head * p.group),
                            (int)(w.q.n.token + (w.tile * (Plan::kRows / 128) + t) * (uint32_t)q_tokens), &sm->q_full);
    };
    // Other groups' rows are copied one by one, by some warps; the copies are complete on return.
    auto copy_q = [&](uint32_t first, uint32_t step) {
        constexpr uint32_t kLanes = D / 8, kAt = 32 / kLanes;    // lanes of a row, rows at a time
        const uint32_t chunk = (uint32_t)lane % kLanes, rows = rows_of(w), end = NS == 2 && rows > 128u ? 256u : 128u;
        const uint16_t *src = p.q + (uint64_t)w.head * p.group * D + 8 * chunk;
#pragma unroll 4
        for (uint32_t row = first * kAt + (uint32_t)lane / kLanes; row < end; row += step * kAt) {
            const bool live = row < rows;
            const uint32_t at = live ? w.tile * Plan::kRows + row : 0u, token = at / p.group, rr = row & 127u;
            copy16(q_tiles + (row >> 7) * kQBytes + (chunk >> 3) * 16384 + rr * 128 + (((chunk & 7u) ^ (rr & 7u)) << 4),
                   src + (uint64_t)(w.q.n.token + token) * p.q_stride + (uint64_t)(at - token * p.group) * D, live);
        }
        copies_done();
        fence_proxy_async();
    };

    if (warp < Plan::kSoftmaxWarps) {
        // ---------------- softmax: thread = row of a stream's tile ----------------
        set_registers<Plan::kSoftmaxRegs, Plan::kLaunched>();
        const int st = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t p_at = tmem + lanes + Plan::kPCol + (uint32_t)st * (BK / 2), o_at = tmem + lanes + Plan::kOCol + (uint32_t)st * D;
        const float scale = p.scale * 1.4426950408889634f;      // scores in powers of two
        uint32_t done = 0, all_ph = 0, it_base = 0, segment = 0;
        bool ok = true, bad_out = false;
        if (tid == 0) p.share[blockIdx.x].rows = 0;
        auto sync_all = [&]() {                                 // every softmax thread of the CTA; bounded like every wait
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm->all);
            ok = ok && mbar_wait_warp(&sm->all, all_ph, abort);
            all_ph ^= 1u;
        };
        w.start(p, start);
        if (w.live() && !q_tokens) {                            // the first item's Q; a warp of its own fetches the others' ahead
            copy_q((uint32_t)warp, Plan::kSoftmaxWarps);
            sync_all();
            if (tid == 0) mbar_arrive(&sm->q_full);
        }
        for (; w.live() && ok; it_base += w.count, w.next(p), ++segment) {
            const uint32_t rows = rows_of(w);
            const bool two = NS == 2 && rows > 128u;            // two tiles of rows
            const uint32_t row0 = w.tile * Plan::kRows + (two ? 128u * st : 0u), item_row = row0 + r;
            const bool live = item_row < w.q.rows;
            const uint32_t token = item_row / p.group;
            const int cached = (int)w.q.n.cached, end = cached + (int)w.q.n.fresh, seen = live ? cached + (int)token + 1 : cached;
            const uint64_t mask = p.tree && live ? p.ancestors[w.q.n.token + token] : 0ull;
            const int safe = safe_keys(w);
            const uint32_t stride = two ? 1u : NS, begin = two ? 0u : (uint32_t)st;
            float m = -INFINITY, l = 0.0f;
            bool any = false;
            for (uint32_t j = begin; j < w.count && ok; j += stride) {
                const uint32_t it = it_base + j;
                const int base = (int)(w.first + j) * BK;
                // (which barrier tells of S: the stream's, or with two buffers for one stream the buffer's)
                const uint32_t full = NS == 1 ? done & 1u : (uint32_t)st, full_ph = NS == 1 ? done >> 1 : done;
                const uint32_t buffer = Plan::kSBuffers == 1 ? 0u : full, s_at = tmem + lanes + buffer * BK;
                ok = mbar_wait_warp(&sm->s_full[full], full_ph & 1u, abort);
                if (!ok) break;
                ++done;
                tc_fence_after();
                float s[BK];
#pragma unroll
                for (int i = 0; i < BK / 32; ++i) tmem_ld32(s_at + 32 * i, reinterpret_cast<uint32_t *>(s) + 32 * i);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm->s_free[buffer]);
                const uint32_t bad = sm->bad_keys[it % Plan::kBadRing];      // groups of 16 keys whose page is none
                if (base + BK > safe || bad) {
                    // ---- keys that not every row sees (their values are looked over by the warp that issues the products)
#pragma unroll
                    for (int i = 0; i < BK / 64; ++i) {
                        uint64_t sees = paged_sees(p.tree, base + 64 * i, cached, seen, mask) & low_bits(end - base - 64 * i);
#pragma unroll
                        for (int g = 0; g < 4; ++g)
                            if ((bad >> (4 * i + g)) & 1u) sees &= ~(0xffffull << (16 * g));
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t x = (uint32_t)(sees >> (32 * h));
                            if (__all_sync(0xffffffffu, x == ~0u)) continue;
#pragma unroll
                            for (int e = 0; e < 32; ++e) s[64 * i + 32 * h + e] = (x >> e) & 1u ? s[64 * i + 32 * h + e] : -INFINITY;
                        }
                    }
                }
                // ---- the block's maximum; O follows it only when it must
                float t[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int i = 4; i + 8 <= BK; i += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) t[e] = fmaxf(fmaxf(t[e], s[i + e]), s[i + 4 + e]);
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = fmaxf(t[e], s[BK - 4 + e]);
                const float top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])) * scale;
                float f = 1.0f;
                if (m == -INFINITY) m = top;                    // nothing seen so far: O is zero
                else if (top > m + kSlack) { f = exp2f(m - top); m = top; }
                if (__any_sync(0xffffffffu, f != 1.0f)) {
                    ok = mbar_wait_warp(&sm->o_done[st], done & 1u, abort);      // O is complete
                    if (!ok) break;
                    tc_fence_after();
                    l *= f;
#pragma unroll 1
                    for (int i = 0; i < D; i += 16) {
                        uint32_t o[16];
                        tmem_ld16(o_at + i, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st16(o_at + i, o);
                    }
                }
                // ---- weights, their sum, and P
                const float shift = (m == -INFINITY ? 0.0f : m) - kLift;
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int b = 0; b < BK / 32; ++b) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 x = fma2(make_float2(s[32 * b + 2 * i], s[32 * b + 2 * i + 1]), scale, -shift);
                        x.x = exp2f(x.x);
                        x.y = exp2f(x.y);
                        add2(sum[i & 1], x);
                        pk[i] = close2<T>(x.x, x.y);
                    }
                    if (b == 0 && any) {                        // the products of the block before have read its P
                        ok = mbar_wait_warp(&sm->o_done[st], done & 1u, abort);
                        tc_fence_after();
                    }
                    tmem_st16(p_at + 16 * b, pk);
                }
                any = true;
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_st_wait();
                if (!ok) break;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm->p_full[st]);
            }
            if (!ok) break;
            // ---- the item's end: the last products, then the rows
            if (any) ok = mbar_wait_warp(&sm->o_done[st], (done - 1u) & 1u, abort);
            ok = ok && mbar_wait_warp(&sm->looked, segment & 1u, abort);
            if (!ok) break;
            tc_fence_after();
            // a row that sees a value which is not finite
            if (p.tree ? (mask & sm->odd_mask) != 0 : sm->odd_first < seen - cached) l = NAN;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm->noted);
            float f0 = 1.0f, f1 = 0.0f;                         // factors of the streams' sums
            uint32_t col = 0, cols = D;                         // columns that this thread writes
            const bool share = NS == 2 && !two;
            if (share) {
                sm->ml[st][0][r] = m;
                sm->ml[st][1][r] = l;
                tc_fence_before();
                sync_all();
                if (!ok) break;
                tc_fence_after();
                const float m0 = sm->ml[0][0][r], m1 = sm->ml[1][0][r], l0 = sm->ml[0][1][r], l1 = sm->ml[1][1][r];
                const float top = fmaxf(m0, m1);
                f0 = m0 == -INFINITY ? 0.0f : exp2f(m0 - top);
                f1 = m1 == -INFINITY ? 0.0f : exp2f(m1 - top);
                l = (m0 == -INFINITY ? l0 : l0 * f0) + (m1 == -INFINITY ? l1 : l1 * f1);
                m = top;
                cols = D / 2;
                col = (uint32_t)st * cols;
            }
            const bool both = share && w.count > 1u, whole = w.begins && w.ends;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const uint32_t slot_row = item_row - w.tile * Plan::kRows;
            float *slot = paged_slot(p, blockIdx.x, w.begins, Plan::kRows, D);
            if (!whole && live && col == 0) *reinterpret_cast<float2 *>(slot + 2 * slot_row) = make_float2(m, l);
            const uint32_t o0 = tmem + lanes + Plan::kOCol + (two ? (uint32_t)st * D : 0u);
            // whole rows go out turned in shared memory, 32 rows x 64 bytes at a time, so that four lanes write a row's 64 bytes instead of one lane
            // its 16: this lane writes rows 8 e + lane / 4 of the warp's 32
            uint4 *turn = sm->staging[warp], *to[4];
            float finite = 0.0f;                                // NaN once a value is not
            if (whole) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t row = row0 + 32u * (warp & 3) + 8u * e + (lane >> 2), t = row / p.group;
                    const uint64_t at = ((uint64_t)(w.q.n.token + t) * p.kv_heads + w.head) * p.group + (row - t * p.group);
                    to[e] = row < w.q.rows ? reinterpret_cast<uint4 *>(p.out + at * D) + (lane & 3) : nullptr;
                }
            }
#pragma unroll 1
            for (uint32_t c = col; c < col + cols; c += 32) {
                uint32_t a[32];
                tmem_ld32(o0 + c, a);
                if (both) {
                    uint32_t b[32];
                    tmem_ld32(o0 + D + c, b);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; ++e) a[e] = __float_as_uint(__uint_as_float(a[e]) * f0 + __uint_as_float(b[e]) * f1);
                } else {
                    tmem_ld_wait();
                    if (share) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) a[e] = __float_as_uint(__uint_as_float(a[e]) * f0);
                    }
                }
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t o[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float y0 = __uint_as_float(a[8 * e + 2 * x]) * inv, y1 = __uint_as_float(a[8 * e + 2 * x + 1]) * inv;
                            finite = fmaf(y0, 0.0f, finite);
                            finite = fmaf(y1, 0.0f, finite);
                            o[x] = close_means<T>(y0, y1);
                        }
                        turn[lane * 4 + (e ^ ((lane >> 1) & 3))] = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int q = 8 * e + (lane >> 2);
                        if (to[e]) to[e][c / 8] = turn[q * 4 + ((lane & 3) ^ ((q >> 1) & 3))];
                    }
                    __syncwarp();
                } else if (live) {
                    float4 *part = reinterpret_cast<float4 *>(slot + 2 * Plan::kRows) + (uint64_t)(c / 4) * Plan::kRows + slot_row;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        part[e * Plan::kRows] = make_float4(__uint_as_float(a[4 * e]), __uint_as_float(a[4 * e + 1]), __uint_as_float(a[4 * e + 2]), __uint_as_float(a[4 * e + 3]));
                }
            }
            bad_out |= live && finite != finite;
            if (tid == 0 && w.begins && !w.ends)
                p.share[blockIdx.x] = PagedShare{w.last_cta(start), (int32_t)rows, (int32_t)w.q.n.token, (int32_t)(w.head * p.group),
                                                 (int32_t)(w.tile * Plan::kRows), {0, 0, 0}};
            if (share) {                                        // either stream's sums may be written again
                tc_fence_before();
                sync_all();
            }
        }
        if (bad_out) raise(p.status, YVEX_B200_STATUS_NUMERIC);
    } else {
    set_registers<Plan::kControlRegs, Plan::kLaunched>();
    w.start(p, start);
    if (warp == Plan::kSoftmaxWarps) {
        // ---------------- TMA producer: a lane per box of a block ----------------
        const int boxes = BK / box_keys;
        const uint32_t nowhere = (uint32_t)(p.pages * p.kv_heads * p.page_size);      // a row past the cache: the box is filled with zeros
        const uint32_t groups = (uint32_t)box_keys / 16u, page_size = (uint32_t)p.page_size;
        bool ok = true, bad_page = false;
        uint32_t it = 0, k_asked = 0, v_asked = 0;
        for (; w.live() && ok; w.next(p)) {
            const uint32_t end = w.q.n.cached + w.q.n.fresh;
            const int32_t *table = p.block_table + (uint64_t)w.request * p.table_width;
            auto row_of = [&](uint32_t j, bool &none) -> uint32_t {      // where this lane's box of block j begins; none: no page holds it
                none = false;
                const uint32_t key = (w.first + j) * BK + (uint32_t)(lane * box_keys);
                if (lane >= boxes || j >= w.count || key >= end) return nowhere;
                const int32_t page = table[key / page_size];
                none = page < 0 || (uint64_t)page >= p.pages;
                return none ? nowhere : ((uint32_t)page * p.kv_heads + w.head) * page_size + key % page_size;
            };
            // K a block ahead of V, which waits for products that come later
            auto copy = [&](uint8_t *tiles, const CUtensorMap *map, uint32_t s, uint32_t y, uint64_t *full) {
                if (lane >= boxes) return;
                for (int h = 0; h < kHalves; ++h) tma_load_2d(tiles + s * kTileBytes + h * BK * 128 + lane * box_keys * 128, map, 64 * h, (int)y, full);
            };
            uint32_t y = 0;
            bool none;
            uint32_t y_next = row_of(0, none);
            for (uint32_t j = 0; j <= w.count && ok; ++j) {
                if (j < w.count) {                              // K of block j
                    const uint32_t at = it + j, s = at % kStages;
                    bad_page |= none;
                    const uint32_t bad = __reduce_or_sync(0xffffffffu, none ? ((1u << groups) - 1u) << (groups * lane) : 0u);
                    ok = mbar_wait_warp(&sm->k_empty[s], ((at / kStages) & 1u) ^ 1u, abort);
                    if (!ok) break;
                    if (lane == 0) { sm->bad_keys[at % Plan::kBadRing] = bad; mbar_expect_tx(&sm->k_full[s], kTileBytes); }
                    __syncwarp();
                    copy(k_tiles, &maps.k, s, y_next, &sm->k_full[s]);
                    k_asked = at + 1;
                }
                const uint32_t y_now = y_next;
                if (j < w.count) y_next = row_of(j + 1, none);
                if (j) {                                        // V of the block before
                    const uint32_t at = it + j - 1, s = at % kStages;
                    ok = mbar_wait_warp(&sm->v_empty[s], ((at / kStages) & 1u) ^ 1u, abort);
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&sm->v_full[s], kTileBytes);
                    __syncwarp();
                    copy(v_tiles, &maps.v, s, y, &sm->v_full[s]);
                    v_asked = at + 1;
                }
                y = y_now;
            }
            it += w.count;
        }
        if (bad_page) raise(p.status, YVEX_B200_STATUS_ARGUMENT);
        if (!ok && lane == 0) {
            // copies in flight must land before the CTA's shared memory is someone else's
            volatile int none = 0;
            for (uint32_t i = k_asked > kStages ? k_asked - kStages : 0; i < k_asked; ++i) mbar_wait(&sm->k_full[i % kStages], (i / kStages) & 1u, &none);
            for (uint32_t i = v_asked > kStages ? v_asked - kStages : 0; i < v_asked; ++i) mbar_wait(&sm->v_full[i % kStages], (i / kStages) & 1u, &none);
        }
        __syncwarp();
    } else if (warp == Plan::kSoftmaxWarps + 1) {
        // ---------------- S = Q K^T, block after block and stream after stream; one lane issues ----------------
        if (elect_one()) {
            constexpr uint32_t kIdesc = idesc_16bit(!kHalfType, false, BK);
            const uint64_t q0 = smem_desc_sw128(smem_u32(q_tiles)), k0 = smem_desc_sw128(smem_u32(k_tiles));
            uint32_t it = 0, segment = 0, used = 0, asked[2] = {0, 0};      // blocks, segments, S so far, S of a stream
            bool ok = true;
            for (; w.live() && ok; w.next(p), ++segment) {
                const bool two = NS == 2 && rows_of(w) > 128u;
                ok = mbar_wait(&sm->q_full, segment & 1u, abort);
                for (uint32_t j = 0; j < w.count && ok; ++j, ++it) {
                    const uint32_t s = it % kStages;
                    const uint64_t kd = k0 + s * (kTileBytes >> 4);
                    ok = mbar_wait(&sm->k_full[s], (it / kStages) & 1u, abort);
#pragma unroll
                    for (uint32_t st = 0; st < NS; ++st) {
                        if (!ok || (!two && NS == 2 && (j & 1u) != st)) continue;
                        const uint32_t n = asked[st]++, full = NS == 1 ? n & 1u : st, b = Plan::kSBuffers == 1 ? 0u : full;
                        // the buffer has been read since it was last used (every phase of a barrier is waited for in turn: parities tell no more)
                        const uint32_t uses = Plan::kSBuffers == 1 ? used : NS == 1 ? n >> 1 : n;
                        if (uses) ok = mbar_wait(&sm->s_free[b], (uses - 1u) & 1u, abort);
                        if (!ok) continue;
                        ++used;
                        tc_fence_after();
                        const uint64_t qd = q0 + (two ? st * (kQBytes >> 4) : 0u);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
                            umma_f16(tmem + b * BK, qd + (k >> 2) * (16384 >> 4) + 2 * (k & 3), kd + (k >> 2) * (BK * 128 >> 4) + 2 * (k & 3), kIdesc, k ? 1u : 0u);
                        umma_commit(&sm->s_full[full]);
                    }
                    if (ok) umma_commit(&sm->k_empty[s]);
                }
                if (ok) umma_commit(&sm->q_free);
            }
            if (!ok) {
                volatile int none = 0;
                umma_commit(&sm->drain[0]);                     // products in flight end before the tensor memory is freed
                mbar_wait(&sm->drain[0], 0u, &none);
            }
        }
    } else if (warp == Plan::kSoftmaxWarps + 2) {
        // ---------------- O += P V in the same order, behind the softmax; one lane issues ----------------
        if (elect_one()) {
            constexpr uint32_t kIdesc = idesc_16bit(!kHalfType, true, D);
            const uint64_t v0 = smem_desc_n_major_sw128(smem_u32(v_tiles), BK * 128);
            uint32_t it = 0, given[2] = {0, 0}, cleaned = 0;      // cleaned: the phase of each stage's barrier, a bit each
            bool ok = true;
            for (; w.live() && ok; w.next(p)) {
                const bool two = NS == 2 && rows_of(w) > 128u;
                const int safe = safe_keys(w);
                for (uint32_t j = 0; j < w.count && ok; ++j, ++it) {
                    const uint32_t s = it % kStages;
                    const uint64_t vd = v0 + s * (kTileBytes >> 4);
                    ok = mbar_wait(&sm->v_full[s], (it / kStages) & 1u, abort);
                    if (ok && (int)(w.first + j + 1) * BK > safe) {
                        ok = mbar_wait(&sm->v_clean[s], (cleaned >> s) & 1u, abort);
                        cleaned ^= 1u << s;
                    }
#pragma unroll
                    for (uint32_t st = 0; st < NS; ++st) {
                        if (!ok || (!two && NS == 2 && (j & 1u) != st)) continue;
                        ok = mbar_wait(&sm->p_full[st], given[st] & 1u, abort);
                        if (!ok) continue;
                        ++given[st];
                        tc_fence_after();
                        const uint32_t first = two || NS == 1 ? j : j >> 1;      // 0: the sums begin
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k)
                            umma_f16_ts(tmem + Plan::kOCol + st * D, tmem + Plan::kPCol + st * (BK / 2) + 8 * k, vd + k * (2048 >> 4), kIdesc, first || k ? 1u : 0u);
                        umma_commit(&sm->o_done[st]);
                    }
                    if (ok) umma_commit(&sm->v_empty[s]);
                }
            }
            if (!ok) {
                volatile int none = 0;
                umma_commit(&sm->drain[1]);
                mbar_wait(&sm->drain[1], 0u, &none);
            }
        }
    } else if (warp == Plan::kSoftmaxWarps + 3) {
        // ---------------- what comes once an item: values that are not finite, and the next item's Q ----------------
        // A weight of zero times an infinity would reach rows that do not see it. So in blocks that not every row sees to the end, values
        // that are not finite are taken out of the V tile before the products, and noted where they are a fresh token's: rows that see it become
        // NaN when the item ends. (The softmax warps did this for 8000 cycles a block, two joint waits among them.)
        bool ok = true;
        uint32_t it = 0, segment = 0;
        if (q_tokens && w.live() && lane == 0) load_q();
        while (w.live() && ok) {
            if (segment) ok = mbar_wait_warp(&sm->noted, (segment - 1u) & 1u, abort);      // the notes on the item before have been read
            if (!ok) break;
            const int cached = (int)w.q.n.cached, end = cached + (int)w.q.n.fresh, safe = safe_keys(w);
            if (lane == 0) { sm->odd_mask = 0ull; sm->odd_first = INT32_MAX; }
            __syncwarp();
            for (uint32_t j = 0; j < w.count && ok; ++j) {
                const uint32_t s = (it + j) % kStages;
                const int base = (int)(w.first + j) * BK;
                // (every tile is waited for and let go here too, so that none can be replaced unseen: a barrier's parity only tells a phase from the next)
                ok = mbar_wait_warp(&sm->v_full[s], ((it + j) / kStages) & 1u, abort);
                if (!ok) break;
                if (base + BK <= safe) {
                    if (lane == 0) mbar_arrive(&sm->v_empty[s]);
                    continue;
                }
                uint4 *tile = reinterpret_cast<uint4 *>(v_tiles + s * kTileBytes);
                // four keys of 128 bytes at a time, a half of D after the other: zeros behind the request's end; of the fresh tokens' values 0 times
                // each is summed, which is NaN once one is not finite
                const int stop = min(BK, max(end - base, 0));
                for (int h = 0; h < kHalves; ++h) {
                    uint4 *half = tile + h * BK * 8 + (lane & 7);
#pragma unroll 4
                    for (int key = stop + (lane >> 3); key < BK; key += 4) half[key * 8] = make_uint4(0, 0, 0, 0);
                    for (int key0 = max(safe - base, 0); key0 < stop; key0 += 32) {
                        typename PairOf<T>::type sum = pair_of<T>(0u);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int key = min(key0 + 4 * e + (lane >> 3), stop - 1);
                            const uint4 v = half[key * 8];
                            sum = __hfma2(pair_of<T>(v.x), pair_of<T>(0u), sum);
                            sum = __hfma2(pair_of<T>(v.y), pair_of<T>(0u), sum);
                            sum = __hfma2(pair_of<T>(v.z), pair_of<T>(0u), sum);
                            sum = __hfma2(pair_of<T>(v.w), pair_of<T>(0u), sum);
                        }
                        if (!odd_halves<T>(*reinterpret_cast<uint32_t *>(&sum))) continue;
                        for (int e = 0; e < 8; ++e) {
                            const int key = key0 + 4 * e + (lane >> 3), fresh = base + key - cached;
                            if (key >= stop) break;
                            const uint4 v = half[key * 8];
                            const uint4 o = make_uint4(odd_halves<T>(v.x), odd_halves<T>(v.y), odd_halves<T>(v.z), odd_halves<T>(v.w));
                            if (!(o.x | o.y | o.z | o.w)) continue;
                            half[key * 8] = make_uint4(without_halves(v.x, o.x), without_halves(v.y, o.y), without_halves(v.z, o.z), without_halves(v.w, o.w));
                            if (fresh < YVEX_B200_TREE_NODES) atomicOr(&sm->odd_mask, 1ull << fresh);
                            atomicMin(&sm->odd_first, fresh);
                        }
                    }
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) { mbar_arrive(&sm->v_clean[s]); mbar_arrive(&sm->v_empty[s]); }
            }
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(&sm->looked);
            it += w.count;
            w.next(p);
            if (!ok || !w.live()) break;
            ok = mbar_wait_warp(&sm->q_free, segment & 1u, abort);
            if (!ok) break;
            if (q_tokens) {
                if (lane == 0) load_q();
            } else {
                copy_q(0, 1);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm->q_full);
            }
            ++segment;
        }
        if (!ok && lane == 0 && q_tokens) {                     // Q in flight must land before the CTA ends
            volatile int none = 0;
            mbar_wait(&sm->q_full, segment & 1u, &none, 1000000ull);
        }
        __syncwarp();
    }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && sm->abort) raise(p.status, YVEX_B200_STATUS_TIMEOUT);
    if (warp == 0) tmem_dealloc(tmem, kTilesTmem);
}

static PFN_cuTensorMapEncodeTiled_v12000 tiles_encode() {
    static std::atomic<void *> found{nullptr};
    void *p = found.load(std::memory_order_acquire);
    if (!p) {
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
        found.store(p, std::memory_order_release);
    }
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
}

// One side of the cache as rows of head_dim values -> boxes of [box_keys rows][64 values], 128-byte swizzle, zeros past the last row.
static int pages_map(CUtensorMap *map, const uint16_t *base, const PagedParams &p, unsigned qtype, uint64_t head_dim, int box_keys) {
    auto fn = tiles_encode();
    if (!fn) return ERR_BACKEND;
    cuuint64_t dims[2] = {head_dim, p.pages * p.kv_heads * p.page_size}, strides[1] = {head_dim * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_keys}, estr[2] = {1, 1};
    const CUresult r = fn(map, qtype == Q_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<uint16_t *>(base), dims,
                          strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? OK : ERR_BACKEND;
}

static int rows_map(CUtensorMap *map, const PagedParams &p, unsigned qtype, uint64_t head_dim) {
    auto fn = tiles_encode();
    if (!fn) return ERR_BACKEND;
    cuuint64_t dims[3] = {head_dim, (cuuint64_t)p.kv_heads * p.group, p.tokens}, strides[2] = {head_dim * 2, p.q_stride * 2};
    cuuint32_t box[3] = {64, p.group, 128 / p.group}, estr[3] = {1, 1, 1};
    const CUresult r = fn(map, qtype == Q_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<uint16_t *>(p.q), dims,
                          strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? OK : ERR_BACKEND;
}

template <class T, int D> static int launch_tiles(const PagedParams &p, unsigned qtype, unsigned ctas, cudaStream_t s) {
    using Plan = TilePlan<D>;
    static SmemOptIn optin;
    constexpr size_t smem = Plan::kStreams * Plan::kQBytes + 2 * Plan::kStages * Plan::kTileBytes + sizeof(TileSmem<D>);
    static_assert(smem <= 227 * 1024, "shared memory plan exceeds the 227 KiB a CTA can have");
    const int rc = optin.ensure(paged_tiles_kernel<T, D>, (int)smem);
    if (rc != OK) return rc;
    int box = 16;                                               // a box stays within a page
    while (box < Plan::kKeys && p.page_size % (2u * box) == 0) box *= 2;
    TileMaps maps;
    const int q_tokens = p.group <= 128 && 128 % p.group == 0 ? (int)(128 / p.group) : 0;
    if (q_tokens && rows_map(&maps.q, p, qtype, D) != OK) return ERR_BACKEND;
    if (pages_map(&maps.k, p.k, p, qtype, D, box) != OK || pages_map(&maps.v, p.v, p, qtype, D, box) != OK) return ERR_BACKEND;
    if (launch_pdl(paged_tiles_kernel<T, D>, dim3(ctas), dim3(Plan::kThreads), smem, s, maps, p, box, q_tokens) != cudaSuccess) return ERR_BACKEND;
    return OK;
}

int launch_paged_tiles(const PagedParams &p, unsigned qtype, uint64_t head_dim, unsigned ctas, cudaStream_t s) {
    const bool bf = qtype == Q_BF16;
    switch (head_dim) {
    case 64: return bf ? launch_tiles<__nv_bfloat16, 64>(p, qtype, ctas, s) : launch_tiles<__half, 64>(p, qtype, ctas, s);
    case 128: return bf ? launch_tiles<__nv_bfloat16, 128>(p, qtype, ctas, s) : launch_tiles<__half, 128>(p, qtype, ctas, s);
    default: return bf ? launch_tiles<__nv_bfloat16, 256>(p, qtype, ctas, s) : launch_tiles<__half, 256>(p, qtype, ctas, s);
    }
}

}  // namespace yb
