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
// weight of up to 2^kSlack costs no precision in f32 sums. f16 weights are lifted by 2^10 so that small ones do not
// become subnormal, and follow the maximum sooner.
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
    uint64_t s_full[2], s_free[2], p_full[2], o_done[2], all, own[2], drain[2];
    PagedScratch<Plan::kThreads> scan;
    float ml[2][2][128];
    uint32_t odd[3][2][4];                       // by stream, or of both
    uint32_t bad_keys[Plan::kBadRing];
    uint32_t tmem_base;
    int abort;
};

struct TileMaps { CUtensorMap k, v; };

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
// 16 bytes global -> shared that complete with the thread's group of copies; zeros where `live` is false
__device__ __forceinline__ void copy16(void *dst, const void *src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(sm100::smem_u32(dst)), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <class T, int D>
__global__ void __launch_bounds__(TilePlan<D>::kThreads, 1) paged_tiles_kernel(const __grid_constant__ TileMaps maps, const PagedParams p, const int box_keys) {
    using namespace sm100;
    using Plan = TilePlan<D>;
    constexpr int BK = Plan::kKeys, NS = Plan::kStreams, kStages = Plan::kStages, kHalves = D / 64;
    constexpr uint32_t kTileBytes = Plan::kTileBytes, kQBytes = Plan::kQBytes;
    constexpr bool kHalfType = std::is_same<T, __half>::value;
    constexpr float kLift = kHalfType ? 10.0f : 0.0f, kSlack = kHalfType ? 4.0f : 8.0f;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    if (smem_u32(smem_raw) & 1023u) {                           // uniform: nothing has been set up yet
        pdl_wait();
        if (threadIdx.x == 0) raise(p.status, YVEX_B200_STATUS_TIMEOUT);
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
            mbar_init(&sm->v_full[i], 1); mbar_init(&sm->v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sm->s_full[i], 1); mbar_init(&sm->s_free[i], 4); mbar_init(&sm->p_full[i], 4); mbar_init(&sm->o_done[i], 1);
            mbar_init(&sm->own[i], 4); mbar_init(&sm->drain[i], 1);
        }
        mbar_init(&sm->all, Plan::kSoftmaxWarps);
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
    auto rows_of = [](const Walk &w) { return min(w.q.rows - w.tile * Plan::kRows, (uint32_t)Plan::kRows); };
    Walk w;

    if (warp < Plan::kSoftmaxWarps) {
        // ---------------- softmax: thread = row of a stream's tile ----------------
        set_registers<Plan::kSoftmaxRegs, Plan::kLaunched>();
        const int st = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t p_at = tmem + lanes + Plan::kPCol + (uint32_t)st * (BK / 2), o_at = tmem + lanes + Plan::kOCol + (uint32_t)st * D;
        const float scale = p.scale * 1.4426950408889634f;      // scores in powers of two
        uint32_t done = 0, all_ph = 0, own_ph = 0, odd_own = 0, odd_all = 0, it_base = 0;
        bool ok = true, bad_out = false;
        if (tid == 0) p.share[blockIdx.x].rows = 0;
        auto sync_all = [&]() {                                 // every softmax thread of the CTA; bounded like every wait
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm->all);
            ok = ok && mbar_wait_warp(&sm->all, all_ph, abort);
            all_ph ^= 1u;
        };
        auto sync_own = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm->own[st]);
            ok = ok && mbar_wait_warp(&sm->own[st], own_ph, abort);
            own_ph ^= 1u;
        };
        for (w.start(p, start); w.live() && ok; it_base += w.count, w.next(p)) {
            const uint32_t rows = rows_of(w);
            const bool two = NS == 2 && rows > 128u;            // two tiles of rows
            const uint32_t row0 = w.tile * Plan::kRows + (two ? 128u * st : 0u), item_row = row0 + r;
            const bool live = item_row < w.q.rows;
            const uint32_t token = item_row / p.group;
            const int cached = (int)w.q.n.cached, end = cached + (int)w.q.n.fresh, seen = live ? cached + (int)token + 1 : cached;
            const uint64_t mask = p.tree && live ? p.ancestors[w.q.n.token + token] : 0ull;
            const int safe = p.tree ? cached : cached + (int)(w.tile * Plan::kRows / p.group) + 1;      // keys before it are seen by every row
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
                    // ---- keys that not every row sees
                    uint32_t sees[BK / 32], odd[BK / 32];
#pragma unroll
                    for (int i = 0; i < BK / 64; ++i) {
                        const uint64_t x = paged_sees(p.tree, base + 64 * i, cached, seen, mask) & low_bits(end - base - 64 * i);
                        sees[2 * i] = (uint32_t)x;
                        sees[2 * i + 1] = (uint32_t)(x >> 32);
                    }
#pragma unroll
                    for (int i = 0; i < BK / 32; ++i) {
                        const uint32_t b2 = (bad >> (2 * i)) & 3u;
                        sees[i] &= ~((b2 & 1u ? 0xffffu : 0u) | (b2 & 2u ? 0xffff0000u : 0u));
                        odd[i] = 0;
                    }
                    if (base + BK > safe) {
                        // A weight of zero times an infinity would reach rows that do not see it, so such values (and whatever lies behind the
                        // request's end) are taken out of the V tile, and rows that see one of the former are marked. Both streams of an item of two tiles
                        // read the tile: they clean it together.
                        uint32_t *found = two ? sm->odd[2][odd_all] : sm->odd[st][odd_own];
                        const int threads = two ? 256 : 128, at = two ? tid : r;
                        if (two) odd_all ^= 1u; else odd_own ^= 1u;
                        if (at < 4) found[at] = 0u;
                        // (the products of the block before have read theirs, so the tile's barrier is in this block's phase)
                        if (any) ok = mbar_wait_warp(&sm->o_done[st], done & 1u, abort);
                        ok = ok && mbar_wait_warp(&sm->v_full[it % kStages], (it / kStages) & 1u, abort);
                        if (two) sync_all(); else sync_own();
                        if (ok) {
                            uint8_t *tile = v_tiles + (it % kStages) * kTileBytes;
#pragma unroll 4
                            for (int i = at; i < (int)(kTileBytes / 16); i += threads) {
                                const int key = (i >> 3) % BK;
                                if (base + key < cached) continue;
                                uint4 *x = reinterpret_cast<uint4 *>(tile) + i;
                                if (base + key >= end) {
                                    *x = make_uint4(0, 0, 0, 0);
                                } else {
                                    const uint4 v = *x;
                                    const uint32_t a = odd_halves<T>(v.x), b = odd_halves<T>(v.y), c = odd_halves<T>(v.z), d = odd_halves<T>(v.w);
                                    if (a | b | c | d) {
                                        atomicOr(&found[key >> 5], 1u << (key & 31));
                                        *x = make_uint4(without_halves(v.x, a), without_halves(v.y, b), without_halves(v.z, c), without_halves(v.w, d));
                                    }
                                }
                            }
                        }
                        fence_proxy_async();
                        if (two) sync_all(); else sync_own();
                        if (!ok) break;
#pragma unroll
                        for (int i = 0; i < BK / 32; ++i) odd[i] = found[i];
                    }
#pragma unroll
                    for (int i = 0; i < BK; ++i) s[i] = (sees[i >> 5] >> (i & 31)) & 1u ? s[i] : -INFINITY;
#pragma unroll
                    for (int i = 0; i < BK / 32; ++i) if (odd[i] & sees[i]) l = NAN;
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
                if (any) {                                      // the products of the block before: P may be written, O is complete
                    ok = mbar_wait_warp(&sm->o_done[st], done & 1u, abort);
                    if (!ok) break;
                    tc_fence_after();
                    if (__any_sync(0xffffffffu, f != 1.0f)) {
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
                }
                any = true;
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
                    tmem_st16(p_at + 16 * b, pk);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm->p_full[st]);
            }
            if (!ok) break;
            // ---- the item's end: the last products, then the rows
            if (any) {
                ok = mbar_wait_warp(&sm->o_done[st], (done - 1u) & 1u, abort);
                if (!ok) break;
                tc_fence_after();
            }
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
            const uint64_t heads = (uint64_t)p.kv_heads * p.group;
            uint4 *turn = sm->staging[warp];
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
                    // 32 rows x 64 bytes turned in shared memory, so that four lanes write a row's 64 bytes instead of one lane its 16
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t o[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float y0 = __uint_as_float(a[8 * e + 2 * x]) * inv, y1 = __uint_as_float(a[8 * e + 2 * x + 1]) * inv;
                            bad_out |= live && (!isfinite(y0) || !isfinite(y1));
                            o[x] = close2<T>(y0, y1);
                        }
                        turn[lane * 4 + (e ^ ((lane >> 1) & 3))] = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int q = 8 * e + (lane >> 2);
                        const uint32_t row = row0 + 32u * (warp & 3) + q;
                        const uint4 x = turn[q * 4 + ((lane & 3) ^ ((q >> 1) & 3))];
                        if (row < w.q.rows)
                            *reinterpret_cast<uint4 *>(p.out + ((w.q.n.token + row / p.group) * heads + (uint64_t)w.head * p.group + row % p.group) * D + c + 8 * (lane & 3)) = x;
                    }
                    __syncwarp();
                } else if (live) {
                    float4 *part = reinterpret_cast<float4 *>(slot + 2 * Plan::kRows) + (uint64_t)(c / 4) * Plan::kRows + slot_row;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        part[e * Plan::kRows] = make_float4(__uint_as_float(a[4 * e]), __uint_as_float(a[4 * e + 1]), __uint_as_float(a[4 * e + 2]), __uint_as_float(a[4 * e + 3]));
                }
            }
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
        uint32_t it = 0, k_asked = 0;
        for (; w.live() && ok; w.next(p)) {
            const uint32_t end = w.q.n.cached + w.q.n.fresh;
            const int32_t *table = p.block_table + (uint64_t)w.request * p.table_width;
            auto row_of = [&](uint32_t j, bool &none) -> uint32_t {      // where this lane's box of block j begins; none: no page holds it
                none = false;
                const uint32_t key = (w.first + j) * BK + (uint32_t)(lane * box_keys);
                if (lane >= boxes || j >= w.count || key >= end) return nowhere;
                const int32_t page = __ldg(table + key / page_size);
                none = page < 0 || (uint64_t)page >= p.pages;
                return none ? nowhere : ((uint32_t)page * p.kv_heads + w.head) * page_size + key % page_size;
            };
            bool none, none_next;
            uint32_t y = row_of(0, none);
            for (uint32_t j = 0; j < w.count && ok; ++j, ++it) {
                const uint32_t y_next = row_of(j + 1, none_next), s = it % kStages, ph = (it / kStages) & 1u;
                bad_page |= none;
                const uint32_t bad = __reduce_or_sync(0xffffffffu, none ? ((1u << groups) - 1u) << (groups * lane) : 0u);
                ok = mbar_wait_warp(&sm->k_empty[s], ph ^ 1u, abort);
                if (!ok) break;
                if (lane == 0) { sm->bad_keys[it % Plan::kBadRing] = bad; mbar_expect_tx(&sm->k_full[s], kTileBytes); }
                __syncwarp();
                if (lane < boxes)
                    for (int h = 0; h < kHalves; ++h)
                        tma_load_2d(k_tiles + s * kTileBytes + h * BK * 128 + lane * box_keys * 128, &maps.k, 64 * h, (int)y, &sm->k_full[s]);
                k_asked = it + 1;
                ok = mbar_wait_warp(&sm->v_empty[s], ph ^ 1u, abort);
                if (!ok) break;
                if (lane == 0) mbar_expect_tx(&sm->v_full[s], kTileBytes);
                __syncwarp();
                if (lane < boxes)
                    for (int h = 0; h < kHalves; ++h)
                        tma_load_2d(v_tiles + s * kTileBytes + h * BK * 128 + lane * box_keys * 128, &maps.v, 64 * h, (int)y, &sm->v_full[s]);
                y = y_next;
                none = none_next;
            }
        }
        if (bad_page) raise(p.status, YVEX_B200_STATUS_ARGUMENT);
        if (!ok && lane == 0) {
            // copies in flight must land before the CTA's shared memory is someone else's
            volatile int none = 0;
            for (uint32_t i = k_asked > kStages ? k_asked - kStages : 0; i < k_asked; ++i) mbar_wait(&sm->k_full[i % kStages], (i / kStages) & 1u, &none);
            for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i) mbar_wait(&sm->v_full[i % kStages], (i / kStages) & 1u, &none);
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
            uint32_t it = 0, given[2] = {0, 0};
            bool ok = true;
            for (; w.live() && ok; w.next(p)) {
                const bool two = NS == 2 && rows_of(w) > 128u;
                for (uint32_t j = 0; j < w.count && ok; ++j, ++it) {
                    const uint32_t s = it % kStages;
                    const uint64_t vd = v0 + s * (kTileBytes >> 4);
                    ok = mbar_wait(&sm->v_full[s], (it / kStages) & 1u, abort);
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
        // ---------------- Q: rows of an item while the one before is being finished, K-major with the 128-byte swizzle ----------------
        constexpr int kLanes = D / 8, kAt = 32 / kLanes;         // lanes of a row, rows at a time
        const uint32_t chunk = (uint32_t)lane % kLanes;
        bool ok = true;
        for (uint32_t segment = 0; w.live() && ok; w.next(p), ++segment) {
            if (segment) ok = mbar_wait_warp(&sm->q_free, (segment - 1u) & 1u, abort);
            if (!ok) break;
            const uint32_t rows = rows_of(w), tiles = NS == 2 && rows > 128u ? 2u : 1u;
#pragma unroll 4
            for (uint32_t row = (uint32_t)lane / kLanes; row < 128u * tiles; row += kAt) {
                const bool live = row < rows;
                const uint32_t at = live ? w.tile * Plan::kRows + row : 0u, token = at / p.group;
                const uint16_t *src = p.q + (uint64_t)(w.q.n.token + token) * p.q_stride + ((uint64_t)w.head * p.group + at % p.group) * D + 8 * chunk;
                const uint32_t rr = row & 127u;
                copy16(q_tiles + (row >> 7) * kQBytes + (chunk >> 3) * 16384 + rr * 128 + (((chunk & 7u) ^ (rr & 7u)) << 4), src, live);
            }
            copies_done();
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm->q_full);
        }
        copies_done();
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
    if (pages_map(&maps.k, p.k, p, qtype, D, box) != OK || pages_map(&maps.v, p.v, p, qtype, D, box) != OK) return ERR_BACKEND;
    if (launch_pdl(paged_tiles_kernel<T, D>, dim3(ctas), dim3(Plan::kThreads), smem, s, maps, p, box) != cudaSuccess) return ERR_BACKEND;
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
