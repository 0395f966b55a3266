// Attention of many rows per (request, kv head) over the paged cache - drafted trees, chunks of prompts - on tcgen05.
//
// Keys and values come page by page by TMA, straight from where they lie (boxes of as many rows as a page's size allows, up to the 128
// keys of a block), scores and the output's sums live in tensor memory, and a thread of the softmax warps owns a row, so its
// maximum and sum need no shuffles. S = Q K^T reads both operands from shared memory; P replaces S in tensor memory, rounded once to the
// cache's type, and is the A operand of O += P V, whose B is the V tile as it lies (N-major). Two streams of softmax warps, each with scores and
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
    static constexpr uint32_t kOCol = kStreams == 2 ? 256 : 64;                          // columns: S of stream 0, S of stream 1, O of each
    static constexpr uint32_t kSPitch = 128, kBadRing = 8;
};
constexpr uint32_t kTilesTmem = 512;

template <int D> struct TileSmem {
    using Plan = TilePlan<D>;
    uint64_t q_full, k_full[Plan::kStages], k_empty[Plan::kStages], v_full[Plan::kStages], v_empty[Plan::kStages];
    uint64_t s_full[2], p_full[2], o_done[2], all, own[2], drain;
    uint64_t scan[Plan::kThreads / 32 + 4];
    float ml[2][2][128];
    uint32_t odd[3][2][4];                       // by stream, or of both
    uint32_t bad_keys[Plan::kBadRing];
    uint32_t tmem_base;
    int abort;
};

struct TileMaps { CUtensorMap k, v; };

// exp2 of a score's distance; the softmax's only transcendental
__device__ __forceinline__ float weight_of(float x) { return exp2f(x); }

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
        mbar_init(&sm->q_full, Plan::kSoftmaxWarps);
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sm->k_full[i], 1); mbar_init(&sm->k_empty[i], 1);
            mbar_init(&sm->v_full[i], 1); mbar_init(&sm->v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) { mbar_init(&sm->s_full[i], 1); mbar_init(&sm->p_full[i], 4); mbar_init(&sm->o_done[i], 1); mbar_init(&sm->own[i], 4); }
        mbar_init(&sm->all, Plan::kSoftmaxWarps);
        mbar_init(&sm->drain, 1);
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
    const PagedStart start = paged_start<Plan::kThreads, Plan::kRows, BK>(p, sm->scan);
    PagedWalk<Plan::kRows, BK> w;
    w.start(p, start);

    // An item of more rows than a stream has is two tiles over the same keys, otherwise the streams take turns with the blocks of keys.
    auto rows_of = [&]() { return min(w.q.rows - w.tile * Plan::kRows, (uint32_t)Plan::kRows); };

    if (warp < Plan::kSoftmaxWarps) {
        // ---------------- softmax: thread = row of a stream's tile ----------------
        set_registers<Plan::kSoftmaxRegs, Plan::kLaunched>();
        const int st = warp >> 2, r = tid & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s_at = tmem + lanes + (uint32_t)st * Plan::kSPitch, o_at = tmem + lanes + Plan::kOCol + (uint32_t)st * D;
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
        for (; w.live() && ok; it_base += w.count, w.next(p)) {
            const uint32_t rows = rows_of();
            const bool two = NS == 2 && rows > 128u;            // two tiles of rows
            const uint32_t item_row = w.tile * Plan::kRows + (two ? 128u * st : 0u) + r;
            const bool live = item_row < w.q.rows;
            const uint32_t token = item_row / p.group;
            // ---- Q into shared memory, K-major with the 128-byte swizzle; one tile shared by both streams is written half by half of its dims
            {
                const uint16_t *src = p.q + (uint64_t)(w.q.n.token + token) * p.q_stride + ((uint64_t)w.head * p.group + item_row % p.group) * D;
                uint8_t *dst = q_tiles + (two ? st * kQBytes : 0u);
                const int chunks = NS == 2 && !two ? D / 16 : D / 8, c0 = NS == 2 && !two ? st * (D / 16) : 0;
#pragma unroll 4
                for (int i = 0; i < chunks; ++i) {
                    const int ch = c0 + i;
                    const uint4 v = live ? __ldg(reinterpret_cast<const uint4 *>(src) + ch) : make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4 *>(dst + (ch >> 3) * 16384 + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm->q_full);
            }
            const int64_t cached = w.q.n.cached, end = cached + w.q.n.fresh, seen = live ? cached + token + 1 : cached;
            const uint64_t mask = p.tree && live ? p.ancestors[w.q.n.token + token] : 0ull;
            const int64_t safe = p.tree ? cached : cached + (w.tile * Plan::kRows) / p.group + 1;      // keys before it are seen by every row
            const uint32_t stride = two ? 1u : NS, begin = two ? 0u : (uint32_t)st;
            float m = -INFINITY, l = 0.0f;
            bool any = false;
            for (uint32_t j = begin; j < w.count && ok; j += stride) {
                const uint32_t it = it_base + j;
                const int64_t base = (int64_t)(w.first + j) * BK;
                ok = mbar_wait_warp(&sm->s_full[st], done & 1u, abort);
                if (!ok) break;
                ++done;
                tc_fence_after();
                float s[BK];
#pragma unroll
                for (int i = 0; i < BK / 32; ++i) tmem_ld32(s_at + 32 * i, reinterpret_cast<uint32_t *>(s) + 32 * i);
                tmem_ld_wait();
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
                        ok = mbar_wait_warp(&sm->v_full[it % kStages], (it / kStages) & 1u, abort);
                        if (two) sync_all(); else sync_own();
                        if (ok) {
                            uint8_t *tile = v_tiles + (it % kStages) * kTileBytes;
                            for (int i = at; i < (int)(kTileBytes / 16); i += threads) {
                                const int key = (i >> 3) % BK;
                                if (base + key < cached) continue;
                                uint4 *x = reinterpret_cast<uint4 *>(tile) + i;
                                uint4 v = *x;
                                if (base + key >= end) {
                                    *x = make_uint4(0, 0, 0, 0);
                                } else {
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
                float t0 = s[0], t1 = s[1], t2 = s[2], t3 = s[3];
#pragma unroll
                for (int i = 4; i < BK; i += 4) { t0 = fmaxf(t0, s[i]); t1 = fmaxf(t1, s[i + 1]); t2 = fmaxf(t2, s[i + 2]); t3 = fmaxf(t3, s[i + 3]); }
                const float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)) * scale;
                float f = 1.0f;
                if (m == -INFINITY) m = top;                    // nothing seen so far: O is zero
                else if (top > m + kSlack) { f = exp2f(m - top); m = top; }
                if (any && __any_sync(0xffffffffu, f != 1.0f)) {
                    // (the scores that were just read came behind the products of the block before: O is complete)
                    l *= f;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) {
                        uint32_t o[32];
                        tmem_ld32(o_at + 32 * i, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_st32(o_at + 32 * i, o);
                    }
                }
                any = true;
                // ---- weights, their sum, and P over S
                const float shift = (m == -INFINITY ? 0.0f : m) - kLift;
                float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
                for (int b = 0; b < BK / 64; ++b) {
                    uint32_t pk[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float x = weight_of(fmaf(s[64 * b + 2 * i], scale, -shift)), y = weight_of(fmaf(s[64 * b + 2 * i + 1], scale, -shift));
                        l0 += x;
                        l1 += y;
                        pk[i] = close2<T>(x, y);
                    }
                    tmem_st32(s_at + 32 * b, pk);
                }
                l += l0 + l1;
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
            float *slot = p.partial + (2ull * blockIdx.x + (w.begins ? 1 : 0)) * Plan::kRows * (D + 2);
            if (!whole && live && col == 0) *reinterpret_cast<float2 *>(slot + 2 * slot_row) = make_float2(m, l);
            const uint32_t o0 = tmem + lanes + Plan::kOCol + (two ? (uint32_t)st * D : 0u);
            uint16_t *out = p.out + ((uint64_t)(w.q.n.token + token) * p.kv_heads * p.group + (uint64_t)w.head * p.group + item_row % p.group) * D;
            float *part = slot + 2 * Plan::kRows + (uint64_t)slot_row * D;
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
                if (!live) continue;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t o[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const float y0 = __uint_as_float(a[e + 2 * x]) * inv, y1 = __uint_as_float(a[e + 2 * x + 1]) * inv;
                            bad_out |= !isfinite(y0) || !isfinite(y1);
                            o[x] = close2<T>(y0, y1);
                        }
                        *reinterpret_cast<uint4 *>(out + c + e) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 2) *reinterpret_cast<float2 *>(part + c + e) = make_float2(__uint_as_float(a[e]), __uint_as_float(a[e + 1]));
                }
            }
            if (tid == 0 && w.begins && !w.ends)
                p.share[blockIdx.x] = PagedShare{w.last_cta(start), (int32_t)rows, (int32_t)w.q.n.token, (int32_t)(w.head * p.group),
                                                 (int32_t)(w.tile * Plan::kRows), {0, 0, 0}};
            tc_fence_before();
            sync_all();                                         // Q and the sums may be written again
            tc_fence_after();
        }
        if (bad_out) raise(p.status, YVEX_B200_STATUS_NUMERIC);
    } else {
    set_registers<Plan::kControlRegs, Plan::kLaunched>();
    if (warp == Plan::kSoftmaxWarps) {
        // ---------------- TMA producer: a lane per box of a block ----------------
        const int boxes = BK / box_keys;
        const uint32_t nowhere = (uint32_t)(p.pages * p.kv_heads * p.page_size);      // a row past the cache: the box is filled with zeros
        const uint32_t groups = (uint32_t)box_keys / 16u, page_size = (uint32_t)p.page_size;
        bool ok = true, bad_page = false;
        uint32_t it = 0;
        for (; w.live() && ok; w.next(p)) {
            const int64_t end = (int64_t)w.q.n.cached + w.q.n.fresh;
            const int32_t *table = p.block_table + (uint64_t)w.request * p.table_width;
            auto row_of = [&](uint32_t j, bool &none) -> uint32_t {      // where this lane's box of block j begins; none: no page holds it
                none = false;
                if (lane >= boxes || j >= w.count) return nowhere;
                const int64_t key = (int64_t)(w.first + j) * BK + (int64_t)lane * box_keys;
                if (key >= end) return nowhere;
                const int32_t page = __ldg(table + (uint32_t)key / page_size);
                none = page < 0 || (uint64_t)page >= p.pages;
                return none ? nowhere : ((uint32_t)page * p.kv_heads + w.head) * page_size + (uint32_t)key % page_size;
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
            for (uint32_t i = it >= kStages ? it - kStages : 0; i < it; ++i) {
                mbar_wait(&sm->k_full[i % kStages], (i / kStages) & 1u, &none);
                mbar_wait(&sm->v_full[i % kStages], (i / kStages) & 1u, &none);
            }
            mbar_wait(&sm->k_full[it % kStages], (it / kStages) & 1u, &none, 1000000ull);      // (a K tile whose V was not asked for)
        }
        __syncwarp();
    } else if (warp == Plan::kSoftmaxWarps + 1 && elect_one()) {
        // ---------------- MMA issuer: whichever stream is ready ----------------
        constexpr uint32_t kIdescS = idesc_16bit(!kHalfType, false, BK), kIdescO = idesc_16bit(!kHalfType, true, D);
        const uint64_t q0 = smem_desc_sw128(smem_u32(q_tiles)), k0 = smem_desc_sw128(smem_u32(k_tiles));
        const uint64_t v0 = smem_desc_n_major_sw128(smem_u32(v_tiles), BK * 128);
        uint32_t it_base = 0, segment = 0, asked[2] = {0, 0}, given[2] = {0, 0};      // S and PV issued per stream so far
        bool ok = true;
        for (; w.live() && ok; it_base += w.count, w.next(p), ++segment) {
            const bool two = NS == 2 && rows_of() > 128u;
            ok = mbar_wait(&sm->q_full, segment & 1u, abort);
            if (!ok) break;
            uint32_t n[2], s_i[2] = {0, 0}, v_i[2] = {0, 0};
            n[0] = two || NS == 1 ? w.count : (w.count + 1) / 2;
            n[1] = NS == 1 ? 0 : two ? w.count : w.count / 2;
            const uint32_t stride = two || NS == 1 ? 1u : 2u;
            uint64_t t0 = 0;
            uint32_t idle = 0;
            while (v_i[0] < n[0] || v_i[1] < n[1]) {
                bool moved = false;
#pragma unroll
                for (int st = 0; st < NS; ++st) {
                    if (s_i[st] == v_i[st]) {
                        if (s_i[st] == n[st]) continue;
                        // S of the stream's next block: its P of the block before has been used, the keys are there
                        const uint32_t it = it_base + (two ? s_i[st] : s_i[st] * stride + st), s = it % kStages;
                        if (given[st] && !mbar_try_wait(&sm->o_done[st], (given[st] - 1u) & 1u)) continue;
                        if (!mbar_try_wait(&sm->k_full[s], (it / kStages) & 1u)) continue;
                        tc_fence_after();
                        const uint64_t qd = q0 + (two ? st * (kQBytes >> 4) : 0u), kd = k0 + s * (kTileBytes >> 4);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
                            umma_f16(tmem + st * Plan::kSPitch, qd + (k >> 2) * (16384 >> 4) + 2 * (k & 3), kd + (k >> 2) * (BK * 128 >> 4) + 2 * (k & 3), kIdescS, k ? 1u : 0u);
                        umma_commit(&sm->s_full[st]);
                        ++s_i[st];
                        ++asked[st];
                        if (!two || s_i[st ^ 1] >= s_i[st]) umma_commit(&sm->k_empty[s]);
                        moved = true;
                    } else {
                        // O += P V of the stream's block
                        const uint32_t it = it_base + (two ? v_i[st] : v_i[st] * stride + st), s = it % kStages;
                        if (!mbar_try_wait(&sm->p_full[st], (asked[st] - 1u) & 1u) || !mbar_try_wait(&sm->v_full[s], (it / kStages) & 1u)) continue;
                        tc_fence_after();
                        const uint64_t vd = v0 + s * (kTileBytes >> 4);
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k)
                            umma_f16_ts(tmem + Plan::kOCol + st * D, tmem + st * Plan::kSPitch + 8 * k, vd + k * (2048 >> 4), kIdescO, v_i[st] | k ? 1u : 0u);
                        umma_commit(&sm->o_done[st]);
                        ++v_i[st];
                        ++given[st];
                        if (!two || v_i[st ^ 1] >= v_i[st]) umma_commit(&sm->v_empty[s]);
                        moved = true;
                    }
                }
                if (moved) { idle = 0; t0 = 0; continue; }
                if ((++idle & 63u) == 0u) {                     // bounded like every wait
                    const uint64_t now = global_ns();
                    if (*abort || (t0 && now - t0 > kWaitLimitNs)) { *abort = 1; ok = false; break; }
                    if (!t0) t0 = now;
                }
            }
        }
        if (!ok) {
            volatile int none = 0;
            umma_commit(&sm->drain);                            // products in flight end before the tensor memory is freed
            mbar_wait(&sm->drain, 0u, &none);
        }
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
