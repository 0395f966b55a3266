// Attention of a step's fresh tokens over the paged cache: softmax(scale q K^T) V with one running maximum and sum per row.
//
// Few rows per (request, kv head) - one token of a group of query heads, a short chain -: bound by HBM, the cache is read once and
// the products hide behind it. Like the contiguous decode kernel, a warp takes 16 keys at a time and does both products on
// mma.sync m16n8k16 with operands built from 16-byte loads as they lie in memory (the k-slots of S are whatever dims, those
// of PV whatever keys a lane holds), so nothing is staged or transposed. 16 keys never straddle a page, and the page
// of a warp's next block is looked up while this one is computed. The weights are rounded once to the cache's type for the second product,
// which adds less to the output's error than its own rounding (an output of f32 would not allow that); their sum stays f32 and unrounded. f16
// weights are lifted by 2^15 before, and their sums with them, so that those down to 2^-29 of the largest keep all their bits and smaller ones are off by at
// most 2^-40 of it: of a million keys that is 2^-20 (unlifted, the many small weights beside one large key were lost: 2^-25 each).
// 64 sessions of 100 to 32768 keys (3.46 GB): 562 us, 6.15 TB/s, 94 % of the copy bandwidth, and 581 us (91 %) with three sets of inputs in rotation,
// at 1740 MHz under the power cap; equal shares of blocks instead of a fixed number of slices per session are what holds that for ragged lengths.
// One session of 1500 keys: 12 us for the two kernels, all latency. Registers: 150 to 189 with 64 dims, 168 (16 bytes spilled, 8 rows) and 248 (16 rows)
// with 128, 255 with 256 (244 bytes spilled).
#include <cuda_bf16.h>
#include <float.h>

#include <initializer_list>

#include "paged_work.cuh"

namespace yb {

int launch_paged_tiles(const PagedParams &p, unsigned qtype, uint64_t head_dim, unsigned ctas, cudaStream_t s);

constexpr int kRowsThreads = 128, kRowsWarps = kRowsThreads / 32;
constexpr int kRowsBlock = 16 * kRowsWarps, kRowsCost = 1;      // keys of a unit of work, 16 a warp; units that an item costs besides

template <class T> __device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// (Not through the read-only path, here and for the tables: the kernel may begin while the one before it still writes what is read after the wait.)
__device__ __forceinline__ uint4 ldg_once(const uint16_t *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// R: rows held, 8 or 16 (the MMA has 16; with 8 the upper ones are zero and their results dropped).
template <class T, int D, int R>
__global__ void __launch_bounds__(kRowsThreads, R == 8 && D <= 128 ? 3 : 2) paged_rows_kernel(const PagedParams p) {
    constexpr int KL = D / 32, VU = D / 64, H = R / 8;
    __shared__ PagedScratch<kRowsThreads> s_scan;
    __shared__ float s_m[kRowsWarps][R], s_l[kRowsWarps][R];
    __shared__ __align__(16) float s_acc[kRowsWarps][R][D + 4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    pdl_trigger();
    pdl_wait();
    const PagedStart start = paged_start<kRowsThreads, R, kRowsBlock, kRowsCost>(p, &s_scan);
    PagedWalk<R, kRowsBlock, kRowsCost> w;
    const uint32_t units_per_page = (uint32_t)(p.page_size / 16);
    const float scale = p.scale * 1.4426950408889634f;          // scores in powers of two
    constexpr float kLift = std::is_same<T, __half>::value ? 32768.0f : 1.0f;
    if (tid == 0) p.share[blockIdx.x].rows = 0;
    bool bad_page = false, bad_out = false;

    for (w.start(p, start); w.live(); w.next(p)) {
        const int64_t cached = w.q.n.cached, end = (int64_t)w.q.n.cached + w.q.n.fresh;
        const int32_t *table = p.block_table + (uint64_t)w.request * p.table_width;
        const uint64_t head_at = (uint64_t)w.head * p.page_size, pitch = (uint64_t)p.kv_heads * p.page_size;
        // ---- the rows: lane (g, c) holds dims 8 (c + 4 i) .. of rows g and g + 8
        uint32_t qa[H][KL][4];
        int64_t seen[H];
        uint64_t mask[H];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const uint32_t row = (uint32_t)(g + 8 * h), token = row / p.group;
            const bool live = row < w.q.rows;
            const uint16_t *src = p.q + (uint64_t)(w.q.n.token + token) * p.q_stride + ((uint64_t)w.head * p.group + row % p.group) * D;
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const uint4 v = live ? reinterpret_cast<const uint4 *>(src)[c + 4 * i] : make_uint4(0, 0, 0, 0);
                qa[h][i][0] = v.x; qa[h][i][1] = v.y; qa[h][i][2] = v.z; qa[h][i][3] = v.w;
            }
            seen[h] = live ? cached + token + 1 : cached;
            mask[h] = p.tree && live ? p.ancestors[w.q.n.token + token] : 0ull;
        }
        float m[H], l[H], acc[VU][8][4];
#pragma unroll
        for (int h = 0; h < H; ++h) { m[h] = -INFINITY; l[h] = 0.0f; }
#pragma unroll
        for (int u = 0; u < VU; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[u][j][e] = 0.0f;

        auto page_of = [&](int64_t base) -> int32_t {           // the page of the 16 keys from base on; -1 past the end
            return base < end ? table[(uint32_t)(base / 16) / units_per_page] : -1;
        };
        int64_t base = (int64_t)w.first * kRowsBlock + 16 * warp;
        int32_t page = page_of(base);
        for (uint32_t i = 0; i < w.count; ++i, base += kRowsBlock) {
            const int32_t ahead = i + 1 < w.count ? page_of(base + kRowsBlock) : -1;
            const bool fine = page >= 0 && (uint64_t)page < p.pages;
            if (base < end && !fine) bad_page = true;
            const int64_t stop = fine ? end : base;             // keys from here on are not read
            const uint64_t at = ((uint64_t)(fine ? page : 0) * pitch + head_at + ((uint32_t)(base / 16) % units_per_page) * 16u) * D;
            const uint16_t *kb = p.k + at, *vb = p.v + at;
            page = ahead;
            if (base >= stop) continue;
            uint4 kr[2][KL], vr[4][VU];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int key = 8 * half + g;
#pragma unroll
                for (int x = 0; x < KL; ++x) kr[half][x] = base + key < stop ? ldg_once(kb + key * D + 8 * (c + 4 * x)) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = 2 * c + (r & 1) + 8 * (r >> 1);
#pragma unroll
                for (int u = 0; u < VU; ++u) vr[r][u] = base + key < stop ? ldg_once(vb + key * D + 8 * (g + 8 * u)) : make_uint4(0, 0, 0, 0);
            }
            // ---- S: sc[half] = scores of rows g (0, 1) and g + 8 (2, 3), keys base + 8 half + 2c, + 1
            float sc[2][4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[half][e] = 0.0f;
#pragma unroll
                for (int x = 0; x < KL; ++x) {
                    const uint32_t b[4] = {kr[half][x].x, kr[half][x].y, kr[half][x].z, kr[half][x].w};
                    mma16816<T>(sc[half], qa[0][x][0], H == 2 ? qa[H - 1][x][0] : 0u, qa[0][x][1], H == 2 ? qa[H - 1][x][1] : 0u, b[0], b[1]);
                    mma16816<T>(sc[half], qa[0][x][2], H == 2 ? qa[H - 1][x][2] : 0u, qa[0][x][3], H == 2 ? qa[H - 1][x][3] : 0u, b[2], b[3]);
                }
            }
            // ---- keys that not every row sees: fresh ones, and the block's end
            uint32_t sees[H], odd = 0;
#pragma unroll
            for (int h = 0; h < H; ++h) sees[h] = 0xffffu;
            if (base + 16 > cached) {
#pragma unroll
                for (int h = 0; h < H; ++h) sees[h] = (uint32_t)(paged_sees(p.tree, base, cached, seen[h], mask[h]) & low_bits(end - base)) & 0xffffu;
                // a weight of zero times an infinity would reach rows that do not see it: such values are taken out, and rows that see them marked
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = 2 * c + (r & 1) + 8 * (r >> 1);
                    if (base + key < cached) continue;
#pragma unroll
                    for (int u = 0; u < VU; ++u) {
                        uint32_t *x = reinterpret_cast<uint32_t *>(&vr[r][u]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t o = odd_halves<T>(x[e]);
                            if (o) { odd |= 1u << key; x[e] = without_halves(x[e], o); }
                        }
                    }
                }
                odd = __reduce_or_sync(0xffffffffu, odd);
            }
            // ---- softmax of the block, P as A fragments
            uint32_t pa[2][2] = {{0u, 0u}, {0u, 0u}};           // [half][rows g, rows g + 8]
#pragma unroll
            for (int h = 0; h < H; ++h) {
                float x[2][2], top = m[h];
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        x[half][e] = (sees[h] >> (8 * half + 2 * c + e)) & 1u ? sc[half][2 * h + e] * scale : -INFINITY;
                        top = fmaxf(top, x[half][e]);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float shift = top == -INFINITY ? 0.0f : top, corr = exp2f(m[h] - shift);
                m[h] = top;
                l[h] *= corr;
                if (corr != 1.0f) {
#pragma unroll
                    for (int u = 0; u < VU; ++u)
#pragma unroll
                        for (int j = 0; j < 8; ++j) { acc[u][j][2 * h] *= corr; acc[u][j][2 * h + 1] *= corr; }
                }
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float p0 = exp2f(x[half][0] - shift) * kLift, p1 = exp2f(x[half][1] - shift) * kLift;     // (exact)
                    pa[half][h] = close2<T>(p0, p1);
                    l[h] += p0 + p1;
                }
                if (odd & sees[h]) l[h] = NAN;
            }
            // ---- O += P V: n-tile (u, j) is dim j of chunks 8u .. 8u + 7, the k-slots are this lane's keys
#pragma unroll
            for (int u = 0; u < VU; ++u) {
                const uint32_t r0[4] = {vr[0][u].x, vr[0][u].y, vr[0][u].z, vr[0][u].w}, r1[4] = {vr[1][u].x, vr[1][u].y, vr[1][u].z, vr[1][u].w};
                const uint32_t r2[4] = {vr[2][u].x, vr[2][u].y, vr[2][u].z, vr[2][u].w}, r3[4] = {vr[3][u].x, vr[3][u].y, vr[3][u].z, vr[3][u].w};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                    mma16816<T>(acc[u][j], pa[0][0], pa[0][1], pa[1][0], pa[1][1], __byte_perm(r0[j >> 1], r1[j >> 1], sel),
                                __byte_perm(r2[j >> 1], r3[j >> 1], sel));
                }
            }
        }
        // ---- the warps' states joined
#pragma unroll
        for (int h = 0; h < H; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if (c == 0) { s_m[warp][g + 8 * h] = m[h]; s_l[warp][g + 8 * h] = l[h]; }
#pragma unroll
            for (int u = 0; u < VU; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) s_acc[warp][g + 8 * h][8 * (2 * c + e + 8 * u) + j] = acc[u][j][2 * h + e];
        }
        __syncthreads();
        const bool whole = w.begins && w.ends;
        float *slot = paged_slot(p, blockIdx.x, w.begins, R, D);
        for (int idx = tid; idx < R * (D / 4); idx += kRowsThreads) {
            const int row = whole ? idx / (D / 4) : idx % R, d = 4 * (whole ? idx % (D / 4) : idx / R);
            if (row >= (int)w.q.rows) continue;
            float top = -INFINITY, sum = 0.0f;
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int x = 0; x < kRowsWarps; ++x) top = fmaxf(top, s_m[x][row]);
#pragma unroll
            for (int x = 0; x < kRowsWarps; ++x) {
                const float f = s_m[x][row] == -INFINITY ? 0.0f : exp2f(s_m[x][row] - top);
                sum += s_m[x][row] == -INFINITY ? s_l[x][row] : s_l[x][row] * f;     // (a NaN sum marks the row whatever its maximum)
                const float4 y = *reinterpret_cast<const float4 *>(&s_acc[x][row][d]);
                a.x += y.x * f; a.y += y.y * f; a.z += y.z * f; a.w += y.w * f;
            }
            if (whole) {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                a.x *= inv; a.y *= inv; a.z *= inv; a.w *= inv;
                bad_out |= !isfinite(a.x) || !isfinite(a.y) || !isfinite(a.z) || !isfinite(a.w);
                const uint64_t token = w.q.n.token + (uint32_t)row / p.group, head = (uint64_t)w.head * p.group + (uint32_t)row % p.group;
                *reinterpret_cast<uint2 *>(p.out + (token * p.kv_heads * p.group + head) * D + d) = make_uint2(close_means<T>(a.x, a.y), close_means<T>(a.z, a.w));
            } else {
                if (d == 0) *reinterpret_cast<float2 *>(slot + 2 * row) = make_float2(top, sum);
                *reinterpret_cast<float4 *>(slot + 2 * R + (d / 4 * R + row) * 4) = a;
            }
        }
        if (tid == 0 && w.begins && !w.ends)
            p.share[blockIdx.x] = PagedShare{w.last_cta(start), (int32_t)w.q.rows, (int32_t)w.q.n.token, (int32_t)(w.head * p.group), 0, {0, 0, 0}};
        __syncthreads();
    }
    if (bad_page) raise(p.status, YVEX_B200_STATUS_ARGUMENT);
    if (bad_out) raise(p.status, YVEX_B200_STATUS_NUMERIC);
}

// Joins the parts of the item that CTA blockIdx.x of the kernel before began and did not end: a CTA takes eight rows, a thread four
// columns of one of them (a warp's 8 rows x 16 columns are whole lines of every part, and whole sectors of the output). One walk over the
// parts with a running maximum, four loads ahead: with a walk for the maximum first, or more loads ahead, it took 1 to 3 us more at 20 parts,
// since the code is fetched anew by every call.
constexpr int kJoinRows = 8;
template <class T, int D>
__global__ void __launch_bounds__(2 * D) paged_join_kernel(const PagedParams p, int slot_rows) {
    pdl_trigger();
    pdl_wait();
    const PagedShare sh = p.share[blockIdx.x];
    const int lane = threadIdx.x & 31, row = (int)blockIdx.y * kJoinRows + (lane >> 2), group = 4 * (threadIdx.x >> 5) + (lane & 3);
    if (row >= sh.rows) return;
    const uint64_t pitch = paged_slot_floats((uint32_t)slot_rows, D);
    const int parts = sh.last - (int)blockIdx.x + 1;
    const float *slot = p.partial + (2ull * blockIdx.x + 1) * pitch;      // the first part; the others are every second slot from the next one on
    const uint32_t ml_at = 2u * row, acc_at = 2u * slot_rows + 4u * (group * slot_rows + row);
    float top = -INFINITY, sum = 0.0f;
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
        const float2 ml = *reinterpret_cast<const float2 *>(slot + ml_at);
        const float4 y = *reinterpret_cast<const float4 *>(slot + acc_at);
        slot += i == 0 ? pitch : 2 * pitch;
        const float most = fmaxf(top, ml.x), shift = most == -INFINITY ? 0.0f : most;
        const float c = exp2f(top - shift), f = exp2f(ml.x - shift);      // (a part that saw nothing: 0, and its sum is 0, or NaN where it marks the row)
        top = most;
        sum = sum * c + (ml.x == -INFINITY ? ml.y : ml.y * f);
        a.x = a.x * c + y.x * f; a.y = a.y * c + y.y * f; a.z = a.z * c + y.z * f; a.w = a.w * c + y.w * f;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    a.x *= inv; a.y *= inv; a.z *= inv; a.w *= inv;
    const uint32_t r = (uint32_t)(sh.first_row + row);
    const uint64_t token = (uint64_t)sh.token + r / p.group, head = (uint64_t)sh.head + r % p.group;
    *reinterpret_cast<uint2 *>(p.out + (token * p.kv_heads * p.group + head) * D + 4 * group) = make_uint2(close_means<T>(a.x, a.y), close_means<T>(a.z, a.w));
    if (!isfinite(a.x) || !isfinite(a.y) || !isfinite(a.z) || !isfinite(a.w)) raise(p.status, YVEX_B200_STATUS_NUMERIC);
}

// Which kernel, for how many rows a slot holds, on how many CTAs. Up to 16 rows fit the MMA of the rows kernel (8 with 256 dims, where
// sixteen rows of Q and O would not fit the registers); beyond that its operands would be read again for every 16 rows, while a tile holds 128.
// Device time in us of the rows kernel and of the tiles kernel for the same calls, bf16, fresh 1: 64 sessions of up to 16384 keys and 4 kv heads; 8
// sessions of up to 4096 and 8; one of 4096 and 8:
//   64 dims,  8 rows    77 107 |  14.9 24.6 |  18.1 15.0      128 dims,  8 rows  133 141 |  25.6 30.0 |  20.7 15.9
//   64 dims, 16 rows   106 107 |  18.0 24.6 |  17.8 15.0      128 dims, 16 rows  147 142 |  27.2 29.6 |  20.6 15.6
//  256 dims,  8 rows   273 249 |  48.6 42.8 |  24.0 17.2      (24 rows, tiles alone: 108, 138, 246 us of the first kind)
// So the border holds for a few sessions and more at 64 and 128 dims (but for 3 % at 16 rows of 128 and 64 sessions); one session would gain 16 to 24 %
// from tiles, 256 dims altogether 9 to 28 %.
struct PagedShape { bool tiles; uint32_t rows; unsigned ctas; };
static PagedShape paged_shape(const yvex_b200_kv_cache *c, const yvex_b200_kv_step *t, uint64_t q_heads) {
    const uint64_t group = q_heads / c->kv_heads, rows = t->longest_fresh * group, D = c->head_dim;
    PagedShape s;
    s.tiles = rows > (D == 256 ? 8u : 16u);
    s.rows = s.tiles ? (D == 256 ? 128u : 256u) : rows <= 8 ? 8u : 16u;
    const uint64_t keys = s.tiles ? (D == 256 ? 64u : 128u) : (uint64_t)kRowsBlock;
    // no more CTAs than there can be units of work
    const uint64_t tiles = (rows + s.rows - 1) / s.rows, blocks = (t->longest + keys - 1) / keys + (s.tiles ? kTilesCost : kRowsCost);
    uint64_t most = (uint64_t)kSmCount * (s.tiles ? 1u : s.rows == 8 && D <= 128 ? 3u : 2u);
    for (uint64_t x : {t->requests, c->kv_heads, tiles, blocks}) if (x >= most) return s.ctas = (unsigned)most, s;
    const uint64_t bound = t->requests * c->kv_heads * tiles * blocks;
    s.ctas = (unsigned)(bound < most ? bound : most);
    return s;
}
static uint64_t paged_partial_bytes(const PagedShape &s, uint64_t head_dim) {
    return (2ull * s.ctas * paged_slot_floats(s.rows, (uint32_t)head_dim) * sizeof(float) + 255) / 256 * 256;
}

template <class T, int D> static int launch_paged(const PagedParams &p, const PagedShape &s, unsigned qtype, cudaStream_t stream) {
    int rc = OK;
    if (s.tiles) {
        rc = launch_paged_tiles(p, qtype, D, s.ctas, stream);
    } else if constexpr (D <= 128) {
        if (launch_pdl(s.rows == 8 ? paged_rows_kernel<T, D, 8> : paged_rows_kernel<T, D, 16>, dim3(s.ctas), dim3(kRowsThreads), 0, stream, p) != cudaSuccess)
            rc = ERR_BACKEND;
    } else if (launch_pdl(paged_rows_kernel<T, D, 8>, dim3(s.ctas), dim3(kRowsThreads), 0, stream, p) != cudaSuccess) {
        rc = ERR_BACKEND;
    }
    if (rc != OK) return rc;
    const uint64_t rows = p.longest_fresh * p.group < s.rows ? p.longest_fresh * p.group : s.rows;
    if (launch_pdl(paged_join_kernel<T, D>, dim3(s.ctas, (unsigned)((rows + kJoinRows - 1) / kJoinRows)), dim3(2 * D), 0, stream, p, (int)s.rows) != cudaSuccess)
        return ERR_BACKEND;
    return launch_status(2);
}

}  // namespace yb

using namespace yb;

static int paged_refusal(const yvex_b200_kv_cache *c, const yvex_b200_kv_step *t, uint64_t q_heads) {
    int rc = check_cache(c);
    if (rc == OK) rc = check_step(t);
    if (rc != OK) return rc;
    if (!q_heads || q_heads % c->kv_heads) return ERR_INVALID_ARG;
    if (q_heads > 65536 || c->pages > (uint64_t)INT32_MAX / (c->kv_heads * c->page_size)) return ERR_BOUNDS;
    return OK;
}

extern "C" uint64_t yvex_b200_attention_paged_workspace_bytes(const yvex_b200_kv_cache *c, const yvex_b200_kv_step *t, uint64_t q_heads) {
    if (paged_refusal(c, t, q_heads) != OK) return 0;
    const PagedShape s = paged_shape(c, t, q_heads);
    return paged_partial_bytes(s, c->head_dim) + s.ctas * sizeof(PagedShare);
}

extern "C" int yvex_b200_attention_paged(const yvex_b200_kv_cache *c, const yvex_b200_kv_step *t, const void *q, uint64_t q_stride, uint64_t q_heads,
                                         float scale, void *out, void *workspace, uint64_t workspace_bytes, int *status, void *stream) {
    const int rc = paged_refusal(c, t, q_heads);
    if (rc != OK) return rc;
    if (!q || !out || !status || !t->cached || !t->offsets || !t->block_table || (t->tree && !t->ancestors)) return ERR_INVALID_ARG;
    if (!(scale >= FLT_MIN) || !isfinite(scale * 1.4426950408889634f)) return ERR_INVALID_ARG;
    if (q_stride < q_heads * c->head_dim) return ERR_BOUNDS;
    if (((uintptr_t)q | (uintptr_t)out) & 15u || q_stride % 8) return ERR_INVALID_ARG;
    const PagedShape s = paged_shape(c, t, q_heads);
    const uint64_t partial = paged_partial_bytes(s, c->head_dim);
    if (!workspace || workspace_bytes < partial + s.ctas * sizeof(PagedShare)) return ERR_NOMEM;
    if ((uintptr_t)workspace & 15u) return ERR_INVALID_ARG;
    const PagedParams p{(const uint16_t *)q, (const uint16_t *)c->k, (const uint16_t *)c->v, (uint16_t *)out, q_stride, c->pages, c->page_size,
                        t->table_width, t->requests, t->tokens, t->longest_fresh, t->longest, (uint32_t)c->kv_heads, (uint32_t)(q_heads / c->kv_heads),
                        t->tree != 0, t->cached, t->offsets, t->block_table, t->ancestors, scale, status, (float *)workspace,
                        (PagedShare *)((char *)workspace + partial)};
    cudaStream_t st = as_stream(stream);
#define YB_PAGED(T) (c->head_dim == 64 ? launch_paged<T, 64>(p, s, c->qtype, st) : c->head_dim == 128 ? launch_paged<T, 128>(p, s, c->qtype, st) \
                                       : launch_paged<T, 256>(p, s, c->qtype, st))
    return c->qtype == Q_BF16 ? YB_PAGED(__nv_bfloat16) : YB_PAGED(__half);
#undef YB_PAGED
}
