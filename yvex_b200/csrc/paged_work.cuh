// How the attention over a paged cache is cut into work, for both of its kernels.
//
// An item is (request, kv head, tile of query rows); a row is (fresh token, query head of the group), row = token * group + head. An
// item's work is counted in blocks of BK keys, as many as its last row sees. The blocks of all items, one behind the other, are cut into
// equal shares, one per CTA, whatever the lengths of the requests: a long session beside short ones, or one session alone, still
// fills the chip, and the host needs no lengths. A CTA's share covers the end of one item, whole items, and the beginning of
// another. Whole items are written out at once; the two others leave their running (maximum, sum, accumulator) in the workspace,
// slot 2c for the item that began in an earlier CTA and 2c + 1 for the one that goes on in a later one, and a second kernel joins them:
// its CTA c takes the item that CTA c began and did not end, which share[c] describes.
#pragma once
#include "paged.cuh"

namespace yb {

struct PagedParams {
    const uint16_t *q, *k, *v;
    uint16_t *out;
    uint64_t q_stride, pages, page_size, table_width, requests, tokens, longest_fresh, longest;
    uint32_t kv_heads, group;
    int tree;
    const int32_t *cached, *offsets, *block_table;
    const uint64_t *ancestors;
    float scale;
    int *status;
    float *partial;                              // [2 * CTAs] slots
    struct PagedShare *share;                    // [CTAs]
};

// What an item costs the tiles kernel besides its blocks of 128 keys (64 with 256 dims), in blocks: the first S waits for Q, the last PV is
// waited for, the sums are read and written, and the code of all that is fetched anew. (16 trees at 100 to 32768 keys with 2, 4, 6 and 8 blocks:
// 276, 270, 265 and 268 us; chunks of two prompts 570, 565, 564 and 579; one tree 22.0, 21.8, 21.7 and 20.9: all at 128 dims, within 3 % of noise.)
constexpr int kTilesCost = 6;

// An item that a CTA began: CTAs c .. last hold its parts. rows 0: none.
struct PagedShare { int32_t last, rows, token, head, first_row, pad[3]; };

// One request's lengths; a request whose numbers cannot be those of a plan counts as one without fresh tokens.
struct PagedLengths { uint32_t cached, fresh, token; bool bad; };
__device__ __forceinline__ PagedLengths paged_lengths(const PagedParams &p, uint64_t r) {
    const int64_t c = p.cached[r], b = p.offsets[r], e = p.offsets[r + 1];
    PagedLengths n;
    n.bad = c < 0 || b < 0 || e < b || e > (int64_t)p.tokens || e - b > (int64_t)p.longest_fresh || c + (e - b) > (int64_t)p.longest ||
            (uint64_t)(c + (e - b)) > p.table_width * p.page_size;
    n.cached = n.bad ? 0u : (uint32_t)c;
    n.fresh = n.bad ? 0u : (uint32_t)(e - b);
    n.token = n.bad ? 0u : (uint32_t)b;
    return n;
}

// Keys that the rows before `rows_end` of a request see at most.
__device__ __forceinline__ uint32_t paged_visible(const PagedParams &p, const PagedLengths &n, uint32_t rows_end) {
    if (p.tree) return n.cached + n.fresh;
    return n.cached + min(n.fresh, (rows_end - 1u) / p.group + 1u);
}

template <int MROWS, int BK> struct PagedRequest {
    PagedLengths n;
    uint32_t rows, tiles;
    __device__ __forceinline__ void open(const PagedParams &p, uint64_t r) {
        n = paged_lengths(p, r);
        rows = n.fresh * p.group;
        tiles = (rows + MROWS - 1) / MROWS;
    }
    __device__ __forceinline__ uint32_t blocks(const PagedParams &p, uint32_t tile) const {
        return (paged_visible(p, n, min(rows, (tile + 1u) * MROWS)) + BK - 1) / BK;
    }
};

// Where a CTA's share begins, found by all its threads (NT of them). COST: what beginning and ending an item costs, in blocks; they
// stand before the item's first block when the shares are cut.
struct PagedStart { uint64_t total, each, from, left; uint32_t more, request, head, tile, skip, ctas; };
// (a 64-bit division takes hundreds of cycles)
__device__ __forceinline__ uint64_t divided(uint64_t a, uint64_t b) { return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b; }
template <int NT> struct PagedScratch {
    uint64_t warps[NT / 32], sum, skip;
    uint32_t request, head, tile, first;
    uint64_t units[NT / 8];
};
template <int NT, int MROWS, int BK, int COST>
__device__ PagedStart paged_start(const PagedParams &p, PagedScratch<NT> *sc) {
    constexpr int W = NT / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    using Request = PagedRequest<MROWS, BK>;
    auto tile_units = [&](const Request &q, uint32_t t) { return t < q.tiles ? q.blocks(p, t) + COST : 0u; };
    auto units = [&](uint64_t r) -> uint64_t {                  // of one request and kv head, by one thread
        if (r >= p.requests) return 0;
        Request q;
        q.open(p, r);
        if (q.n.bad && blockIdx.x == 0) raise(p.status, YVEX_B200_STATUS_ARGUMENT);
        if (p.tree) return (uint64_t)q.tiles * tile_units(q, 0);
        uint64_t sum = 0;
        for (uint32_t t = 0; t < q.tiles; ++t) sum += tile_units(q, t);
        return sum;
    };
    auto scan = [&](uint64_t v) {                               // inclusive prefix over the block's threads; the sum in sc->sum
        uint64_t s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t a = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += a;
        }
        if (lane == 31) sc->warps[warp] = s;
        __syncthreads();
        uint64_t before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) before += sc->warps[w];
            all += sc->warps[w];
        }
        if (tid == 0) sc->sum = all;
        __syncthreads();
        return s + before;
    };
    PagedStart st;
    // A few requests of many tiles (a prompt) are counted by a warp each, many requests by a thread each.
    const bool few = !p.tree && p.longest_fresh * p.group > (uint64_t)MROWS && p.requests <= NT / 8, single = p.requests <= NT;
    uint64_t first;
    if (few) {
        for (uint32_t r = warp; r < (uint32_t)p.requests; r += W) {
            Request q;
            q.open(p, r);
            if (q.n.bad && blockIdx.x == 0 && lane == 0) raise(p.status, YVEX_B200_STATUS_ARGUMENT);
            uint64_t sum = 0;
            for (uint32_t t = lane; t < q.tiles; t += 32) sum += tile_units(q, t);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) sc->units[r] = sum;
        }
        __syncthreads();
        first = tid < (int)p.requests ? sc->units[tid] : 0;
    } else {
        first = units((uint64_t)tid);
    }
    uint64_t v = first;
    if (!single)
        for (uint64_t r = (uint64_t)tid + NT; r < p.requests; r += NT) v += units(r);
    uint64_t prefix = scan(v);
    st.total = sc->sum * p.kv_heads;
    st.ctas = (uint32_t)min((uint64_t)gridDim.x, st.total);     // every CTA that has a share has a unit at least
    // `more` CTAs have one unit more than `each`
    st.each = st.ctas ? divided(st.total, st.ctas) : 0;
    st.more = (uint32_t)(st.total - st.each * st.ctas);
    const uint64_t u0 = blockIdx.x < st.ctas ? st.each * blockIdx.x + min(blockIdx.x, st.more) : st.total;
    st.from = u0;
    st.left = blockIdx.x < st.ctas ? st.each + (blockIdx.x < st.more ? 1 : 0) : 0;
    uint64_t base = 0;
    for (uint64_t chunk = 0; chunk < p.requests && st.left; chunk += NT) {
        if (!single) {
            __syncthreads();
            v = chunk ? units(chunk + tid) : first;
            prefix = scan(v);
        }
        const uint64_t begin = (base + prefix - v) * p.kv_heads;
        if (v && u0 >= begin && u0 < begin + v * p.kv_heads) {
            const uint64_t skip = u0 - begin, head = divided(skip, v);
            sc->request = (uint32_t)(chunk + tid);
            sc->head = (uint32_t)head;
            sc->skip = skip - head * v;
        }
        base += sc->sum;
        if (base * p.kv_heads > u0) break;
    }
    __syncthreads();
    if (warp == 0 && st.left) {                                 // the tile of that request: the first whose units reach past what is skipped
        Request q;
        q.open(p, sc->request);
        uint64_t skip = sc->skip;
        for (uint32_t t0 = 0; t0 < q.tiles; t0 += 32) {
            const uint32_t mine = tile_units(q, t0 + lane);
            uint64_t s = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint64_t a = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += a;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, s > skip);
            if (past) {
                if (lane == __ffs((int)past) - 1) { sc->tile = t0 + lane; sc->first = (uint32_t)(skip - (s - mine)); }
                break;
            }
            skip -= __shfl_sync(0xffffffffu, s, 31);
        }
    }
    __syncthreads();
    st.request = sc->request;
    st.head = sc->head;
    st.tile = sc->tile;
    st.skip = sc->first;
    return st;
}

// The segments of a CTA's share, one after the other; every role of a CTA walks them by itself.
template <int MROWS, int BK, int COST> struct PagedWalk {
    PagedRequest<MROWS, BK> q;
    uint64_t left, at;                           // units of the share still to come; place of the next one among all units
    uint32_t request, head, tile, first, count, blocks, rest;
    bool begins, ends;                           // the segment holds the item's first block, its last
    __device__ __forceinline__ void start(const PagedParams &p, const PagedStart &s) {
        left = s.left;
        at = s.from;
        request = s.request;
        head = s.head;
        tile = s.tile;
        count = 0;
        if (!left) return;
        q.open(p, request);
        cut(p, s.skip);
    }
    __device__ __forceinline__ void cut(const PagedParams &p, uint32_t from) {
        blocks = q.blocks(p, tile);
        const uint32_t to = (uint32_t)min((uint64_t)(blocks + COST), from + left), units = to - from;
        first = from > COST ? from - COST : 0u;
        count = (to > COST ? to - COST : 0u) - first;           // 0 only where the share ends within the cost of an item's beginning
        begins = first == 0;
        ends = first + count == blocks;
        rest = blocks + COST - to;
        left -= units;
        at += units;
    }
    __device__ __forceinline__ bool live() const { return count != 0; }
    __device__ __forceinline__ void next(const PagedParams &p) {
        count = 0;
        if (!left) return;
        if (++tile == q.tiles) {
            tile = 0;
            if (++head == p.kv_heads) {
                head = 0;
                do q.open(p, ++request); while (q.rows == 0);   // (there is work left, so there is such a request)
            }
        }
        cut(p, 0);
    }
    // The CTA that holds the item's last block; of a segment that does not end its item.
    __device__ __forceinline__ int32_t last_cta(const PagedStart &s) const {
        const uint64_t u = at + rest - 1, larger = s.more * (s.each + 1);
        return (int32_t)(u < larger ? divided(u, s.each + 1) : s.more + divided(u - larger, s.each));
    }
};

// A slot of the workspace: (maximum, sum) of every row, then the accumulators in groups of four columns, [head_dim / 4][rows][4], so that
// threads with a row each write whole lines.
__host__ __device__ constexpr uint64_t paged_slot_floats(uint32_t rows, uint32_t head_dim) { return (uint64_t)rows * (head_dim + 2); }
__device__ __forceinline__ float *paged_slot(const PagedParams &p, uint32_t cta, bool began, uint32_t rows, uint32_t head_dim) {
    return p.partial + (2ull * cta + (began ? 1 : 0)) * paged_slot_floats(rows, head_dim);
}

// Which of the keys base .. base + 63 a row sees, as bits. chain: keys below `seen`; tree: keys below `cached`, and of those from
// there on (base may lie before or behind) the bits of `mask`.
__device__ __forceinline__ uint64_t low_bits(int64_t n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; }
__device__ __forceinline__ uint64_t paged_sees(bool tree, int64_t base, int64_t cached, int64_t seen, uint64_t mask) {
    if (!tree) return low_bits(seen - base);
    const int64_t d = cached - base;
    return low_bits(d) | (d >= 64 || d <= -64 ? 0ull : d >= 0 ? mask << d : mask >> -d);
}

template <class T> __device__ __forceinline__ uint32_t close2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
}
// The same of means of values. In f16, weights that were rounded up can lift a mean over the largest number, by up to 2^-11: it is no infinity.
template <class T> __device__ __forceinline__ uint32_t close_means(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) {
        auto within = [](float x) { return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x; };
        return close2<T>(within(a), within(b));
    } else {
        return close2<T>(a, b);
    }
}
// The words' halves that are infinities or NaN (bit 15 and 31 of the result), and the words without them.
template <class T> __device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
    constexpr uint32_t e = std::is_same<T, __half>::value ? 0x7c007c00u : 0x7f807f80u, one = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
    return ((w & e) + one) & 0x80008000u;        // an exponent of all ones carries into the sign's place
}
__device__ __forceinline__ uint32_t without_halves(uint32_t w, uint32_t odd) {
    const uint32_t m = odd >> 15;                // bits 0 and 16
    return w & ~(m * 0xffffu);
}

}  // namespace yb
