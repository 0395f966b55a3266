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
    float *partial;                              // [2 * CTAs] slots of rows x (maximum, sum), then rows x head_dim
    struct PagedShare *share;                    // [CTAs]
};

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
    __device__ void open(const PagedParams &p, uint64_t r) {
        n = paged_lengths(p, r);
        rows = n.fresh * p.group;
        tiles = (rows + MROWS - 1) / MROWS;
    }
    __device__ uint32_t blocks(const PagedParams &p, uint32_t tile) const {
        return (paged_visible(p, n, min(rows, (tile + 1u) * MROWS)) + BK - 1) / BK;
    }
    __device__ uint64_t blocks_per_head(const PagedParams &p) const {
        if (p.tree || tiles <= 1u) return tiles ? (uint64_t)tiles * blocks(p, 0) : 0ull;
        uint64_t sum = 0;
        for (uint32_t t = 0; t < tiles; ++t) sum += blocks(p, t);
        return sum;
    }
};

// Where a CTA's share begins, found by all its threads (NT of them; `scratch`: NT / 32 + 4 words of shared memory).
struct PagedStart { uint64_t total, from, left, skip; uint32_t request, ctas; };
template <int NT, int MROWS, int BK>
__device__ PagedStart paged_start(const PagedParams &p, uint64_t *scratch) {
    constexpr int W = NT / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    auto units = [&](uint64_t r) -> uint64_t {
        if (r >= p.requests) return 0;
        PagedRequest<MROWS, BK> q;
        q.open(p, r);
        if (q.n.bad && blockIdx.x == 0) raise(p.status, YVEX_B200_STATUS_ARGUMENT);
        return q.blocks_per_head(p) * p.kv_heads;
    };
    auto sum_warps = [&](uint64_t v) {                          // inclusive prefix over the block's threads; the sum in scratch[W]
        uint64_t s = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t a = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += a;
        }
        if (lane == 31) scratch[warp] = s;
        __syncthreads();
        uint64_t before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) before += scratch[w];
            all += scratch[w];
        }
        if (tid == 0) scratch[W] = all;
        return s + before;
    };
    PagedStart st;
    const bool single = p.requests <= NT;                       // one request a thread
    const uint64_t first = units((uint64_t)tid);
    uint64_t v = first;
    if (!single)
        for (uint64_t r = (uint64_t)tid + NT; r < p.requests; r += NT) v += units(r);
    uint64_t prefix = sum_warps(v);
    __syncthreads();
    st.total = scratch[W];
    st.ctas = (uint32_t)min((uint64_t)gridDim.x, st.total);     // every CTA that has a share has a block at least
    const uint64_t u0 = blockIdx.x < st.ctas ? st.total * blockIdx.x / st.ctas : st.total;
    const uint64_t u1 = blockIdx.x < st.ctas ? st.total * (blockIdx.x + 1ull) / st.ctas : st.total;
    st.from = u0;
    st.left = u1 - u0;
    uint64_t base = 0;
    for (uint64_t chunk = 0; chunk < p.requests; chunk += NT) {
        if (!single) {
            __syncthreads();
            v = chunk ? units(chunk + tid) : first;
            prefix = sum_warps(v);
            __syncthreads();
        }
        const uint64_t begin = base + prefix - v;
        if (v && u0 >= begin && u0 < begin + v) { scratch[W + 1] = chunk + tid; scratch[W + 2] = u0 - begin; }
        base += scratch[W];
        if (base > u0) break;
    }
    __syncthreads();
    st.request = st.left ? (uint32_t)scratch[W + 1] : 0u;
    st.skip = st.left ? scratch[W + 2] : 0ull;
    __syncthreads();
    return st;
}

// The segments of a CTA's share, one after the other; every role of a CTA walks them by itself.
template <int MROWS, int BK> struct PagedWalk {
    PagedRequest<MROWS, BK> q;
    uint64_t left, at;                           // blocks of the share still to come; place of the next one among all blocks
    uint32_t request, head, tile, first, count, blocks;
    bool begins, ends;                           // the segment holds the item's first block, its last
    __device__ void start(const PagedParams &p, const PagedStart &s) {
        left = s.left;
        at = s.from;
        request = s.request;
        count = 0;
        if (!left) return;
        q.open(p, request);
        const uint64_t per_head = q.blocks_per_head(p);
        uint64_t skip = s.skip;
        head = (uint32_t)(skip / per_head);
        skip -= head * per_head;
        tile = 0;
        if (p.tree) { blocks = q.blocks(p, 0); tile = (uint32_t)(skip / blocks); skip -= (uint64_t)tile * blocks; }
        else for (; (blocks = q.blocks(p, tile)) <= skip; ++tile) skip -= blocks;
        first = (uint32_t)skip;
        cut();
    }
    __device__ void cut() {
        count = (uint32_t)min((uint64_t)(blocks - first), left);
        begins = first == 0;
        ends = first + count == blocks;
        left -= count;
        at += count;
    }
    __device__ bool live() const { return count != 0; }
    __device__ void next(const PagedParams &p) {
        count = 0;
        if (!left) return;
        if (++tile == q.tiles) {
            tile = 0;
            if (++head == p.kv_heads) {
                head = 0;
                do q.open(p, ++request); while (q.rows == 0);   // (there is work left, so there is such a request)
            }
        }
        blocks = q.blocks(p, tile);
        first = 0;
        cut();
    }
    // The CTA that holds the item's last block; of a segment that does not end its item.
    __device__ int32_t last_cta(const PagedStart &s) const {
        const uint64_t u = at + (blocks - first - count) - 1;   // `at` is behind the segment
        return (int32_t)(((u + 1) * s.ctas - 1) / s.total);
    }
};

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
