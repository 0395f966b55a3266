// The paged cache of a serving step: the plan made on the device from the requests' lengths, and the rows written into pages.
#include "paged.cuh"

namespace yb {

// ---- plan ---------------------------------------------------------------------------------------------------------------
// offsets = exclusive prefix of fresh; first_page = exclusive prefix of ceil((cached + fresh) / S) - ceil(cached / S). A page
// that a request gains starts with one of its fresh tokens (its first token has an index >= cached), so every row can be planned
// by itself, table entry included, once the prefixes are known.
// 64 sessions 3.7 us, 512 trees (24 K nodes) 4.9, launch included.
//
// Latency is all there is to it (a step of 64 requests moves 2 KB): one launch, and instead of a second kernel or a wait between
// CTAs every CTA scans the lengths itself, 512 requests at a time, and keeps what concerns its own rows. Rows of a tree need their
// ancestors, all of the same request and at most 63 rows before: a CTA reads the parents of 64 rows before its own too and follows
// them by pointer doubling in shared memory (at most six rounds for 64 nodes, against 63 dependent loads).
constexpr int kPlanThreads = 512, kPlanHalo = YVEX_B200_TREE_NODES;

struct PlanParams {
    uint64_t pages, page_size, requests, tokens, table_width, longest_fresh, longest, free_count;
    int tree;
    const int32_t *cached, *fresh, *parents, *free_pages;
    int32_t *block_table, *offsets;
    int64_t *slots;
    int32_t *positions, *row_request;
    uint64_t *ancestors;
    int32_t *pages_used;
    int *status;
};

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const PlanParams p) {
    __shared__ int64_t s_row[kPlanThreads], s_page[kPlanThreads];
    __shared__ int64_t s_warp[2][kPlanThreads / 32];
    __shared__ uint64_t s_mask[2][kPlanThreads];
    __shared__ int s_up[2][kPlanThreads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int halo = p.tree ? kPlanHalo : 0;
    const int64_t row = (int64_t)blockIdx.x * (kPlanThreads - halo) + tid - halo;
    const uint32_t S = (uint32_t)p.page_size;
    int64_t rows_before = 0, pages_before = 0, index = 0, first_page = 0;
    int request = -1;
    bool bad = false;

    // Lengths that no step can have: the request's rows get no slot and the request no pages.
    auto impossible = [&](int32_t cs, int32_t fs) {
        return cs < 0 || fs < 0 || (uint64_t)fs > p.longest_fresh || (uint64_t)cs + (uint64_t)fs > p.longest || (p.tree && fs > kPlanHalo);
    };

    pdl_trigger();
    pdl_wait();
    int parent = -1;
    if (p.tree && row >= 0 && row < (int64_t)p.tokens) parent = p.parents[row];
    for (uint64_t chunk = 0; chunk < p.requests; chunk += kPlanThreads) {
        const uint64_t r = chunk + tid;
        uint32_t c = 0, f = 0;
        bool none = false;
        if (r < p.requests) {
            const int32_t cs = p.cached[r], fs = p.fresh[r];
            none = impossible(cs, fs);
            bad |= none;
            c = cs < 0 ? 0u : (uint32_t)cs;
            f = fs < 0 ? 0u : (uint32_t)fs;
        }
        const uint32_t need = none ? 0u : (uint32_t)(((uint64_t)c + f + S - 1) / S) - (uint32_t)(((uint64_t)c + S - 1) / S);
        int64_t rows = f, pages = need;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t a = __shfl_up_sync(0xffffffffu, rows, o), b = __shfl_up_sync(0xffffffffu, pages, o);
            if (lane >= o) { rows += a; pages += b; }
        }
        if (lane == 31) { s_warp[0][warp] = rows; s_warp[1][warp] = pages; }
        __syncthreads();
        int64_t row_sum = 0, page_sum = 0;
#pragma unroll
        for (int w = 0; w < kPlanThreads / 32; ++w) {
            const int64_t a = s_warp[0][w], b = s_warp[1][w];
            if (w < warp) { rows += a; pages += b; }
            row_sum += a;
            page_sum += b;
        }
        s_row[tid] = rows_before + rows - f;
        s_page[tid] = pages_before + pages - need;
        if (r < p.requests && (chunk / kPlanThreads) % gridDim.x == blockIdx.x)
            p.offsets[r] = (int32_t)(s_row[tid] < INT32_MAX ? s_row[tid] : INT32_MAX);
        __syncthreads();
        if (row >= rows_before && row < rows_before + row_sum) {
            int lo = 0, hi = kPlanThreads - 1;              // the last request that starts at or before the row
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_row[mid] <= row) lo = mid; else hi = mid - 1;
            }
            request = (int)(chunk + lo);                    // (those behind the chunk's last one have no rows and start past this one)
            index = row - s_row[lo];
            first_page = s_page[lo];
        }
        rows_before += row_sum;
        pages_before += page_sum;
        __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.offsets[p.requests] = (int32_t)(rows_before < INT32_MAX ? rows_before : INT32_MAX);
        *p.pages_used = (int32_t)(pages_before < INT32_MAX ? pages_before : INT32_MAX);
        bad |= rows_before > (int64_t)p.tokens || pages_before > (int64_t)p.free_count;
    }

    uint64_t mask = 0;
    if (p.tree) {
        // s_up: the thread whose mask is still to be added, -1 for none. A row's mask and its pointer double their reach each round.
        bool wrong = false;
        if (request >= 0 && parent != -1) {
            wrong = parent < -1 || parent >= index || index >= kPlanHalo;
            bad |= wrong && tid >= halo;
        }
        mask = request >= 0 && index < kPlanHalo ? 1ull << index : 0ull;
        int up = request >= 0 && parent >= 0 && !wrong ? tid - (int)(index - parent) : -1;
        if (up < 0) up = -1;                                // (a row before the halo: only rows that are not this CTA's have such parents)
        int b = 0;
        s_mask[0][tid] = mask;
        s_up[0][tid] = up;
        while (__syncthreads_or(up >= 0)) {
            if (up >= 0) {
                mask |= s_mask[b][up];
                up = s_up[b][up];
            }
            b ^= 1;
            s_mask[b][tid] = mask;
            s_up[b][tid] = up;
        }
    }

    if (tid >= halo && row < (int64_t)p.tokens) {
        int64_t slot = -1;
        int32_t position = 0;
        if (request >= 0) {
            const int32_t cs = p.cached[request];
            const uint32_t c = (uint32_t)max(cs, 0);
            const uint64_t at = (uint64_t)c + (uint64_t)index, col = at / S;
            const uint64_t held = ((uint64_t)c + S - 1) / S;
            int32_t page = -1;
            if (col < p.table_width && !impossible(cs, p.fresh[request])) {
                int32_t *entry = p.block_table + (uint64_t)request * p.table_width + col;
                if (col < held) {
                    page = *entry;
                } else {
                    const uint64_t k = (uint64_t)first_page + (col - held);
                    if (k < p.free_count) page = p.free_pages[k];
                    if (at % S == 0 && page >= 0 && (uint64_t)page < p.pages) *entry = page;
                }
            }
            if (page >= 0 && (uint64_t)page < p.pages) slot = (int64_t)page * S + (int64_t)(at % S);
            else bad = true;
            const uint64_t pos = (uint64_t)c + (p.tree ? (uint64_t)max(__popcll(mask) - 1, 0) : (uint64_t)index);
            position = (int32_t)(pos < INT32_MAX ? pos : INT32_MAX);
        }
        p.slots[row] = slot;
        p.positions[row] = position;
        p.row_request[row] = request;
        if (p.tree) p.ancestors[row] = mask;
    }
    if (bad) raise(p.status, YVEX_B200_STATUS_ARGUMENT);
}

// ---- append -------------------------------------------------------------------------------------------------------------
// A copy with one rounding, bound by HBM (16384 tokens x 8 heads x 128, bf16: 134 MB in 20.8 us, 6.4 TB/s). A warp takes one row of one side (kv_heads * head_dim values, 16 bytes of the cache per
// lane at a time, four of them in flight), so that the slot is read and divided once per row. (No __restrict__: the compiler would read what the
// kernel before this one may still be writing through the read-only path.)
constexpr int kAppendWarps = 8;

template <class Out> __device__ __forceinline__ uint32_t pack2(float a, float b, bool &bad) {
    if constexpr (std::is_same<Out, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        const uint32_t w = *reinterpret_cast<const uint32_t *>(&h);
        bad |= (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u;
        return w;
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        const uint32_t w = *reinterpret_cast<const uint32_t *>(&h);
        bad |= (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
        return w;
    }
}
template <class In> __device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (std::is_same<In, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <class In> struct AppendVec { uint4 w[sizeof(In) / 2]; };      // eight values of the source

template <class In, class Out>
__global__ void __launch_bounds__(32 * kAppendWarps) kv_append_kernel(const int64_t *slots, uint64_t tokens, const In *k, uint64_t k_stride, const In *v,
                                                                      uint64_t v_stride, uint64_t total_slots, uint32_t page_size, uint32_t kv_heads,
                                                                      uint32_t dim_vecs, uint4 *k_pages, uint4 *v_pages, int *status) {
    const uint64_t job = (uint64_t)blockIdx.x * kAppendWarps + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31u;
    pdl_trigger();
    pdl_wait();
    if (job >= 2 * tokens) return;
    const uint64_t t = job >> 1;
    const int64_t slot = slots[t];
    if (slot < 0) return;
    if ((uint64_t)slot >= total_slots) { raise(status, YVEX_B200_STATUS_ARGUMENT); return; }
    const In *src = job & 1 ? v + t * v_stride : k + t * k_stride;
    const uint64_t page = (uint64_t)slot / page_size;
    const uint32_t at = (uint32_t)((uint64_t)slot - page * page_size);
    uint4 *dst = (job & 1 ? v_pages : k_pages) + (page * kv_heads * page_size + at) * dim_vecs;
    const uint32_t vecs = kv_heads * dim_vecs, head_pitch = page_size * dim_vecs, shift = 31u - (uint32_t)__clz((int)dim_vecs);
    bool bad = false;
    for (uint32_t i0 = lane; i0 < vecs; i0 += 128) {
        AppendVec<In> x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t i = i0 + 32u * j;
            if (i < vecs) {
#pragma unroll
                for (int e = 0; e < (int)(sizeof(In) / 2); ++e) x[j].w[e] = __ldcs(reinterpret_cast<const uint4 *>(src + 8ull * i) + e);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t i = i0 + 32u * j;
            if (i >= vecs) continue;
            uint4 o;
            if constexpr (sizeof(In) == 4) {
                o.x = pack2<Out>(__uint_as_float(x[j].w[0].x), __uint_as_float(x[j].w[0].y), bad);
                o.y = pack2<Out>(__uint_as_float(x[j].w[0].z), __uint_as_float(x[j].w[0].w), bad);
                o.z = pack2<Out>(__uint_as_float(x[j].w[1].x), __uint_as_float(x[j].w[1].y), bad);
                o.w = pack2<Out>(__uint_as_float(x[j].w[1].z), __uint_as_float(x[j].w[1].w), bad);
            } else {
                const uint32_t w[4] = {x[j].w[0].x, x[j].w[0].y, x[j].w[0].z, x[j].w[0].w};
                uint32_t r[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) { const float2 f = unpack2<In>(w[e]); r[e] = pack2<Out>(f.x, f.y, bad); }
                o = make_uint4(r[0], r[1], r[2], r[3]);
            }
            const uint32_t h = i >> shift;
            dst[(uint64_t)h * head_pitch + (i & (dim_vecs - 1u))] = o;
        }
    }
    if (bad) raise(status, YVEX_B200_STATUS_NUMERIC);
}

template <class In, class Out>
static int launch_append(const yvex_b200_kv_cache *c, const int64_t *slots, uint64_t tokens, const void *k, uint64_t ks, const void *v, uint64_t vs,
                         int *status, cudaStream_t s) {
    const uint64_t ctas = (2 * tokens + kAppendWarps - 1) / kAppendWarps;
    if (launch_pdl(kv_append_kernel<In, Out>, dim3((unsigned)ctas), dim3(32 * kAppendWarps), 0, s, slots, tokens, (const In *)k, ks, (const In *)v, vs,
                   c->pages * c->page_size, (uint32_t)c->page_size, (uint32_t)c->kv_heads, (uint32_t)(c->head_dim / 8), (uint4 *)c->k, (uint4 *)c->v,
                   status) != cudaSuccess)
        return ERR_BACKEND;
    return launch_status(1);
}

int check_cache(const yvex_b200_kv_cache *c) {
    if (!c || !c->k || !c->v || !c->pages || !c->kv_heads) return ERR_INVALID_ARG;
    if (c->qtype != Q_F16 && c->qtype != Q_BF16) return ERR_UNSUPPORTED;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return ERR_UNSUPPORTED;
    if (!c->page_size || c->page_size % 16) return ERR_UNSUPPORTED;
    if (c->page_size > (1u << 24) || c->pages > INT32_MAX || c->kv_heads > 1024) return ERR_BOUNDS;
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15u) return ERR_INVALID_ARG;
    return OK;
}

int check_step(const yvex_b200_kv_step *t) {
    if (!t || !t->requests || !t->tokens || !t->table_width || !t->longest_fresh || !t->longest) return ERR_INVALID_ARG;
    if (t->requests >= INT32_MAX || t->tokens >= INT32_MAX || t->table_width > INT32_MAX || t->longest > (1u << 30) || t->longest_fresh > t->longest)
        return ERR_BOUNDS;
    if (t->tree && t->longest_fresh > YVEX_B200_TREE_NODES) return ERR_BOUNDS;
    return OK;
}

}  // namespace yb

using namespace yb;

extern "C" int yvex_b200_kv_plan(const yvex_b200_kv_cache *c, const yvex_b200_kv_step *t, const int32_t *free_pages, uint64_t free_count,
                                 int32_t *pages_used, int *status, void *stream) {
    if (!c || !c->pages || !c->page_size || !pages_used || !status || (!free_pages && free_count)) return ERR_INVALID_ARG;
    if (c->page_size > (1u << 24) || c->pages > INT32_MAX) return ERR_BOUNDS;
    const int rc = check_step(t);
    if (rc != OK) return rc;
    if (!t->cached || !t->fresh || !t->block_table || !t->offsets || !t->slots || !t->positions || !t->row_request) return ERR_INVALID_ARG;
    if (t->tree && (!t->parents || !t->ancestors)) return ERR_INVALID_ARG;
    PlanParams p{c->pages, c->page_size, t->requests, t->tokens, t->table_width, t->longest_fresh, t->longest, free_count, t->tree != 0,
                 t->cached, t->fresh, t->parents, free_pages, t->block_table, t->offsets, t->slots, t->positions, t->row_request, t->ancestors,
                 pages_used, status};
    const uint64_t own = kPlanThreads - (t->tree ? kPlanHalo : 0), ctas = (t->tokens + own - 1) / own;
    if (launch_pdl(kv_plan_kernel, dim3((unsigned)ctas), dim3(kPlanThreads), 0, as_stream(stream), p) != cudaSuccess) return ERR_BACKEND;
    return launch_status(1);
}

extern "C" int yvex_b200_kv_append(const yvex_b200_kv_cache *c, const int64_t *slots, uint64_t tokens, unsigned int qtype, const void *k,
                                   uint64_t k_stride, const void *v, uint64_t v_stride, int *status, void *stream) {
    const int rc = check_cache(c);
    if (rc != OK) return rc;
    if (!slots || !k || !v || !status || !tokens) return ERR_INVALID_ARG;
    if (qtype != Q_F32 && qtype != Q_F16 && qtype != Q_BF16) return ERR_UNSUPPORTED;
    const uint64_t width = c->kv_heads * c->head_dim, unit = qtype == Q_F32 ? 4 : 8;
    if (tokens >= INT32_MAX || k_stride < width || v_stride < width) return ERR_BOUNDS;
    if (((uintptr_t)k | (uintptr_t)v) & 15u || k_stride % unit || v_stride % unit) return ERR_INVALID_ARG;
    cudaStream_t s = as_stream(stream);
#define YB_APPEND(In) (c->qtype == Q_BF16 ? launch_append<In, __nv_bfloat16>(c, slots, tokens, k, k_stride, v, v_stride, status, s) \
                                          : launch_append<In, __half>(c, slots, tokens, k, k_stride, v, v_stride, status, s))
    return qtype == Q_F32 ? YB_APPEND(float) : qtype == Q_BF16 ? YB_APPEND(__nv_bfloat16) : YB_APPEND(__half);
#undef YB_APPEND
}
