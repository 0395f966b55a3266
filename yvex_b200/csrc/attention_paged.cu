// Attention of a step's fresh tokens over the paged cache: softmax(scale q K^T) V with one running maximum and sum per row.
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
};

template <class T> __device__ __forceinline__ float2 open2(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T> __device__ __forceinline__ uint32_t close2(float a, float b) {
    if constexpr (std::is_same<T, __half>::value) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }
}

// One warp per (row, query head), one key after the other.
template <class T, int D>
__global__ void __launch_bounds__(256) paged_rows_kernel(const PagedParams p) {
    constexpr int W = D / 64;                           // 32-bit words of a row per lane
    pdl_trigger();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31u, q_heads = p.kv_heads * p.group;
    const uint64_t job = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const uint64_t row = job / q_heads;
    const uint32_t head = (uint32_t)(job % q_heads), kvh = head / p.group;
    if (row >= p.tokens) return;
    uint64_t lo = 0, hi = p.requests - 1;
    if ((int64_t)row >= p.offsets[p.requests]) return;
    while (lo < hi) {
        const uint64_t mid = (lo + hi + 1) / 2;
        if (p.offsets[mid] <= (int64_t)row) lo = mid; else hi = mid - 1;
    }
    const int64_t begin = p.offsets[lo], fresh = p.offsets[lo + 1] - begin, cached = max(p.cached[lo], 0), index = (int64_t)row - begin;
    bool bad = p.cached[lo] < 0 || begin < 0 || index < 0 || fresh > (int64_t)p.longest_fresh || cached + fresh > (int64_t)p.longest || index >= fresh;
    const int64_t room = (int64_t)(p.table_width * p.page_size);
    bad |= cached + fresh > room;
    if (bad) { if (lane == 0) raise(p.status, YVEX_B200_STATUS_ARGUMENT); return; }
    const uint64_t mask = p.tree ? p.ancestors[row] : 0ull;
    const int64_t visible = p.tree ? cached + fresh : cached + index + 1;
    float2 q[W], acc[W];
    const uint32_t *qr = reinterpret_cast<const uint32_t *>(p.q + row * p.q_stride + (uint64_t)head * D);
#pragma unroll
    for (int i = 0; i < W; ++i) { q[i] = open2<T>(qr[lane + 32 * i]); acc[i] = make_float2(0.0f, 0.0f); }
    float m = -INFINITY, l = 0.0f;
    for (int64_t j = 0; j < visible; ++j) {
        if (p.tree && j >= cached && (j - cached > 63 || !((mask >> (j - cached)) & 1ull))) continue;
        const int32_t page = p.block_table[lo * p.table_width + (uint64_t)j / p.page_size];
        if (page < 0 || (uint64_t)page >= p.pages) { bad = true; continue; }
        const uint64_t at = (((uint64_t)page * p.kv_heads + kvh) * p.page_size + (uint64_t)j % p.page_size) * D;
        const uint32_t *kr = reinterpret_cast<const uint32_t *>(p.k + at), *vr = reinterpret_cast<const uint32_t *>(p.v + at);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) { const float2 x = open2<T>(kr[lane + 32 * i]); s += q[i].x * x.x + q[i].y * x.y; }
        s = warp_sum(s) * p.scale;
        const float top = fmaxf(m, s);
        if (s != s || top == INFINITY) { l = NAN; continue; }
        if (top == -INFINITY) continue;
        const float c = expf(m - top), w = expf(s - top);
        m = top;
        l = l * c + w;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float2 x = open2<T>(vr[lane + 32 * i]);
            acc[i].x = acc[i].x * c + w * x.x;
            acc[i].y = acc[i].y * c + w * x.y;
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    bool odd = false;
    uint32_t *o = reinterpret_cast<uint32_t *>(p.out + (row * q_heads + head) * D);
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float x = acc[i].x * inv, y = acc[i].y * inv;
        odd |= !isfinite(x) || !isfinite(y);
        o[lane + 32 * i] = close2<T>(x, y);
    }
    if (bad) raise(p.status, YVEX_B200_STATUS_ARGUMENT);
    if (odd) raise(p.status, YVEX_B200_STATUS_NUMERIC);
}

template <class T, int D> static int launch_rows(const PagedParams &p, cudaStream_t s) {
    const uint64_t warps = p.tokens * p.kv_heads * p.group;
    if (launch_pdl(paged_rows_kernel<T, D>, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, s, p) != cudaSuccess) return ERR_BACKEND;
    return launch_status(1);
}

}  // namespace yb

using namespace yb;

static int paged_refusal(const yvex_b200_kv_cache *c, const yvex_b200_kv_step *t, uint64_t q_heads) {
    int rc = check_cache(c);
    if (rc == OK) rc = check_step(t);
    if (rc != OK) return rc;
    if (!q_heads || q_heads % c->kv_heads) return ERR_INVALID_ARG;
    if (q_heads > 65536) return ERR_BOUNDS;
    return OK;
}

extern "C" uint64_t yvex_b200_attention_paged_workspace_bytes(const yvex_b200_kv_cache *c, const yvex_b200_kv_step *t, uint64_t q_heads) {
    return paged_refusal(c, t, q_heads) == OK ? 256 : 0;
}

extern "C" int yvex_b200_attention_paged(const yvex_b200_kv_cache *c, const yvex_b200_kv_step *t, const void *q, uint64_t q_stride, uint64_t q_heads,
                                         float scale, void *out, void *workspace, uint64_t workspace_bytes, int *status, void *stream) {
    const int rc = paged_refusal(c, t, q_heads);
    if (rc != OK) return rc;
    if (!q || !out || !status || !t->cached || !t->offsets || !t->block_table || (t->tree && !t->ancestors)) return ERR_INVALID_ARG;
    if (!isfinite(scale) || scale <= 0.0f) return ERR_INVALID_ARG;
    if (q_stride < q_heads * c->head_dim) return ERR_BOUNDS;
    if (((uintptr_t)q | (uintptr_t)out) & 15u || q_stride % 8) return ERR_INVALID_ARG;
    if (!workspace || workspace_bytes < yvex_b200_attention_paged_workspace_bytes(c, t, q_heads)) return ERR_NOMEM;
    if ((uintptr_t)workspace & 15u) return ERR_INVALID_ARG;
    PagedParams p{(const uint16_t *)q, (const uint16_t *)c->k, (const uint16_t *)c->v, (uint16_t *)out, q_stride, c->pages, c->page_size, t->table_width,
                  t->requests, t->tokens, t->longest_fresh, t->longest, (uint32_t)c->kv_heads, (uint32_t)(q_heads / c->kv_heads), t->tree != 0, t->cached,
                  t->offsets, t->block_table, t->ancestors, scale, status};
    cudaStream_t s = as_stream(stream);
#define YB_ROWS(T) (c->head_dim == 64 ? launch_rows<T, 64>(p, s) : c->head_dim == 128 ? launch_rows<T, 128>(p, s) : launch_rows<T, 256>(p, s))
    return c->qtype == Q_BF16 ? YB_ROWS(__nv_bfloat16) : YB_ROWS(__half);
#undef YB_ROWS
}
