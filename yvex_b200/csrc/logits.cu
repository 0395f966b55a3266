// Edits of the output head's rows: penalties for words that occurred, biases, grammar masks.
//
// One pass over the logits, bound by HBM (8 bytes a word for f32 rows) once there are a few rows, by launch latency for one. A CTA
// owns a slice of the vocabulary for several rows: it counts the words of the request's history that fall into its slice in
// shared memory (one 32-bit word each: bit 31 occurs in the prompt, bit 30 has a bias, the rest how often it was generated),
// then streams the rows' slices; the drafted words of a row's path are counted in before the row and, for trees, out again after
// it. Counters are integers, so the order of the atomics does not show. Nearly every word has a zero counter: those only
// meet the grammar's bit.
#include "paged.cuh"

namespace yb {

constexpr int kLogitsThreads = 256;
constexpr uint32_t kSeen = 1u << 31, kBiased = 1u << 30, kCount = kBiased - 1u;
constexpr uint32_t kLeastSlice = 1024, kMostSlice = 4096;

struct LogitsParams {
    yvex_b200_logits_policy p;
    yvex_b200_logits_drafts d;
    const void *logits;
    uint64_t logits_stride;
    const uint32_t *grammar;
    uint64_t grammar_stride;
    void *out;
    uint64_t out_stride;
    uint32_t slice, rows_per_cta;
    int *status;
};

template <class T> struct LogitsVec {
    static constexpr int kN = 16 / sizeof(T);
    __device__ static void open(const uint4 &w, float (&x)[kN]) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                x[i] = __uint_as_float(v[i]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&v[i]));
                x[2 * i] = f.x; x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(v[i] << 16); x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
            }
        }
    }
    __device__ static uint4 close(const float (&x)[kN]) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __float_as_uint(x[i]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                v[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                v[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        return make_uint4(v[0], v[1], v[2], v[3]);
    }
    __device__ static float get(const T *p) {
        if constexpr (sizeof(T) == 4) return *p;
        else if constexpr (std::is_same<T, __half>::value) return __half2float(*p);
        else return __bfloat162float(*p);
    }
    __device__ static void put(T *p, float x) {
        if constexpr (sizeof(T) == 4) *p = x;
        else if constexpr (std::is_same<T, __half>::value) *p = __float2half_rn(x);
        else *p = __float2bfloat16_rn(x);
    }
};

template <class T>
__global__ void __launch_bounds__(kLogitsThreads) logits_edit_kernel(const LogitsParams a) {
    extern __shared__ uint32_t table[];                 // [slice] counters, then [slice] index of the bias entry + 1
    constexpr int N = LogitsVec<T>::kN, kInFlight = 4;
    const int tid = threadIdx.x;
    const int64_t lo = (int64_t)blockIdx.x * a.slice, hi = min((int64_t)a.p.vocabulary, lo + a.slice);
    const uint32_t words = (uint32_t)(hi - lo);
    uint32_t *bias_at = table + a.slice;
    const uint64_t first_row = (uint64_t)blockIdx.y * a.rows_per_cta, last_row = min(a.d.rows, first_row + a.rows_per_cta);
    bool bad_arg = false, bad_num = false;
    pdl_trigger();
    pdl_wait();

    // counts word w in (or out); whether it is one at all
    auto count = [&](int64_t w, bool in) {
        if (w >= (int64_t)a.p.vocabulary) { bad_arg = true; return; }
        if (w < lo || w >= hi) return;
        if (in) atomicAdd(&table[w - lo], 1u); else atomicSub(&table[w - lo], 1u);
    };

    int64_t current = -1, before = -1;                  // the request whose history is in the table, and its row whose chain is
    float rep = 1.0f, presence = 0.0f, frequency = 0.0f;
    int64_t begin = 0, end = 0;                         // its rows
    for (uint64_t row = first_row; row < last_row; ++row) {
        const int64_t r = a.d.row_request ? (int64_t)a.d.row_request[row] : (int64_t)row;
        if (r < 0) continue;
        if (r >= (int64_t)a.p.requests) { bad_arg = true; continue; }
        const bool fresh = r != current || (a.d.drafted && !a.d.tree && (int64_t)row != before + 1);
        before = (int64_t)row;
        if (fresh) {
            current = r;
            __syncthreads();
            for (uint32_t i = tid; i < words; i += kLogitsThreads) {
                table[i] = 0u;
                if (a.p.bias_tokens) bias_at[i] = 0u;
            }
            __syncthreads();
            if (a.p.history) {
                const int64_t from = a.p.history_offsets[r], to = a.p.history_offsets[r + 1];
                const int64_t prompt = from + (a.p.prompt_lengths ? max(a.p.prompt_lengths[r], 0) : 0);
                const bool sound = from >= 0 && to >= from && to <= (int64_t)a.p.history_tokens;
                bad_arg |= !sound;
                for (int64_t i = from + tid; sound && i < to; i += kLogitsThreads) {
                    const int64_t w = a.p.history[i];
                    if (w >= (int64_t)a.p.vocabulary) bad_arg = true;
                    else if (w >= lo && w < hi) {
                        if (i >= prompt) atomicAdd(&table[w - lo], 1u);
                        else if (!(table[w - lo] & kSeen)) atomicOr(&table[w - lo], kSeen);
                    }
                }
            }
            if (a.p.bias_tokens) {
                const int64_t from = a.p.bias_offsets[r], to = a.p.bias_offsets[r + 1];
                const bool sound = from >= 0 && to >= from && to <= (int64_t)a.p.bias_entries;
                bad_arg |= !sound;
                for (int64_t i = from + tid; sound && i < to; i += kLogitsThreads) {
                    const int64_t w = a.p.bias_tokens[i];
                    if (w >= (int64_t)a.p.vocabulary) bad_arg = true;
                    else if (w >= lo && w < hi) {
                        atomicOr(&table[w - lo], kBiased);
                        atomicMax(&bias_at[w - lo], (uint32_t)(i - from) + 1u);     // the last entry of a word counts
                    }
                }
            }
            rep = a.p.repetition ? a.p.repetition[r] : 1.0f;
            if (!(rep > 0.0f) || isinf(rep)) { bad_arg = true; rep = 1.0f; }
            presence = a.p.presence ? a.p.presence[r] : 0.0f;
            frequency = a.p.frequency ? a.p.frequency[r] : 0.0f;
            begin = end = 0;
            if (a.d.drafted) {
                begin = a.d.offsets[r];
                end = a.d.offsets[r + 1];
                if (begin < 0 || end < begin || end > (int64_t)a.d.rows) { bad_arg = true; begin = end = 0; }
            }
        }
        // ---- the row's path
        const int64_t index = (int64_t)row - begin;
        const bool has_path = a.d.drafted && index >= 0 && (int64_t)row < end;
        bad_arg |= a.d.drafted && !has_path;
        uint64_t mask = 0;
        if (has_path) {
            if (a.d.tree) {
                mask = a.d.ancestors[row];
                if (end - begin < 64) mask &= (1ull << (end - begin)) - 1ull;
                if (tid < 64 && (mask >> tid) & 1ull) count(a.d.drafted[begin + tid], true);
            } else if (fresh) {
                for (int64_t i = begin + tid; i <= (int64_t)row; i += kLogitsThreads) count(a.d.drafted[i], true);
            } else if (tid == 0) {
                count(a.d.drafted[row], true);          // the row before was the chain's word before this one
            }
        }
        __syncthreads();

        // ---- the row
        const T *in = static_cast<const T *>(a.logits) + row * a.logits_stride;
        T *out = static_cast<T *>(a.out) + row * a.out_stride;
        const uint32_t *allowed = a.grammar ? a.grammar + row * a.grammar_stride : nullptr;
        auto edit = [&](float x, uint32_t w, int64_t e) {
            if (w) {
                if (w & (kSeen | kCount)) {
                    x = x > 0.0f ? x / rep : x * rep;
                    const uint32_t n = w & kCount;
                    if (n) x -= frequency * (float)n + presence;
                }
                if (w & kBiased) x += a.p.bias_values[(int64_t)a.p.bias_offsets[r] + bias_at[e - lo] - 1u];
            }
            return x;
        };
        const int64_t skew = (int64_t)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % N);
        const bool together = (reinterpret_cast<uintptr_t>(out) / sizeof(T)) % N == (uint64_t)skew;     // 16-byte loads and stores fall together
        const int64_t e0 = lo - (lo + skew) % N;
        for (int64_t eb = e0 + (int64_t)tid * N; eb < hi; eb += (int64_t)kLogitsThreads * N * kInFlight) {
            uint4 raw[kInFlight];
            uint32_t bits[kInFlight];
#pragma unroll
            for (int j = 0; j < kInFlight; ++j) {
                const int64_t e = eb + (int64_t)j * kLogitsThreads * N;
                if (together && e >= lo && e + N <= hi) {
                    raw[j] = __ldcs(reinterpret_cast<const uint4 *>(in + e));
                    bits[j] = ~0u;
                    if (allowed) {
                        const uint32_t s = (uint32_t)e & 31u;
                        bits[j] = allowed[e >> 5] >> s;
                        if (s + N > 32u) bits[j] |= allowed[(e >> 5) + 1] << (32u - s);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kInFlight; ++j) {
                const int64_t e = eb + (int64_t)j * kLogitsThreads * N;
                if (together && e >= lo && e + N <= hi) {
                    float x[N];
                    uint32_t w[N];
                    LogitsVec<T>::open(raw[j], x);
                    uint32_t any = 0;
#pragma unroll
                    for (int i = 0; i < N; ++i) { w[i] = table[e - lo + i]; any |= w[i]; }
                    if (any) {
#pragma unroll
                        for (int i = 0; i < N; ++i) x[i] = edit(x[i], w[i], e + i);
                    }
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        if (!((bits[j] >> i) & 1u)) x[i] = -INFINITY;
                        bad_num |= x[i] != x[i];
                    }
                    __stcs(reinterpret_cast<uint4 *>(out + e), LogitsVec<T>::close(x));
                } else {
                    for (int i = 0; i < N; ++i) {
                        const int64_t ei = e + i;
                        if (ei < lo || ei >= hi) continue;
                        float x = edit(LogitsVec<T>::get(in + ei), table[ei - lo], ei);
                        if (allowed && !((allowed[ei >> 5] >> (ei & 31)) & 1u)) x = -INFINITY;
                        bad_num |= x != x;
                        LogitsVec<T>::put(out + ei, x);
                    }
                }
            }
        }
        if (has_path && a.d.tree) {
            __syncthreads();
            if (tid < 64 && (mask >> tid) & 1ull) count(a.d.drafted[begin + tid], false);
        }
        __syncthreads();
    }
    if (bad_arg) raise(a.status, YVEX_B200_STATUS_ARGUMENT);
    if (bad_num) raise(a.status, YVEX_B200_STATUS_NUMERIC);
}

template <class T> static int launch_logits(const LogitsParams &a, cudaStream_t s) {
    static SmemOptIn optin;
    const int smem = (int)(a.slice * sizeof(uint32_t) * (a.p.bias_tokens ? 2 : 1));
    const int rc = optin.ensure(logits_edit_kernel<T>, (int)(kMostSlice * 2 * sizeof(uint32_t)));
    if (rc != OK) return rc;
    const uint64_t slices = (a.p.vocabulary + a.slice - 1) / a.slice, chunks = (a.d.rows + a.rows_per_cta - 1) / a.rows_per_cta;
    if (launch_pdl(logits_edit_kernel<T>, dim3((unsigned)slices, (unsigned)chunks), dim3(kLogitsThreads), (size_t)smem, s, a) != cudaSuccess) return ERR_BACKEND;
    return launch_status(1);
}

}  // namespace yb

using namespace yb;

extern "C" int yvex_b200_logits_edit(const yvex_b200_logits_policy *p, const yvex_b200_logits_drafts *d, unsigned int qtype, const void *logits,
                                     uint64_t logits_stride, const uint32_t *grammar, uint64_t grammar_stride, void *out, uint64_t out_stride,
                                     int *status, void *stream) {
    if (!p || !d || !logits || !out || !status || !p->vocabulary || !p->requests || !d->rows) return ERR_INVALID_ARG;
    if (qtype != Q_F32 && qtype != Q_F16 && qtype != Q_BF16) return ERR_UNSUPPORTED;
    if (p->vocabulary > INT32_MAX || p->requests >= INT32_MAX || d->rows >= INT32_MAX || p->history_tokens > INT32_MAX || p->bias_entries > INT32_MAX)
        return ERR_BOUNDS;
    if (logits_stride < p->vocabulary || out_stride < p->vocabulary || (grammar && grammar_stride < (p->vocabulary + 31) / 32)) return ERR_BOUNDS;
    if ((p->history && !p->history_offsets) || (p->bias_tokens && (!p->bias_values || !p->bias_offsets))) return ERR_INVALID_ARG;
    if (!d->row_request && d->rows > p->requests) return ERR_BOUNDS;
    if (d->drafted && (!d->offsets || !d->row_request || (d->tree && !d->ancestors))) return ERR_INVALID_ARG;
    const uintptr_t size = qtype == Q_F32 ? 4 : 2;
    if (((uintptr_t)logits | (uintptr_t)out) % size || (uintptr_t)grammar % 4) return ERR_INVALID_ARG;
    LogitsParams a{*p, *d, logits, logits_stride, grammar, grammar_stride, out, out_stride, 0, 0, status};
    // A slice for every SM while the vocabulary gives them, then as many rows per slice as fill the chip a few times over.
    const uint64_t even = (p->vocabulary + kSmCount - 1) / kSmCount, unit = 256;
    uint64_t slice = (even + unit - 1) / unit * unit;
    slice = d->rows > 4 ? kMostSlice : slice < kLeastSlice ? kLeastSlice : slice > kMostSlice ? kMostSlice : slice;
    a.slice = (uint32_t)slice;
    const uint64_t slices = (p->vocabulary + slice - 1) / slice, want = ((uint64_t)kSmCount * 6 + slices - 1) / slices;
    a.rows_per_cta = (uint32_t)((d->rows + want - 1) / want);
    if ((d->rows + a.rows_per_cta - 1) / a.rows_per_cta > 65535) a.rows_per_cta = (uint32_t)((d->rows + 65534) / 65535);
    cudaStream_t s = as_stream(stream);
    return qtype == Q_F32 ? launch_logits<float>(a, s) : qtype == Q_BF16 ? launch_logits<__nv_bfloat16>(a, s) : launch_logits<__half>(a, s);
}
