// Edits of the output head's rows: penalties for words that occurred, biases, grammar masks.
//
// Bound by HBM (8 bytes a word for f32 rows) once there are a few rows, by launch latency for one. A CTA owns a share of the
// vocabulary for several rows. It counts the words of the request's history that fall into its share in shared memory (one 32-bit
// word each: bit 31 occurs in the prompt, bit 30 has a bias, the rest how often it was generated) and lists those that occur at all; the drafted
// words of a row's path are counted in before the row and, for trees, out again after it. Then the row's share streams through with
// nothing but the grammar's mask, and the listed words, a few in a hundred, are edited behind it while their lines are still on the chip.
// (With the edits in the stream nearly every warp met a counted word among its 128 and spent 200 instructions on them: 204 us for 376 rows of
// 129280 words.) Counters are integers, so the order of the atomics does not show. Shares are dealt out in groups of 32 x 16 bytes, one a warp
// at a time: frequent words have low ids, and with shares in one piece the first CTA had most of the edits.
#include "paged.cuh"

namespace yb {

constexpr int kLogitsThreads = 256, kCtas = 4;
constexpr uint32_t kSeen = 1u << 31, kBiased = 1u << 30, kCount = kBiased - 1u;
constexpr int kGroups = 32, kBiases = 256;              // groups of a share, and bias entries that a CTA lists
template <class T> constexpr int kGroupWords = 512 / sizeof(T);

struct LogitsParams {
    yvex_b200_logits_policy p;
    yvex_b200_logits_drafts d;
    const void *logits;
    uint64_t logits_stride;
    const uint32_t *grammar;
    uint64_t grammar_stride;
    void *out;
    uint64_t out_stride;
    uint32_t shares_log2, groups, rows_per_cta;         // groups: of the largest share
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
__global__ void __launch_bounds__(kLogitsThreads, kCtas) logits_edit_kernel(const LogitsParams a) {
    extern __shared__ __align__(16) uint32_t table[];   // counters, then the list of those that are not zero (16 bits each)
    __shared__ int2 biases[kBiases];                    // the share's bias entries: where the word is counted, index of the entry
    __shared__ int bias_count, list_count;
    constexpr int N = LogitsVec<T>::kN, W = kGroupWords<T>, kWarps = kLogitsThreads / 32, kMost = kGroups / kWarps;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t share = blockIdx.x, last_share = (1u << a.shares_log2) - 1u, vocabulary = (uint32_t)a.p.vocabulary;
    uint16_t *list = reinterpret_cast<uint16_t *>(table + a.groups * W);
    const uint64_t first_row = (uint64_t)blockIdx.y * a.rows_per_cta, last_row = min(a.d.rows, first_row + a.rows_per_cta);
    bool bad_arg = false, bad_num = false;
    pdl_trigger();
    pdl_wait();

    // Where word w is counted: -1 in another share (or nowhere: negative words are padding, others are reported).
    auto place = [&](int32_t w) -> int {
        if (w < 0) return -1;
        if ((uint32_t)w >= vocabulary) { bad_arg = true; return -1; }
        const uint32_t g = (uint32_t)w / W;
        return (g & last_share) == share ? (int)((g >> a.shares_log2) * W + (uint32_t)w % W) : -1;
    };
    auto word_at = [&](int i) { return ((((uint32_t)i / W) << a.shares_log2) + share) * W + (uint32_t)i % W; };
    auto noted = [&](int i, uint32_t old) {             // the counter at i was `old` before
        if (!old) list[atomicAdd(&list_count, 1)] = (uint16_t)i;
    };

    // A row's part of the share: group k of the warp begins with word word_at(W * (warp + 8 k)), this lane's 16 bytes of it `skew` words before their
    // place, so that they are aligned. What follows from the skew alone is kept from row to row: the word of k = 0, which k lie within
    // their group and the vocabulary, and whether the mask's bits lie in two words.
    uint4 raw[kMost];
    uint32_t bits[kMost], first_at = 0, whole = 0;
    const uint32_t step = (uint32_t)(kWarps * W) << a.shares_log2;
    const T *in;
    T *out;
    const uint32_t *allowed;
    int skew = -1;
    bool together, two_words = false;
    int64_t r_next = -1;
    uint64_t mask_next = 0;
    auto fetch = [&](uint64_t row) {
        r_next = a.d.row_request ? (int64_t)a.d.row_request[row] : (int64_t)row;
        if (a.d.tree) mask_next = a.d.ancestors[row];
        in = static_cast<const T *>(a.logits) + row * a.logits_stride;
        out = static_cast<T *>(a.out) + row * a.out_stride;
        allowed = a.grammar ? a.grammar + row * a.grammar_stride : nullptr;
        const int off = (int)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % N);
        together = (int)((reinterpret_cast<uintptr_t>(out) / sizeof(T)) % N) == off;      // 16-byte loads and stores fall together
        if (off != skew) {
            skew = off;
            const int e = lane * N - skew;
            first_at = word_at(W * warp) + (uint32_t)e;
            two_words = (first_at & 31u) + N > 32u;
            whole = 0;
#pragma unroll
            for (int k = 0; k < kMost; ++k)
                if (warp + kWarps * k < (int)a.groups && e >= 0 && first_at + k * step + N <= vocabulary) whole |= 1u << k;
        }
        if (!together) return;
#pragma unroll
        for (int k = 0; k < kMost; ++k) {
            if (!((whole >> k) & 1u)) continue;
            const uint32_t at = first_at + k * step;
            raw[k] = *reinterpret_cast<const uint4 *>(in + at);
            if (allowed) {
                bits[k] = allowed[at >> 5] >> (at & 31u);
                if (two_words) bits[k] |= allowed[(at >> 5) + 1u] << (32u - (at & 31u));
            }
        }
    };
    auto masked = [&](float x, uint32_t at) {
        if (allowed && !((allowed[at >> 5] >> (at & 31u)) & 1u)) return -INFINITY;
        bad_num |= x != x;
        return x;
    };

    const bool ragged = vocabulary % N != 0;
    int64_t current = -1, before = -1;                  // the request whose history is in the table, and its row whose chain is
    float rep = 1.0f, presence = 0.0f, frequency = 0.0f;
    int64_t bias_from = 0, bias_to = 0, begin = 0, end = 0;      // its bias entries, its rows
    int node = -1;                                      // where this thread's node of its tree is counted
    if (first_row < last_row) fetch(first_row);
    for (uint64_t row = first_row; row < last_row; ++row) {
        const int64_t r = r_next;
        uint64_t mask = mask_next;
        if (r < 0 || r >= (int64_t)a.p.requests) {
            bad_arg |= r >= 0;
            if (row + 1 < last_row) fetch(row + 1);
            continue;
        }
        const bool fresh = r != current || (a.d.drafted && !a.d.tree && (int64_t)row != before + 1);
        before = (int64_t)row;
        if (fresh) {
            current = r;
            __syncthreads();
            for (uint32_t i = tid; i < a.groups * (W / 4); i += kLogitsThreads) reinterpret_cast<uint4 *>(table)[i] = make_uint4(0, 0, 0, 0);
            if (tid == 0) { bias_count = 0; list_count = 0; }
            __syncthreads();
            if (a.p.history) {
                const int64_t from = a.p.history_offsets[r], to = a.p.history_offsets[r + 1];
                const int64_t prompt = from + (a.p.prompt_lengths ? max(a.p.prompt_lengths[r], 0) : 0);
                const bool sound = from >= 0 && to >= from && to <= (int64_t)a.p.history_tokens;
                bad_arg |= !sound;
                for (int64_t t0 = from + tid; sound && t0 < to; t0 += 8 * kLogitsThreads) {
                    int32_t w[8];                       // (eight words on their way at a time)
#pragma unroll
                    for (int q = 0; q < 8; ++q) w[q] = t0 + q * kLogitsThreads < to ? a.p.history[t0 + q * kLogitsThreads] : -1;
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const int i = place(w[q]);
                        if (i < 0) continue;
                        if (t0 + q * kLogitsThreads >= prompt) noted(i, atomicAdd(&table[i], 1u));
                        else if (!(table[i] & kSeen)) noted(i, atomicOr(&table[i], kSeen));
                    }
                }
            }
            if (a.p.bias_tokens) {
                const int64_t from = a.p.bias_offsets[r], to = a.p.bias_offsets[r + 1];
                const bool sound = from >= 0 && to >= from && to <= (int64_t)a.p.bias_entries;
                bad_arg |= !sound;
                bias_from = sound ? from : 0;
                bias_to = sound ? to : 0;
                for (int64_t t = bias_from + tid; t < bias_to; t += kLogitsThreads) {
                    const int i = place(a.p.bias_tokens[t]);
                    if (i < 0) continue;
                    noted(i, atomicOr(&table[i], kBiased));
                    const int n = atomicAdd(&bias_count, 1);
                    if (n < kBiases) biases[n] = make_int2(i, (int)t);
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
            node = a.d.tree && tid < end - begin && tid < YVEX_B200_TREE_NODES ? place(a.d.drafted[begin + tid]) : -1;
            __syncthreads();
        }
        // ---- the row's path
        const bool has_path = a.d.drafted && (int64_t)row >= begin && (int64_t)row < end, goes = has_path && a.d.tree;
        bad_arg |= a.d.drafted && !has_path;
        const int lasting = list_count;
        const bool mine = goes && node >= 0 && (mask >> tid) & 1ull;      // this thread's node is on the path
        if (has_path) {
            __syncthreads();                            // (`lasting` has been read)
            if (a.d.tree) {
                if (mine) noted(node, atomicAdd(&table[node], 1u));
            } else {
                for (int64_t i = fresh ? begin + tid : tid == 0 ? (int64_t)row : end; i <= (int64_t)row; i += kLogitsThreads) {
                    const int at = place(a.d.drafted[i]);      // (the row before was the chain's word before this one)
                    if (at >= 0) noted(at, atomicAdd(&table[at], 1u));
                }
            }
        }

        if (has_path) __syncthreads();
        // (the first of this thread's listed words is on its way while the row streams)
        const int n = list_count, first = tid < n ? list[tid] : 0;
        const T ahead = in[tid < n ? word_at(first) : 0u];
        // ---- the row but for the listed words
        if (together) {
#pragma unroll
            for (int k = 0; k < kMost; ++k) {
                if (!((whole >> k) & 1u)) continue;
                float x[N];
                LogitsVec<T>::open(raw[k], x);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (allowed && !((bits[k] >> i) & 1u)) x[i] = -INFINITY;
                    bad_num |= x[i] != x[i];
                }
                *reinterpret_cast<uint4 *>(out + (first_at + k * step)) = LogitsVec<T>::close(x);
            }
        }
        if (skew || !together || ragged)                // the edges of groups, and rows that are aligned in one place only
            for (int k = 0; k < kMost; ++k) {
                const uint32_t g = word_at(W * (warp + kWarps * k));
                if (warp + kWarps * k >= (int)a.groups || g >= vocabulary) continue;
                // (words of the group that the lanes above did not take)
                for (int i = lane; i < W && g + (uint32_t)i < vocabulary; i += 32) {
                    const int e = (i + skew) / N * N - skew;      // where the 16 bytes of word i begin
                    if (together && e >= 0 && e + N <= W && g + (uint32_t)(e + N) <= vocabulary) continue;
                    LogitsVec<T>::put(out + g + i, masked(LogitsVec<T>::get(in + g + i), g + i));
                }
            }
        __syncthreads();
        // ---- the listed words (in place, the stream has left them as they were, or -inf where the grammar forbids them)
        for (int t = tid; t < n; t += kLogitsThreads) {
            const int i = t == tid ? first : list[t];
            const uint32_t w = table[i], at = word_at(i), times = w & kCount;
            float x = t == tid ? LogitsVec<T>::get(&ahead) : LogitsVec<T>::get(in + at);
            if (w & (kSeen | kCount)) {
                x = x > 0.0f ? x / rep : x * rep;
                if (times) x -= frequency * (float)times + presence;
            }
            if (w & kBiased) {                          // the last entry of a word counts
                int last = -1;
                if (bias_count <= kBiases) {
                    for (int b = 0; b < bias_count; ++b) if (biases[b].x == i) last = max(last, biases[b].y);
                } else {                                // more than the list holds
                    for (int64_t b = bias_to - 1; b >= bias_from && last < 0; --b) if (place(a.p.bias_tokens[b]) == i) last = (int)b;
                }
                x += a.p.bias_values[last];
            }
            LogitsVec<T>::put(out + at, masked(x, at));
        }
        if (row + 1 < last_row) fetch(row + 1);
        __syncthreads();
        if (goes) {
            if (mine) atomicSub(&table[node], 1u);
            if (tid == 0) list_count = lasting;
            __syncthreads();
        }
    }
    if (bad_arg) raise(a.status, YVEX_B200_STATUS_ARGUMENT);
    if (bad_num) raise(a.status, YVEX_B200_STATUS_NUMERIC);
}

template <class T> static int launch_logits(LogitsParams &a, cudaStream_t s) {
    // As few shares as hold the vocabulary in their tables, for one or a few rows as many as there are SMs; then as many rows a
    // CTA as let all of them run at once.
    static SmemOptIn optin;
    constexpr uint64_t W = kGroupWords<T>;
    const uint64_t groups = (a.p.vocabulary + W - 1) / W;
    a.shares_log2 = 0;
    while ((groups + (1ull << a.shares_log2) - 1) >> a.shares_log2 > (uint64_t)kGroups) ++a.shares_log2;
    while ((a.d.rows << a.shares_log2) * 2 <= kSmCount && groups > 1ull << a.shares_log2) ++a.shares_log2;
    const uint64_t shares = 1ull << a.shares_log2, slots = (uint64_t)kSmCount * kCtas, want = slots > shares ? slots / shares : 1;
    a.groups = (uint32_t)((groups + shares - 1) / shares);
    a.rows_per_cta = (uint32_t)((a.d.rows + want - 1) / want);
    const uint64_t least = (a.d.rows + 65534) / 65535;
    if (a.rows_per_cta < least) a.rows_per_cta = (uint32_t)least;
    if (shares > INT32_MAX) return ERR_BOUNDS;
    constexpr size_t most = (size_t)kGroups * W * (sizeof(uint32_t) + sizeof(uint16_t));
    const size_t smem = (size_t)a.groups * W * (sizeof(uint32_t) + sizeof(uint16_t));
    const int rc = optin.ensure(logits_edit_kernel<T>, (int)most);
    if (rc != OK) return rc;
    const uint64_t chunks = (a.d.rows + a.rows_per_cta - 1) / a.rows_per_cta;
    if (launch_pdl(logits_edit_kernel<T>, dim3((unsigned)shares, (unsigned)chunks), dim3(kLogitsThreads), smem, s, a) != cudaSuccess) return ERR_BACKEND;
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
    LogitsParams a{*p, *d, logits, logits_stride, grammar, grammar_stride, out, out_stride, 0, 0, 0, status};
    cudaStream_t s = as_stream(stream);
    return qtype == Q_F32 ? launch_logits<float>(a, s) : qtype == Q_BF16 ? launch_logits<__nv_bfloat16>(a, s) : launch_logits<__half>(a, s);
}
