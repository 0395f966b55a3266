// Edits of the output head's rows: penalties for words that occurred, biases, grammar masks.
//
// Two kernels. The first streams the rows through with nothing but the grammar's mask: bound by HBM (8 bytes a word for f32 rows). The
// second edits the words that occur in a request's history, on a row's path or among its biases, a few in a hundred, in place: a CTA
// takes several rows of a request, counts its words in a hash table in shared memory (key, and one 32-bit counter: bit 31 occurs in the
// prompt, the rest how often it was generated), and then visits the table's words for every row. Biased words enter the table first, so that they are
// the first of its list and their last entries an array beside it (a place for them in every slot, 229 KB of shared memory in place of 160, took 24 us
// more at 419 rows). With few rows the table is built while the
// stream runs; with many the two follow one another, since an edit CTA's registers (57344 of an SM's 65536) only fit an SM that the stream has left.
// Counters are integers, so the order of the atomics does not show. Requests with more words than the table holds are done in
// parts of the words, halved until they fit. (One kernel with counters for a share of the vocabulary and the edits in the stream took 204 us for
// 419 rows of 129280 words, with the edits behind the stream 175: nearly every warp meets a counted word among its 128, and every share
// of the vocabulary counts the whole history.) Now 148 with one set of inputs, 152 with three: the stream 92 (435 MB, 4.7 TB/s), the edits 56. One row
// is 7.9 us of device time, two launches; as one kernel it took 6, but there is no rule yet that would choose that form for few rows.
#include "paged.cuh"

namespace yb {

constexpr int kStreamThreads = 256, kStreamLoads = 4, kStreamCtas = 4;      // of the stream: loads of 16 bytes, CTAs an SM
constexpr int kEditThreads = 1024, kEditsAhead = 4;       // of the edits: words a thread has on their way
constexpr uint32_t kSeen = 1u << 31, kCount = kSeen - 1u;
constexpr uint32_t kLeastTable = 1024, kMostTable = 16384, kFewBiased = 2560, kMostBiased = 8192;      // slots; biased words of a table

struct LogitsParams {
    yvex_b200_logits_policy p;
    yvex_b200_logits_drafts d;
    const void *logits;
    uint64_t logits_stride;
    const uint32_t *grammar;
    uint64_t grammar_stride;
    void *out;
    uint64_t out_stride;
    uint32_t table_log2, biased, rows_per_cta;         // biased: places for biased words
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

// The request of a row; -1 for a row that is left alone.
__device__ __forceinline__ int64_t request_of(const LogitsParams &a, uint64_t row, bool &bad) {
    const int64_t r = a.d.row_request ? (int64_t)a.d.row_request[row] : (int64_t)row;
    bad |= r >= (int64_t)a.p.requests;
    return r < (int64_t)a.p.requests ? r : -1;
}
__device__ __forceinline__ bool allows(const uint32_t *allowed, uint32_t word) { return !allowed || (allowed[word >> 5] >> (word & 31u)) & 1u; }

// blockIdx.x: a piece of a row, blockIdx.y: the rows. What the edits need besides the rows is complete when this kernel lets them start.
template <class T>
__global__ void __launch_bounds__(kStreamThreads, kStreamCtas) logits_stream_kernel(const LogitsParams a) {
    constexpr int N = LogitsVec<T>::kN, kPiece = kStreamThreads * kStreamLoads * N;
    pdl_wait();
    pdl_trigger();
    const uint32_t vocabulary = (uint32_t)a.p.vocabulary, lo = blockIdx.x * (uint32_t)kPiece, hi = min(vocabulary, lo + (uint32_t)kPiece);
    bool bad_arg = false, bad_num = false;
    for (uint64_t row = blockIdx.y; row < a.d.rows; row += gridDim.y) {
        const int64_t r = request_of(a, row, bad_arg);          // (looked at when the row's loads are on their way)
        const T *in = static_cast<const T *>(a.logits) + row * a.logits_stride + lo;
        T *out = static_cast<T *>(a.out) + row * a.out_stride + lo;
        const uint32_t *allowed = a.grammar ? a.grammar + row * a.grammar_stride : nullptr;
        const int skew = (int)((reinterpret_cast<uintptr_t>(in) / sizeof(T)) % N), words = (int)(hi - lo);
        const bool together = (int)((reinterpret_cast<uintptr_t>(out) / sizeof(T)) % N) == skew;      // 16-byte loads and stores fall together
        auto one = [&](int e) {
            float x = LogitsVec<T>::get(in + e);
            if (!allows(allowed, lo + (uint32_t)e)) x = -INFINITY;
            bad_num |= x != x;
            LogitsVec<T>::put(out + e, x);
        };
        if (!together) {
            for (int e = threadIdx.x; e < words && r >= 0; e += kStreamThreads) one(e);
            continue;
        }
        uint4 raw[kStreamLoads];
        uint32_t bits[kStreamLoads];
        const int first = (int)threadIdx.x * N - skew;
        const uint32_t shift = (lo + (uint32_t)first) & 31u;    // (the same for all of the thread's loads)
        const uint32_t *mask = allowed ? allowed + (((int64_t)lo + first) >> 5) : nullptr;
#pragma unroll
        for (int j = 0; j < kStreamLoads; ++j) {
            const int e = first + j * kStreamThreads * N;
            if (e < 0 || e + N > words) continue;
            raw[j] = __ldcs(reinterpret_cast<const uint4 *>(in + e));
            if (allowed) {
                bits[j] = mask[j * (kStreamThreads * N / 32)] >> shift;
                if (shift + N > 32u) bits[j] |= mask[j * (kStreamThreads * N / 32) + 1] << (32u - shift);
            }
        }
        if (r < 0) continue;
#pragma unroll
        for (int j = 0; j < kStreamLoads; ++j) {
            const int e = first + j * kStreamThreads * N;
            if (e >= 0 && e + N <= words) {
                float x[N];
                LogitsVec<T>::open(raw[j], x);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (allowed && !((bits[j] >> i) & 1u)) x[i] = -INFINITY;
                    bad_num |= x[i] != x[i];
                }
                __stcg(reinterpret_cast<uint4 *>(out + e), LogitsVec<T>::close(x));
            } else {
                for (int i = max(e, 0); i < min(e + N, words); ++i) one(i);
            }
        }
        if (skew && (int)threadIdx.x < skew && kPiece - skew + (int)threadIdx.x < words) one(kPiece - skew + (int)threadIdx.x);
    }
    if (bad_arg) raise(a.status, YVEX_B200_STATUS_ARGUMENT);
    if (bad_num) raise(a.status, YVEX_B200_STATUS_NUMERIC);
}

// blockIdx.x: the rows, blockIdx.y of gridDim.y (a power of two): the words.
template <class T>
__global__ void __launch_bounds__(kEditThreads) logits_edit_kernel(const LogitsParams a) {
    extern __shared__ __align__(16) uint32_t keys[];    // words (~0: none), their counters, the list of those in use, the last bias entries of the list's first
    __shared__ int list_count;
    const int tid = threadIdx.x;
    const uint32_t slots = 1u << a.table_log2, limit = slots / 4 * 3, vocabulary = (uint32_t)a.p.vocabulary;
    uint32_t *counters = keys + slots;
    uint16_t *list = reinterpret_cast<uint16_t *>(counters + slots);
    int *last_bias = reinterpret_cast<int *>(list + limit);
    const uint64_t first_row = (uint64_t)blockIdx.x * a.rows_per_cta, last_row = min(a.d.rows, first_row + a.rows_per_cta);
    bool bad_arg = false, bad_num = false, waited = false;
    uint32_t parts = gridDim.y, part = blockIdx.y;      // words of that part are in the table

    auto hash = [](uint32_t w) { return w * 0x9E3779B1u; };
    // Parts nest: of a power of two of them, part p falls into 2p and 2p + 1 of twice as many, whatever the words are. The high bits of a
    // second hash say which, so that neither a step between the words (their low bits alone make the low bits of the first) nor
    // the place in the table, which the first one's high bits give, tells the part.
    auto part_of = [&](uint32_t h) { return __umulhi(hash(h ^ (h >> 15)), parts); };
    // The slot of word w, which is entered if it is not there (`numbered`: with its place in the list as its counter); -1 for padding, words of
    // other parts, and when the table is full.
    auto slot_of = [&](int32_t w, bool numbered) -> int {
        if (w < 0) return -1;
        if ((uint32_t)w >= vocabulary) { bad_arg = true; return -1; }
        const uint32_t h = hash((uint32_t)w);
        if (parts != 1u && part_of(h) != part) return -1;
        uint32_t s = h >> (32u - a.table_log2);
        for (uint32_t tries = 0; tries < slots; ++tries, s = (s + 1u) & (slots - 1u)) {
            uint32_t k = *(volatile uint32_t *)&keys[s];
            if (k == ~0u) {
                if (*(volatile int *)&list_count >= (int)limit) { list_count = (int)limit + 1; return -1; }
                k = atomicCAS(&keys[s], ~0u, (uint32_t)w);
                if (k == ~0u) {                         // (one addition for the lanes that got here together: thousands on one word would queue)
                    const uint32_t m = __activemask(), leader = (uint32_t)__ffs((int)m) - 1u, lane = (uint32_t)tid & 31u;
                    int n = 0;
                    if (lane == leader) n = atomicAdd(&list_count, __popc(m));
                    n = __shfl_sync(m, n, (int)leader) + __popc(m & ((1u << lane) - 1u));
                    if (n < (int)limit) list[n] = (uint16_t)s;
                    if (numbered) counters[s] = (uint32_t)n;
                    return (int)s;
                }
            }
            if (k == (uint32_t)w) return (int)s;
        }
        return -1;
    };

    uint64_t row = first_row;
    while (row < last_row) {
        // ---- the rows of one request
        const int64_t r = request_of(a, row, bad_arg);
        if (r < 0) { ++row; continue; }
        uint64_t stop = row + 1;
        while (stop < last_row && request_of(a, stop, bad_arg) == r) ++stop;
        float rep = a.p.repetition ? a.p.repetition[r] : 1.0f;
        if (!(rep > 0.0f) || isinf(rep)) { bad_arg = true; rep = 1.0f; }
        const float presence = a.p.presence ? a.p.presence[r] : 0.0f, frequency = a.p.frequency ? a.p.frequency[r] : 0.0f;
        int64_t begin = 0, end = 0, from = 0, to = 0, bias_from = 0, bias_to = 0;
        if (a.d.drafted) {
            begin = a.d.offsets[r];
            end = a.d.offsets[r + 1];
            if (begin < 0 || end < begin || end > (int64_t)a.d.rows || (int64_t)row < begin || (int64_t)stop > end) { bad_arg = true; begin = end = 0; }
        }
        if (a.p.history) {
            from = a.p.history_offsets[r];
            to = a.p.history_offsets[r + 1];
            if (from < 0 || to < from || to > (int64_t)a.p.history_tokens) { bad_arg = true; from = to = 0; }
        }
        const int64_t prompt = from + (a.p.prompt_lengths ? max(a.p.prompt_lengths[r], 0) : 0);
        if (a.p.bias_tokens) {
            bias_from = a.p.bias_offsets[r];
            bias_to = a.p.bias_offsets[r + 1];
            if (bias_from < 0 || bias_to < bias_from || bias_to > (int64_t)a.p.bias_entries) { bad_arg = true; bias_from = bias_to = 0; }
        }
        const int64_t paths_end = a.d.tree ? min(end, begin + YVEX_B200_TREE_NODES) : min(end, (int64_t)stop);      // words that a path may have

        const int32_t first_biased = bias_from + tid < bias_to ? a.p.bias_tokens[bias_from + tid] : -1;      // (on its way while the table is cleared)
        parts = gridDim.y;
        part = blockIdx.y;
        for (;;) {
            // ---- the table
            __syncthreads();
            for (uint32_t i = tid; i < slots / 2; i += kEditThreads)
                reinterpret_cast<uint4 *>(keys)[i] = i < slots / 4 ? make_uint4(~0u, ~0u, ~0u, ~0u) : make_uint4(0, 0, 0, 0);
            for (uint32_t i = tid; i < a.biased; i += kEditThreads) last_bias[i] = -1;
            if (tid == 0) list_count = 0;
            __syncthreads();
            int biased = 0;                             // the list's words up to here have biases
            if (bias_to > bias_from) {
                const int first = slot_of(first_biased, true);
                for (int64_t t = bias_from + tid + kEditThreads; t < bias_to; t += kEditThreads) slot_of(a.p.bias_tokens[t], true);
                __syncthreads();
                biased = list_count;
                if (biased > (int)min(limit, a.biased)) { parts *= 2u; part *= 2u; continue; }      // too many words: half of them first
                if (first >= 0) atomicMax(&last_bias[counters[first]], (int)(bias_from + tid));
                for (int64_t t = bias_from + tid + kEditThreads; t < bias_to; t += kEditThreads) {
                    const int s = slot_of(a.p.bias_tokens[t], true);      // (every word is there now)
                    if (s >= 0) atomicMax(&last_bias[counters[s]], (int)t);
                }
                __syncthreads();
                for (int i = tid; i < biased; i += kEditThreads) counters[list[i]] = 0;
                __syncthreads();
            }
            for (int64_t t0 = from + tid; t0 < to; t0 += 4 * kEditThreads) {
                int32_t w[4];                           // (four words on their way at a time)
#pragma unroll
                for (int q = 0; q < 4; ++q) w[q] = t0 + q * kEditThreads < to ? a.p.history[t0 + q * kEditThreads] : -1;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int s = slot_of(w[q], false);
                    if (s < 0) continue;
                    if (t0 + q * kEditThreads >= prompt) atomicAdd(&counters[s], 1u);
                    else if (!(counters[s] & kSeen)) atomicOr(&counters[s], kSeen);
                }
            }
            // drafted words have their slots before the first row; a tree's nodes keep a thread each
            int node = -1;
            for (int64_t t = begin + tid; t < paths_end; t += kEditThreads) {
                const int s = slot_of(a.d.drafted[t], false);
                if (a.d.tree) node = s;
                else if (t < (int64_t)row && s >= 0) atomicAdd(&counters[s], 1u);      // (the chain before the first row)
            }
            __syncthreads();
            const int n = list_count;
            if (n > (int)limit) { parts *= 2u; part *= 2u; continue; }

            if (!waited) { pdl_wait(); waited = true; }                     // the stream has written the rows
            for (uint64_t t = row; t < stop; ++t) {
                const T *in = static_cast<const T *>(a.logits) + t * a.logits_stride;
                T *out = static_cast<T *>(a.out) + t * a.out_stride;
                const uint32_t *allowed = a.grammar ? a.grammar + t * a.grammar_stride : nullptr;
                bool on = false;                        // this thread's node is on the path
                if (a.d.drafted && end > begin) {
                    if (a.d.tree) on = node >= 0 && (a.d.ancestors[t] >> tid) & 1ull;
                    else if (tid == 0) node = slot_of(a.d.drafted[t], false), on = node >= 0;
                    if (on) atomicAdd(&counters[node], 1u);
                    __syncthreads();
                }
                for (int i0 = tid; i0 < n; i0 += kEditsAhead * kEditThreads) {
                    float x[kEditsAhead];
                    int slot[kEditsAhead];
#pragma unroll
                    for (int q = 0; q < kEditsAhead; ++q) {     // (in place, the stream has left the words as they were, or -inf where the grammar forbids them)
                        const int i = i0 + q * kEditThreads;
                        slot[q] = i < n ? list[i] : -1;
                        if (slot[q] >= 0 && i >= biased && !counters[slot[q]]) slot[q] = -1;
                        if (slot[q] >= 0) x[q] = LogitsVec<T>::get(in + keys[slot[q]]);
                    }
#pragma unroll
                    for (int q = 0; q < kEditsAhead; ++q) {
                        const int s = slot[q];
                        if (s < 0) continue;
                        const uint32_t c = counters[s], word = keys[s], times = c & kCount;
                        float y = x[q];
                        if (c) {
                            y = y > 0.0f ? y / rep : y * rep;
                            if (times) y -= frequency * (float)times + presence;
                        }
                        if (const int i = i0 + q * kEditThreads; i < biased) y += a.p.bias_values[last_bias[i]];      // the last entry of a word counts
                        if (!allows(allowed, word)) y = -INFINITY;
                        bad_num |= y != y;
                        LogitsVec<T>::put(out + word, y);
                    }
                }
                if (a.d.drafted && end > begin && a.d.tree) {
                    __syncthreads();
                    if (on) atomicSub(&counters[node], 1u);
                    __syncthreads();
                } else {
                    __syncthreads();
                }
            }
            // the next part: the other half of the one that was split, or what follows once both are done
            ++part;
            while (parts > gridDim.y && !(part & 1u)) { part >>= 1; parts >>= 1; }
            if (parts == gridDim.y) break;
        }
        row = stop;
    }
    if (!waited) pdl_wait();
    if (bad_arg) raise(a.status, YVEX_B200_STATUS_ARGUMENT);
    if (bad_num) raise(a.status, YVEX_B200_STATUS_NUMERIC);
}

template <class T> static int launch_logits(LogitsParams &a, cudaStream_t s) {
    constexpr uint64_t kPiece = (uint64_t)kStreamThreads * kStreamLoads * LogitsVec<T>::kN;
    const uint64_t pieces = (a.p.vocabulary + kPiece - 1) / kPiece;
    if (launch_pdl(logits_stream_kernel<T>, dim3((unsigned)pieces, (unsigned)(a.d.rows < 65535 ? a.d.rows : 65535)), dim3(kStreamThreads), 0, s, a) != cudaSuccess)
        return ERR_BACKEND;
    if (!a.p.history && !a.p.bias_tokens && !a.d.drafted) return launch_status(1);
    // A table for twice the words there can be, within limits; for few rows several CTAs that share the words; then as many rows a
    // CTA as leave one or two CTAs for every SM.
    static SmemOptIn optin;
    const uint64_t all = a.p.history_tokens + a.p.bias_entries + (a.d.drafted ? a.d.rows : 0), words = all < a.p.vocabulary ? all : a.p.vocabulary;
    uint32_t slots = kLeastTable;
    a.table_log2 = 10;
    while (slots < 2 * words && slots < kMostTable) { slots *= 2; ++a.table_log2; }
    constexpr uint64_t four_slots = 4 * 2 * sizeof(uint32_t) + 3 * sizeof(uint16_t);
    // Places for 2560 biased words leave the shared memory at 164 KB and the rest as cache; more are taken where a request has more on average, whose
    // words would else be counted in more parts (416 rows of 16 requests, us with 2560 and with 8192: 300 biases each 142 and 145, 1000 163
    // and 167, 2000 187 and 192, 4000 266 and 237, 10000 582 and 468).
    const uint64_t places = a.p.bias_entries > kFewBiased * a.p.requests ? kMostBiased : kFewBiased;
    a.biased = a.p.bias_tokens ? (uint32_t)(a.p.bias_entries < places ? a.p.bias_entries : places) : 0u;
    const int rc = optin.ensure(logits_edit_kernel<T>, (int)(kMostTable / 4 * four_slots + kMostBiased * sizeof(int)));
    if (rc != OK) return rc;
    uint64_t parts = 1;
    while (a.d.rows * parts * 2 <= kSmCount && parts * 128 < words) parts *= 2;
    const uint64_t ctas = (uint64_t)kSmCount * (slots >= kMostTable ? 1 : 2) / parts;
    a.rows_per_cta = (uint32_t)((a.d.rows + ctas - 1) / ctas);
    const uint64_t chunks = (a.d.rows + a.rows_per_cta - 1) / a.rows_per_cta;
    if (launch_pdl(logits_edit_kernel<T>, dim3((unsigned)chunks, (unsigned)parts), dim3(kEditThreads), (size_t)(slots / 4 * four_slots + a.biased * sizeof(int)), s, a) != cudaSuccess) return ERR_BACKEND;
    return launch_status(2);
}

// Whether a row at `a` and one at `b` (of `width` bytes, strides in bytes, a stride at least the width) have a byte in common.
static bool rows_meet(uintptr_t a, __int128 a_stride, uintptr_t b, __int128 b_stride, __int128 width, __int128 rows) {
    const __int128 apart = (__int128)b - (__int128)a;
    if (apart >= (rows - 1) * a_stride + width || -apart >= (rows - 1) * b_stride + width) return false;
    if (a_stride == b_stride) {                                 // row i + k of a lies `rest` before row i of b, row i + k + 1 so much behind that
        const __int128 k = apart >= 0 ? apart / a_stride : -((-apart + a_stride - 1) / a_stride), rest = apart - k * a_stride;
        auto there = [&](__int128 d) { return d < rows && -d < rows; };
        return (there(k) && rest < width) || (there(k + 1) && a_stride - rest < width);
    }
    for (__int128 i = 0, j = 0; i < rows && j < rows;) {
        const __int128 d = apart + j * b_stride - i * a_stride;
        if (d < width && -d < width) return true;
        if (d > 0) ++i; else ++j;
    }
    return false;
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
    if (p->history_tokens > (uint64_t)kCount - d->rows) return ERR_BOUNDS;      // (a word's counter has 31 bits, for the history and a path)
    if (logits_stride < p->vocabulary || out_stride < p->vocabulary || (grammar && grammar_stride < (p->vocabulary + 31) / 32)) return ERR_BOUNDS;
    if ((p->history && !p->history_offsets) || (p->bias_tokens && (!p->bias_values || !p->bias_offsets))) return ERR_INVALID_ARG;
    if (!d->row_request && d->rows > p->requests) return ERR_BOUNDS;
    if (d->drafted && (!d->offsets || !d->row_request || (d->tree && !d->ancestors))) return ERR_INVALID_ARG;
    const uintptr_t size = qtype == Q_F32 ? 4 : 2;
    if (((uintptr_t)logits | (uintptr_t)out) % size || (uintptr_t)grammar % 4) return ERR_INVALID_ARG;
    if ((logits != out || (logits_stride != out_stride && d->rows > 1)) &&
        rows_meet((uintptr_t)logits, (__int128)logits_stride * size, (uintptr_t)out, (__int128)out_stride * size, (__int128)p->vocabulary * size, d->rows))
        return ERR_INVALID_ARG;
    LogitsParams a{*p, *d, logits, logits_stride, grammar, grammar_stride, out, out_stride, 0, 0, 0, status};
    cudaStream_t s = as_stream(stream);
    return qtype == Q_F32 ? launch_logits<float>(a, s) : qtype == Q_BF16 ? launch_logits<__nv_bfloat16>(a, s) : launch_logits<__half>(a, s);
}
