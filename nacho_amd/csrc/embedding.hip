// Rows of a table by number, scaled, and the gradient of the table.
//
// lookup: rows[t] = scale table[id[t]].  Bound by the bytes of the rows.
//
// Its gradient is the product of a sparse matrix (words x tokens, one entry a token) and the rows'
// gradients: dtable[w] = scale sum of dout[t] over the tokens t of word w.  The entries are sorted
// by word, in order of the token within one, which gives every sum a fixed order; runs of kChunk
// sorted entries are summed by one workgroup each, whatever their words, so that a word that half
// of a batch has costs no more than others.  A word whose entries lie in more than one run gets its
// parts joined by a second launch, in their order.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <new>
#include <type_traits>

#include "dense_rows.hpp"
#include "runtime.hpp"

namespace nacho {
namespace embedding {

using dense::element_aligned;
using dense::item_of;
using dense::load_piece;
using dense::Piece;
using dense::pieces;
using dense::store_piece;

constexpr int kThreads = 256;

struct Ids {
    const void *ids;
    int bytes;     // 4 or 8
    int64_t words;

    // Word of a token, -1 for one that is none.
    __device__ __forceinline__ int64_t operator()(int64_t t) const {
        const int64_t id = bytes == 8 ? static_cast<const int64_t *>(ids)[t]
                                      : static_cast<const int32_t *>(ids)[t];
        return id >= 0 && id < words ? id : -1;
    }
};

// LANES threads per token, each with STEP pieces of its row on their way.
template <typename T, int N, int LANES>
__global__ __launch_bounds__(kThreads) void lookup_kernel(Ids ids, int64_t tokens, int64_t width,
                                                          float scale,
                                                          const T *__restrict__ table,
                                                          int64_t stride, T *__restrict__ rows) {
    constexpr int kPer = kThreads / LANES, kStep = 4;
    int64_t token = blockIdx.x * static_cast<int64_t>(kPer) +
                    __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
    for (; token < tokens; token += gridDim.x * static_cast<int64_t>(kPer)) {
        const int64_t id = ids(token);
        const T *from = table + (id < 0 ? 0 : id) * stride;
        T *to = rows + token * width;
        for (int64_t col0 = static_cast<int64_t>(threadIdx.x % LANES) * N; col0 < width;
             col0 += LANES * N * kStep) {
            Piece<T, N> piece[kStep];
#pragma unroll
            for (int s = 0; s < kStep; ++s) {
                const int64_t col = col0 + s * LANES * N;
                if (col < width) {
                    if (id >= 0) {
                        piece[s] = *reinterpret_cast<const Piece<T, N> *>(from + col);
                    } else {
                        for (int j = 0; j < N; ++j) piece[s].v[j] = static_cast<T>(0.0f);
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < kStep; ++s) {
                const int64_t col = col0 + s * LANES * N;
                if (col < width) {
                    if (scale != 1.0f && id >= 0) {
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            piece[s].v[j] =
                                static_cast<T>(scale * static_cast<float>(piece[s].v[j]));
                        }
                    }
                    store_piece<T, N>(to + col, piece[s]);
                }
            }
        }
    }
}

// ---- tokens in order of (word, token) ---------------------------------------------------
//
// keys[place] and order[place]: the word and the token at a place; tokens without a word are behind
// with the key `words`.

// Up to kRankMost tokens: a token's place is the number of tokens before it, counted.  A workgroup
// has 64 tokens, one a lane, and its wavefronts share the tokens to count.
constexpr int kRankMost = 8192;
constexpr int kRankThreads = 1024;
constexpr int kRankWaves = kRankThreads / dev::kWave;

__global__ __launch_bounds__(kRankThreads) void rank_kernel(Ids ids, int tokens,
                                                            int *__restrict__ keys,
                                                            int *__restrict__ order) {
    __shared__ __attribute__((aligned(16))) int s_key[kRankMost];
    __shared__ int s_before[kRankWaves][dev::kWave];
    const int lane = dev::lane(), wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int none = static_cast<int>(ids.words);
    // (past the tokens: a key that is before no other)
    const int filled = (tokens + 4 * kRankWaves - 1) / (4 * kRankWaves) * (4 * kRankWaves);
    for (int t = threadIdx.x; t < filled; t += kRankThreads) {
        const int64_t id = t < tokens ? ids(t) : -1;
        s_key[t] = t >= tokens ? INT_MAX : id < 0 ? none : static_cast<int>(id);
    }
    __syncthreads();
    const int mine = static_cast<int>(blockIdx.x) * dev::kWave + lane;
    const int key = mine < tokens ? s_key[mine] : none;
    const int per = filled / kRankWaves;
    int before = 0;
    for (int t = wave * per; t < wave * per + per; t += 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int other = s_key[t + j];
            before += other < key || (other == key && t + j < mine) ? 1 : 0;
        }
    }
    s_before[wave][lane] = before;
    __syncthreads();
    if (wave == 0 && mine < tokens) {
        int at = 0;
        for (int w = 0; w < kRankWaves; ++w) at += s_before[w][lane];
        keys[at] = key;
        order[at] = mine;
    }
}

// More tokens: a stable counting sort by kDigitBits bits at a time, lowest first.  Tokens are cut
// into runs of kRun, one wavefront each: counts per (digit, run), their exclusive scan, and each
// token's place from its run's offset and the equal digits before it in the run.
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kRun = 512;
constexpr int kRunSteps = kRun / dev::kWave;
constexpr int kRunWaves = kThreads / dev::kWave;

struct Pass {
    Ids ids;             // the first pass: tokens in their own order
    const int *keys_in;  // else the last one's
    const int *order_in;
    int tokens, runs, shift;
    int *keys, *order;
};

__device__ __forceinline__ int pass_key(const Pass &p, int i) {
    if (p.keys_in) return p.keys_in[i];
    const int64_t id = p.ids(i);
    return id < 0 ? static_cast<int>(p.ids.words) : static_cast<int>(id);
}

__device__ __forceinline__ int digit_of(int key, int shift) {
    return key >> shift & (kDigits - 1);
}

__global__ __launch_bounds__(kThreads) void count_kernel(Pass p, int *__restrict__ counts) {
    __shared__ int s_count[kRunWaves][kDigits];
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave, lane = dev::lane();
    const int run = static_cast<int>(blockIdx.x) * kRunWaves + wave;
    for (int i = lane; i < kDigits; i += dev::kWave) s_count[wave][i] = 0;
    dev::wave_sync();
    if (run >= p.runs) return;
    for (int step = 0; step < kRunSteps; ++step) {
        const int i = run * kRun + step * dev::kWave + lane;
        // (only the count matters here: the order of these additions decides nothing)
        if (i < p.tokens) atomicAdd(&s_count[wave][digit_of(pass_key(p, i), p.shift)], 1);
    }
    dev::wave_sync();
    for (int i = lane; i < kDigits; i += dev::kWave) {
        counts[static_cast<int64_t>(run) * kDigits + i] = s_count[wave][i];
    }
}

// counts[run][digit] become the offsets of each run's tokens within their digit, and totals[digit]
// the digit's tokens: a workgroup per 64 digits, its wavefronts over the runs.
__global__ __launch_bounds__(1024) void scan_kernel(int runs, int *__restrict__ counts,
                                                    int *__restrict__ totals) {
    constexpr int kParts = 1024 / dev::kWave;
    __shared__ int s_part[kParts][dev::kWave];
    const int lane = dev::lane(), part = static_cast<int>(threadIdx.x) / dev::kWave;
    int *mine = counts + blockIdx.x * dev::kWave + lane;
    const int per = (runs + kParts - 1) / kParts;
    const int from = min(runs, part * per), to = min(runs, from + per);
    int sum = 0;
#pragma unroll 8
    for (int r = from; r < to; ++r) sum += mine[static_cast<int64_t>(r) * kDigits];
    s_part[part][lane] = sum;
    __syncthreads();
    int at = 0, all = 0;
    for (int q = 0; q < kParts; ++q) {
        at += q < part ? s_part[q][lane] : 0;
        all += s_part[q][lane];
    }
#pragma unroll 8
    for (int r = from; r < to; ++r) {
        const int n = mine[static_cast<int64_t>(r) * kDigits];
        mine[static_cast<int64_t>(r) * kDigits] = at;
        at += n;
    }
    if (part == 0) totals[blockIdx.x * dev::kWave + lane] = all;
}

__global__ __launch_bounds__(kThreads) void place_kernel(Pass p, const int *__restrict__ counts,
                                                         const int *__restrict__ totals) {
    __shared__ int s_next[kRunWaves][kDigits];
    __shared__ int s_first[kDigits];
    __shared__ int s_sums[kRunWaves];
    int carry = 0;
    for (int x0 = 0; x0 < kDigits; x0 += kThreads) {
        const int x = x0 + static_cast<int>(threadIdx.x);
        int total = 0;
        s_first[x] = carry + dev::block_exclusive_sum<kThreads>(totals[x], s_sums, total);
        carry += total;
    }
    __syncthreads();
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave, lane = dev::lane();
    const int run = static_cast<int>(blockIdx.x) * kRunWaves + wave;
    if (run >= p.runs) return;
    int *next = s_next[wave];
    for (int i = lane; i < kDigits; i += dev::kWave) {
        next[i] = s_first[i] + counts[static_cast<int64_t>(run) * kDigits + i];
    }
    dev::wave_sync();
    for (int step = 0; step < kRunSteps; ++step) {
        const int i = run * kRun + step * dev::kWave + lane;
        const bool there = i < p.tokens;
        const int key = there ? pass_key(p, i) : 0;
        // (a lane past the tokens is no one's peer: digits have kDigitBits bits)
        const int digit = there ? digit_of(key, p.shift) : kDigits;
        const unsigned long long peers = dev::peers_of(digit, kDigitBits + 1);
        const int rank = __popcll(peers & ((1ull << lane) - 1ull));
        const int at = there ? next[digit] + rank : 0;
        dev::wave_sync();
        if (there && rank == 0) next[digit] += __popcll(peers);
        dev::wave_sync();
        if (there) {
            p.keys[at] = key;
            p.order[at] = p.order_in ? p.order_in[i] : i;
        }
    }
}

// ---- sums over sorted tokens ------------------------------------------------------------

constexpr int kChunk = 32;  // sorted tokens of a run

struct Sums {
    const int *keys, *order;
    int tokens, words;
    int64_t width;
    float scale;
    float *parts;  // [run][2][width]: sums of the run's first and last word, where these have
                   // tokens before and behind the run
};

template <typename T, int N>
__device__ __forceinline__ void store_sum(T *to, const float (&sum)[N], float scale) {
    Piece<T, N> o;
#pragma unroll
    for (int j = 0; j < N; ++j) o.v[j] = static_cast<T>(scale * sum[j]);
    *reinterpret_cast<Piece<T, N> *>(to) = o;
}

template <int N>
__device__ __forceinline__ void store_part(float *to, const float (&sum)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) to[j] = sum[j];
}

template <typename T, int N>
__global__ __launch_bounds__(kThreads) void sum_kernel(Sums a, const T *__restrict__ dout,
                                                       int64_t stride, T *__restrict__ dtable) {
    constexpr int kStep = 8;
    const int first = static_cast<int>(blockIdx.x) * kChunk;
    const int end = min(first + kChunk, a.tokens);
    const int64_t col =
        (blockIdx.y * static_cast<int64_t>(kThreads) + threadIdx.x) * N;
    if (col >= a.width) return;
    const int before = first > 0 ? a.keys[first - 1] : -1;
    const int behind = end < a.tokens ? a.keys[end] : -1;
    float sum[N] = {};
    for (int e0 = first; e0 < end; e0 += kStep) {
        Piece<T, N> piece[kStep];
        int key[kStep + 1];
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int e = min(e0 + s, end - 1);
            key[s] = a.keys[e];
            piece[s] = load_piece<T, N>(dout + a.order[e] * stride + col);
        }
        key[kStep] = e0 + kStep < end ? a.keys[e0 + kStep] : behind;
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int e = e0 + s;
            if (e >= end || key[s] >= a.words) return;  // (behind all words)
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] += static_cast<float>(piece[s].v[j]);
            const int next = e + 1 == end ? behind : key[s + 1];
            if (next == key[s] && e + 1 < end) continue;
            // the word's last token in this run
            if (key[s] == before) {
                store_part<N>(a.parts + (blockIdx.x * 2ll) * a.width + col, sum);
            } else if (next == key[s]) {
                store_part<N>(a.parts + (blockIdx.x * 2ll + 1) * a.width + col, sum);
            } else {
                store_sum<T, N>(dtable + static_cast<int64_t>(key[s]) * a.width + col, sum,
                                a.scale);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] = 0.0f;
        }
    }
}

// Words that begin in a run and go on behind it: their parts in the order of the runs.
template <typename T, int N>
__global__ __launch_bounds__(kThreads) void join_kernel(Sums a, T *__restrict__ dtable) {
    constexpr int kStep = 8;
    const int first = static_cast<int>(blockIdx.x) * kChunk, end = first + kChunk;
    if (end >= a.tokens) return;
    const int key = a.keys[end - 1];
    if (key >= a.words || a.keys[end] != key || (first > 0 && a.keys[first - 1] == key)) return;
    const int64_t col =
        (blockIdx.y * static_cast<int64_t>(kThreads) + threadIdx.x) * N;
    if (col >= a.width) return;
    // the word's last token: keys are sorted
    int lo = end, hi = a.tokens - 1;
    while (lo < hi) {
        const int mid = lo + (hi - lo + 1) / 2;
        if (a.keys[mid] == key) {
            lo = mid;
        } else {
            hi = mid - 1;
        }
    }
    const int64_t last = lo / kChunk;
    float sum[N];
    const float *mine = a.parts + (blockIdx.x * 2ll + 1) * a.width + col;
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = mine[j];
    for (int64_t run = blockIdx.x + 1ll; run <= last; run += kStep) {
        float part[kStep][N];
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const float *from = a.parts + min(run + s, last) * 2 * a.width + col;
#pragma unroll
            for (int j = 0; j < N; ++j) part[s][j] = from[j];
        }
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] += run + s <= last ? part[s][j] : 0.0f;
        }
    }
    store_sum<T, N>(dtable + static_cast<int64_t>(key) * a.width + col, sum, a.scale);
}

// ---- host -----------------------------------------------------------------------------

int check(int32_t dtype, int64_t tokens, int64_t words, int64_t width, float scale,
          const void *ids, int32_t id_bytes) {
    if (dtype < NACHO_F32 || dtype > NACHO_BF16 || tokens < 0 || words < 0 || width < 0 ||
        !(scale - scale == 0.0f) || (id_bytes != 4 && id_bytes != 8)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if (words > NACHO_MAX_WORDS || tokens > INT32_MAX - kRun * kRunWaves) {
        return NACHO_ERR_INDEX_OVERFLOW;
    }
    if (tokens > 0 && (!ids || !element_aligned(ids, id_bytes))) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    return NACHO_OK;
}

// Calls f with the element type and the elements of a piece.
template <typename F>
int with_type(int32_t dtype, bool whole, F f) {
    auto typed = [&](auto type) {
        using T = decltype(type);
        if (whole) return f(type, std::integral_constant<int, 16 / sizeof(T)>{});
        return f(type, std::integral_constant<int, 1>{});
    };
    if (dtype == NACHO_F32) return typed(float{});
    if (dtype == NACHO_F16) return typed(_Float16{});
    return typed(__bf16{});
}

int lookup(int32_t dtype, int64_t tokens, int64_t words, int64_t width, float scale,
           const void *ids, int32_t id_bytes, const void *table, int64_t stride, void *rows,
           void *stream) {
    NACHO_TRY(check(dtype, tokens, words, width, scale, ids, id_bytes));
    if (tokens == 0 || width == 0) return NACHO_OK;
    const int item = item_of(dtype);
    if ((words > 0 && !table) || !rows || !element_aligned(table, item) ||
        !element_aligned(rows, item)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    const Ids of{ids, id_bytes, words};
    const bool whole = pieces(table, stride, width, item) && pieces(rows, width, width, item);
    return with_type(dtype, whole, [&](auto type, auto n) -> int {
        using T = decltype(type);
        auto launch = [&](auto lanes) -> int {
            const int64_t groups = (tokens * lanes() + kThreads - 1) / kThreads;
            const unsigned grid = static_cast<unsigned>(
                groups < dense::kMostGroups ? groups : dense::kMostGroups);
            lookup_kernel<T, n(), lanes()><<<grid, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                of, tokens, width, scale, static_cast<const T *>(table), stride,
                static_cast<T *>(rows));
            NACHO_TRY_HIP(hipGetLastError());
            return NACHO_OK;
        };
        if (width * item <= 2048) return launch(std::integral_constant<int, dev::kWave>{});
        return launch(std::integral_constant<int, kThreads>{});
    });
}

// The tokens sorted by word into keys and order.
int sort_tokens(Call &call, const Ids &ids, int tokens, int *keys, int *order) {
    const hipStream_t s = call.stream();
    if (tokens <= kRankMost) {
        rank_kernel<<<ceil_div(static_cast<size_t>(tokens), dev::kWave), kRankThreads, 0, s>>>(
            ids, tokens, keys, order);
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    }
    const int runs = (tokens + kRun - 1) / kRun;
    int bits = 1;
    while (ids.words >> bits) ++bits;  // of the key `words`
    const int passes = (bits + kDigitBits - 1) / kDigitBits;
    int *counts = nullptr, *totals = nullptr, *other_keys = nullptr, *other_order = nullptr;
    NACHO_TRY(call.scratch_n(static_cast<size_t>(runs) * kDigits, &counts));
    NACHO_TRY(call.scratch_n(static_cast<size_t>(kDigits), &totals));
    if (passes > 1) {
        NACHO_TRY(call.scratch_n(static_cast<size_t>(tokens), &other_keys));
        NACHO_TRY(call.scratch_n(static_cast<size_t>(tokens), &other_order));
    }
    const unsigned groups = ceil_div(static_cast<size_t>(runs), kRunWaves);
    Pass p{ids, nullptr, nullptr, tokens, runs, 0, nullptr, nullptr};
    for (int i = 0; i < passes; ++i) {
        const bool to_result = (passes - i) % 2 == 1;
        p.keys = to_result ? keys : other_keys;
        p.order = to_result ? order : other_order;
        p.shift = i * kDigitBits;
        count_kernel<<<groups, kThreads, 0, s>>>(p, counts);
        NACHO_TRY_HIP(hipGetLastError());
        scan_kernel<<<kDigits / dev::kWave, 1024, 0, s>>>(runs, counts, totals);
        NACHO_TRY_HIP(hipGetLastError());
        place_kernel<<<groups, kThreads, 0, s>>>(p, counts, totals);
        NACHO_TRY_HIP(hipGetLastError());
        p.keys_in = p.keys;
        p.order_in = p.order;
    }
    return NACHO_OK;
}

int backward(int32_t dtype, int64_t tokens, int64_t words, int64_t width, float scale,
             const void *ids, int32_t id_bytes, const void *dout, int64_t stride, void *dtable,
             void *stream, const nacho_allocator *alloc) {
    NACHO_TRY(check(dtype, tokens, words, width, scale, ids, id_bytes));
    if (words == 0 || width == 0) return NACHO_OK;
    const int item = item_of(dtype);
    if ((tokens > 0 && !dout) || !dtable || !element_aligned(dout, item) ||
        !element_aligned(dtable, item)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    const bool whole = pieces(dout, stride, width, item) && pieces(dtable, width, width, item);
    const int64_t chunks = (tokens + kChunk - 1) / kChunk;
    const int64_t per = whole ? kThreads * (16 / item) : kThreads;
    const int64_t slices = (width + per - 1) / per;
    if (slices > 65535 || chunks * slices > dense::kMostGroups) return NACHO_ERR_INDEX_OVERFLOW;
    Call call(stream, alloc);
    const hipStream_t s = call.stream();
    return with_type(dtype, whole, [&](auto type, auto n) -> int {
        using T = decltype(type);
        NACHO_TRY(dense::clear(s, static_cast<T *>(dtable), words * width));
        if (tokens == 0) return NACHO_OK;
        int *keys = nullptr, *order = nullptr;
        float *parts = nullptr;
        NACHO_TRY(call.scratch_n(static_cast<size_t>(tokens), &keys));
        NACHO_TRY(call.scratch_n(static_cast<size_t>(tokens), &order));
        if (chunks > 1) NACHO_TRY(call.scratch_n(static_cast<size_t>(chunks * 2 * width), &parts));
        NACHO_TRY(sort_tokens(call, Ids{ids, id_bytes, words}, static_cast<int>(tokens), keys,
                              order));
        const Sums a{keys, order, static_cast<int>(tokens), static_cast<int>(words),
                     width, scale, parts};
        const dim3 all(static_cast<unsigned>(chunks), static_cast<unsigned>(slices));
        sum_kernel<T, n()><<<all, kThreads, 0, s>>>(a, static_cast<const T *>(dout), stride,
                                                    static_cast<T *>(dtable));
        NACHO_TRY_HIP(hipGetLastError());
        if (chunks > 1) {
            join_kernel<T, n()><<<all, kThreads, 0, s>>>(a, static_cast<T *>(dtable));
            NACHO_TRY_HIP(hipGetLastError());
        }
        return NACHO_OK;
    });
}

}  // namespace embedding
}  // namespace nacho

extern "C" int nacho_embedding(int32_t dtype, int64_t tokens, int64_t words, int64_t width,
                               float scale, const void *ids, int32_t id_bytes, const void *table,
                               int64_t stride, void *rows, void *stream) {
    return nacho::embedding::lookup(dtype, tokens, words, width, scale, ids, id_bytes, table,
                                    stride, rows, stream);
}

extern "C" int nacho_embedding_backward(int32_t dtype, int64_t tokens, int64_t words,
                                        int64_t width, float scale, const void *ids,
                                        int32_t id_bytes, const void *dout, int64_t stride,
                                        void *dtable, void *stream,
                                        const nacho_allocator *alloc) {
    try {
        return nacho::embedding::backward(dtype, tokens, words, width, scale, ids, id_bytes, dout,
                                          stride, dtable, stream, alloc);
    } catch (const std::bad_alloc &) {
        return NACHO_ERR_OUT_OF_MEMORY;
    }
}
