// Rows of a table by number, scaled, and the gradient of the table.
//
// lookup: rows[t] = scale table[id[t]].  Bound by the bytes of the rows.
//
// Its gradient is the product of a sparse matrix (words x tokens, one entry a token) and the rows'
// gradients: dtable[w] = scale sum of dout[t] over the tokens t of word w.  The entries are sorted
// by word, in order of the token within one, which gives every sum a fixed order; runs of kChunk
// sorted entries are summed by one workgroup each, whatever their words, so that a word that half
// of a batch has costs no more than others.  A word whose entries lie in more than one run gets its
// parts joined by another launch, in their order, for which many runs' parts are first added up in
// groups, by workgroups of their own (262144 tokens of 2048 bfloat16, none, half and all of them of one word:
// 300, 291 and 266 us; without such groups 299, 617 and 931).
//
// Measured, bfloat16: the lookup of 65536 rows of 4096 124 us, 5.7 TB/s; the gradient of 16384 tokens
// of 2048 and 65537 words 78 us traced, of which sorting them beside clearing the table 47 (5.7 TB/s of
// zeros), sums 21, groups of parts 5, joins 6.
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

constexpr int kThreads = 256;

// Pieces of rows that start anywhere.
template <typename T, int N>
using Piece = dense::Piece<T, N, sizeof(T)>;

// Where the piece that starts at col < width lies: a row's last piece ends with the row, over
// elements that the one before has too (and both give them the same value).
template <int N>
__device__ __forceinline__ int64_t within(int64_t col, int64_t width) {
    return min(col, width - N);
}

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
                        piece[s] = *reinterpret_cast<const Piece<T, N> *>(
                            from + within<N>(col, width));
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
                    dense::store_piece(to + within<N>(col, width), piece[s]);
                }
            }
        }
    }
}

// ---- tokens in order of (word, token) ---------------------------------------------------
//
// keys[place] and order[place]: the word and the token at a place; tokens without a word are behind
// with the key `words`.  Sorting keeps a few workgroups busy with waits for memory; the others of
// its launches clear the table's gradient meanwhile, each launch a share of it.

struct Clear {
    dense::u32x4 *pieces;
    int64_t from, to;      // of 16 bytes, in this launch
    unsigned first;        // the first workgroup that clears
    uint16_t *ends[2];     // before and behind all pieces, in the launch that clears the first
    int in_ends[2];

    // Whether the workgroup is one of those, and has done its part.
    __device__ __forceinline__ bool done() const {
        if (blockIdx.x < first) return false;
        const dense::u32x4 zero{0u, 0u, 0u, 0u};
        const int64_t all = (gridDim.x - first) * static_cast<int64_t>(blockDim.x);
        for (int64_t i = from + (blockIdx.x - first) * static_cast<int64_t>(blockDim.x) +
                         threadIdx.x; i < to; i += all) {
            pieces[i] = zero;
        }
        if (from == 0 && blockIdx.x == first) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (static_cast<int>(threadIdx.x) < in_ends[e]) ends[e][threadIdx.x] = 0;
            }
        }
        return true;
    }
};

// Up to kRankMost tokens: a token's place is the number of tokens before it, counted.  A workgroup
// has 64 tokens, one a lane, and its wavefronts share the tokens to count.
constexpr int kRankMost = 16384;
constexpr int kRankThreads = 1024;
constexpr int kRankWaves = kRankThreads / dev::kWave;

__global__ __launch_bounds__(kRankThreads) void rank_kernel(Ids ids, int tokens,
                                                            int *__restrict__ keys,
                                                            int *__restrict__ order,
                                                            Clear clear) {
    __shared__ __attribute__((aligned(16))) int s_key[kRankMost];
    __shared__ int s_before[kRankWaves][dev::kWave];
    if (clear.done()) return;
    const int lane = dev::lane();
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / dev::kWave);
    const int none = static_cast<int>(ids.words);
    // (past the tokens: a key that is before no other)
    constexpr int kStep = 8;
    const int filled = (tokens + kStep * kRankWaves - 1) / (kStep * kRankWaves) *
                       (kStep * kRankWaves);
    for (int t0 = threadIdx.x; t0 < filled; t0 += kRankThreads * kStep) {
        int64_t id[kStep];
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int t = t0 + s * kRankThreads;
            id[s] = t < tokens ? ids(t) : -1;
        }
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int t = t0 + s * kRankThreads;
            if (t < filled) {
                s_key[t] = t >= tokens ? INT_MAX : id[s] < 0 ? none : static_cast<int>(id[s]);
            }
        }
    }
    __syncthreads();
    const int group = static_cast<int>(blockIdx.x) * dev::kWave;
    const int mine = group + lane;
    const int key = mine < tokens ? s_key[mine] : none;
    const int per = filled / kRankWaves;
    const int from = wave * per, to = from + per;
    // Tokens before this group's count with an equal key too, those behind without; among its own
    // 64 the lane decides.
    auto count = [&](int a, int b, auto before) {
        int n = 0;
        for (int t = a; t < b; t += kStep) {
            int other[kStep];
#pragma unroll
            for (int j = 0; j < kStep; ++j) other[j] = s_key[t + j];
#pragma unroll
            for (int j = 0; j < kStep; ++j) n += before(other[j], t + j) ? 1 : 0;
        }
        return n;
    };
    const int a = min(max(group, from), to), b = min(max(group + dev::kWave, from), to);
    int n = count(from, a, [&](int other, int) { return other <= key; });
    n += count(a, b, [&](int other, int t) { return other < key || (other == key && t < mine); });
    n += count(b, to, [&](int other, int) { return other < key; });
    s_before[wave][lane] = n;
    __syncthreads();
    if (wave == 0 && mine < tokens) {
        int at = 0;
#pragma unroll
        for (int w = 0; w < kRankWaves; ++w) at += s_before[w][lane];
        keys[at] = key;
        order[at] = mine;
    }
}

// More tokens: a stable counting sort by kDigitBits bits at a time, lowest first.  A workgroup has
// a block of kBlock tokens, its wavefronts runs of kRun of them.  A token's place is its digit's
// first, and the equal digits of the blocks before, of the block's runs before, and before it in
// its run.
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / dev::kWave;
constexpr int kRunSteps = 2;
constexpr int kRun = kRunSteps * dev::kWave;
constexpr int kBlock = kRun * kSortWaves;
// Up to so many blocks, the workgroups that place tokens add up the blocks' counts themselves.
constexpr int kFewBlocks = 256;

struct Pass {
    Ids ids;             // the first pass: tokens in their own order
    const int *keys_in;  // else the last one's
    const int *order_in;
    int tokens, blocks, shift;
    int *keys, *order;
};

// Keys of a wavefront's run; -1 past the tokens.
__device__ __forceinline__ void run_keys(const Pass &p, int first, int (&keys)[kRunSteps]) {
#pragma unroll
    for (int step = 0; step < kRunSteps; ++step) {
        const int i = first + step * dev::kWave + dev::lane();
        keys[step] = -1;
        if (i < p.tokens) {
            if (p.keys_in) {
                keys[step] = p.keys_in[i];
            } else {
                const int64_t id = p.ids(i);
                keys[step] = static_cast<int>(id < 0 ? p.ids.words : id);
            }
        }
    }
}

__device__ __forceinline__ int run_first() {
    return static_cast<int>(blockIdx.x) * kBlock +
           static_cast<int>(threadIdx.x) / dev::kWave * kRun;
}

__device__ __forceinline__ int digit_of(int key, int shift) {
    return key >> shift & (kDigits - 1);
}

// counts[block][digit]
__global__ __launch_bounds__(kSortThreads) void count_kernel(Pass p, int *__restrict__ counts,
                                                             Clear clear) {
    __shared__ int s_count[kDigits];
    if (clear.done()) return;
    int keys[kRunSteps];
    run_keys(p, run_first(), keys);
    if (threadIdx.x < kDigits) s_count[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int step = 0; step < kRunSteps; ++step) {
        // (only the count matters here: the order of these additions decides nothing)
        if (keys[step] >= 0) atomicAdd(&s_count[digit_of(keys[step], p.shift)], 1);
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
        counts[static_cast<int64_t>(blockIdx.x) * kDigits + threadIdx.x] = s_count[threadIdx.x];
    }
}

// counts[block][digit] become the tokens of the digit in the blocks before, and totals[digit] the
// digit's tokens: a workgroup per 64 digits, its wavefronts over the blocks.
__global__ __launch_bounds__(1024) void scan_kernel(int blocks, int *__restrict__ counts,
                                                    int *__restrict__ totals, Clear clear) {
    constexpr int kParts = 1024 / dev::kWave;
    __shared__ int s_part[kParts][dev::kWave];
    if (clear.done()) return;
    const int lane = dev::lane(), part = static_cast<int>(threadIdx.x) / dev::kWave;
    int *mine = counts + blockIdx.x * dev::kWave + lane;
    const int per = (blocks + kParts - 1) / kParts;
    const int from = min(blocks, part * per), to = min(blocks, from + per);
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

// totals: null for few blocks, whose counts are as counted.
__global__ __launch_bounds__(kSortThreads) void place_kernel(Pass p,
                                                             const int *__restrict__ counts,
                                                             const int *__restrict__ totals,
                                                             Clear clear) {
    __shared__ int s_next[kSortWaves][kDigits];
    __shared__ int s_half[2][2][kDigits];
    __shared__ int s_sums[kSortWaves];
    if (clear.done()) return;
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave, lane = dev::lane();
    const int block = static_cast<int>(blockIdx.x);
    int keys[kRunSteps];
    run_keys(p, run_first(), keys);
    for (int i = threadIdx.x; i < kSortWaves * kDigits; i += kSortThreads) {
        (&s_next[0][0])[i] = 0;
    }
    // The digits' sizes, and their tokens in the blocks before: every digit has two threads, which
    // take the blocks in turn.
    static_assert(kSortThreads == 2 * kDigits, "two threads a digit");
    const int digit = static_cast<int>(threadIdx.x) % kDigits;
    const int half = static_cast<int>(threadIdx.x) / kDigits;
    int before = 0, size = 0;
    if (totals) {
        if (half == 0) {
            before = counts[static_cast<int64_t>(block) * kDigits + digit];
            size = totals[digit];
        }
    } else {
#pragma unroll 8
        for (int b = half; b < p.blocks; b += 2) {
            const int n = counts[static_cast<int64_t>(b) * kDigits + digit];
            before += b < block ? n : 0;
            size += n;
        }
    }
    s_half[half][0][digit] = before;
    s_half[half][1][digit] = size;
    __syncthreads();
    int *mine = s_next[wave];
#pragma unroll
    for (int step = 0; step < kRunSteps; ++step) {
        if (keys[step] >= 0) atomicAdd(&mine[digit_of(keys[step], p.shift)], 1);
    }
    size = half == 0 ? s_half[0][1][digit] + s_half[1][1][digit] : 0;
    int all = 0;
    int at = dev::block_exclusive_sum<kSortThreads>(size, s_sums, all);
    if (half == 0) {
        at += s_half[0][0][digit] + s_half[1][0][digit];
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const int n = s_next[w][digit];
            s_next[w][digit] = at;
            at += n;
        }
    }
    __syncthreads();
#pragma unroll
    for (int step = 0; step < kRunSteps; ++step) {
        const int i = run_first() + step * dev::kWave + lane;
        const bool there = keys[step] >= 0;
        const int x = digit_of(keys[step], p.shift);
        // (a lane past the tokens is no one's peer)
        const unsigned long long peers = dev::peers_of(x, kDigitBits) & __ballot(there);
        const int rank = __popcll(peers & ((1ull << lane) - 1ull));
        const int place = mine[x] + rank;
        dev::wave_sync();
        if (there && rank == 0) mine[x] += __popcll(peers);
        dev::wave_sync();
        if (there) {
            p.keys[place] = keys[step];
            p.order[place] = p.order_in ? p.order_in[i] : i;
        }
    }
}

// ---- sums over sorted tokens ------------------------------------------------------------

constexpr int kChunk = 32;  // sorted tokens of a run

struct Sums {
    const int *keys, *order;
    int tokens, words, chunks;
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

// The run of this thread, of which LANES threads have a slice of the columns each, and the thread's
// first column.
template <int N, int LANES>
struct Part {
    int run;
    int64_t col;
    bool there;

    __device__ __forceinline__ explicit Part(const Sums &a)
        : run(static_cast<int>(blockIdx.x) * (kThreads / LANES) +
              __builtin_amdgcn_readfirstlane(threadIdx.x / LANES)),
          col((blockIdx.y * static_cast<int64_t>(LANES) + threadIdx.x % LANES) * N),
          there(run < a.chunks && col < a.width) {
        col = within<N>(col, a.width);
    }
};

template <typename T, int N, int LANES>
__global__ __launch_bounds__(kThreads) void sum_kernel(Sums a, const T *__restrict__ dout,
                                                       int64_t stride, T *__restrict__ dtable) {
    constexpr int kStep = 16;
    const Part<N, LANES> part(a);
    if (!part.there) return;
    const int first = part.run * kChunk, end = min(first + kChunk, a.tokens);
    const int64_t col = part.col;
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
            piece[s] = dense::load_piece<T, N, sizeof(T)>(dout + a.order[e] * stride + col);
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
                store_part<N>(a.parts + (part.run * 2ll) * a.width + col, sum);
            } else if (next == key[s]) {
                store_part<N>(a.parts + (part.run * 2ll + 1) * a.width + col, sum);
            } else {
                store_sum<T, N>(dtable + static_cast<int64_t>(key[s]) * a.width + col, sum,
                                a.scale);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] = 0.0f;
        }
    }
}

// Runs that a workgroup of fold_kernel adds up.
constexpr int kFold = 64;

// Groups of kFold runs, the first at a multiple of kFold, that begin with a word that the run before
// ends with, all of them: their parts' sum goes into the first's second place.  (It has no second part,
// as it has no other word.  Not into the first place, which is read: threads whose pieces share columns
// would read each other's sums.)
template <int N, int LANES>
__global__ __launch_bounds__(kThreads) void fold_kernel(Sums a) {
    constexpr int kStep = 16;
    const Part<N, LANES> own(a);
    // (the first group's first run has none before it)
    const int64_t first = (own.run + 1) * static_cast<int64_t>(kFold), last = first + kFold - 1;
    if (last >= a.chunks || !own.there) return;
    const int key = a.keys[first * kChunk];
    if (key >= a.words || a.keys[first * kChunk - 1] != key || a.keys[last * kChunk] != key) return;
    float sum[N] = {};
    const float *const mine = a.parts + first * 2 * a.width + own.col;
    for (int r0 = 0; r0 < kFold; r0 += kStep) {
        float part[kStep][N];
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
#pragma unroll
            for (int j = 0; j < N; ++j) part[s][j] = mine[(r0 + s) * 2 * a.width + j];
        }
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] += part[s][j];
        }
    }
    store_part<N>(a.parts + (first * 2 + 1) * a.width + own.col, sum);
}

// Words that begin in a run and go on behind it: their parts in the order of the runs, groups of them
// in one where they are folded.
template <typename T, int N, int LANES>
__global__ __launch_bounds__(kThreads) void join_kernel(Sums a, bool folded,
                                                        T *__restrict__ dtable) {
    constexpr int kStep = 8;
    const Part<N, LANES> own(a);
    if (own.run + 1 >= a.chunks) return;
    const int first = own.run * kChunk, end = first + kChunk;
    const int key = a.keys[end - 1];
    if (key >= a.words || a.keys[end] != key || (first > 0 && a.keys[first - 1] == key)) return;
    // The last run that begins with the word: keys are sorted, and the lanes look at 64 runs at a
    // time, the same number apart.
    int last = own.run + 1, most = a.chunks - 1;
    while (last < most) {
        const int step = (most - last) / dev::kWave + 1;
        const int64_t run = last + static_cast<int64_t>(dev::lane()) * step;
        const bool with = run <= most && a.keys[run * kChunk] == key;
        const int n = __popcll(__ballot(with));  // (1 or more: `last` begins with the word)
        last += (n - 1) * step;
        most = min(most, last + step - 1);
    }
    if (!own.there) return;
    const int64_t col = own.col;
    float sum[N];
    const float *mine = a.parts + (own.run * 2ll + 1) * a.width + col;
#pragma unroll
    for (int j = 0; j < N; ++j) sum[j] = mine[j];
    // Single runs before the first whole group, groups, and single runs behind the last.
    int next = own.run + 1;
    const int whole = (next + kFold - 1) / kFold * kFold, behind = (last + 1) / kFold * kFold;
    const bool groups = folded && whole < behind;
#pragma unroll 1  // (one copy of the loop: three of them were a tenth slower)
    while (next <= last) {
        const bool group = groups && next == whole;
        const int end = group ? behind : groups && next < whole ? whole : last + 1;
        const int n = group ? (end - next) / kFold : end - next;
        const float *from = a.parts + (next * 2ll + (group ? 1 : 0)) * a.width + col;
        const int64_t step = (group ? kFold * 2ll : 2ll) * a.width;
        for (int i = 0; i < n; i += kStep) {
            float part[kStep][N];
#pragma unroll
            for (int s = 0; s < kStep; ++s) {
#pragma unroll
                for (int j = 0; j < N; ++j) part[s][j] = from[j];
                from += i + s + 1 < n ? step : 0;
            }
#pragma unroll
            for (int s = 0; s < kStep; ++s) {
#pragma unroll
                for (int j = 0; j < N; ++j) sum[j] += i + s < n ? part[s][j] : 0.0f;
            }
        }
        next = end;
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
    if (words > NACHO_MAX_WORDS || tokens > INT32_MAX - kBlock) {
        return NACHO_ERR_INDEX_OVERFLOW;
    }
    if (tokens > 0 && (!ids || !element_aligned(ids, id_bytes))) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    return NACHO_OK;
}

// Calls f with the element type and the elements of a piece.  (In us with pieces of 16 bytes and of
// one element: 30001 rows of 333 float32, lookup 11 and 12, sums 14 and 20.)
template <typename F>
int with_type(int32_t dtype, int64_t width, F f) {
    auto typed = [&](auto type) {
        using T = decltype(type);
        if (width * static_cast<int64_t>(sizeof(T)) >= 16) return f(type, std::integral_constant<int, 16 / sizeof(T)>{});
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
    return with_type(dtype, width, [&](auto type, auto n) -> int {
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

// Memory that is cleared: 16-byte pieces, and what is before and behind them in units of 2 bytes.
struct Cleared {
    dense::u32x4 *pieces;
    int64_t n;
    uint16_t *ends[2];
    int in_ends[2];

    Cleared(void *p, int64_t bytes) {
        char *const at = static_cast<char *>(p);
        int64_t head = static_cast<int64_t>(-reinterpret_cast<uintptr_t>(p) & 15);
        if (head > bytes) head = bytes;
        n = (bytes - head) / 16;
        pieces = reinterpret_cast<dense::u32x4 *>(at + head);
        ends[0] = reinterpret_cast<uint16_t *>(at);
        ends[1] = reinterpret_cast<uint16_t *>(at + head + 16 * n);
        in_ends[0] = static_cast<int>(head / 2);
        in_ends[1] = static_cast<int>((bytes - head - 16 * n) / 2);
    }
};

// The tokens sorted by word: keys of all places, then their tokens.  Clears `all` meanwhile.
int sort_tokens(Call &call, const Ids &ids, int tokens, const Cleared &all, int **sorted) {
    const hipStream_t s = call.stream();
    // Launch i of n: its share of the pieces, and a grid with workgroups for them.
    auto share = [&](unsigned groups, int threads, int i, int n, unsigned *grid) {
        const Clear c{all.pieces, all.n * i / n, all.n * (i + 1) / n, groups,
                      {all.ends[0], all.ends[1]}, {all.in_ends[0], all.in_ends[1]}};
        // (16 bytes a thread: 1.5 GB of zeros take 216 us so, and 290 us with as many workgroups as
        // run at a time)
        const int64_t want = (c.to - c.from + threads - 1) / threads;
        const int64_t most = dense::kMostGroups * 256 / threads - groups;
        *grid = groups + static_cast<unsigned>(want < 1 ? 1 : want < most ? want : most);
        return c;
    };
    unsigned grid = 0;
    const size_t n = static_cast<size_t>(tokens);
    if (tokens <= kRankMost) {
        NACHO_TRY(call.scratch_n(2 * n, sorted));
        const Clear clear = share(ceil_div(n, dev::kWave), kRankThreads, 0, 1, &grid);
        rank_kernel<<<grid, kRankThreads, 0, s>>>(ids, tokens, *sorted, *sorted + n, clear);
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    }
    const int blocks = (tokens + kBlock - 1) / kBlock;
    int bits = 1;
    while (ids.words >> bits) ++bits;  // of the key `words`
    const int passes = (bits + kDigitBits - 1) / kDigitBits;
    const bool few = blocks <= kFewBlocks;
    const int launches = passes * (few ? 2 : 3);
    const size_t n_counts = static_cast<size_t>(blocks) * kDigits;
    NACHO_TRY(call.scratch_n(4 * n + n_counts + kDigits, sorted));
    int *const other = *sorted + 2 * n;
    int *const counts = other + 2 * n, *const totals = few ? nullptr : counts + n_counts;
    const unsigned groups = static_cast<unsigned>(blocks);
    Pass p{ids, nullptr, nullptr, tokens, blocks, 0, nullptr, nullptr};
    for (int i = 0, launch = 0; i < passes; ++i) {
        const bool to_result = (passes - i) % 2 == 1;
        p.keys = to_result ? *sorted : other;
        p.order = p.keys + n;
        p.shift = i * kDigitBits;
        Clear clear = share(groups, kSortThreads, launch++, launches, &grid);
        count_kernel<<<grid, kSortThreads, 0, s>>>(p, counts, clear);
        NACHO_TRY_HIP(hipGetLastError());
        if (!few) {
            clear = share(kDigits / dev::kWave, 1024, launch++, launches, &grid);
            scan_kernel<<<grid, 1024, 0, s>>>(blocks, counts, totals, clear);
            NACHO_TRY_HIP(hipGetLastError());
        }
        clear = share(groups, kSortThreads, launch++, launches, &grid);
        place_kernel<<<grid, kSortThreads, 0, s>>>(p, counts, totals, clear);
        NACHO_TRY_HIP(hipGetLastError());
        p.keys_in = p.keys;
        p.order_in = p.order;
    }
    return NACHO_OK;
}

// Runs from which on fold_kernel is launched.  (us with it and without it, half of the tokens of one word,
// and none: 8192 tokens of 2048 bfloat16 49 and 47, 42 and 41; 16384 68 and 77, 60 and 59; 262144 291 and
// 617, 300 and 299; 1048576 of 64 float32 161 and 961, 160 and 158.)
constexpr int64_t kFoldChunks = 512;

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
    const int64_t chunks = (tokens + kChunk - 1) / kChunk;
    // Threads of a run: a row's pieces, if they are few.
    const int64_t row = width * item >= 16 ? (width * item + 15) / 16 : width;
    const int lanes = row <= 64 ? 64 : row <= 128 ? 128 : kThreads;
    const int64_t slices = (row + lanes - 1) / lanes;
    const int64_t groups_x = (chunks * lanes + kThreads - 1) / kThreads;
    if (slices > 65535 || groups_x * slices > dense::kMostGroups) return NACHO_ERR_INDEX_OVERFLOW;
    Call call(stream, alloc);
    const hipStream_t s = call.stream();
    return with_type(dtype, width, [&](auto type, auto n) -> int {
        using T = decltype(type);
        if (tokens == 0) return dense::clear(s, static_cast<T *>(dtable), words * width);
        int *sorted = nullptr;
        float *parts = nullptr;
        if (chunks > 1) NACHO_TRY(call.scratch_n(static_cast<size_t>(chunks * 2 * width), &parts));
        T *const table = static_cast<T *>(dtable);
        NACHO_TRY(sort_tokens(call, Ids{ids, id_bytes, words}, static_cast<int>(tokens),
                              Cleared(table, words * width * item), &sorted));
        const Sums a{sorted, sorted + tokens, static_cast<int>(tokens), static_cast<int>(words),
                     static_cast<int>(chunks), width, scale, parts};
        const dim3 groups(static_cast<unsigned>(groups_x), static_cast<unsigned>(slices));
        auto sums = [&](auto of) -> int {
            sum_kernel<T, n(), of()><<<groups, kThreads, 0, s>>>(a, static_cast<const T *>(dout),
                                                                 stride, table);
            NACHO_TRY_HIP(hipGetLastError());
            const bool fold = chunks >= kFoldChunks;
            if (fold) {
                const int64_t folds = (chunks / kFold * of() + kThreads - 1) / kThreads;
                fold_kernel<n(), of()><<<dim3(static_cast<unsigned>(folds), groups.y), kThreads, 0,
                                         s>>>(a);
                NACHO_TRY_HIP(hipGetLastError());
            }
            if (chunks > 1) {
                join_kernel<T, n(), of()><<<groups, kThreads, 0, s>>>(a, fold, table);
                NACHO_TRY_HIP(hipGetLastError());
            }
            return NACHO_OK;
        };
        if (lanes == 64) return sums(std::integral_constant<int, 64>{});
        if (lanes == 128) return sums(std::integral_constant<int, 128>{});
        return sums(std::integral_constant<int, kThreads>{});
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
