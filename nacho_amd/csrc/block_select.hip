// Which blocks of keys a query attends to: each block's mean key, every query's scores against
// the means, and the blocks of the highest scores.
//
// means: bound by reading k once.  A workgroup per (sequence, block, head): 16 lanes read a key
// (16 bytes or 32 each), 16 keys at a time; float32 sums.  8192 keys of 8 heads of 128 in bfloat16
// (17 MB): 5 us, a launch and 3 us of reads.
//
// scores: scale (sum of the group's heads of q) . mean, in float32 throughout: they are
// compared with each other, and the product is small (one row per group and one column per
// block of keys), so it runs on the float32 matrix instruction. A workgroup sums 16 queries'
// heads into LDS and goes over the blocks 64 at a time, 16 to a wavefront. 8192 queries of 32
// heads of 128 against 128 blocks: 30 us, where reading q and writing the scores would take 18.
// 48 sequences' tokens against the 320 of 512 blocks that they have on average (63 MB of means): 15
// to 17 us, 4 TB/s, where a copy's rate would take 11.3: a workgroup's first means are on their way
// only when q's heads are summed, and each step's only when the step before is multiplied.  32 or
// 64 queries to a workgroup are no faster for many queries and 1.3 us slower there.
//
// select: a wavefront per query and key head. Scores become unsigned numbers of the same order,
// and a threshold that the wanted number of them reaches is found with ballots: no sort, and
// ties are counted off from the lowest id. 65,536 rows of 128 blocks: 28 us, bound by
// instructions, about ten counts a row; reading the scores would take 7.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <new>
#include <type_traits>

#include "dense_tiles.hpp"
#include "runtime.hpp"

namespace nacho {
namespace select {

using namespace dense;

constexpr int kThreads = 256;

__device__ __forceinline__ int length_of(const int *lengths, int b, int keys) {
    return lengths ? min(max(lengths[b], 0), keys) : keys;
}

// ---- means ----------------------------------------------------------------------------

struct MeansArgs {
    int64_t groups;  // batch * blocks * heads, each a workgroup's
    int keys, heads, dim, block, blocks;
    int64_t batch_stride, row_stride, head_stride;
    const int *lengths;
    float *means;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void means_kernel(MeansArgs a, const T *__restrict__ k) {
    constexpr int kSlices = kThreads / 16;
    __shared__ float s_sum[kSlices][128 + 1];
    const int thread = static_cast<int>(threadIdx.x);
    const int piece = thread % 16, slice = thread / 16;
    for (int64_t group = blockIdx.x; group < a.groups; group += gridDim.x) {  // uniform
        const int h = static_cast<int>(group % a.heads);
        const int64_t bj = group / a.heads;
        const int j = static_cast<int>(bj % a.blocks), b = static_cast<int>(bj / a.blocks);
        const int first = j * a.block;
        const int there = min(max(length_of(a.lengths, b, a.keys) - first, 0), a.block);
        float sum[8] = {};
        if (8 * piece < a.dim) {
            const T *p =
                k + b * a.batch_stride + first * a.row_stride + h * a.head_stride + 8 * piece;
#pragma unroll 4
            for (int key = slice; key < there; key += kSlices) {
                const Frag<T> f = row_frag<T>(p + key * a.row_stride);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += static_cast<float>(f[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) s_sum[slice][8 * piece + i] = sum[i];
        __syncthreads();
        if (thread < a.dim) {
            float total = 0.0f;
#pragma unroll
            for (int x = 0; x < kSlices; ++x) total += s_sum[x][thread];
            a.means[(bj * a.heads + h) * a.dim + thread] =
                there > 0 ? total / static_cast<float>(there) : 0.0f;
        }
        __syncthreads();
    }
}

// ---- scores ---------------------------------------------------------------------------

struct ScoresArgs {
    int queries, keys, heads, group, dim, block, blocks, causal;
    float scale;
    int64_t batch_stride, row_stride, head_stride;
    const float *means;
    const int *lengths;
    float *scores;
    int tiles;     // of TOKENS queries
    int per_part;  // steps of 64 blocks that a workgroup takes
};

template <typename T, int DP, int TOKENS>
__global__ __launch_bounds__(kThreads) void scores_kernel(ScoresArgs a, const T *__restrict__ q,
                                                          int sequences) {
    constexpr int kRow = kTileRow<float, DP>;
    __shared__ __align__(16) float s_q[TOKENS * kRow];
    const int heads = sequences * a.heads;
    const int bh = static_cast<int>(blockIdx.x) % heads;
    const int rest = static_cast<int>(blockIdx.x) / heads;
    const int tile = rest % a.tiles, part = rest / a.tiles;
    const int b = bh / a.heads, h = bh % a.heads;
    const int t0 = TOKENS * tile, tokens = min(TOKENS, a.queries - t0);
    const int length = length_of(a.lengths, b, a.keys);
    const int place0 = length - a.queries + t0;
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
    // the group's heads, summed
    constexpr int kPieces = DP / 8;
    for (int x = threadIdx.x; x < TOKENS * kPieces; x += kThreads) {
        const int r = x / kPieces, col = x % kPieces * 8;
        float sum[8] = {};
        if (r < tokens && col < a.dim) {
            const T *p = q + b * a.batch_stride + (t0 + r) * a.row_stride +
                         static_cast<int64_t>(h) * a.group * a.head_stride + col;
#pragma unroll 4
            for (int i = 0; i < a.group; ++i) {
                const Frag<T> f = row_frag<T>(p + i * a.head_stride);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += static_cast<float>(f[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s_q[r * kRow + col + j] = sum[j] * a.scale;
    }
    __syncthreads();
    const int row_tiles = (tokens + 15) / 16;
    // the last block that some query of the tile may see
    const int last_place = place0 + tokens - 1;
    const int last = last_place < 0 ? -1 : (a.causal ? last_place : length - 1);
    const int steps = (a.blocks + 63) / 64;
    const int end = min(steps, (part + 1) * a.per_part);
    const int64_t next_row = static_cast<int64_t>(a.heads) * a.blocks;
    for (int step = part * a.per_part; step < end; ++step) {
        const int j = 64 * step + 16 * wave + c;
        if (64 * step + 16 * wave >= a.blocks) continue;
        f32x4 acc[TOKENS / 16];
#pragma unroll
        for (int t = 0; t < TOKENS / 16; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (static_cast<int64_t>(64 * step + 16 * wave) * a.block <= last) {  // uniform
            f32x8 m[DP / 32];
            const int64_t row = (static_cast<int64_t>(b) * a.blocks + j) * a.heads + h;
            load_row_frags<float, DP>(j < a.blocks ? a.means + row * a.dim : nullptr, a.dim, g, m);
#pragma unroll
            for (int t = 0; t < TOKENS / 16; ++t) {
                if (t < row_tiles) {
#pragma unroll
                    for (int kk = 0; kk < DP / 32; ++kk) {
                        acc[t] = mma(row_frag<float>(s_q + (16 * t + c) * kRow + 32 * kk + 8 * g),
                                     m[kk], acc[t]);
                    }
                }
            }
        }
        if (j >= a.blocks) continue;
        float *p = a.scores + ((static_cast<int64_t>(b) * a.queries + t0 + 4 * g) * a.heads + h) *
                                  a.blocks + j;
        // (queries whose place is before the block's first key do not see it)
        const int64_t unseen = static_cast<int64_t>(j) * a.block - place0;
#pragma unroll
        for (int t = 0; t < TOKENS / 16; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 16 * t + 4 * g + i;
                const bool sees = a.causal ? r >= unseen
                                           : place0 + r >= 0 && unseen < length - place0;
                if (r < tokens) p[(16 * t + i) * next_row] = sees ? acc[t][i] : kNegInf;
            }
        }
    }
}

// ---- selection ------------------------------------------------------------------------

struct SelectArgs {
    int64_t rows;
    unsigned first;  // row of the launch
    int queries, heads, keys, shift, blocks, count, sink, local, causal;  // block = 2^shift
    const float *scores;
    const int *lengths;
    int *ids;
};

constexpr int kMaxForced = 1 << 20;  // of sink and of local: fits above the infinity's number

// A number that orders like the score: 0 for a block that is not to be taken, the forced blocks'
// above every score's, in the order in which they are taken.  (Selects, not branches.)
constexpr unsigned kHighestScore = 0xff800000u;  // of an infinity

__device__ __forceinline__ unsigned order_of(const SelectArgs &a, float score, int j, int own) {
    const unsigned u = __float_as_uint(score + 0.0f);  // -0 as 0
    unsigned x = u ^ (static_cast<unsigned>(static_cast<int>(u) >> 31) | 0x80000000u);
    x = score > kNegInf ? x : 0u;  // (NaN too)
    x = j < a.sink ? UINT_MAX - static_cast<unsigned>(a.local) - static_cast<unsigned>(j) : x;
    x = own - j < a.local ? UINT_MAX - static_cast<unsigned>(own - j) : x;
    return j > own ? 0u : x;
}

// Selects for one row, whose scores are in `held_score` (NR > 0) or read again each time.
template <int NR>
__device__ __forceinline__ void select_row(const SelectArgs &a, unsigned row32, const float *scores,
                                           const float (&held_score)[NR ? NR : 1]) {
    const int lane = dev::lane();
    const int chunks = NR ? NR : (a.blocks + dev::kWave - 1) / dev::kWave;
    const int64_t row = row32;
    const unsigned bt = row32 / static_cast<unsigned>(a.heads);
    const int t = static_cast<int>(bt % static_cast<unsigned>(a.queries));
    const int b = static_cast<int>(bt / static_cast<unsigned>(a.queries));
    const int length = length_of(a.lengths, b, a.keys);
    const int place = length - a.queries + t;
    const int own = place < 0 ? -1 : (a.causal ? place : length - 1) >> a.shift;
    unsigned held[NR ? NR : 1];
    if constexpr (NR > 0) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            held[r] = order_of(a, held_score[r], r * dev::kWave + lane, own);
        }
    }
    auto key = [&](int r) {
        if constexpr (NR > 0) {
            return held[r];
        } else {
            const int j = r * dev::kWave + lane;
            return j < a.blocks ? order_of(a, scores[j], j, own) : 0u;
        }
    };
    auto at_least = [&](unsigned x) {
        int n = 0;
#pragma unroll NR ? NR : 1
        for (int r = 0; r < chunks; ++r) n += __popcll(__ballot(key(r) >= x));
        return n;
    };
    // The largest threshold that `count` numbers reach, or 0 where no more than `count` are to be
    // had: between lo, which that many reach, and hi, which they do not.  A float's number falls
    // by 2^23 when it is halved, so lo is a step or two of that below the highest score's, and
    // half of what is between them is where the count is met, most often after a few halvings.
    unsigned threshold = 0u;
    int above = 0;  // how many are over the threshold
    if (at_least(1u) > a.count) {
        unsigned top = 0u;
#pragma unroll NR ? NR : 1
        for (int r = 0; r < chunks; ++r) {
            const unsigned x = key(r);
            top = max(top, x <= kHighestScore ? x : 0u);
        }
        top = __builtin_amdgcn_readlane(dev::wave_inclusive_umax_dpp(top), dev::kWave - 1);
        unsigned lo = 0u, hi = top + 1u;
        int n = at_least(hi);
        above = n;
        if (n >= a.count) {  // forced blocks alone
            lo = hi;
            hi = UINT_MAX;
            above = at_least(hi);
            if (above >= a.count) {  // (count = 1: the latest block's number is the highest)
                lo = hi;
                n = above;
            }
        } else {
            for (unsigned width = 1u << 23;; width *= 2u) {
                lo = hi > width ? hi - width : 1u;
                n = at_least(lo);
                if (n >= a.count || width > UINT_MAX / 2u) break;
                above = n;
                hi = lo;
            }
        }
        while (n != a.count && hi - lo > 1u) {
            const unsigned mid = lo + (hi - lo) / 2u;
            const int m = at_least(mid);
            if (m >= a.count) {
                lo = mid;
                n = m;
            } else {
                hi = mid;
                above = m;
            }
        }
        threshold = lo;
        if (n == a.count) above = -1;  // no ties to break
    }
    // those over the threshold, and of those at it the lowest ids that there is room for
    int ties = above < 0 || threshold == 0u ? INT_MAX : a.count - above;
    const unsigned least = max(threshold, 1u);
    int *ids = a.ids + row * a.count;
    const unsigned long long before = (1ull << lane) - 1ull;
    int at = 0;
#pragma unroll NR ? NR : 1
    for (int r = 0; r < chunks; ++r) {
        const unsigned x = key(r);
        unsigned long long taken = __ballot(x >= least);
        if (ties != INT_MAX) {  // uniform
            const unsigned long long equal = __ballot(x == least);
            const bool extra = x == least && static_cast<int>(__popcll(equal & before)) >= ties;
            taken &= ~__ballot(extra);
            ties -= min(ties, static_cast<int>(__popcll(equal)));
        }
        if (taken >> lane & 1ull) ids[at + __popcll(taken & before)] = r * dev::kWave + lane;
        at += __popcll(taken);
    }
    for (int i = at + lane; i < a.count; i += dev::kWave) ids[i] = -1;
}

// A wavefront per row (four rows each, so that their loads are on the way together, took 30 us
// instead of 28 for 65,536 rows of 128 blocks). NR registers a lane hold a row of 64 NR blocks;
// NR = 0, for longer ones, reads it again each time. Empty registers cost as much as full ones:
// 32,768 rows of 64 blocks 13 us with one, 15 with two, 19 with four, 26 with eight; 384 rows
// of 1024 blocks 8 with 16, 14 with 32, 53 with none.
template <int NR>
__global__ __launch_bounds__(kThreads) void select_kernel(SelectArgs a) {
    // (a wavefront's number in scalar registers: the divisions are a few scalar instructions)
    const unsigned row = a.first + __builtin_amdgcn_readfirstlane(
        blockIdx.x * (kThreads / dev::kWave) + threadIdx.x / dev::kWave);
    if (row >= static_cast<unsigned>(a.rows)) return;
    const float *scores = a.scores + static_cast<int64_t>(row) * a.blocks;
    float held[NR ? NR : 1];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int j = r * dev::kWave + dev::lane();
        held[r] = j < a.blocks ? scores[j] : kNegInf;
    }
    select_row<NR>(a, row, scores, held);
}

// ---- host -----------------------------------------------------------------------------

bool aligned(const nacho_heads *h, int dtype, bool optional) {
    if (!h) return false;
    if (!h->data) return optional;
    const int64_t per = dtype == NACHO_F32 ? 4 : 8;
    return reinterpret_cast<uintptr_t>(h->data) % 16 == 0 && h->batch_stride % per == 0 &&
           h->row_stride % per == 0 && h->head_stride % per == 0;
}

bool good_dim(int32_t dim) { return dim >= 8 && dim <= 128 && dim % 8 == 0; }
bool good_block(int32_t block) { return block == 32 || block == 64 || block == 128; }
bool good_type(int32_t dtype) { return dtype >= NACHO_F32 && dtype <= NACHO_BF16; }

int means(int32_t dtype, int32_t batch, int32_t keys, int32_t heads, int32_t dim, int32_t block,
          const nacho_heads *k, const int32_t *lengths, float *out, void *stream) {
    const bool empty = batch == 0 || keys == 0;
    if (!good_type(dtype) || batch < 0 || keys < 0 || heads < 1 || !good_dim(dim) ||
        !good_block(block) || !aligned(k, dtype, empty) || (!out && !empty)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if (empty) return NACHO_OK;
    const int64_t blocks = (static_cast<int64_t>(keys) + block - 1) / block;
    const int64_t groups = blocks * batch * heads;
    if (groups > INT32_MAX) return NACHO_ERR_INDEX_OVERFLOW;
    const MeansArgs a{groups,
                      keys,
                      heads,
                      dim,
                      block,
                      static_cast<int>(blocks),
                      k->batch_stride,
                      k->row_stride,
                      k->head_stride,
                      lengths,
                      out};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned n = static_cast<unsigned>(groups < kMostGroups ? groups : kMostGroups);
    if (dtype == NACHO_F32) {
        means_kernel<float><<<n, kThreads, 0, s>>>(a, static_cast<const float *>(k->data));
    } else if (dtype == NACHO_F16) {
        means_kernel<_Float16><<<n, kThreads, 0, s>>>(a, static_cast<const _Float16 *>(k->data));
    } else {
        means_kernel<__bf16><<<n, kThreads, 0, s>>>(a, static_cast<const __bf16 *>(k->data));
    }
    NACHO_TRY_HIP(hipGetLastError());
    return NACHO_OK;
}

constexpr int kScoreTokens = 16;

template <typename T>
int launch_scores(const ScoresArgs &a, const void *q, int batch, unsigned grid, hipStream_t s) {
    const T *data = static_cast<const T *>(q);
    if (a.dim <= 64) {
        scores_kernel<T, 64, kScoreTokens><<<grid, kThreads, 0, s>>>(a, data, batch);
    } else {
        scores_kernel<T, 128, kScoreTokens><<<grid, kThreads, 0, s>>>(a, data, batch);
    }
    NACHO_TRY_HIP(hipGetLastError());
    return NACHO_OK;
}

int scores(int32_t dtype, int32_t batch, int32_t queries, int32_t keys, int32_t q_heads,
           int32_t kv_heads, int32_t dim, int32_t block, int32_t causal, float scale,
           const nacho_heads *q, const float *mean, const int32_t *lengths, float *out,
           void *stream) {
    const bool empty = batch == 0 || queries == 0 || keys == 0;
    if (!good_type(dtype) || batch < 0 || queries < 0 || keys < 0 || q_heads < 1 || kv_heads < 1 ||
        q_heads % kv_heads != 0 || !good_dim(dim) || !good_block(block) ||
        (causal != 0 && causal != 1) || !std::isfinite(scale) || !aligned(q, dtype, empty) ||
        reinterpret_cast<uintptr_t>(mean) % 16 != 0 || ((!mean || !out) && !empty)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if (empty) return NACHO_OK;
    const int64_t blocks = (static_cast<int64_t>(keys) + block - 1) / block;
    const int64_t tiles = (static_cast<int64_t>(queries) + kScoreTokens - 1) / kScoreTokens;
    const int64_t groups = tiles * batch * kv_heads;
    const int64_t steps = (blocks + 63) / 64;
    if (groups * steps > INT32_MAX) return NACHO_ERR_INDEX_OVERFLOW;
    // Enough workgroups for every CU to have four, while each sums its queries' heads once.  48
    // tokens of 8 key heads against 512 blocks, in us by the workgroups aimed at (256, 512, 1024,
    // 2048): 21.3 17.9 16.2 17.7.
    int64_t parts = (1024 + groups - 1) / groups;
    if (parts > steps) parts = steps;
    if (groups * parts > kMostGroups) return NACHO_ERR_INDEX_OVERFLOW;
    const int64_t per_part = (steps + parts - 1) / parts;
    const ScoresArgs a{queries,
                       keys,
                       kv_heads,
                       q_heads / kv_heads,
                       dim,
                       block,
                       static_cast<int>(blocks),
                       causal,
                       scale,
                       q->batch_stride,
                       q->row_stride,
                       q->head_stride,
                       mean,
                       lengths,
                       out,
                       static_cast<int>(tiles),
                       static_cast<int>(per_part)};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(groups * parts);
    switch (dtype) {
        case NACHO_F32: return launch_scores<float>(a, q->data, batch, grid, s);
        case NACHO_F16: return launch_scores<_Float16>(a, q->data, batch, grid, s);
        default: return launch_scores<__bf16>(a, q->data, batch, grid, s);
    }
}

int select(int32_t batch, int32_t queries, int32_t heads, int32_t keys, int32_t block,
           int32_t count, int32_t sink, int32_t local, int32_t causal, const float *score,
           const int32_t *lengths, int32_t *ids, void *stream) {
    if (batch < 0 || queries < 0 || heads < 1 || keys < 0 || !good_block(block) || count < 0 ||
        sink < 0 || local < 0 || sink > kMaxForced || local > kMaxForced ||
        (causal != 0 && causal != 1)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    const int64_t rows = static_cast<int64_t>(batch) * queries * heads;
    if (rows == 0 || count == 0) return NACHO_OK;
    if (!ids || (!score && keys > 0)) return NACHO_ERR_INVALID_ARGUMENT;
    const int64_t blocks = (static_cast<int64_t>(keys) + block - 1) / block;
    const int64_t grid = (rows + 3) / 4;
    // (a wavefront goes over its row's ids 64 at a time)
    if (rows > INT32_MAX || count > INT32_MAX - dev::kWave) return NACHO_ERR_INDEX_OVERFLOW;
    const int shift = block == 32 ? 5 : block == 64 ? 6 : 7;
    SelectArgs a{rows,  0,     queries, heads, keys,  shift,   static_cast<int>(blocks), count,
                 sink,  local, causal,  score, lengths, ids};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = [&](auto nr) {
        // (rows in a loop of the kernel's: 65,536 of 128 blocks take 29.3 us instead of 28.1)
        for (int64_t done = 0; done < grid; done += kMostGroups) {
            const unsigned n = static_cast<unsigned>(min(grid - done, kMostGroups));
            a.first = static_cast<unsigned>(done * (kThreads / dev::kWave));
            select_kernel<nr()><<<n, kThreads, 0, s>>>(a);
        }
    };
    if (blocks <= dev::kWave) {
        launch(std::integral_constant<int, 1>{});
    } else if (blocks <= 2 * dev::kWave) {
        launch(std::integral_constant<int, 2>{});
    } else if (blocks <= 4 * dev::kWave) {
        launch(std::integral_constant<int, 4>{});
    } else if (blocks <= 8 * dev::kWave) {
        launch(std::integral_constant<int, 8>{});
    } else if (blocks <= 16 * dev::kWave) {
        launch(std::integral_constant<int, 16>{});
    } else if (blocks <= 32 * dev::kWave) {
        launch(std::integral_constant<int, 32>{});
    } else {
        launch(std::integral_constant<int, 0>{});
    }
    NACHO_TRY_HIP(hipGetLastError());
    return NACHO_OK;
}

}  // namespace select
}  // namespace nacho

extern "C" int nacho_block_means(int32_t dtype, int32_t batch, int32_t keys, int32_t kv_heads,
                                 int32_t head_dim, int32_t block, const nacho_heads *k,
                                 const int32_t *lengths, float *means, void *stream) {
    return nacho::select::means(dtype, batch, keys, kv_heads, head_dim, block, k, lengths, means,
                                stream);
}

extern "C" int nacho_block_scores(int32_t dtype, int32_t batch, int32_t queries, int32_t keys,
                                  int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                  int32_t block, int32_t causal, float scale,
                                  const nacho_heads *q, const float *means,
                                  const int32_t *lengths, float *scores, void *stream) {
    return nacho::select::scores(dtype, batch, queries, keys, q_heads, kv_heads, head_dim, block,
                                 causal, scale, q, means, lengths, scores, stream);
}

extern "C" int nacho_block_select(int32_t batch, int32_t queries, int32_t kv_heads, int32_t keys,
                                  int32_t block, int32_t count, int32_t sink, int32_t local,
                                  int32_t causal, const float *scores, const int32_t *lengths,
                                  int32_t *ids, void *stream) {
    return nacho::select::select(batch, queries, kv_heads, keys, block, count, sink, local, causal,
                                 scores, lengths, ids, stream);
}
