// Tokens sorted by expert and back: a router's choices as sparse structure (experts x tokens),
// and dense rows moved through it.
//
// route: a stable counting sort.  Entries are cut into runs of 256, one wavefront each: counts
// per (run, expert), their exclusive scan in order of (expert, run), and then each entry's place
// is its run's offset plus the number of equal experts before it in the run, found with one
// ballot per bit of the expert's number.  No atomics decide an order.  Up to kSmall entries are
// one launch of one workgroup, larger inputs three launches.
//
// dispatch, combine and their gradients are bound by the bytes of the rows that they move.  All
// go token by token: a token's row is read once whatever its number of experts, and the rows of
// its places are written or read whole (going place by place, with the tokens' rows read again for
// each, dispatch took 166 us instead of 140).
//
// 16384 tokens of 4096 bfloat16 to 4 of 64 experts, in us and TB/s of what each has to move:
// route 18; dispatch 139, 4.8; combine 111, 5.9; its gradients 240, 5.0.  A large copy reaches 5.7.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <new>
#include <type_traits>

#include "dense_rows.hpp"
#include "dense_tiles.hpp"
#include "runtime.hpp"

namespace nacho {
namespace routing {

using dense::element_aligned;
using dense::item_of;
using dense::load_piece;
using dense::Piece;
using dense::pieces;
using dense::store_piece;
using dev::bits_for;
using dev::peers_of;

constexpr int kThreads = 256;
constexpr int kRun = 256;  // entries that one wavefront ranks
constexpr int kRunSteps = kRun / dev::kWave;
constexpr int kRunWaves = kThreads / dev::kWave;

struct RouteArgs {
    const void *experts;
    int id_bytes;
    int entries, n_experts;
    int *pos, *order, *slot;
};

// Expert of an entry; n_experts for one that is dropped or not there.
__device__ __forceinline__ int expert_of(const RouteArgs &a, int e) {
    if (e >= a.entries) return a.n_experts;
    const long long id = a.id_bytes == 8 ? static_cast<const long long *>(a.experts)[e]
                                         : static_cast<const int *>(a.experts)[e];
    return id >= 0 && id < a.n_experts ? static_cast<int>(id) : a.n_experts;
}

// A run's entries, counted into the wavefront's own counters in LDS.
__device__ void count_run(const RouteArgs &a, int first, int bits, int *counters) {
    for (int step = 0; step < kRunSteps; ++step) {
        const int e = first + step * dev::kWave + dev::lane();
        const int x = expert_of(a, e);
        const unsigned long long peers = peers_of(x, bits);
        // entries past the end count as dropped ones, behind all others; they get no place
        if ((peers & ((1ull << dev::lane()) - 1ull)) == 0ull) counters[x] += __popcll(peers);
        dev::wave_sync();
    }
}

// The run's entries to their places; counters hold the run's next place per expert.
__device__ void place_run(const RouteArgs &a, int first, int bits, int *counters) {
    for (int step = 0; step < kRunSteps; ++step) {
        const int e = first + step * dev::kWave + dev::lane();
        const int x = expert_of(a, e);
        const unsigned long long peers = peers_of(x, bits);
        const int rank = __popcll(peers & ((1ull << dev::lane()) - 1ull));
        const int at = counters[x] + rank;
        dev::wave_sync();
        if (rank == 0) counters[x] += __popcll(peers);
        dev::wave_sync();
        if (e < a.entries) {
            a.order[at] = e;
            a.slot[e] = x < a.n_experts ? at : -1;
        }
    }
}

constexpr int kSmallBlock = 1024;

// Everything in one workgroup: counters[wave][expert] in LDS.
__global__ __launch_bounds__(kSmallBlock) void route_small_kernel(RouteArgs a) {
    extern __shared__ int s_count[];
    __shared__ int s_sums[kSmallBlock / dev::kWave];
    const int buckets = a.n_experts + 1;
    const int runs = (a.entries + kRun - 1) / kRun;
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int bits = bits_for(a.n_experts);
    for (int i = threadIdx.x; i < runs * buckets; i += kSmallBlock) s_count[i] = 0;
    __syncthreads();
    if (wave < runs) count_run(a, wave * kRun, bits, s_count + wave * buckets);
    __syncthreads();
    int carry = 0;
    for (int x0 = 0; x0 < buckets; x0 += kSmallBlock) {  // uniform
        const int x = x0 + static_cast<int>(threadIdx.x);
        int mine = 0;
        if (x < buckets) {
            for (int w = 0; w < runs; ++w) mine += s_count[w * buckets + x];
        }
        int total = 0;
        int at = carry + dev::block_exclusive_sum<kSmallBlock>(mine, s_sums, total);
        carry += total;
        if (x < buckets) {
            a.pos[x] = at;
            for (int w = 0; w < runs; ++w) {
                const int n = s_count[w * buckets + x];
                s_count[w * buckets + x] = at;
                at += n;
            }
        }
    }
    __syncthreads();
    if (wave < runs) place_run(a, wave * kRun, bits, s_count + wave * buckets);
}

// counts[run][bucket]
__global__ __launch_bounds__(kThreads) void count_kernel(RouteArgs a, int runs,
                                                         int *__restrict__ counts) {
    extern __shared__ int s_count[];
    const int buckets = a.n_experts + 1;
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int run = static_cast<int>(blockIdx.x) * kRunWaves + wave;
    int *mine = s_count + wave * buckets;
    for (int i = dev::lane(); i < buckets; i += dev::kWave) mine[i] = 0;
    dev::wave_sync();
    if (run >= runs) return;
    count_run(a, run * kRun, bits_for(a.n_experts), mine);
    dev::wave_sync();
    for (int i = dev::lane(); i < buckets; i += dev::kWave) {
        counts[static_cast<int64_t>(run) * buckets + i] = mine[i];
    }
}

// counts[run][bucket] become the offsets of each run's entries within its bucket, and
// totals[bucket] the bucket's entries: a workgroup per 64 buckets, its wavefronts over the runs.
__global__ __launch_bounds__(1024) void scan_runs_kernel(int runs, int buckets,
                                                         int *__restrict__ counts,
                                                         int *__restrict__ totals) {
    constexpr int kParts = 1024 / dev::kWave;
    __shared__ int s_part[kParts][dev::kWave];
    const int lane = dev::lane(), part = static_cast<int>(threadIdx.x) / dev::kWave;
    const int x = static_cast<int>(blockIdx.x) * dev::kWave + lane;
    const int per = (runs + kParts - 1) / kParts;
    const int from = part * per, to = min(runs, from + per);
    int sum = 0;
    if (x < buckets) {
#pragma unroll 8
        for (int r = from; r < to; ++r) sum += counts[static_cast<int64_t>(r) * buckets + x];
    }
    s_part[part][lane] = sum;
    __syncthreads();
    int at = 0, all = 0;
    for (int p = 0; p < kParts; ++p) {
        at += p < part ? s_part[p][lane] : 0;
        all += s_part[p][lane];
    }
    if (x >= buckets) return;
    for (int r = from; r < to; ++r) {
        int &n = counts[static_cast<int64_t>(r) * buckets + x];
        const int mine = n;
        n = at;
        at += mine;
    }
    if (part == 0) totals[x] = all;
}

__global__ __launch_bounds__(kThreads) void place_kernel(RouteArgs a, int runs,
                                                         const int *__restrict__ counts,
                                                         const int *__restrict__ totals) {
    extern __shared__ int s_count[];
    __shared__ int s_sums[kRunWaves];
    const int buckets = a.n_experts + 1;
    int *s_pos = s_count + kRunWaves * buckets;
    int carry = 0;
    for (int x0 = 0; x0 < buckets; x0 += kThreads) {  // uniform
        const int x = x0 + static_cast<int>(threadIdx.x);
        const int mine = x < buckets ? totals[x] : 0;
        int total = 0;
        const int at = carry + dev::block_exclusive_sum<kThreads>(mine, s_sums, total);
        carry += total;
        if (x < buckets) {
            s_pos[x] = at;
            if (blockIdx.x == 0) a.pos[x] = at;
        }
    }
    __syncthreads();
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int run = static_cast<int>(blockIdx.x) * kRunWaves + wave;
    if (run >= runs) return;
    int *mine = s_count + wave * buckets;
    for (int i = dev::lane(); i < buckets; i += dev::kWave) {
        mine[i] = s_pos[i] + counts[static_cast<int64_t>(run) * buckets + i];
    }
    dev::wave_sync();
    place_run(a, run * kRun, bits_for(a.n_experts), mine);
}

// ---- rows -----------------------------------------------------------------------------

struct Rows {
    int64_t tokens, width;
    int per_token, n_experts;
    const int *pos, *slot;
    unsigned token_groups;  // workgroups that go over tokens; the others clear the rows behind
};

// The workgroup's part of the rows behind the last expert's entries is set to zero.
template <typename T, int N>
__device__ void clear_behind(const Rows &a, T *__restrict__ rows) {
    const int64_t first = a.pos[a.n_experts];
    const int64_t pieces = (a.tokens * a.per_token - first) * (a.width / N);
    Piece<T, N> zero;
#pragma unroll
    for (int j = 0; j < N; ++j) zero.v[j] = static_cast<T>(0.0f);
    const int64_t groups = gridDim.x - a.token_groups;
    for (int64_t i = (blockIdx.x - a.token_groups) * static_cast<int64_t>(kThreads) + threadIdx.x;
         i < pieces; i += groups * kThreads) {
        reinterpret_cast<Piece<T, N> *>(rows + first * a.width)[i] = zero;
    }
}

// Calls f with each token of the threads' own, in scalar registers (LANES is a multiple of a
// wavefront): one, where a launch can have as many workgroups as that takes.
template <int LANES, typename F>
__device__ __forceinline__ void each_token(const Rows &a, F f) {
    constexpr int kPer = kThreads / LANES;
    int64_t token = blockIdx.x * static_cast<int64_t>(kPer) +
                    __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
    for (; token < a.tokens; token += a.token_groups * static_cast<int64_t>(kPer)) f(token);
}

// LANES threads per token.
template <typename T, int N, int LANES>
__global__ __launch_bounds__(kThreads) void dispatch_kernel(Rows a, const T *__restrict__ x,
                                                            int64_t x_stride,
                                                            T *__restrict__ rows) {
    if (blockIdx.x >= a.token_groups) return clear_behind<T, N>(a, rows);
    each_token<LANES>(a, [&](int64_t token) {
        const int *slots = a.slot + token * a.per_token;
        for (int64_t col = static_cast<int64_t>(threadIdx.x % LANES) * N; col < a.width;
             col += LANES * N) {
            const auto piece = *reinterpret_cast<const Piece<T, N> *>(x + token * x_stride + col);
            for (int i = 0; i < a.per_token; ++i) {
                const int64_t at = slots[i];
                if (at >= 0) store_piece<T, N>(rows + at * a.width + col, piece);
            }
        }
    });
}

// The rows of STEP experts are on their way together; a dropped entry's stand-in is row 0, whose
// values are passed over.
template <typename T, int N, int LANES>
__global__ __launch_bounds__(kThreads) void combine_kernel(Rows a, const T *__restrict__ rows,
                                                           int64_t row_stride,
                                                           const float *__restrict__ weights,
                                                           T *__restrict__ out) {
    constexpr int kStep = 4;
    each_token<LANES>(a, [&](int64_t token) {
        const int64_t e = token * a.per_token;
        for (int64_t col = static_cast<int64_t>(threadIdx.x % LANES) * N; col < a.width;
             col += LANES * N) {
            float sum[N] = {};
            for (int i0 = 0; i0 < a.per_token; i0 += kStep) {
                Piece<T, N> piece[kStep];
                float w[kStep];
                bool there[kStep];
#pragma unroll
                for (int i = 0; i < kStep; ++i) {
                    const bool listed = i0 + i < a.per_token;
                    const int64_t at = listed ? a.slot[e + i0 + i] : -1;
                    there[i] = at >= 0;
                    w[i] = weights && listed ? weights[e + i0 + i] : 1.0f;
                    piece[i] = load_piece<T, N>(rows + (there[i] ? at : 0) * row_stride + col);
                }
#pragma unroll
                for (int i = 0; i < kStep; ++i) {
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float x = static_cast<float>(piece[i].v[j]);
                        sum[j] = there[i] ? __builtin_fmaf(w[i], x, sum[j]) : sum[j];
                    }
                }
            }
            Piece<T, N> o;
#pragma unroll
            for (int j = 0; j < N; ++j) o.v[j] = static_cast<T>(sum[j]);
            *reinterpret_cast<Piece<T, N> *>(out + token * a.width + col) = o;
        }
    });
}

template <typename T, int N, int LANES>
__global__ __launch_bounds__(kThreads) void combine_backward_kernel(
    Rows a, const T *__restrict__ rows, int64_t row_stride, const float *__restrict__ weights,
    const T *__restrict__ dout, int64_t dout_stride, T *__restrict__ drows,
    float *__restrict__ dweights) {
    if (blockIdx.x >= a.token_groups) return clear_behind<T, N>(a, drows);
    constexpr int kWavesPer = LANES / dev::kWave;
    __shared__ float s_sum[kThreads / dev::kWave];
    // (with barriers below, a workgroup has one token; else its wavefronts do not wait)
    each_token<LANES>(a, [&](int64_t token) {
        for (int i = 0; i < a.per_token; ++i) {
            const int64_t e = token * a.per_token + i;
            const int64_t at = a.slot[e];
            float dot = 0.0f;
            if (at >= 0) {
                const float w = weights[e];
                for (int64_t col = static_cast<int64_t>(threadIdx.x % LANES) * N; col < a.width;
                     col += LANES * N) {
                    const auto d =
                        *reinterpret_cast<const Piece<T, N> *>(dout + token * dout_stride + col);
                    const auto y = load_piece<T, N>(rows + at * row_stride + col);
                    Piece<T, N> o;
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const float x = static_cast<float>(d.v[j]);
                        dot = __builtin_fmaf(x, static_cast<float>(y.v[j]), dot);
                        o.v[j] = static_cast<T>(w * x);
                    }
                    store_piece<T, N>(drows + at * a.width + col, o);
                }
            }
            dot = dev::wave_sum(dot);
            if constexpr (kWavesPer > 1) {
                if (dev::lane() == 0) s_sum[threadIdx.x / dev::kWave] = dot;
                __syncthreads();
                dot = 0.0f;
                for (int w = 0; w < kWavesPer; ++w) dot += s_sum[w];
                __syncthreads();
            }
            if (threadIdx.x % LANES == 0) dweights[e] = dot;
        }
    });
}

// ---- host -----------------------------------------------------------------------------

// (512 to 4096 entries: 19 us a call, of which most is the host's, and 27 with three launches)
constexpr int kSmall = kRun * (kSmallBlock / dev::kWave);
constexpr int kSmallCounters = 8192;  // 32 KB
// (entries are counted in 32 bits, whole workgroups' runs and a token's by fours)
constexpr int kMostEntries = INT32_MAX - kRun * kRunWaves;

int route(const void *experts, int32_t id_bytes, int64_t tokens, int32_t per_token,
          int32_t n_experts, int32_t *pos, int32_t *order, int32_t *slot, void *stream,
          const nacho_allocator *alloc) {
    if ((id_bytes != 4 && id_bytes != 8) || tokens < 0 || per_token < 1 || n_experts < 1 ||
        n_experts > NACHO_MAX_EXPERTS || !pos) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if (tokens > kMostEntries / per_token) return NACHO_ERR_INDEX_OVERFLOW;
    const int entries = static_cast<int>(tokens * per_token);
    if (entries > 0 && (!experts || !order || !slot ||
                        reinterpret_cast<uintptr_t>(experts) % static_cast<unsigned>(id_bytes))) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    Call call(stream, alloc);
    const hipStream_t s = call.stream();
    const int buckets = n_experts + 1;
    const int runs = (entries + kRun - 1) / kRun;
    const RouteArgs a{experts, id_bytes, entries, n_experts, pos, order, slot};
    if (entries <= kSmall && runs * buckets <= kSmallCounters) {
        const size_t lds = static_cast<size_t>(runs) * buckets * sizeof(int);
        route_small_kernel<<<1, kSmallBlock, lds, s>>>(a);
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    }
    int *counts = nullptr, *totals = nullptr;
    NACHO_TRY(call.scratch_n(static_cast<size_t>(runs) * buckets, &counts));
    NACHO_TRY(call.scratch_n(static_cast<size_t>(buckets), &totals));
    const unsigned groups = ceil_div(static_cast<size_t>(runs), kRunWaves);
    const size_t lds = static_cast<size_t>(kRunWaves) * buckets * sizeof(int);
    count_kernel<<<groups, kThreads, lds, s>>>(a, runs, counts);
    NACHO_TRY_HIP(hipGetLastError());
    scan_runs_kernel<<<ceil_div(static_cast<size_t>(buckets), dev::kWave), 1024, 0, s>>>(
        runs, buckets, counts, totals);
    NACHO_TRY_HIP(hipGetLastError());
    place_kernel<<<groups, kThreads, lds + buckets * sizeof(int), s>>>(a, runs, counts, totals);
    NACHO_TRY_HIP(hipGetLastError());
    return NACHO_OK;
}

int check_rows(int32_t dtype, int64_t tokens, int32_t per_token, int64_t width) {
    if (dtype < NACHO_F32 || dtype > NACHO_BF16 || tokens < 0 || per_token < 1 || width < 0) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if (tokens > kMostEntries / per_token) return NACHO_ERR_INDEX_OVERFLOW;
    return NACHO_OK;
}

// Calls f with the element type, the elements of a piece and the threads per token: a wavefront
// for rows of up to 2 KB, else a workgroup.  16384 tokens to 4 of 64 experts with gradients, in us
// with a wavefront and a workgroup each, by a row's bytes (2048, 2560, 4096, 8192): 162 176,
// 210 211, 339 309, 664 621; 65536 tokens, rows of 512 and 1024 bytes: 182 345, 320 437.
template <typename F>
int with_rows(int32_t dtype, int64_t width, bool whole, F f) {
    auto lanes = [&](auto type, auto n) {
        constexpr int kN = decltype(n)::value;
        using T = decltype(type);
        const int64_t bytes = width * static_cast<int64_t>(sizeof(T));
        if (bytes <= 2048 || kN == 1) {
            return f(type, n, std::integral_constant<int, dev::kWave>{});
        }
        return f(type, n, std::integral_constant<int, kThreads>{});
    };
    auto typed = [&](auto type) {
        using T = decltype(type);
        if (whole) return lanes(type, std::integral_constant<int, 16 / sizeof(T)>{});
        return lanes(type, std::integral_constant<int, 1>{});
    };
    if (dtype == NACHO_F32) return typed(float{});
    if (dtype == NACHO_F16) return typed(_Float16{});
    return typed(__bf16{});
}

constexpr unsigned kClearGroups = 64;  // workgroups for the rows behind: few in ordinary use

unsigned token_groups(int64_t tokens, int lanes) {
    const int64_t n = (tokens * lanes + kThreads - 1) / kThreads;
    const int64_t most = dense::kMostGroups - kClearGroups;
    return static_cast<unsigned>(n < most ? n : most);
}

int dispatch(int32_t dtype, int64_t tokens, int32_t per_token, int32_t n_experts, int64_t width,
             const void *x, int64_t x_stride, const int32_t *pos, const int32_t *slot, void *rows,
             void *stream) {
    NACHO_TRY(check_rows(dtype, tokens, per_token, width));
    if (tokens == 0 || width == 0) return NACHO_OK;
    const int item = item_of(dtype);
    if (n_experts < 1 || !x || !pos || !slot || !rows || !element_aligned(x, item) ||
        !element_aligned(rows, item)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    const bool whole = pieces(x, x_stride, width, item) && pieces(rows, width, width, item);
    return with_rows(dtype, width, whole, [&](auto type, auto n, auto lanes) -> int {
        using T = decltype(type);
        const Rows a{tokens, width, per_token,
                     n_experts, pos, slot, token_groups(tokens, lanes())};
        dispatch_kernel<T, n(), lanes()>
            <<<a.token_groups + kClearGroups, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                a, static_cast<const T *>(x), x_stride, static_cast<T *>(rows));
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    });
}

int combine(int32_t dtype, int64_t tokens, int32_t per_token, int64_t width, const void *rows,
            int64_t row_stride, const float *weights, const int32_t *slot, void *out,
            void *stream) {
    NACHO_TRY(check_rows(dtype, tokens, per_token, width));
    if (tokens == 0 || width == 0) return NACHO_OK;
    const int item = item_of(dtype);
    if (!rows || !slot || !out || !element_aligned(rows, item) || !element_aligned(out, item)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    const bool whole = pieces(rows, row_stride, width, item) && pieces(out, width, width, item);
    return with_rows(dtype, width, whole, [&](auto type, auto n, auto lanes) -> int {
        using T = decltype(type);
        const Rows a{tokens, width, per_token, 0, nullptr, slot, token_groups(tokens, lanes())};
        combine_kernel<T, n(), lanes()>
            <<<a.token_groups, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                a, static_cast<const T *>(rows), row_stride, weights, static_cast<T *>(out));
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    });
}

int combine_backward(int32_t dtype, int64_t tokens, int32_t per_token, int32_t n_experts,
                     int64_t width, const void *rows, int64_t row_stride, const float *weights,
                     const int32_t *pos, const int32_t *slot, const void *dout,
                     int64_t dout_stride, void *drows, float *dweights, void *stream) {
    NACHO_TRY(check_rows(dtype, tokens, per_token, width));
    if (tokens == 0) return NACHO_OK;
    const int item = item_of(dtype);
    if (n_experts < 1 || !weights || !pos || !slot || !dweights ||
        (width > 0 && (!rows || !dout || !drows)) || !element_aligned(rows, item) ||
        !element_aligned(dout, item) || !element_aligned(drows, item)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    const bool whole = pieces(rows, row_stride, width, item) &&
                       pieces(dout, dout_stride, width, item) &&
                       pieces(drows, width, width, item);
    return with_rows(dtype, width, whole, [&](auto type, auto n, auto lanes) -> int {
        using T = decltype(type);
        const Rows a{tokens, width, per_token,
                     n_experts, pos, slot, token_groups(tokens, lanes())};
        combine_backward_kernel<T, n(), lanes()>
            <<<a.token_groups + kClearGroups, kThreads, 0, static_cast<hipStream_t>(stream)>>>(
                a, static_cast<const T *>(rows), row_stride, weights, static_cast<const T *>(dout),
                dout_stride, static_cast<T *>(drows), dweights);
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    });
}

}  // namespace routing
}  // namespace nacho

extern "C" int nacho_route(const void *experts, int32_t id_bytes, int64_t tokens,
                           int32_t per_token, int32_t n_experts, int32_t *pos, int32_t *order,
                           int32_t *slot, void *stream, const nacho_allocator *alloc) {
    try {
        return nacho::routing::route(experts, id_bytes, tokens, per_token, n_experts, pos, order,
                                     slot, stream, alloc);
    } catch (const std::bad_alloc &) {
        return NACHO_ERR_OUT_OF_MEMORY;
    }
}

extern "C" int nacho_dispatch(int32_t dtype, int64_t tokens, int32_t per_token, int32_t n_experts,
                              int64_t width, const void *x, int64_t x_stride, const int32_t *pos,
                              const int32_t *slot, void *rows, void *stream) {
    return nacho::routing::dispatch(dtype, tokens, per_token, n_experts, width, x, x_stride, pos,
                                    slot, rows, stream);
}

extern "C" int nacho_combine(int32_t dtype, int64_t tokens, int32_t per_token, int64_t width,
                             const void *rows, int64_t row_stride, const float *weights,
                             const int32_t *slot, void *out, void *stream) {
    return nacho::routing::combine(dtype, tokens, per_token, width, rows, row_stride, weights,
                                   slot, out, stream);
}

extern "C" int nacho_combine_backward(int32_t dtype, int64_t tokens, int32_t per_token,
                                      int32_t n_experts, int64_t width, const void *rows,
                                      int64_t row_stride, const float *weights,
                                      const int32_t *pos, const int32_t *slot, const void *dout,
                                      int64_t dout_stride, void *drows, float *dweights,
                                      void *stream) {
    return nacho::routing::combine_backward(dtype, tokens, per_token, n_experts, width, rows,
                                            row_stride, weights, pos, slot, dout, dout_stride,
                                            drows, dweights, stream);
}
