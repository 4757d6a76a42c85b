// The loss of rows over a vocabulary, and its gradients, without the logits in memory.
//
// With z = scale x w^T (tokens x words), a token's loss is log s + (m - z[target]) where m is its
// greatest logit and s the sum of exp(z - m); dz = (exp(z - m) / s - [word is target]) c with the
// gradient c of the token's loss; dx = scale dz w, dw = scale dz^T x.
//
// Tokens without a target are left out before anything else: the others' rows are gathered, and
// all products have as many rows as there are targets (a number that only the device knows; tiles
// past it end at once).  What the rows left out hold never counts.
//
// forward: one product, whose tiles of logits are reduced to m and s where they stand in
// registers, words in the result's rows: a lane has one token's logits, and only two exchanges and
// one pass through LDS join them.  Tiles' parts are joined by a second kernel, token by token.
// backward: the words are taken in pieces.  A piece's logits are worked out again and become dz in
// the rows' type, in scratch; two more products take it from there.  dx is summed in float32 over
// the pieces.
//
// Rounding: sums, m, s and losses are float32 (the sum of the losses float64).  dz reaches the
// gradients' products in the rows' type, without c's size: mean and sum have the factor c in
// common, which the results are multiplied by in float32, and else the largest |c| is taken out.
// float16 takes 2^14 dz: probabilities down to 2^-28 keep their bits, and below 2^-38 add nothing.  That
// is relative to the token's own gradient for dx: float16 has dz twice where tokens have gradients of
// their own, without these for dx, and with them, over the largest, for dtable, whose sums join the
// tokens (both gradients of 1000 tokens of 1024 and 50,001 words take 472 us instead of 413 with one
// dz, of 8192 of 2048 and 131,072 words 14.2 ms instead of 12.4).
// A rounded dz of a token's target is what the gradients lose most by: bfloat16 ones are up to 0.0024 of
// their norms off, of which rounding the results alone is 0.0017 (float16 0.0003 and 0.0002).  Up to
// kPartsMost tokens with a target, of 16 bits, have dz in two parts and lose nothing: a row for what the
// first has rounded away behind all first ones, and the gathered rows a second time with it.
//
// Bound by the matrix cores, and by the table's bytes for few tokens.  Measured, bfloat16: 8192 tokens
// of 2048, 131072 words, loss and gradients 15.05 to 15.35 ms; traced, the forward product 1.26
// PFLOP/s, dz 1.11, the gradients 1.06.  One token of 4096, its loss alone: 183 to 185 us, 5.8 TB/s.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <new>
#include <type_traits>

#include "dense_product.hpp"
#include "dense_rows.hpp"
#include "runtime.hpp"

namespace nacho {
namespace cross_entropy {

using dense::Across;
using dense::AcrossPairs;
using dense::Along;
using dense::element_aligned;
using dense::f32x4;
using dense::item_of;
using dense::kLog2e;
using dense::kNegInf;
using dense::Matrix;
using dense::Product;
using dense::Shape;

constexpr int kThreads = 256;

// ---- the tokens that have a target ------------------------------------------------------

struct Targets {
    const void *ids;
    int bytes;  // 4 or 8
    int64_t words;

    // Word of a token, -1 for one without.
    __device__ __forceinline__ int operator()(int64_t t) const {
        const int64_t id = bytes == 8 ? static_cast<const int64_t *>(ids)[t]
                                      : static_cast<const int32_t *>(ids)[t];
        return id >= 0 && id < words ? static_cast<int>(id) : -1;
    }
};

// What the kernels know of the tokens: `held` of them have a target.
struct Held {
    int *count;     // [2]: and a counter that starts at 0
    int *slot;      // [tokens]: place among them, -1 for one without a target
    int *token;     // [held]
    int *target;    // [held]
    float *factor;  // [held]: gradient of the token's loss over `common` (the backward pass)
    float *common;  // [1]
};

// The parts of dz, of which a token's gathered row has as many copies, by the tokens that have a target;
// and the rows that all of them take at most.  The number decides what two parts cost, not what they
// bring: both gradients of 100 tokens of 1024 and 32,000 words take 115 us with two and 90 with one, of
// 129 139 and 111, of 512 250 and 177, of 2000 790 and 457; bfloat16 targets of probabilities of 0.13 on
// average leave them 0.00166 and 0.0019 to 0.0020 of their norms off, at 100 tokens as at 2000.
constexpr int kPartsMost = 128;
template <typename T>
__device__ __forceinline__ int copies_of(int held) {
    return sizeof(T) == 2 && held <= kPartsMost ? 2 : 1;
}
template <typename T>
int64_t most_copies(int64_t tokens) {
    const int64_t few = tokens < kPartsMost ? tokens : kPartsMost;
    return sizeof(T) == 2 && 2 * few > tokens ? 2 * few : tokens;
}

enum Reduction { kNone = NACHO_LOSS_NONE, kMean = NACHO_LOSS_MEAN, kSum = NACHO_LOSS_SUM };

// The gradient of each token's loss from that of their mean or sum.  (Of no token: 0, so that sums of
// nothing are that whatever the gradient.)
__device__ __forceinline__ float common_of(int held, int reduction, float dloss) {
    if (held == 0) return 0.0f;
    return reduction == kMean ? dloss / static_cast<float>(held) : dloss;
}

constexpr int kListThreads = 1024;
constexpr int kListPer = 8;  // tokens of a thread and step

// One workgroup: places in order of the tokens and, with dloss, the gradients' factors.
__global__ __launch_bounds__(kListThreads) void list_kernel(Targets targets, int tokens,
                                                            int reduction,
                                                            const float *__restrict__ dloss,
                                                            Held held) {
    __shared__ int s_sums[kListThreads / dev::kWave];
    __shared__ float s_max[kListThreads / dev::kWave];
    int carry = 0;
    float most = 0.0f;
    for (int64_t t0 = 0; t0 < tokens; t0 += kListThreads * kListPer) {
        const int64_t first = t0 + static_cast<int>(threadIdx.x) * kListPer;
        int id[kListPer];
        int mine = 0;
#pragma unroll
        for (int i = 0; i < kListPer; ++i) {
            id[i] = first + i < tokens ? targets(first + i) : -1;
            mine += id[i] >= 0 ? 1 : 0;
        }
        int total = 0;
        int at = carry + dev::block_exclusive_sum<kListThreads>(mine, s_sums, total);
        carry += total;
#pragma unroll
        for (int i = 0; i < kListPer; ++i) {
            const int64_t t = first + i;
            if (t < tokens) held.slot[t] = id[i] >= 0 ? at : -1;
            if (id[i] >= 0) {
                held.token[at] = static_cast<int>(t);
                held.target[at] = id[i];
                if (dloss && reduction == kNone) {
                    const float c = fabsf(dloss[t]);
                    most = c < dense::kInf ? fmaxf(most, c) : most;
                }
                ++at;
            }
        }
    }
    if (threadIdx.x == 0) {
        held.count[0] = carry;
        held.count[1] = 0;
    }
    if (!dloss) return;
    float common = 0.0f;
    if (reduction == kNone) {
#pragma unroll
        for (int off = dev::kWave / 2; off > 0; off >>= 1) {
            most = fmaxf(most, __shfl_xor(most, off, dev::kWave));
        }
        if (dev::lane() == 0) s_max[threadIdx.x / dev::kWave] = most;
        __syncthreads();
        for (int w = 0; w < kListThreads / dev::kWave; ++w) common = fmaxf(common, s_max[w]);
        if (common == 0.0f) common = 1.0f;
    } else {
        common = common_of(carry, reduction, dloss[0]);
    }
    if (threadIdx.x == 0) *held.common = common;
    if (reduction != kNone) return;
    for (int64_t t = threadIdx.x; t < tokens; t += kListThreads) {
        const int id = targets(t);
        if (id >= 0) held.factor[held.slot[t]] = dloss[t] / common;
    }
}

// A row of `width` elements, with zeros behind them up to `padded`, by LANES threads.
template <typename T, int LANES>
__device__ __forceinline__ void copy_row(const T *__restrict__ from, int64_t width,
                                         T *__restrict__ to, int64_t padded, int lane) {
    constexpr int kN = 16 / sizeof(T);
    typedef T piece_t __attribute__((ext_vector_type(kN)));
    // (a row starts anywhere: loads of 16 bytes take any address)
    typedef piece_t any_t __attribute__((aligned(sizeof(T))));
    for (int64_t col = static_cast<int64_t>(lane) * kN; col < padded; col += LANES * kN) {
        piece_t v;
        if (col + kN <= width) {
            v = *reinterpret_cast<const any_t *>(from + col);
        } else {
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                v[j] = col + j < width ? from[col + j] : static_cast<T>(0.0f);
            }
        }
        *reinterpret_cast<piece_t *>(to + col) = v;
    }
}

// Those of the listed tokens (token), with copies for the parts of dz, or the first `rows` (null).
template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void gather_kernel(const int *__restrict__ count,
                                                          const int *__restrict__ token,
                                                          bool parts, int64_t rows, int64_t width,
                                                          int64_t padded,
                                                          const T *__restrict__ from,
                                                          int64_t stride, T *__restrict__ to,
                                                          int64_t to_stride) {
    constexpr int kPer = kThreads / LANES;
    const int64_t there = count ? *count : rows;
    int64_t row = blockIdx.x * static_cast<int64_t>(kPer) +
                  __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
    const int copies = parts ? copies_of<T>(static_cast<int>(there)) : 1;
    for (; row < there; row += gridDim.x * static_cast<int64_t>(kPer)) {
        const T *mine = from + (token ? token[row] : row) * stride;
        for (int c = 0; c < copies; ++c) {
            copy_row<T, LANES>(mine, width, to + (c * there + row) * to_stride, padded,
                               threadIdx.x % LANES);
        }
    }
}

// Both of the above for up to kListMost tokens: every workgroup counts the targets before its own
// kListRows tokens.  (8192 tokens of 2048 bfloat16: 29 us, and 27 for the two; 3000 of 776: 9 and 9;
// few: a launch less, 5 us.)
constexpr int kListMost = 2048;
constexpr int kListRows = 8;

template <typename T>
__global__ __launch_bounds__(kThreads) void list_rows_kernel(Targets targets, int tokens,
                                                             int reduction,
                                                             const float *__restrict__ dloss,
                                                             Held held, int64_t width,
                                                             int64_t padded,
                                                             const T *__restrict__ from,
                                                             int64_t stride, T *__restrict__ to,
                                                             int64_t to_stride, bool parts) {
    constexpr int kWaves = kThreads / dev::kWave, kStep = 8;
    __shared__ int s_before[kWaves], s_all[kWaves], s_token[kListRows];
    __shared__ float s_most[kWaves];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / dev::kWave), lane = dev::lane();
    const int first = static_cast<int>(blockIdx.x) * kListRows;
    const bool each = dloss && reduction == kNone;
    int before = 0, all = 0;
    float most = 0.0f;
    for (int t0 = threadIdx.x; t0 < tokens; t0 += kThreads * kStep) {
        int id[kStep];
        float c[kStep];
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int t = t0 + s * kThreads;
            id[s] = t < tokens ? targets(t) : -1;
            c[s] = each && t < tokens ? fabsf(dloss[t]) : 0.0f;
        }
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int t = t0 + s * kThreads;
            if (id[s] >= 0) {
                ++all;
                before += t < first ? 1 : 0;
                most = c[s] < dense::kInf ? fmaxf(most, c[s]) : most;
            }
        }
    }
    before = dev::wave_sum(before);
    all = dev::wave_sum(all);
#pragma unroll
    for (int off = dev::kWave / 2; off > 0; off >>= 1) {
        most = fmaxf(most, __shfl_xor(most, off, dev::kWave));
    }
    if (lane == 0) {
        s_before[wave] = before;
        s_all[wave] = all;
        s_most[wave] = most;
    }
    __syncthreads();
    before = all = 0;
    float common = 0.0f;
    for (int w = 0; w < kWaves; ++w) {
        before += s_before[w];
        all += s_all[w];
        common = fmaxf(common, s_most[w]);
    }
    if (each) {
        if (common == 0.0f) common = 1.0f;
    } else if (dloss) {
        common = common_of(all, reduction, dloss[0]);
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        held.count[0] = all;
        held.count[1] = 0;
        if (dloss) *held.common = common;
    }
    // the workgroup's own tokens, a lane each
    if (wave == 0) {
        const int t = first + lane;
        const int id = lane < kListRows && t < tokens ? targets(t) : -1;
        const unsigned long long there = __ballot(id >= 0);
        const int at = before + __popcll(there & ((1ull << lane) - 1ull));
        if (lane < kListRows && t < tokens) held.slot[t] = id >= 0 ? at : -1;
        if (id >= 0) {
            held.token[at] = t;
            held.target[at] = id;
            if (each) held.factor[at] = dloss[t] / common;
        }
        if (lane < kListRows) s_token[lane] = id >= 0 ? at : -1;
    }
    __syncthreads();
    const int copies = parts ? copies_of<T>(all) : 1;
    for (int i = wave; i < kListRows; i += kWaves) {
        const int at = s_token[i];
        if (at >= 0) {
            for (int c = 0; c < copies; ++c) {
                copy_row<T, dev::kWave>(from + (first + i) * stride, width,
                                        to + (c * all + at) * to_stride, padded, lane);
            }
        }
    }
}

// ---- tiles ------------------------------------------------------------------------------

// Workgroups that run at a time, one a compute unit.
constexpr unsigned kUnits = 256;

// All tiles are of 512 threads.  Wide ones are those of calls with many tokens, whose products bound
// them; a tile at the end of the tokens, the words or the columns takes as little of each as it
// needs.
constexpr int kTileThreads = 512;
template <int BM, int BN>
struct TileOf;
template <> struct TileOf<256, 256> { using type = Shape<256, 256, 2, 4>; };
template <> struct TileOf<256, 192> { using type = Shape<256, 192, 2, 4>; };
template <> struct TileOf<256, 128> { using type = Shape<256, 128, 4, 2>; };
template <> struct TileOf<256, 64> { using type = Shape<256, 64, 4, 2>; };
template <> struct TileOf<256, 16> { using type = Shape<256, 16, 8, 1>; };
template <> struct TileOf<128, 256> { using type = Shape<128, 256, 2, 4>; };
template <> struct TileOf<128, 192> { using type = Shape<128, 192, 2, 4>; };
template <> struct TileOf<128, 128> { using type = Shape<128, 128, 2, 4>; };
template <> struct TileOf<128, 64> { using type = Shape<128, 64, 4, 2>; };
template <> struct TileOf<64, 256> { using type = Shape<64, 256, 1, 8>; };
template <> struct TileOf<64, 16> { using type = Shape<64, 16, 4, 1>; };
template <int BM, int BN>
using Tile = typename TileOf<BM, BN>::type;
template <int N>
using Number = std::integral_constant<int, N>;

// ---- logits -----------------------------------------------------------------------------

struct Logits {
    const int *held;
    int64_t width;         // of the gathered rows, and of the table's
    const void *rows;      // [held][rows_stride]
    int64_t rows_stride;
    const void *table;
    int64_t table_stride;
    int words;             // of this piece
    int first;             // its first word
    const int *target;
    float scale;
    // the forward pass
    unsigned m_tiles;
    float2 *parts;         // [held][m_tiles]: m and s of a tile's words
    float *mine;           // [held]: the target's logit
    // the backward pass
    const float *most;     // m by token of the whole batch
    const float *total;    // s
    const int *token;
    const float *factor;   // null: 1
    void *dz;              // [parts][held][dz_stride]; null: only the next
    void *own_dz;          // the same without the factors, for dx; null: dz serves
    int64_t dz_stride;     // at least the piece's tiles: words past the piece's get zeros
};

template <typename T>
constexpr float kDzScale = __is_same(T, _Float16) ? 0x1p14f : 1.0f;

// Calls f(shape, first word, its tile, first token) for this workgroup's tile of BM x BN.
//
// Where BN is 256 the tiles of the last round, if they are few, are cut along the tokens so that
// more compute units have one: 1000 tokens of 50001 words are 784 tiles, three rounds and 16 tiles.
template <int BM, int BN, typename F>
__device__ __forceinline__ void with_tile(int words, int held, F f) {
    const unsigned m_tiles = (words + BM - 1) / BM, n_tiles = (held + BN - 1) / BN;
    const unsigned all = m_tiles * n_tiles;
    unsigned mt = 0, nt = 0;
    if constexpr (BN == 256) {
        const unsigned rest = all % kUnits;
        const unsigned cut = rest == 0 ? 1 : rest <= kUnits / 4 ? 4 : rest <= kUnits / 2 ? 2 : 1;
        const unsigned whole = cut == 1 ? all : all - rest;
        const unsigned late = blockIdx.x - whole;
        int wide = 256, n0 = 0;
        if (blockIdx.x < whole) {
            dense::tile_of(dense::order_of(blockIdx.x, whole), m_tiles, n_tiles, mt, nt);
        } else {
            if (cut == 1 || late >= rest * cut) return;
            dense::tile_of(whole + late / cut, m_tiles, n_tiles, mt, nt);
            wide = 256 / static_cast<int>(cut);
            n0 = static_cast<int>(late % cut) * wide;
        }
        n0 += static_cast<int>(nt) * 256;
        const int left = held - n0;
        if (left <= 0) return;
        const int64_t v0 = static_cast<int64_t>(mt) * BM;
        if (wide <= 64 || left <= 64) {
            f(Tile<BM, 64>{}, v0, mt, n0);
        } else if (wide <= 128 || left <= 128) {
            f(Tile<BM, 128>{}, v0, mt, n0);
        } else if (left <= 192) {
            f(Tile<BM, 192>{}, v0, mt, n0);
        } else {
            f(Tile<BM, 256>{}, v0, mt, n0);
        }
    } else {
        if (blockIdx.x >= all) return;
        dense::tile_of(dense::order_of(blockIdx.x, all), m_tiles, n_tiles, mt, nt);
        f(Tile<BM, BN>{}, static_cast<int64_t>(mt) * BM, mt, static_cast<int>(nt) * BN);
    }
}

// The tile's product of table and rows.
template <typename T, typename S>
__device__ __forceinline__ void logits_of(const Logits &a, int64_t v0, int64_t n0, int held,
                                          T *lds, f32x4 (&z)[S::MT][S::NT]) {
    const Matrix<T> table{static_cast<const T *>(a.table) + (a.first + v0) * a.table_stride,
                          a.table_stride};
    const Matrix<T> rows{static_cast<const T *>(a.rows) + n0 * a.rows_stride, a.rows_stride};
    Product<T, S, Along, Along>::run(
        table, static_cast<int>(min(a.words - v0, static_cast<int64_t>(S::BM))), rows,
        static_cast<int>(min(held - n0, static_cast<int64_t>(S::BN))), a.width, lds, z);
}

// m and s of a tile's words for each of its tokens, and the logits of targets among them.
template <typename T, typename S>
__device__ __forceinline__ void tile_parts(const Logits &a, int64_t v0, unsigned mt, int64_t n0,
                                           int held, T *lds) {
    const int wave = threadIdx.x / dev::kWave, lane = dev::lane(), g = lane >> 4, c = lane & 15;
    const int wm = wave / S::WN, wn = wave % S::WN;
    const float scale = a.scale;
    int target[S::NT];  // among the tile's words
#pragma unroll
    for (int t = 0; t < S::NT; ++t) {
        const int64_t n = n0 + (wn * S::NT + t) * 16 + c;
        target[t] = n < held ? static_cast<int>(a.target[n] - v0) : -1;
    }
    f32x4 z[S::MT][S::NT];
    logits_of<T, S>(a, v0, n0, held, lds, z);
    float(*s_most)[S::BN] = reinterpret_cast<float(*)[S::BN]>(lds);
    float(*s_total)[S::BN] = s_most + S::WM;
    __syncthreads();  // (the tiles have been read)
#pragma unroll
    for (int t = 0; t < S::NT; ++t) {
        const int col = (wn * S::NT + t) * 16 + c;
        // (a wavefront seldom has a token's target: it looks for one only then)
        const int there = target[t] - wm * S::MT * 16 - 4 * g;
        const bool mine = there >= 0 && there < S::MT * 16 && (there & 15) < 4;
        if (__ballot(mine)) {
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < S::MT; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x = 16 * i + j == there ? z[i][t][j] : x;
            }
            if (mine) a.mine[n0 + col] = x * scale;
        }
#pragma unroll
        for (int i = 0; i < S::MT; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) z[i][t][j] *= scale;
        }
        if (v0 + S::BM > a.words) {  // words that there are not
#pragma unroll
            for (int i = 0; i < S::MT; ++i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (v0 + (wm * S::MT + i) * 16 + 4 * g + j >= a.words) z[i][t][j] = kNegInf;
                }
            }
        }
        float most = kNegInf;
#pragma unroll
        for (int i = 0; i < S::MT; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) most = fmaxf(most, z[i][t][j]);
        }
        most = dense::column_max(most);
        // (with no finite logit: exp(-inf) of each)
        const float base = most == kNegInf ? 0.0f : most;
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < S::MT; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) total += dense::exp2_fast((z[i][t][j] - base) * kLog2e);
        }
        total = dense::column_sum(total);
        if (g == 0) {
            s_most[wm][col] = most;
            s_total[wm][col] = total;
        }
    }
    __syncthreads();
    for (int col = threadIdx.x; col < S::BN; col += S::kThreads) {
        if (n0 + col >= held) break;
        float most = kNegInf, total = 0.0f;
#pragma unroll
        for (int w = 0; w < S::WM; ++w) most = fmaxf(most, s_most[w][col]);
        const float base = most == kNegInf ? 0.0f : most;
#pragma unroll
        for (int w = 0; w < S::WM; ++w) {
            total += s_total[w][col] * dense::exp2_fast((s_most[w][col] - base) * kLog2e);
        }
        a.parts[(n0 + col) * a.m_tiles + mt] = float2{most, total};
    }
}

// LDS of the largest tile that a kernel of BM x BN tiles has.
template <typename T, int BM, int BN, template <typename, int, int> class A,
          template <typename, int, int> class B>
constexpr int kLds = Product<T, Tile<BM, BN>, A, B>::kLdsElements;

template <typename T, int BM, int BN>
__global__ __launch_bounds__((Tile<BM, BN>::kThreads)) void parts_kernel(Logits a) {
    __shared__ __attribute__((aligned(16))) T lds[kLds<T, BM, BN, Along, Along>];
    const int held = *a.held;
    with_tile<BM, BN>(a.words, held, [&](auto shape, int64_t v0, unsigned mt, int n0) {
        tile_parts<T, decltype(shape)>(a, v0, mt, n0, held, lds);
    });
}

// The sum of the threads' values, over a number if there is one, as a float.
template <int THREADS>
__device__ __forceinline__ void store_sum(double all, const int *count, float *to) {
    __shared__ double s_sum[THREADS / dev::kWave];
    all = dev::wave_sum(all);
    if (dev::lane() == 0) s_sum[threadIdx.x / dev::kWave] = all;
    __syncthreads();
    if (threadIdx.x != 0) return;
    all = 0.0;
    for (int w = 0; w < THREADS / dev::kWave; ++w) all += s_sum[w];
    *to = static_cast<float>(count ? all / max(*count, 1) : all);
}

// A token's tiles' parts to m, s and the loss, by a wavefront.
__device__ __forceinline__ void join_token(const float2 *__restrict__ from, unsigned tiles,
                                           const float *__restrict__ mine, float *most_of,
                                           float *total_of, float *loss) {
    float most = kNegInf, total = 0.0f;
#pragma unroll 4
    for (unsigned i = dev::lane(); i < tiles; i += dev::kWave) {
        const float2 p = from[i];
        const float higher = fmaxf(most, p.x);
        const float base = higher == kNegInf ? 0.0f : higher;
        total = total * dense::exp2_fast((most - base) * kLog2e) +
                p.y * dense::exp2_fast((p.x - base) * kLog2e);
        most = higher;
    }
#pragma unroll
    for (int off = dev::kWave / 2; off > 0; off >>= 1) {
        const float other = __shfl_xor(most, off, dev::kWave);
        const float other_total = __shfl_xor(total, off, dev::kWave);
        const float higher = fmaxf(most, other);
        const float base = higher == kNegInf ? 0.0f : higher;
        total = total * dense::exp2_fast((most - base) * kLog2e) +
                other_total * dense::exp2_fast((other - base) * kLog2e);
        most = higher;
    }
    if (dev::lane() == 0) {
        *most_of = most;
        *total_of = total;
        *loss = logf(total) + (most - *mine);
    }
}

// A wavefront per token; with `sum`, for up to kJoinMost tokens, also the sum of the losses or (mean)
// their mean.  (What makes the losses of all workgroups visible to the last costs each of them:
// 5 us less than two launches for 64 tokens, 49 us more for 3001.)
constexpr int64_t kJoinMost = 64;

__global__ __launch_bounds__(kThreads) void join_kernel(const int *__restrict__ slot,
                                                        int tokens, unsigned tiles,
                                                        const float2 *__restrict__ parts,
                                                        const float *__restrict__ mine,
                                                        float *__restrict__ most_of,
                                                        float *__restrict__ total_of, float *each,
                                                        int *count, int mean, float *sum) {
    constexpr int kPer = kThreads / dev::kWave;
    int64_t t = blockIdx.x * static_cast<int64_t>(kPer) +
                __builtin_amdgcn_readfirstlane(threadIdx.x / dev::kWave);
    for (; t < tokens; t += gridDim.x * static_cast<int64_t>(kPer)) {
        const int at = slot[t];
        if (at >= 0) {
            join_token(parts + static_cast<int64_t>(at) * tiles, tiles, mine + at, most_of + t,
                       total_of + t, each + t);
        } else if (dev::lane() == 0) {
            most_of[t] = 0.0f;
            total_of[t] = 1.0f;
            each[t] = 0.0f;
        }
    }
    if (!sum) return;
    // The workgroup that finds all others done adds the losses up, in their order.
    __shared__ int s_last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        s_last = atomicAdd(count + 1, 1) == static_cast<int>(gridDim.x) - 1;
        __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
    double all = 0.0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < tokens; i += kThreads) {
        all += static_cast<double>(
            __hip_atomic_load(each + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    }
    store_sum<kThreads>(all, mean ? count : nullptr, sum);
}

// The sum of the losses, or their mean over the tokens that have a target.
__global__ __launch_bounds__(1024) void sum_kernel(const int *__restrict__ count, int64_t tokens,
                                                   const float *__restrict__ each, int mean,
                                                   float *__restrict__ loss) {
    double all = 0.0;
#pragma unroll 8
    for (int64_t t = threadIdx.x; t < tokens; t += 1024) all += static_cast<double>(each[t]);
    store_sum<1024>(all, mean ? count : nullptr, loss);
}

// Four results of a row, or those of them that are within its width.
template <typename T>
__device__ __forceinline__ void store_row4(T *row, int64_t d, int64_t width, f32x4 v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    typedef t4 any_t __attribute__((aligned(sizeof(T))));
    if (d + 4 <= width) {
        t4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = static_cast<T>(v[j]);
        *reinterpret_cast<any_t *>(row + d) = o;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (d + j < width) row[d + j] = static_cast<T>(v[j]);
        }
    }
}

template <typename T>
__device__ __forceinline__ void store_row8(T *row, int64_t d, int64_t width, f32x4 lo, f32x4 hi) {
    if constexpr (sizeof(T) == 2) {
        typedef T t8 __attribute__((ext_vector_type(8)));
        typedef t8 any_t __attribute__((aligned(sizeof(T))));
        if (d + 8 <= width) {
            t8 o;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                o[j] = static_cast<T>(lo[j]);
                o[4 + j] = static_cast<T>(hi[j]);
            }
            *reinterpret_cast<any_t *>(row + d) = o;
            return;
        }
    }
    store_row4<T>(row, d, width, lo);
    store_row4<T>(row, d + 4, width, hi);
}

// Four words' dz of a token, and what its first part has rounded away.
template <typename T>
__device__ __forceinline__ void store_dz(const Logits &a, T *to, int held, f32x4 d) {
    dense::store4<T>(to, d);
    if constexpr (sizeof(T) == 2) {
        if (copies_of<T>(held) == 2) {
            f32x4 rest;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                rest[j] = d[j] - static_cast<float>(static_cast<T>(d[j]));
                // (of an infinity or what is no number: nothing)
                if (rest[j] != rest[j]) rest[j] = 0.0f;
            }
            dense::store4<T>(to + held * a.dz_stride, rest);
        }
    }
}

// dz of a tile's words and tokens.
template <typename T, typename S>
__device__ __forceinline__ void tile_dz(const Logits &a, int64_t v0, int64_t n0, int held,
                                        T *lds) {
    const int wave = threadIdx.x / dev::kWave, lane = dev::lane(), g = lane >> 4, c = lane & 15;
    const int wm = wave / S::WN, wn = wave % S::WN;
    const bool own = __is_same(T, _Float16) && a.own_dz;
    // (on their way before the product: nothing is left to wait for behind it)
    int target[S::NT];
    float most[S::NT], part[S::NT], factor[S::NT];
#pragma unroll
    for (int t = 0; t < S::NT; ++t) {
        const int64_t n = min(n0 + (wn * S::NT + t) * 16 + c, static_cast<int64_t>(held - 1));
        const int token = a.token[n];
        target[t] = static_cast<int>(a.target[n] - a.first - v0);
        most[t] = a.most[token];
        factor[t] = kDzScale<T> * (a.factor && !own ? a.factor[n] : 1.0f);
        part[t] = factor[t] / a.total[token];
    }
    f32x4 z[S::MT][S::NT];
    logits_of<T, S>(a, v0, n0, held, lds, z);
#pragma unroll
    for (int t = 0; t < S::NT; ++t) {
        const int64_t n = n0 + (wn * S::NT + t) * 16 + c;
        // the target's probability less 1, where the wavefront has a target
        const int there = target[t] - wm * S::MT * 16 - 4 * g;
        const bool some = __ballot(there >= 0 && there < S::MT * 16 && (there & 15) < 4) != 0;
        const int64_t at = n * a.dz_stride + v0;
        const float weight = own ? a.factor[min(n, static_cast<int64_t>(held - 1))] : 1.0f;
#pragma unroll
        for (int i = 0; i < S::MT; ++i) {
            const int v = (wm * S::MT + i) * 16 + 4 * g;
            f32x4 d;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = z[i][t][j] * a.scale;
                d[j] = dense::exp2_fast((x - most[t]) * kLog2e) * part[t];
            }
            if (some) {
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] -= 16 * i + j == there ? factor[t] : 0.0f;
            }
            if (v0 + S::BM > a.words) {  // words that there are not
#pragma unroll
                for (int j = 0; j < 4; ++j) d[j] = v0 + v + j < a.words ? d[j] : 0.0f;
            }
            if (n >= held) continue;
            if constexpr (__is_same(T, _Float16)) {
                if (own) {
                    store_dz<T>(a, static_cast<T *>(a.own_dz) + at + v, held, d);
                    if (!a.dz) continue;
                    d *= weight;  // (words that there are not are in no result of it)
                }
            }
            store_dz<T>(a, static_cast<T *>(a.dz) + at + v, held, d);
        }
    }
}

template <typename T, int BM, int BN>
__global__ __launch_bounds__((Tile<BM, BN>::kThreads)) void dz_kernel(Logits a) {
    __shared__ __attribute__((aligned(16))) T lds[kLds<T, BM, BN, Along, Along>];
    const int held = *a.held;
    with_tile<BM, BN>(a.words, held, [&](auto shape, int64_t v0, unsigned, int n0) {
        tile_dz<T, decltype(shape)>(a, v0, n0, held, lds);
    });
}

// ---- the gradients' products ------------------------------------------------------------

struct Gradients {
    const int *held;
    const void *dz;       // [parts][held][dz_stride], for dtable
    const void *dx_dz;    // for dx: the same, or (own) without the tokens' gradients
    const float *own;     // these gradients, by token; null: dx's are `common`
    int64_t dz_stride;
    const void *rows;     // gathered
    const void *table;    // of the piece
    int64_t table_stride;
    int64_t words, width; // of the piece; of the results
    int64_t padded;       // columns that the operands' rows have
    int64_t rows_stride;
    int64_t piece;        // words of a whole piece
    int64_t most_rows;    // that the sums have room for, at least all tokens
    float *sums;          // [split][parts][held][sums_stride]; null: no dx
    int64_t sums_stride;
    int first;            // whether the piece is the first
    int64_t most_parts;   // splits that `parts` has room for; 1 without it
    float *parts;         // [split][piece][sums_stride]: dtable's
    const float *common;
    float scale;
    void *dtable;         // of the piece, [words][width]; null: none
};

// How the gradients' products are split: dx's tiles, of its columns by the tokens, over the words,
// and dtable's, of its columns by the words, over the tokens.  An item is at most about three
// quarters of a compute unit's work, that of both where one launch has both, so that the units' work
// is even.
// The same for every piece, and known to the device alone.
struct Splits {
    unsigned m_tiles, n_tiles, count;
    int64_t depth;  // words, or tokens, of a split

    __device__ __forceinline__ unsigned tiles() const { return m_tiles * n_tiles; }
    __device__ __forceinline__ unsigned items() const { return tiles() * count; }
};

constexpr unsigned kMostItems = 512, kMostSplits = 64;

// Tenths of a tile of 256 columns that the width takes: one at the end, of 64 or of 128 columns, takes
// 0.4 or 0.6 as long as a whole one.
__device__ __host__ __forceinline__ int64_t tenths_of(int64_t width) {
    const int64_t rest = width % 256;
    return width / 256 * 10 + (rest == 0 ? 0 : rest <= 64 ? 4 : rest <= 128 ? 6 : 10);
}

// n rows by the width, over `depth`, in whole steps, of a load of `load` steps; most: splits that
// the sums have room for.
__device__ __forceinline__ Splits split_up(int64_t n, int bn, int64_t width, int64_t depth,
                                           int step, int64_t load, int64_t most) {
    Splits s;
    s.m_tiles = static_cast<unsigned>((width + 255) / 256);
    s.n_tiles = static_cast<unsigned>((n + bn - 1) / bn);
    const int64_t steps = (depth + step - 1) / step;
    const int64_t wanted = load * 3 / (4 * static_cast<int64_t>(kUnits));
    const int64_t per = wanted < 8 ? 8 : wanted;
    int64_t k = (steps + per - 1) / per;
    // (a few more make a round of all units: a step of 2048 tokens of 16384 words 1287 us instead of 1350)
    const int64_t round = 10 * static_cast<int64_t>(kUnits) /
                          max(s.n_tiles * tenths_of(width), int64_t{1});
    if (k > 1 && k < round && 2 * round <= 3 * k) k = round;
    k = min(k, static_cast<int64_t>(kMostItems) / max(static_cast<int64_t>(s.tiles()), int64_t{1}));
    k = max(min(min(k, static_cast<int64_t>(kMostSplits)), most), int64_t{1});
    s.depth = max((steps + k - 1) / k, int64_t{1}) * step;
    s.count = static_cast<unsigned>(max((depth + s.depth - 1) / s.depth, int64_t{1}));
    return s;
}

// The steps of dx's and of dtable's products, in those of whole tiles.
template <typename T, int BN>
__device__ __forceinline__ int64_t load_of(const Gradients &a, int held, bool dx, bool dtable) {
    constexpr int kStep = dense::kStepK<T>, kBN = BN <= 64 ? 64 : BN;
    const int64_t x = (held + BN - 1) / BN * ((a.piece + kStep - 1) / kStep);
    const int64_t t = (a.piece + kBN - 1) / kBN * ((held + kStep - 1) / kStep);
    return ((dx ? x : 0) + (dtable ? t : 0)) * tenths_of(a.width) / 10;
}

template <typename T, int BN>
__device__ __forceinline__ Splits dx_splits(const Gradients &a, int held, int64_t load) {
    return split_up(held, BN, a.width, a.piece, dense::kStepK<T>, load,
                    a.most_rows / max(held, 1));
}

template <typename T, int BN>
__device__ __forceinline__ Splits dtable_splits(const Gradients &a, int held, int64_t load) {
    return split_up(a.piece, BN <= 64 ? 64 : BN, a.width, held, dense::kStepK<T>, load,
                    a.most_parts);
}

// A tile of dx's sums: columns of the table's rows by the tokens, over the words of a split.
template <typename T, typename S>
__device__ __forceinline__ void tile_dx(const Gradients &a, int64_t d0, int64_t n0, unsigned split,
                                        int64_t v0, int64_t words, int held, T *lds) {
    const Matrix<T> table{static_cast<const T *>(a.table) + v0 * a.table_stride + d0,
                          a.table_stride};
    const Matrix<T> dz{static_cast<const T *>(a.dx_dz) + n0 * a.dz_stride + v0, a.dz_stride};
    f32x4 sums[S::MT][S::NT];
    Product<T, S, Across, Along>::run(
        table, static_cast<int>(min(a.padded - d0, static_cast<int64_t>(S::BM))), dz,
        static_cast<int>(min(held - n0, static_cast<int64_t>(S::BN))), words, lds, sums);
    const int wave = threadIdx.x / dev::kWave, lane = dev::lane(), g = lane >> 4, c = lane & 15;
    const int wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
    for (int t = 0; t < S::NT; ++t) {
        const int64_t n = n0 + (wn * S::NT + t) * 16 + c;
        if (n >= held) continue;
        float *to = a.sums + (static_cast<int64_t>(split) * held + n) * a.sums_stride;
#pragma unroll
        for (int i = 0; i < S::MT; ++i) {
            const int64_t d = d0 + (wm * S::MT + i) * 16 + 4 * g;
            if (d < a.sums_stride) {
                f32x4 *p = reinterpret_cast<f32x4 *>(to + d);
                *p = a.first ? sums[i][t] : *p + sums[i][t];
            }
        }
    }
}

// A tile of dtable: columns of the gathered rows by the words, over the tokens or (not whole) those
// of a split.
template <typename T, typename S, bool PAIRS>
__device__ __forceinline__ void tile_dtable(const Gradients &a, int64_t d0, int64_t v0,
                                            unsigned split, int64_t t0, int64_t tokens,
                                            bool whole, T *lds) {
    const Matrix<T> rows{static_cast<const T *>(a.rows) + t0 * a.rows_stride + d0, a.rows_stride};
    const Matrix<T> dz{static_cast<const T *>(a.dz) + t0 * a.dz_stride + v0, a.dz_stride};
    f32x4 sums[S::MT][S::NT];
    // Words up to a whole 16 bytes are zeros in dz; behind them nothing has been written (or by another
    // piece), and a product of float32 would be worked out again for what is no number there.
    constexpr int64_t kN = 16 / sizeof(T);
    const int64_t there = (a.words + kN - 1) / kN * kN;
    // (few tokens are bound by the stores of the results: 8 elements together)
    using P = std::conditional_t<PAIRS, Product<T, S, AcrossPairs, Across>,
                                 Product<T, S, Across, Across>>;
    P::run(
        rows, static_cast<int>(min(a.padded - d0, static_cast<int64_t>(S::BM))), dz,
        static_cast<int>(min(there - v0, static_cast<int64_t>(S::BN))), tokens, lds, sums);
    const float factor = *a.common * a.scale * (1.0f / kDzScale<T>);
    const int wave = threadIdx.x / dev::kWave, lane = dev::lane(), g = lane >> 4, c = lane & 15;
    const int wm = wave / S::WN, wn = wave % S::WN;
#pragma unroll
    for (int t = 0; t < S::NT; ++t) {
        const int64_t v = v0 + (wn * S::NT + t) * 16 + c;
        if (v >= a.words) continue;
        T *to = static_cast<T *>(a.dtable) + v * a.width;
        float *part = a.parts + (split * a.piece + v) * a.sums_stride;
        if constexpr (PAIRS) {
#pragma unroll
            for (int i = 0; i < S::MT; i += 2) {
                const int64_t d = d0 + (wm * S::MT + i) * 16 + 8 * g;
                store_row8<T>(to, d, a.width, sums[i][t] * factor, sums[i + 1][t] * factor);
            }
            continue;
        }
#pragma unroll
        for (int i = 0; i < S::MT; ++i) {
            const int64_t d = d0 + (wm * S::MT + i) * 16 + 4 * g;
            if (whole) {
                store_row4<T>(to, d, a.width, sums[i][t] * factor);
            } else if (d < a.sums_stride) {
                *reinterpret_cast<f32x4 *>(part + d) = sums[i][t];
            }
        }
    }
}

// Calls f with the tile of at most 256 x BN that `m` by `n` need.
template <int BN, bool ALONG, typename F>
__device__ __forceinline__ void with_ends(int64_t m, int64_t n, F f) {
    if constexpr (BN <= 64) {
        f(Tile<256, BN>{});
    } else {
        if (n <= 64) return f(Tile<256, 64>{});
        if (m <= 64) return f(Tile<64, 256>{});
        if (m <= 128) return f(Tile<128, 256>{});
        if (n <= 128) return f(Tile<256, 128>{});
        if constexpr (ALONG) {
            if (n <= 192) return f(Tile<256, 192>{});
        }
        f(Tile<256, 256>{});
    }
}

// dx's items, then dtable's: one launch for calls of many tokens (BN 256), else one for each.
template <typename T, int BN, bool DX, bool DTABLE>
__global__ __launch_bounds__(kTileThreads) void gradients_kernel(Gradients a) {
    constexpr int kLdsX = DX ? kLds<T, 256, BN, Across, Along> : 0;
    constexpr int kLdsT = DTABLE ? kLds<T, 256, (BN <= 64 ? 64 : BN), Across, Across> : 0;
    __shared__ __attribute__((aligned(16))) T lds[kLdsX > kLdsT ? kLdsX : kLdsT];
    const int held = *a.held * copies_of<T>(*a.held);
    const int64_t load = load_of<T, BN>(a, held, DX, DTABLE);
    unsigned at = blockIdx.x, mt = 0, nt = 0;
    if constexpr (DX) {
        const Splits s = dx_splits<T, BN>(a, held, load);
        if (at < s.items()) {
            at = dense::order_of(at, s.items());
            const unsigned split = at / s.tiles();
            dense::tile_of(at % s.tiles(), s.m_tiles, s.n_tiles, mt, nt);
            const int64_t d0 = mt * int64_t{256}, n0 = nt * static_cast<int64_t>(BN);
            const int64_t v0 = split * s.depth;
            // (a short last piece has fewer splits; a first one's sums are all written)
            if (v0 >= a.words && !a.first) return;
            with_ends<BN, true>(a.padded - d0, held - n0, [&](auto shape) {
                tile_dx<T, decltype(shape)>(a, d0, n0, split, v0, min(s.depth, a.words - v0), held,
                                            lds);
            });
            return;
        }
        at -= s.items();
    }
    if constexpr (DTABLE) {
        const Splits s = dtable_splits<T, BN>(a, held, load);
        if (at >= s.items()) return;
        at = dense::order_of(at, s.items());
        const unsigned split = at / s.tiles();
        dense::tile_of(at % s.tiles(), s.m_tiles, s.n_tiles, mt, nt);
        constexpr int kBN = BN <= 64 ? 64 : BN;
        const int64_t d0 = mt * int64_t{256}, v0 = nt * static_cast<int64_t>(kBN);
        const int64_t t0 = split * s.depth;
        if (v0 >= a.words) return;
        with_ends<kBN, false>(a.padded - d0, a.words - v0, [&](auto shape) {
            // (with few tokens never split)
            tile_dtable<T, decltype(shape), BN <= 64>(a, d0, v0, split, t0,
                                                      min(s.depth, held - t0), s.count == 1, lds);
        });
    }
}

// Four sums of the splits, `stride` apart, in their order; kStep of them on their way at a time.
__device__ __forceinline__ f32x4 splits_sum(const float *from, int64_t stride, unsigned splits) {
    constexpr unsigned kStep = 8;
    f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
    for (unsigned s0 = 0; s0 < splits; s0 += kStep) {
        f32x4 x[kStep];
#pragma unroll
        for (unsigned s = 0; s < kStep; ++s) {
            x[s] = *reinterpret_cast<const f32x4 *>(from + min(s0 + s, splits - 1) * stride);
        }
#pragma unroll
        for (unsigned s = 0; s < kStep; ++s) {
            if (s0 + s < splits) sum += x[s];
        }
    }
    return sum;
}

// dtable of a piece whose products were split: the splits' sums in their order.
template <typename T, int BN>
__global__ __launch_bounds__(kThreads) void dtable_join_kernel(Gradients a, bool both) {
    const int held = *a.held * copies_of<T>(*a.held);
    const unsigned splits =
        dtable_splits<T, BN>(a, held, load_of<T, BN>(a, held, both, true)).count;
    if (splits == 1) return;
    const float factor = *a.common * a.scale * (1.0f / kDzScale<T>);
    constexpr int kPer = kThreads / dev::kWave;
    int64_t v = blockIdx.x * static_cast<int64_t>(kPer) +
                __builtin_amdgcn_readfirstlane(threadIdx.x / dev::kWave);
    for (; v < a.words; v += gridDim.x * static_cast<int64_t>(kPer)) {
        const float *from = a.parts + v * a.sums_stride;
        for (int64_t d = 4ll * dev::lane(); d < a.width; d += 4 * dev::kWave) {
            const f32x4 sum = splits_sum(from + d, a.piece * a.sums_stride, splits);
            store_row4<T>(static_cast<T *>(a.dtable) + v * a.width, d, a.width, sum * factor);
        }
    }
}

// dx of every token: the splits' sums in their order, and 0 for a token without a target.
template <typename T, int BN, int LANES>
__global__ __launch_bounds__(kThreads) void dx_join_kernel(Gradients a,
                                                           const int *__restrict__ slot,
                                                           int64_t tokens, bool both,
                                                           T *__restrict__ dx) {
    const int copies = copies_of<T>(*a.held), held = *a.held * copies;
    const unsigned splits = dx_splits<T, BN>(a, held, load_of<T, BN>(a, held, true, both)).count;
    constexpr int kPer = kThreads / LANES;
    int64_t t = blockIdx.x * static_cast<int64_t>(kPer) +
                __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
    for (; t < tokens; t += gridDim.x * static_cast<int64_t>(kPer)) {
        const int at = slot[t];
        const float factor = (a.own ? a.own[t] : *a.common) * a.scale * (1.0f / kDzScale<T>);
        for (int64_t d = 4ll * (threadIdx.x % LANES); d < a.width; d += 4 * LANES) {
            f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
            if (at >= 0) {
                const float *from = a.sums + at * a.sums_stride + d;
                sum = splits_sum(from, held * a.sums_stride, splits);
                if (copies == 2) {
                    sum += splits_sum(from + held / 2 * a.sums_stride, held * a.sums_stride, splits);
                }
                sum *= factor;
            }
            store_row4<T>(dx + t * a.width, d, a.width, sum);
        }
    }
}

// ---- host -----------------------------------------------------------------------------

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Elements from row to row of a matrix in scratch: an odd number of 128-byte lines.  (Rows a power of
// two apart share few of the memory's channels, and a tile reads 256 rows at the same column.)
template <typename T>
int64_t scratch_stride(int64_t width) {
    const int64_t line = 128 / static_cast<int64_t>(sizeof(T));
    return up(width, line) / line % 2 ? up(width, line) : up(width, line) + line;
}

struct Args {
    int32_t dtype;
    int64_t tokens, words, width;
    float scale;
    int32_t reduction;
    const void *x;
    int64_t x_stride;
    const void *table;
    int64_t table_stride;
    const void *targets;
    int32_t id_bytes;
};

int check(const Args &a) {
    if (a.dtype < NACHO_F32 || a.dtype > NACHO_BF16 || a.tokens < 0 || a.words < 1 ||
        a.width < 1 || !(a.scale - a.scale == 0.0f) || a.reduction < NACHO_LOSS_NONE ||
        a.reduction > NACHO_LOSS_SUM || (a.id_bytes != 4 && a.id_bytes != 8)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if (a.words > NACHO_MAX_WORDS || a.tokens > NACHO_MAX_WORDS || a.width > NACHO_MAX_LOSS_WIDTH) {
        return NACHO_ERR_INDEX_OVERFLOW;
    }
    const int item = item_of(a.dtype);
    if (!a.table || !element_aligned(a.table, item) || a.table_stride < a.width) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if (a.tokens > 0 && (!a.x || !a.targets || !element_aligned(a.x, item) ||
                         !element_aligned(a.targets, a.id_bytes))) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    return NACHO_OK;
}

// A call's scratch: one allocation for all that it asks for.
struct Wanted {
    struct Piece {
        void **to;
        size_t bytes;
    } pieces[12];
    int n = 0;

    template <typename T>
    void add(T **to, int64_t count) {
        pieces[n++] = {reinterpret_cast<void **>(to), static_cast<size_t>(count) * sizeof(T)};
    }
    int get(Call &call) {
        size_t all = 0;
        for (int i = 0; i < n; ++i) all += (pieces[i].bytes + 255) / 256 * 256;
        char *p = nullptr;
        NACHO_TRY(call.scratch(all, reinterpret_cast<void **>(&p)));
        for (int i = 0; i < n; ++i) {
            *pieces[i].to = p;
            p += (pieces[i].bytes + 255) / 256 * 256;
        }
        return NACHO_OK;
    }
};

// The operands as the kernels take them: rows gathered and, where a table's rows are not whole
// aligned pieces, a copy of it whose are.
template <typename T>
struct Operands {
    Held held{};
    T *rows = nullptr;
    const T *table = nullptr;
    T *copy = nullptr;
    int64_t width = 0;  // of rows, a multiple of a piece
    int64_t rows_stride = 0;
    int64_t table_stride = 0;
    bool copied = false;
    bool parts = false;  // whether rows may have copies

    // (256 rows of a tile within the loads' 2 GB)
    static constexpr int64_t kMostStride = int64_t{1} << 22;

    void want(Wanted &wanted, const Args &a, const float *dloss) {
        width = up(a.width, 16 / sizeof(T));
        rows_stride = scratch_stride<T>(width);
        wanted.add(&held.count, 2);
        wanted.add(&held.slot, a.tokens);
        wanted.add(&held.token, a.tokens);
        wanted.add(&held.target, a.tokens);
        if (dloss) wanted.add(&held.common, 1);
        if (dloss && a.reduction == NACHO_LOSS_NONE) wanted.add(&held.factor, a.tokens);
        parts = dloss;
        wanted.add(&rows, (parts ? most_copies<T>(a.tokens) : a.tokens) * rows_stride);
        table = static_cast<const T *>(a.table);
        table_stride = a.table_stride;
        copied = !dense::pieces(a.table, a.table_stride, a.width, sizeof(T)) ||
                 table_stride * static_cast<int64_t>(sizeof(T)) > kMostStride;
        if (copied) {
            table_stride = scratch_stride<T>(width);
            wanted.add(&copy, a.words * table_stride);
        }
    }

    int start(hipStream_t s, const Args &a, const float *dloss) {
        const Targets targets{a.targets, a.id_bytes, a.words};
        const int tokens = static_cast<int>(a.tokens);
        const T *x = static_cast<const T *>(a.x);
        if (tokens <= kListMost) {
            list_rows_kernel<T><<<ceil_div(static_cast<size_t>(tokens), kListRows), kThreads, 0,
                                  s>>>(targets, tokens, a.reduction, dloss, held, a.width, width,
                                       x, a.x_stride, rows, rows_stride, parts);
            NACHO_TRY_HIP(hipGetLastError());
        } else {
            list_kernel<<<1, kListThreads, 0, s>>>(targets, tokens, a.reduction, dloss, held);
            NACHO_TRY_HIP(hipGetLastError());
            NACHO_TRY(gather(s, held.count, held.token, parts, a.tokens, a.width, x, a.x_stride, rows,
                             rows_stride));
        }
        if (copied) {
            NACHO_TRY(gather(s, nullptr, nullptr, false, a.words, a.width, table, a.table_stride,
                             copy, table_stride));
            table = copy;
        }
        return NACHO_OK;
    }

    int gather(hipStream_t s, const int *count, const int *token, bool with_parts, int64_t n,
               int64_t columns, const T *from, int64_t stride, T *to, int64_t to_stride) const {
        auto launch = [&](auto lanes) -> int {
            const int64_t groups = (n * lanes() + kThreads - 1) / kThreads;
            const unsigned grid = static_cast<unsigned>(groups < (1 << 20) ? groups : 1 << 20);
            gather_kernel<T, lanes()><<<grid, kThreads, 0, s>>>(
                count, token, with_parts, n, columns, width, from, stride, to, to_stride);
            NACHO_TRY_HIP(hipGetLastError());
            return NACHO_OK;
        };
        if (width * static_cast<int64_t>(sizeof(T)) <= 4096) return launch(Number<dev::kWave>{});
        return launch(Number<kThreads>{});
    }
};

// Calls f with the words and the tokens of a tile of logits, by the number of tokens: a tile's
// products of a few tokens would be of nothing.  Few tokens are bound by the table's bytes, of which
// small tiles of a small vocabulary have more on their way; and tiles are smaller where there are
// fewer than compute units.
//
// Measured, us of the loss / of both gradients (bfloat16 unless float32 is said), tokens x words x
// width, the tile that is taken and the other:
// - 16 tokens and 64.  8 x 5000 x 1024: 18 / 43 and 20 / 47; float32 25 / 58 and 49 / 90.
//   24 x 131072 x 4096 (of 64, or the table read twice): 191 / 765 and 205 / 776.  Not so for float32,
//   513 / 1772 and 430 / 1689, and small tables: 24 x 5000 x 1024 20 / 51 and 19 / 48.
// - 64 words and 256, up to 16 tokens.  1 x 16384 x 2048: 26 / 69 and 32 / 76; 1 x 65536 x 2048 (of 256)
//   49 / 241 and 50 / 239, 1 x 100000 x 2048 104 / 342 and 112 / 350.
// - 64 tokens and 256.  100 x 32768 x 2048: 38 / 169 and 38 / 188; 192 (of 256) 43 / 180 and 46 / 163,
//   float32 168 / 503 and 216 / 664; float32 of 100 is better off with 256, 149 / 465 and 134 / 384.
// - 128 words and 256, of 64 tokens, by two rounds of tiles.  64 x 32768 x 1024: 24 / 104 and 28 / 110;
//   128 x 65536 x 1024 (of 256) 34 / 193 and 40 / 206.
// - 128 words and 256, of 256 tokens, by one round.  256 x 5000 x 1024: 23 / 54 and 26 / 59;
//   256 x 65536 x 1024 (of 256) 44 / 205 and 52 / 215.  Just under a round 256 words are better: 256 x
//   50000 x 1024 49 / 200 and 42 / 184.
template <typename F>
int with_shape(int64_t tokens, int64_t words, F f) {
    auto tiles = [&](int64_t bn) { return up(words, 256) / 256 * (up(tokens, bn) / bn); };
    if (tokens <= 16) {
        if (words < 65536) return f(Number<64>{}, Number<16>{});
        return f(Number<256>{}, Number<16>{});
    }
    if (tokens <= 128) {
        if (tiles(64) < 2 * kUnits) return f(Number<128>{}, Number<64>{});
        return f(Number<256>{}, Number<64>{});
    }
    if (tiles(256) < kUnits) return f(Number<128>{}, Number<256>{});
    return f(Number<256>{}, Number<256>{});
}

// The same, and the columns of the gradients' tiles, whose rows are `columns` with the parts of dz.
template <typename F>
int with_shapes(int64_t tokens, int64_t columns, int64_t words, F f) {
    return with_shape(tokens, words, [&](auto bm, auto bn) -> int {
        if constexpr (bn() == 16) {
            if (columns <= 16) return f(bm, bn, Number<16>{});
            return f(bm, bn, Number<64>{});
        } else {
            return f(bm, bn, bn);
        }
    });
}

template <typename F>
int with_type(int32_t dtype, F f) {
    if (dtype == NACHO_F32) return f(float{});
    if (dtype == NACHO_F16) return f(_Float16{});
    return f(__bf16{});
}

// Workgroups of a launch, and of those at the end that cut tiles make; 0 for more than a launch has.
unsigned groups_of(int64_t m, int64_t bm, int64_t n, int64_t bn, int64_t more) {
    const int64_t all = up(m, bm) / bm * (up(n, bn) / bn) + more;
    return all < (int64_t{1} << 32) / kTileThreads ? static_cast<unsigned>(all) : 0u;
}

int forward(const Args &a, float *loss, float *stats, void *stream, const nacho_allocator *alloc) {
    NACHO_TRY(check(a));
    if (!loss && (a.tokens > 0 || a.reduction != NACHO_LOSS_NONE)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if (a.tokens == 0 && a.reduction == NACHO_LOSS_NONE) return NACHO_OK;
    Call call(stream, alloc);
    const hipStream_t s = call.stream();
    return with_type(a.dtype, [&](auto type) -> int {
        using T = decltype(type);
        return with_shape(a.tokens, a.words, [&](auto bm, auto bn) -> int {
            const unsigned m_tiles = static_cast<unsigned>(up(a.words, bm()) / bm());
            const unsigned groups =
                groups_of(a.words, bm(), a.tokens, bn(), bn() == 256 ? kUnits : 0);
            if (a.tokens > 0 && groups == 0) return NACHO_ERR_INDEX_OVERFLOW;
            if (a.tokens == 0) {  // (a reduction of none)
                sum_kernel<<<1, 1024, 0, s>>>(nullptr, 0, nullptr, 0, loss);
                NACHO_TRY_HIP(hipGetLastError());
                return NACHO_OK;
            }
            const int64_t n = a.tokens;
            const bool sums = a.reduction != NACHO_LOSS_NONE;
            Operands<T> ops;
            Wanted wanted;
            float2 *parts = nullptr;
            float *mine = nullptr, *most = stats, *each = loss;
            ops.want(wanted, a, nullptr);
            wanted.add(&parts, n * m_tiles);
            wanted.add(&mine, n);
            if (!stats) wanted.add(&most, 2 * n);
            if (sums) wanted.add(&each, n);
            NACHO_TRY(wanted.get(call));
            NACHO_TRY(ops.start(s, a, nullptr));
            Logits l{};
            l.held = ops.held.count;
            l.width = ops.width;
            l.rows = ops.rows;
            l.rows_stride = ops.rows_stride;
            l.table = ops.table;
            l.table_stride = ops.table_stride;
            l.words = static_cast<int>(a.words);
            l.m_tiles = m_tiles;
            l.target = ops.held.target;
            l.scale = a.scale;
            l.parts = parts;
            l.mine = mine;
            constexpr int kShapeThreads = Tile<bm(), bn()>::kThreads;
            parts_kernel<T, bm(), bn()><<<groups, kShapeThreads, 0, s>>>(l);
            NACHO_TRY_HIP(hipGetLastError());
            const int mean = a.reduction == NACHO_LOSS_MEAN;
            const int64_t joins = up(n, kThreads / dev::kWave) / (kThreads / dev::kWave);
            join_kernel<<<static_cast<unsigned>(joins < (1 << 20) ? joins : 1 << 20), kThreads, 0,
                          s>>>(ops.held.slot, static_cast<int>(n), m_tiles, parts, mine, most,
                               most + n, each, ops.held.count, mean,
                               sums && n <= kJoinMost ? loss : nullptr);
            NACHO_TRY_HIP(hipGetLastError());
            if (sums && n > kJoinMost) {
                sum_kernel<<<1, 1024, 0, s>>>(ops.held.count, n, each, mean, loss);
                NACHO_TRY_HIP(hipGetLastError());
            }
            return NACHO_OK;
        });
    });
}

// Words of a piece whose dz has `bytes` a word: all where that is little, or equal pieces that stay in
// the cache that the dies share.  (8192 tokens of 131072 words of 2048, us a step with pieces of 64 MB,
// which have too few tiles a launch, 16,550, of 128 MB 15,050, of 256 MB 15,600, of 512 MB 15,720;
// 3001 of 32003 words of 776, 192 MB, in one piece 440, in one of 128 MB and a rest 589.)
constexpr int64_t kPieceBytes = int64_t{128} << 20;
constexpr int64_t kPieceWords = 2048;

int64_t piece_of(int64_t words, int64_t bytes) {
    const int64_t all = up(words, 256);
    if (all * bytes <= 2 * kPieceBytes) return all;
    const int64_t pieces = (all * bytes + kPieceBytes - 1) / kPieceBytes;
    const int64_t piece = up((words + pieces - 1) / pieces, 256);
    return piece < kPieceWords ? (kPieceWords < all ? kPieceWords : all) : piece;
}

int backward(const Args &a, const float *stats, const float *dloss, void *dx, void *dtable,
             void *stream, const nacho_allocator *alloc) {
    NACHO_TRY(check(a));
    const int item = item_of(a.dtype);
    if (!element_aligned(dx, item) || !element_aligned(dtable, item) ||
        (a.tokens > 0 && (!stats || !dloss))) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if ((!dx || a.tokens == 0) && !dtable) return NACHO_OK;
    Call call(stream, alloc);
    const hipStream_t s = call.stream();
    return with_type(a.dtype, [&](auto type) -> int {
        using T = decltype(type);
        if (a.tokens == 0) {
            return dense::clear(s, static_cast<T *>(dtable), a.words * a.width);
        }
        const int64_t columns = most_copies<T>(a.tokens);
        return with_shapes(a.tokens, columns, a.words, [&](auto bm, auto tokens, auto bn) -> int {
            // of the logits' tiles, and of the gradients'
            constexpr int kBM = bm(), kTokens = tokens(), kBN = bn();
            // dz by the tokens' own gradients, and without them for dx
            const bool own = __is_same(T, _Float16) && a.reduction == NACHO_LOSS_NONE && dx;
            const int64_t piece = piece_of(a.words, columns * item);
            const int64_t cut = kTokens == 256 ? kUnits : 0;
            const unsigned dx_groups = groups_of(a.width, 256, columns, kBN, kMostItems);
            if (!groups_of(piece, kBM, a.tokens, kTokens, cut) || !dx_groups ||
                !groups_of(a.width, 256, piece, 64, dx_groups + kMostItems)) {
                return NACHO_ERR_INDEX_OVERFLOW;
            }
            Operands<T> ops;
            Wanted wanted;
            Logits l{};
            Gradients d{};
            T *dz = nullptr, *own_dz = nullptr;
            ops.want(wanted, a, dloss);
            l.dz_stride = d.dz_stride = scratch_stride<T>(piece);
            if (dtable || !own) wanted.add(&dz, columns * l.dz_stride);
            if (own) wanted.add(&own_dz, columns * l.dz_stride);
            d.sums_stride = up(a.width, 4);
            // Room for the sums of as many splits as are made: tiles of 256 columns by kBN tokens,
            // at most kMostItems of them where they are split; the same for dtable.
            const int64_t m_tiles = up(a.width, 256) / 256;
            const int64_t most = kMostItems / m_tiles * kBN;
            d.most_rows = columns * kMostSplits < most ? columns * kMostSplits : most;
            if (d.most_rows < columns) d.most_rows = columns;
            if (dx) wanted.add(&d.sums, d.most_rows * d.sums_stride);
            const int64_t tiles = m_tiles * (up(piece, 256) / 256);
            const int64_t deep = up(columns, 512) / 512;  // (splits are 8 steps or more)
            d.most_parts = kMostItems / tiles < deep ? kMostItems / tiles : deep;
            if (d.most_parts > kMostSplits) d.most_parts = kMostSplits;
            // (dx's products are as many: with both, or enough of one, no split is worth its while)
            const int64_t full = up(piece, 256) / 256 * tenths_of(a.width) / 10;
            const bool both = kBN == 256 && dx && dtable;
            if (full * (both ? 2 : 1) * 3 >= 4 * kUnits) d.most_parts = 1;
            if (kBN < 256 || d.most_parts < 2) d.most_parts = 1;
            if (dtable && d.most_parts > 1) {
                wanted.add(&d.parts, d.most_parts * piece * d.sums_stride);
            }
            NACHO_TRY(wanted.get(call));
            NACHO_TRY(ops.start(s, a, dloss));
            l.held = d.held = ops.held.count;
            l.width = d.padded = ops.width;
            l.rows = d.rows = ops.rows;
            l.rows_stride = d.rows_stride = ops.rows_stride;
            l.table_stride = d.table_stride = ops.table_stride;
            l.target = ops.held.target;
            l.scale = d.scale = a.scale;
            l.most = stats;
            l.total = stats + a.tokens;
            l.token = ops.held.token;
            l.factor = ops.held.factor;
            l.dz = dz;
            l.own_dz = own_dz;
            d.dz = dz;
            d.dx_dz = own ? own_dz : dz;
            d.own = own ? dloss : nullptr;
            l.table = ops.table;
            d.width = a.width;
            d.piece = piece;
            d.common = ops.held.common;
            for (int64_t v = 0; v < a.words; v += piece) {
                const int64_t words = a.words - v < piece ? a.words - v : piece;
                l.first = static_cast<int>(v);
                l.words = static_cast<int>(words);
                dz_kernel<T, kBM, kTokens><<<groups_of(words, kBM, a.tokens, kTokens, cut),
                                             Tile<kBM, kTokens>::kThreads, 0, s>>>(l);
                NACHO_TRY_HIP(hipGetLastError());
                d.words = words;
                d.table = ops.table + v * ops.table_stride;
                d.first = v == 0;
                if (dtable) d.dtable = static_cast<T *>(dtable) + v * a.width;
                const unsigned dtable_groups = groups_of(
                    a.width, 256, piece, kBN <= 64 ? 64 : kBN, d.most_parts > 1 ? kMostItems : 0);
                if (both) {
                    gradients_kernel<T, 256, true, true>
                        <<<dx_groups + dtable_groups, kTileThreads, 0, s>>>(d);
                    NACHO_TRY_HIP(hipGetLastError());
                }
                if (dx && !both) {
                    gradients_kernel<T, kBN, true, false><<<dx_groups, kTileThreads, 0, s>>>(d);
                    NACHO_TRY_HIP(hipGetLastError());
                }
                if (dtable && !both) {
                    gradients_kernel<T, kBN, false, true>
                        <<<dtable_groups, kTileThreads, 0, s>>>(d);
                    NACHO_TRY_HIP(hipGetLastError());
                }
                if (dtable && d.most_parts > 1) {
                    const int64_t rows = (words + 3) / 4;
                    dtable_join_kernel<T, kBN>
                        <<<static_cast<unsigned>(rows < (1 << 20) ? rows : 1 << 20), kThreads, 0,
                           s>>>(d, both);
                    NACHO_TRY_HIP(hipGetLastError());
                }
            }
            if (dx) {
                auto join = [&](auto lanes) -> int {
                    const int64_t groups = (a.tokens * lanes() + kThreads - 1) / kThreads;
                    dx_join_kernel<T, kBN, lanes()>
                        <<<static_cast<unsigned>(groups < (1 << 20) ? groups : 1 << 20), kThreads,
                           0, s>>>(d, ops.held.slot, a.tokens, both, static_cast<T *>(dx));
                    NACHO_TRY_HIP(hipGetLastError());
                    return NACHO_OK;
                };
                NACHO_TRY(a.width <= 1024 ? join(Number<dev::kWave>{}) : join(Number<kThreads>{}));
            }
            return NACHO_OK;
        });
    });
}

}  // namespace cross_entropy
}  // namespace nacho

extern "C" int nacho_linear_cross_entropy(int32_t dtype, int64_t tokens, int64_t words,
                                          int64_t width, float scale, int32_t reduction,
                                          const void *x, int64_t x_stride, const void *table,
                                          int64_t table_stride, const void *targets,
                                          int32_t id_bytes, float *loss, float *stats,
                                          void *stream, const nacho_allocator *alloc) {
    try {
        return nacho::cross_entropy::forward({dtype, tokens, words, width, scale, reduction, x,
                                              x_stride, table, table_stride, targets, id_bytes},
                                             loss, stats, stream, alloc);
    } catch (const std::bad_alloc &) {
        return NACHO_ERR_OUT_OF_MEMORY;
    }
}

extern "C" int nacho_linear_cross_entropy_backward(
    int32_t dtype, int64_t tokens, int64_t words, int64_t width, float scale, int32_t reduction,
    const void *x, int64_t x_stride, const void *table, int64_t table_stride, const void *targets,
    int32_t id_bytes, const float *stats, const float *dloss, void *dx, void *dtable,
    void *stream, const nacho_allocator *alloc) {
    try {
        return nacho::cross_entropy::backward({dtype, tokens, words, width, scale, reduction, x,
                                               x_stride, table, table_stride, targets, id_bytes},
                                              stats, dloss, dx, dtable, stream, alloc);
    } catch (const std::bad_alloc &) {
        return NACHO_ERR_OUT_OF_MEMORY;
    }
}
