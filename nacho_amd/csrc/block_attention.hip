// Attention over blocks of keys selected per query, forward and backward.
//
// out = softmax(scale q K^T) V over the keys of the query's blocks, in one pass with a running
// maximum m and sum l per row.  The heads of a key head's group share the blocks, so a tile's
// rows are (token, head) pairs of consecutive tokens and one key head, and a tile goes over the
// union of its tokens' blocks: each block has a mask of the tokens that selected it, and the
// scores of other rows are -inf there.  Neighbouring tokens select much the same blocks, so the
// union is little longer than one token's list; a wavefront none of whose rows selected a block
// passes over it.
//
// Products are transposed: S^T = K Q^T puts a row's keys into the four lanes of its column, so
// the row's maximum is two lane exchanges, and P^T already lies as the operand of
// O^T = V^T P^T (dense_tiles.hpp).  Probabilities are rounded to the operands' type for that
// product, as its operand has to be; their sum l is of the unrounded ones in float32.
//
// Backward, with delta = dout . out and p from the stored lse: ds = p (dout . v - delta),
// dq = scale ds K goes tile by tile as the forward pass; dk = scale ds^T Q and dv = p^T dout go
// block by block over the tokens that selected the block, found from a bit matrix [block][token],
// the transpose of the lists; so no sum depends on an order of atomics.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <new>
#include <type_traits>

#include "dense_tiles.hpp"
#include "runtime.hpp"

namespace nacho {
namespace attention {

using namespace dense;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / dev::kWave;
constexpr int kWindow = 512;  // blocks whose masks are in LDS at a time

struct Shape {
    int batch, queries, keys, q_heads, kv_heads, dim, block, count, causal;
    int group;   // q_heads / kv_heads
    int blocks;  // ceil(keys / block)
    float scale;
};

template <typename T>
struct Heads {
    T *data;
    int64_t batch_stride, row_stride, head_stride;
    __device__ __forceinline__ T *row(int b, int64_t r, int h) const {
        return data + b * batch_stride + r * row_stride + h * head_stride;
    }
};

template <typename T>
Heads<T> heads(const nacho_heads &h) {
    return Heads<T>{static_cast<T *>(h.data), h.batch_stride, h.row_stride, h.head_stride};
}

template <typename T>
struct Args {
    Shape s;
    Heads<T> q, k, v, out, dout, dq, dk, dv;
    const int *lengths;
    const int *ids;
    float *lse;
};

__device__ __forceinline__ int length_of(const Shape &s, const int *lengths, int b) {
    return lengths ? min(max(lengths[b], 0), s.keys) : s.keys;
}

// The rows of a tile of R rows: `tokens` consecutive tokens times the group's heads, or part of
// one token's heads where the group is larger than the tile.
struct Tiling {
    int tokens;    // tokens of a tile
    int parts;     // tiles of one token
    int per_head;  // tiles of a (sequence, key head)
};

__host__ __device__ inline Tiling tiling(const Shape &s, int rows) {
    Tiling t;
    t.tokens = s.group <= rows ? rows / s.group : 1;
    t.parts = s.group <= rows ? 1 : (s.group + rows - 1) / rows;
    t.per_head = ((s.queries + t.tokens - 1) / t.tokens) * t.parts;
    return t;
}

template <int R>
struct Tile {
    int b, h, t0, head0, tokens;  // tokens: those that exist
    int length, place0;           // place of token t0

    // heads: sequences x key heads; the fastest index, so that workgroups that follow each
    // other, which go to different XCDs, read different heads' keys.
    __device__ __forceinline__ Tile(const Shape &s, const int *lengths, int index) {
        const Tiling tl = tiling(s, R);
        const int heads = s.batch * s.kv_heads;
        const int bh = index % heads;
        const int tile = tl.per_head - 1 - index / heads;  // the longest lists first
        b = bh / s.kv_heads;
        h = bh % s.kv_heads;
        t0 = tile / tl.parts * tl.tokens;
        head0 = tile % tl.parts * R;
        tokens = min(tl.tokens, s.queries - t0);
        length = length_of(s, lengths, b);
        place0 = length - s.queries + t0;
    }
    // Row r: its token in the tile and head of q; false where the tile has none.
    __device__ __forceinline__ bool row(const Shape &s, int r, int &token, int &head) const {
        if (s.group <= R) {
            token = r / s.group;
            head = h * s.group + r % s.group;
            return token < tokens;
        }
        token = 0;
        head = h * s.group + head0 + r;
        return head0 + r < s.group;
    }
    // Last key that token sees (-1: none).
    __device__ __forceinline__ int last_key(const Shape &s, int token) const {
        const int place = place0 + token;
        if (place < 0) return -1;
        return s.causal ? place : length - 1;
    }
};

// The union of the tile's blocks within [first, first + kWindow): mask[] by block of the
// window, and the numbers of the blocks with a token, ascending, in ids[0 .. returned).
struct Lists {
    unsigned long long mask[kWindow];
    unsigned short ids[kWindow];
    int sums[kWaves];
};

template <int R>
__device__ int window_lists(const Shape &s, const int *__restrict__ ids, const Tile<R> &tile,
                            int first, Lists &lists) {
    __syncthreads();  // (the lists of the window before are done with)
    for (int i = threadIdx.x; i < kWindow; i += kThreads) lists.mask[i] = 0ull;
    __syncthreads();
    for (int i = threadIdx.x; i < tile.tokens * s.count; i += kThreads) {
        const int token = i / s.count, x = i - token * s.count;
        const int last = tile.last_key(s, token);
        const int64_t row =
            (static_cast<int64_t>(tile.b) * s.queries + tile.t0 + token) * s.kv_heads + tile.h;
        const int id = ids[row * s.count + x];
        // (unsigned: an id < 0 is past the last one)
        if (last >= 0 && static_cast<unsigned>(id) <= static_cast<unsigned>(last / s.block) &&
            id >= first && id < first + kWindow) {
            atomicOr(&lists.mask[id - first], 1ull << token);
        }
    }
    __syncthreads();
    constexpr int kPer = kWindow / kThreads;
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) mine += lists.mask[threadIdx.x * kPer + j] != 0ull;
    int total = 0;
    int at = dev::block_exclusive_sum<kThreads>(mine, lists.sums, total);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = threadIdx.x * kPer + j;
        if (lists.mask[i] != 0ull) lists.ids[at++] = static_cast<unsigned short>(i);
    }
    __syncthreads();
    return total;
}

// ---- forward, tiles of 64 rows --------------------------------------------------------

// One online-softmax step for a row (a lane's column) over 16 N keys: s are the products, at
// most the first `limit` keys from the step's first (this lane's g included) are seen.  Updates
// the running maximum and sum and returns the factor for what was summed before.
template <int N>
__device__ __forceinline__ float softmax_step(f32x4 (&s)[N], float scale2, int limit, float &m,
                                              float &l) {
    if (!__all(limit >= 16 * N)) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[t][i] = 16 * t + i < limit ? s[t][i] * scale2 : kNegInf;
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < N; ++t) s[t] *= scale2;
    }
    float top = kNegInf;
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][i]);
    }
    const float now = fmaxf(m, column_max(top));
    const float base = now == kNegInf ? 0.0f : now;
    const float factor = exp2_fast(m - base);
    m = now;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[t][i] = exp2_fast(s[t][i] - base);
            sum += s[t][i];
        }
    }
    l = l * factor + sum;
    return factor;
}

// The keys of a step that a row sees, as softmax_step's limit.
__device__ __forceinline__ int step_limit(bool selected, int last_key, int first_key, int g) {
    return selected ? last_key + 1 - first_key - 4 * g : 0;
}

template <typename T, int DP, int BN>
__global__ __launch_bounds__(kThreads) void tile_kernel(Args<T> a) {
    constexpr int kRow = kTileRow<T, DP>;
    __shared__ __align__(16) T s_k[BN * kRow];
    __shared__ __align__(16) T s_v[BN * kRow];
    __shared__ Lists s_lists;
    const Shape &s = a.s;
    const Tile<64> tile(s, a.lengths, static_cast<int>(blockIdx.x));
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
    int token, head;
    const bool exists = tile.row(s, 16 * wave + c, token, head);
    const int last_key = exists ? tile.last_key(s, token) : -1;
    Frag<T> q[DP / 32];
    load_row_frags<T, DP>(exists ? a.q.row(tile.b, tile.t0 + token, head) : nullptr, s.dim, g, q);
    f32x4 o[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = kNegInf, l = 0.0f;
    const float scale2 = s.scale * kLog2e;
    const T *k_base = a.k.row(tile.b, 0, tile.h), *v_base = a.v.row(tile.b, 0, tile.h);
    const int end = tile.last_key(s, tile.tokens - 1) + 1;  // keys that some row sees
    const int steps_of = s.block / BN;
    TileLoad<T, DP, BN, kThreads> k_next, v_next;
    for (int first = 0; first * s.block < end; first += kWindow) {  // uniform
        const int steps = window_lists(s, a.ids, tile, first, s_lists) * steps_of;
        auto first_key = [&](int step) {
            return (first + s_lists.ids[step / steps_of]) * s.block + step % steps_of * BN;
        };
        auto load = [&](int step) {
            const int key = first_key(step);
            k_next.load(threadIdx.x, s.dim, [&](int r) -> const T * {
                return key + r < tile.length ? k_base + (key + r) * a.k.row_stride : nullptr;
            });
            v_next.load(threadIdx.x, s.dim, [&](int r) -> const T * {
                return key + r < tile.length ? v_base + (key + r) * a.v.row_stride : nullptr;
            });
        };
        if (steps > 0) load(0);
        for (int step = 0; step < steps; ++step) {
            __syncthreads();
            k_next.store(threadIdx.x, s_k);
            v_next.store(threadIdx.x, s_v);
            __syncthreads();
            if (step + 1 < steps) load(step + 1);
            const unsigned long long tokens = s_lists.mask[s_lists.ids[step / steps_of]];
            const bool selected = exists && (tokens >> token & 1ull);
            const int limit = step_limit(selected, last_key, first_key(step), g);
            if (!__any(limit > 0)) continue;
            f32x4 p[BN / 16];
#pragma unroll
            for (int t = 0; t < BN / 16; ++t) {
                p[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int kk = 0; kk < DP / 32; ++kk) {
                    p[t] = mma(row_frag<T>(s_k + (16 * t + c) * kRow + 32 * kk + 8 * g), q[kk],
                               p[t]);
                }
            }
            const float factor = softmax_step<BN / 16>(p, scale2, limit, m, l);
            if (!__all(factor == 1.0f)) {
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) o[i] *= factor;
            }
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) {
                const Frag<T> pf = result_frag<T>(p[2 * u], p[2 * u + 1]);
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    o[i] = mma(column_frag<kRow>(s_v + 32 * u * kRow, 16 * i, g, c), pf, o[i]);
                }
            }
        }
    }
    l = column_sum(l);
    if (!exists) return;
    const float inverse = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;  // (NaN stays)
    T *out = a.out.row(tile.b, tile.t0 + token, head);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        const int col = 16 * i + 4 * g;
        if (col < s.dim) store4<T>(out + col, o[i] * inverse);
    }
    if (a.lse && g == 0) {
        a.lse[(static_cast<int64_t>(tile.b) * s.queries + tile.t0 + token) * s.q_heads + head] =
            l == 0.0f ? kNegInf : (m + log2_fast(l)) * kLn2;
    }
}

// ---- forward, few rows: tiles of 16 rows, their blocks split over wavefronts -----------

// Partial results of a split: per row its maximum and sum (base 2) and its sum of p v.
struct Partials {
    float *ml;  // [tile][split][16][2]
    float *o;   // [tile][split][16][DP]
};

constexpr int kSplitKeys = 32;  // keys of a step

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void split_kernel(Args<T> a, int splits, Partials part) {
    constexpr int kRow = kTileRow<T, DP>;
    constexpr int kJoin = DP + 4;  // floats of a row of o in LDS
    constexpr int kTileBytes = kSplitKeys * kRow * static_cast<int>(sizeof(T));
    constexpr int kJoinBytes = 16 * kJoin * 4;
    constexpr int kWaveBytes = kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes;
    __shared__ __align__(16) unsigned char s_wave[kWaves][kWaveBytes];
    __shared__ float s_m[kWaves][16], s_l[kWaves][16];
    __shared__ Lists s_lists;
    const Shape &s = a.s;
    const int split = static_cast<int>(blockIdx.x) % splits;
    const int index = static_cast<int>(blockIdx.x) / splits;
    const Tile<16> tile(s, a.lengths, index);
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
    T *s_v = reinterpret_cast<T *>(s_wave[wave]);
    int token, head;
    const bool exists = tile.row(s, c, token, head);
    const int last_key = exists ? tile.last_key(s, token) : -1;
    Frag<T> q[DP / 32];
    load_row_frags<T, DP>(exists ? a.q.row(tile.b, tile.t0 + token, head) : nullptr, s.dim, g, q);
    f32x4 o[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = kNegInf, l = 0.0f;
    const float scale2 = s.scale * kLog2e;
    const T *k_base = a.k.row(tile.b, 0, tile.h), *v_base = a.v.row(tile.b, 0, tile.h);
    const int end = tile.last_key(s, tile.tokens - 1) + 1;
    const int steps_of = s.block / kSplitKeys;
    const int stride = splits * kWaves;
    TileLoad<T, DP, kSplitKeys, dev::kWave> v_next;
    Frag<T> k_next[2][DP / 32];
    for (int first = 0; first * s.block < end; first += kWindow) {  // uniform
        const int steps = window_lists(s, a.ids, tile, first, s_lists) * steps_of;
        auto first_key = [&](int step) {
            return (first + s_lists.ids[step / steps_of]) * s.block + step % steps_of * kSplitKeys;
        };
        auto load = [&](int step) {
            const int key = first_key(step);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int r = key + 16 * t + c;
                load_row_frags<T, DP>(r < tile.length ? k_base + r * a.k.row_stride : nullptr,
                                      s.dim, g, k_next[t]);
            }
            v_next.load(lane, s.dim, [&](int r) -> const T * {
                return key + r < tile.length ? v_base + (key + r) * a.v.row_stride : nullptr;
            });
        };
        int step = split * kWaves + wave;
        if (step < steps) load(step);
        for (; step < steps; step += stride) {  // the wavefront's own
            const unsigned long long tokens = s_lists.mask[s_lists.ids[step / steps_of]];
            const bool selected = exists && (tokens >> token & 1ull);
            const int limit = step_limit(selected, last_key, first_key(step), g);
            f32x4 p[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                p[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int kk = 0; kk < DP / 32; ++kk) p[t] = mma(k_next[t][kk], q[kk], p[t]);
            }
            dev::wave_sync();  // the reads of the step before
            v_next.store(lane, s_v);
            dev::wave_sync();
            if (step + stride < steps) load(step + stride);
            if (!__any(limit > 0)) continue;
            const float factor = softmax_step<2>(p, scale2, limit, m, l);
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) o[i] *= factor;
            const Frag<T> pf = result_frag<T>(p[0], p[1]);
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                o[i] = mma(column_frag<kRow>(s_v, 16 * i, g, c), pf, o[i]);
            }
        }
    }
    l = column_sum(l);
    // Join the wavefronts: each row's sums are brought to the largest maximum.
    dev::wave_sync();
    float *s_o = reinterpret_cast<float *>(s_wave[wave]);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        *reinterpret_cast<f32x4 *>(s_o + c * kJoin + 16 * i + 4 * g) = o[i];
    }
    if (g == 0) {
        s_m[wave][c] = m;
        s_l[wave][c] = l;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * DP; x += kThreads) {
        const int r = x / DP, col = x % DP;
        int t, hd;
        if (!tile.row(s, r, t, hd)) continue;
        float top = kNegInf;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_m[w][r]);
        const float base = top == kNegInf ? 0.0f : top;
        float sum = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = exp2_fast(s_m[w][r] - base);
            sum += f * s_l[w][r];
            v += f * reinterpret_cast<const float *>(s_wave[w])[r * kJoin + col];
        }
        if (splits > 1) {
            const int64_t at = (static_cast<int64_t>(index) * splits + split) * 16 + r;
            part.o[at * DP + col] = v;
            if (col == 0) {
                part.ml[2 * at] = top;
                part.ml[2 * at + 1] = sum;
            }
            continue;
        }
        const float inverse = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
        if (col < s.dim) {
            a.out.row(tile.b, tile.t0 + t, hd)[col] = static_cast<T>(v * inverse);
        }
        if (col == 0 && a.lse) {
            a.lse[(static_cast<int64_t>(tile.b) * s.queries + tile.t0 + t) * s.q_heads + hd] =
                sum == 0.0f ? kNegInf : (top + log2_fast(sum)) * kLn2;
        }
    }
}

// Joins the splits of a row: a workgroup of DP threads per row of a tile.
template <typename T, int DP>
__global__ __launch_bounds__(DP) void join_kernel(Args<T> a, int splits, Partials part) {
    const Shape &s = a.s;
    const int index = static_cast<int>(blockIdx.x) / 16, r = static_cast<int>(blockIdx.x) % 16;
    const Tile<16> tile(s, a.lengths, index);
    int t, hd;
    if (!tile.row(s, r, t, hd)) return;
    const int64_t at = static_cast<int64_t>(index) * splits * 16 + r;
    float top = kNegInf;
    for (int i = 0; i < splits; ++i) top = fmaxf(top, part.ml[2 * (at + 16 * i)]);
    const float base = top == kNegInf ? 0.0f : top;
    float sum = 0.0f, v = 0.0f;
    const int col = static_cast<int>(threadIdx.x);
    for (int i = 0; i < splits; ++i) {
        const int64_t x = at + 16 * i;
        const float f = exp2_fast(part.ml[2 * x] - base);
        sum += f * part.ml[2 * x + 1];
        v += f * part.o[x * DP + col];
    }
    const float inverse = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
    if (col < s.dim) a.out.row(tile.b, tile.t0 + t, hd)[col] = static_cast<T>(v * inverse);
    if (col == 0 && a.lse) {
        a.lse[(static_cast<int64_t>(tile.b) * s.queries + tile.t0 + t) * s.q_heads + hd] =
            sum == 0.0f ? kNegInf : (top + log2_fast(sum)) * kLn2;
    }
}

// ---- backward -------------------------------------------------------------------------

// delta[b][t][head] = dout . out: 16 lanes per row.
template <typename T>
__global__ __launch_bounds__(kThreads) void delta_kernel(Args<T> a, float *__restrict__ delta) {
    const Shape &s = a.s;
    const int64_t rows = static_cast<int64_t>(s.batch) * s.queries * s.q_heads;
    const int64_t r = blockIdx.x * static_cast<int64_t>(kThreads / 16) + threadIdx.x / 16;
    const int c = threadIdx.x % 16;
    float v = 0.0f;
    if (r < rows) {
        const int head = static_cast<int>(r % s.q_heads);
        const int64_t bt = r / s.q_heads;
        const int t = static_cast<int>(bt % s.queries), b = static_cast<int>(bt / s.queries);
        const T *x = a.dout.row(b, t, head), *y = a.out.row(b, t, head);
        for (int col = 8 * c; col < s.dim; col += 128) {
            const Frag<T> fx = row_frag<T>(x + col), fy = row_frag<T>(y + col);
#pragma unroll
            for (int j = 0; j < 8; ++j) v += static_cast<float>(fx[j]) * static_cast<float>(fy[j]);
        }
    }
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) v += __shfl_xor(v, off, dev::kWave);
    if (r < rows && c == 0) delta[r] = v;
}

// bits[b][h][block][token / 32]: the tokens that see something of the block through their ids.
__global__ __launch_bounds__(kThreads) void mark_kernel(Shape s, const int *__restrict__ lengths,
                                                        const int *__restrict__ ids, int words,
                                                        unsigned *__restrict__ bits) {
    const int64_t n = static_cast<int64_t>(s.batch) * s.queries * s.kv_heads * s.count;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int id = ids[i];
        const int64_t row = i / s.count;
        const int h = static_cast<int>(row % s.kv_heads);
        const int64_t bt = row / s.kv_heads;
        const int t = static_cast<int>(bt % s.queries), b = static_cast<int>(bt / s.queries);
        const int length = length_of(s, lengths, b);
        const int place = length - s.queries + t;
        const int last = place < 0 ? -1 : s.causal ? place : length - 1;
        if (last < 0 || static_cast<unsigned>(id) > static_cast<unsigned>(last / s.block)) continue;
        const int64_t at = (static_cast<int64_t>(b) * s.kv_heads + h) * s.blocks + id;
        atomicOr(&bits[at * words + t / 32], 1u << (t % 32));
    }
}

__global__ __launch_bounds__(kThreads) void clear_kernel(unsigned *__restrict__ words, int64_t n) {
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        words[i] = 0u;
    }
}

// Gradient of the scores from the products s = q . k and dp = dout . v of 16 N keys: ds (without
// the scale) replaces dp, and the probabilities s.
template <int N>
__device__ __forceinline__ void score_gradient(f32x4 (&s)[N], f32x4 (&dp)[N], float scale2,
                                               float lse2, float delta, int limit) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool seen = 16 * t + i < limit;
            s[t][i] = seen ? exp2_fast(s[t][i] * scale2 - lse2) : 0.0f;
            dp[t][i] = seen ? s[t][i] * (dp[t][i] - delta) : 0.0f;
        }
    }
}

template <typename T, int DP, int BN>
__global__ __launch_bounds__(kThreads) void dq_kernel(Args<T> a, const float *__restrict__ delta) {
    constexpr int kRow = kTileRow<T, DP>;
    __shared__ __align__(16) T s_k[BN * kRow];
    __shared__ __align__(16) T s_v[BN * kRow];
    __shared__ Lists s_lists;
    const Shape &s = a.s;
    const Tile<64> tile(s, a.lengths, static_cast<int>(blockIdx.x));
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
    int token, head;
    const bool exists = tile.row(s, 16 * wave + c, token, head);
    const int last_key = exists ? tile.last_key(s, token) : -1;
    Frag<T> q[DP / 32], dout[DP / 32];
    load_row_frags<T, DP>(exists ? a.q.row(tile.b, tile.t0 + token, head) : nullptr, s.dim, g, q);
    load_row_frags<T, DP>(exists ? a.dout.row(tile.b, tile.t0 + token, head) : nullptr, s.dim, g,
                          dout);
    const int64_t at =
        (static_cast<int64_t>(tile.b) * s.queries + tile.t0 + token) * s.q_heads + head;
    const float lse = exists ? a.lse[at] : 0.0f;
    const float lse2 = lse == kNegInf ? 0.0f : lse * kLog2e;
    const float row_delta = exists ? delta[at] : 0.0f;
    f32x4 o[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const float scale2 = s.scale * kLog2e;
    const T *k_base = a.k.row(tile.b, 0, tile.h), *v_base = a.v.row(tile.b, 0, tile.h);
    const int end = tile.last_key(s, tile.tokens - 1) + 1;
    const int steps_of = s.block / BN;
    TileLoad<T, DP, BN, kThreads> k_next, v_next;
    for (int first = 0; first * s.block < end; first += kWindow) {  // uniform
        const int steps = window_lists(s, a.ids, tile, first, s_lists) * steps_of;
        auto first_key = [&](int step) {
            return (first + s_lists.ids[step / steps_of]) * s.block + step % steps_of * BN;
        };
        auto load = [&](int step) {
            const int key = first_key(step);
            k_next.load(threadIdx.x, s.dim, [&](int r) -> const T * {
                return key + r < tile.length ? k_base + (key + r) * a.k.row_stride : nullptr;
            });
            v_next.load(threadIdx.x, s.dim, [&](int r) -> const T * {
                return key + r < tile.length ? v_base + (key + r) * a.v.row_stride : nullptr;
            });
        };
        if (steps > 0) load(0);
        for (int step = 0; step < steps; ++step) {
            __syncthreads();
            k_next.store(threadIdx.x, s_k);
            v_next.store(threadIdx.x, s_v);
            __syncthreads();
            if (step + 1 < steps) load(step + 1);
            const unsigned long long tokens = s_lists.mask[s_lists.ids[step / steps_of]];
            const bool selected = exists && (tokens >> token & 1ull);
            const int limit = step_limit(selected, last_key, first_key(step), g);
            if (!__any(limit > 0)) continue;
            f32x4 p[BN / 16], dp[BN / 16];
#pragma unroll
            for (int t = 0; t < BN / 16; ++t) {
                p[t] = dp[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int kk = 0; kk < DP / 32; ++kk) {
                    const int x = (16 * t + c) * kRow + 32 * kk + 8 * g;
                    p[t] = mma(row_frag<T>(s_k + x), q[kk], p[t]);
                    dp[t] = mma(row_frag<T>(s_v + x), dout[kk], dp[t]);
                }
            }
            score_gradient<BN / 16>(p, dp, scale2, lse2, row_delta, limit);
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) {
                const Frag<T> ds = result_frag<T>(dp[2 * u], dp[2 * u + 1]);
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    o[i] = mma(column_frag<kRow>(s_k + 32 * u * kRow, 16 * i, g, c), ds, o[i]);
                }
            }
        }
    }
    if (!exists) return;
    T *dq = a.dq.row(tile.b, tile.t0 + token, head);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        const int col = 16 * i + 4 * g;
        if (col < s.dim) store4<T>(dq + col, o[i] * s.scale);
    }
}

constexpr int kTokenWords = 64;  // words of a block's bits that are listed at a time
constexpr int kRows = 32;        // (token, head) rows of a step

// dk and dv of 16 x WAVES keys of a block: each wavefront has 16 keys' columns, and all go over
// the rows of the tokens that selected the block.
template <typename T, int DP, int WAVES>
__global__ __launch_bounds__(WAVES *dev::kWave) void dkv_kernel(
    Args<T> a, const float *__restrict__ delta, int words, const unsigned *__restrict__ bits) {
    constexpr int kBlock = WAVES * dev::kWave;
    constexpr int kRow = kTileRow<T, DP>;
    __shared__ __align__(16) T s_q[kRows * kRow];
    __shared__ __align__(16) T s_do[kRows * kRow];
    __shared__ __align__(16) float s_lse[kRows], s_delta[kRows];
    __shared__ __align__(16) int s_last[kRows];
    __shared__ unsigned short s_tokens[kTokenWords * 32];
    __shared__ int s_sums[WAVES];
    const Shape &s = a.s;
    const int heads = s.batch * s.kv_heads;
    const int parts = s.block / (16 * WAVES);
    const int bh = static_cast<int>(blockIdx.x) % heads;
    const int part = static_cast<int>(blockIdx.x) / heads;
    const int id = part / parts;
    const int b = bh / s.kv_heads, h = bh % s.kv_heads;
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
    const int length = length_of(s, a.lengths, b);
    const int key = id * s.block + part % parts * 16 * WAVES + 16 * wave + c;
    const bool exists = key < length;
    Frag<T> k[DP / 32], v[DP / 32];
    load_row_frags<T, DP>(exists ? a.k.row(b, key, h) : nullptr, s.dim, g, k);
    load_row_frags<T, DP>(exists ? a.v.row(b, key, h) : nullptr, s.dim, g, v);
    f32x4 dk[DP / 16], dv[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) dk[i] = dv[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const float scale2 = s.scale * kLog2e;
    const int place0 = length - s.queries;
    const unsigned *row_bits = bits + (static_cast<int64_t>(bh) * s.blocks + id) * words;
    TileLoad<T, DP, kRows, kBlock> q_next, do_next;
    for (int w0 = 0; w0 < words; w0 += kTokenWords) {  // uniform
        // the tokens of these words, ascending
        __syncthreads();
        const int w = static_cast<int>(threadIdx.x);
        unsigned mine = w < kTokenWords && w0 + w < words ? row_bits[w0 + w] : 0u;
        int total = 0;
        int at = dev::block_exclusive_sum<kBlock>(static_cast<int>(__popc(mine)), s_sums,
                                                   total);
        for (; mine; mine &= mine - 1u) {
            s_tokens[at++] = static_cast<unsigned short>(32 * w + __ffs(mine) - 1);
        }
        __syncthreads();
        const int rows = total * s.group;
        auto token_of = [&](int r) { return 32 * w0 + s_tokens[r / s.group]; };
        auto load = [&](int r0) {
            q_next.load(threadIdx.x, s.dim, [&](int r) -> const T * {
                const int x = r0 + r;
                return x < rows ? a.q.row(b, token_of(x), h * s.group + x % s.group) : nullptr;
            });
            do_next.load(threadIdx.x, s.dim, [&](int r) -> const T * {
                const int x = r0 + r;
                return x < rows ? a.dout.row(b, token_of(x), h * s.group + x % s.group) : nullptr;
            });
        };
        if (rows > 0) load(0);
        for (int r0 = 0; r0 < rows; r0 += kRows) {
            __syncthreads();
            q_next.store(threadIdx.x, s_q);
            do_next.store(threadIdx.x, s_do);
            if (threadIdx.x < kRows) {
                const int x = r0 + static_cast<int>(threadIdx.x);
                float lse = 0.0f, d = 0.0f;
                int last = -1;
                if (x < rows) {
                    const int t = token_of(x);
                    const int64_t i = (static_cast<int64_t>(b) * s.queries + t) * s.q_heads +
                                      h * s.group + x % s.group;
                    lse = a.lse[i];
                    lse = lse == kNegInf ? 0.0f : lse * kLog2e;
                    d = delta[i];
                    last = s.causal ? place0 + t : length - 1;
                }
                s_lse[threadIdx.x] = lse;
                s_delta[threadIdx.x] = d;
                s_last[threadIdx.x] = last;
            }
            __syncthreads();
            if (r0 + kRows < rows) load(r0 + kRows);
            f32x4 p[kRows / 16], dp[kRows / 16];
#pragma unroll
            for (int t = 0; t < kRows / 16; ++t) {
                p[t] = dp[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int kk = 0; kk < DP / 32; ++kk) {
                    const int x = (16 * t + c) * kRow + 32 * kk + 8 * g;
                    p[t] = mma(row_frag<T>(s_q + x), k[kk], p[t]);
                    dp[t] = mma(row_frag<T>(s_do + x), v[kk], dp[t]);
                }
                // this lane's rows 16 t + 4 g + i, its key in each
                const f32x4 lse = *reinterpret_cast<const f32x4 *>(s_lse + 16 * t + 4 * g);
                const f32x4 d = *reinterpret_cast<const f32x4 *>(s_delta + 16 * t + 4 * g);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool seen = key <= s_last[16 * t + 4 * g + i];
                    p[t][i] = seen ? exp2_fast(p[t][i] * scale2 - lse[i]) : 0.0f;
                    dp[t][i] = seen ? p[t][i] * (dp[t][i] - d[i]) : 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < kRows / 32; ++u) {
                const Frag<T> pf = result_frag<T>(p[2 * u], p[2 * u + 1]);
                const Frag<T> ds = result_frag<T>(dp[2 * u], dp[2 * u + 1]);
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    dv[i] = mma(column_frag<kRow>(s_do + 32 * u * kRow, 16 * i, g, c), pf, dv[i]);
                    dk[i] = mma(column_frag<kRow>(s_q + 32 * u * kRow, 16 * i, g, c), ds, dk[i]);
                }
            }
        }
    }
    if (key >= s.keys) return;  // (keys past the length have gradients: zeros)
    T *out_k = a.dk.row(b, key, h), *out_v = a.dv.row(b, key, h);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        const int col = 16 * i + 4 * g;
        if (col < s.dim) {
            store4<T>(out_k + col, dk[i] * s.scale);
            store4<T>(out_v + col, dv[i]);
        }
    }
}

// ---- host -----------------------------------------------------------------------------

bool aligned(const nacho_heads &h, int item, bool optional = false) {
    if (!h.data) return optional;
    const int64_t per = 16 / item;
    return reinterpret_cast<uintptr_t>(h.data) % 16 == 0 && h.batch_stride % per == 0 &&
           h.row_stride % per == 0 && h.head_stride % per == 0;
}

int check(const nacho_block_attention_args *p, bool backward, Shape *s) {
    if (!p || p->dtype < NACHO_F32 || p->dtype > NACHO_BF16) return NACHO_ERR_INVALID_ARGUMENT;
    if (p->batch < 0 || p->queries < 0 || p->keys < 0 || p->q_heads < 1 || p->kv_heads < 1 ||
        p->q_heads % p->kv_heads != 0 || p->head_dim < 8 || p->head_dim > 128 ||
        p->head_dim % 8 != 0 || (p->block != 32 && p->block != 64 && p->block != 128) ||
        p->count < 0 || (p->causal != 0 && p->causal != 1) || !std::isfinite(p->scale)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    const int64_t rows = static_cast<int64_t>(p->batch) * p->queries * p->q_heads;
    const int64_t blocks = (static_cast<int64_t>(p->keys) + p->block - 1) / p->block;
    const int64_t parts = blocks * (p->block / 32) * p->batch * p->kv_heads;
    if (rows > INT32_MAX / 16 || parts > INT32_MAX || p->keys > INT32_MAX - 256 ||
        p->count > INT32_MAX / 64) {
        return NACHO_ERR_INDEX_OVERFLOW;
    }
    const int item = p->dtype == NACHO_F32 ? 4 : 2;
    const bool no_rows = rows == 0, no_keys = p->batch == 0 || p->keys == 0;
    if (!aligned(p->q, item, no_rows) || !aligned(p->k, item, no_keys) ||
        !aligned(p->v, item, no_keys) || !aligned(p->out, item, no_rows) ||
        (!p->blocks && !no_rows && p->count > 0)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    if (backward && (!aligned(p->dout, item, no_rows) || !aligned(p->dq, item, no_rows) ||
                     !aligned(p->dk, item, no_keys) || !aligned(p->dv, item, no_keys) ||
                     (!p->lse && !no_rows))) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    *s = Shape{p->batch,    p->queries,  p->keys,  p->q_heads,
               p->kv_heads, p->head_dim, p->block, p->count,
               p->causal,   p->q_heads / p->kv_heads, static_cast<int>(blocks), p->scale};
    return NACHO_OK;
}

template <typename T>
Args<T> args_of(const nacho_block_attention_args &p, const Shape &s) {
    return Args<T>{s,
                   heads<T>(p.q),
                   heads<T>(p.k),
                   heads<T>(p.v),
                   heads<T>(p.out),
                   heads<T>(p.dout),
                   heads<T>(p.dq),
                   heads<T>(p.dk),
                   heads<T>(p.dv),
                   p.lengths,
                   p.blocks,
                   p.lse};
}

// Calls f with the keys of a step: 64, or 32 where the block or float32's tiles (twice as large:
// 32 keys keep two workgroups on a CU) want it.
template <typename T, typename F>
void with_step(const Shape &s, F f) {
    if constexpr (sizeof(T) == 2) {
        if (s.block % 64 == 0) return f(std::integral_constant<int, 64>{});
    }
    f(std::integral_constant<int, 32>{});
}

constexpr int kFullGrid = 256;  // workgroups that occupy the device: one per CU

template <typename T, int DP>
int forward(Call &call, const Args<T> &a) {
    const Shape &s = a.s;
    const hipStream_t stream = call.stream();
    const int heads = s.batch * s.kv_heads;
    const int tiles = tiling(s, 64).per_head * heads;
    if (tiles >= kFullGrid) {
        with_step<T>(s, [&](auto keys) {
            tile_kernel<T, DP, keys()><<<static_cast<unsigned>(tiles), kThreads, 0, stream>>>(a);
        });
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    }
    const Tiling small = tiling(s, 16);
    const int64_t few = static_cast<int64_t>(small.per_head) * heads;
    const int64_t listed = static_cast<int64_t>(small.tokens) * s.count;
    const int64_t steps = (listed < s.blocks ? listed : s.blocks) * (s.block / kSplitKeys);
    int64_t splits = (2 * kFullGrid + few - 1) / few;
    const int64_t most = (steps + kWaves - 1) / kWaves;
    if (splits > most) splits = most;
    if (splits < 1) splits = 1;
    Partials part{};
    if (splits > 1) {
        const size_t rows = static_cast<size_t>(few) * static_cast<size_t>(splits) * 16;
        NACHO_TRY(call.scratch_n(2 * rows, &part.ml));
        NACHO_TRY(call.scratch_n(rows * DP, &part.o));
    }
    split_kernel<T, DP><<<static_cast<unsigned>(few * splits), kThreads, 0, stream>>>(
        a, static_cast<int>(splits), part);
    NACHO_TRY_HIP(hipGetLastError());
    if (splits > 1) {
        join_kernel<T, DP><<<static_cast<unsigned>(few * 16), DP, 0, stream>>>(
            a, static_cast<int>(splits), part);
        NACHO_TRY_HIP(hipGetLastError());
    }
    return NACHO_OK;
}

unsigned grid_for(int64_t n, int per) {
    const int64_t want = (n + per - 1) / per;
    return static_cast<unsigned>(want < 1 ? 1 : want > 65536 ? 65536 : want);
}

template <typename T, int DP>
int backward(Call &call, const Args<T> &a) {
    const Shape &s = a.s;
    const hipStream_t stream = call.stream();
    const int heads = s.batch * s.kv_heads;
    const int64_t rows = static_cast<int64_t>(s.batch) * s.queries * s.q_heads;
    const int words = (s.queries + 31) / 32;
    const int64_t all_words = static_cast<int64_t>(heads) * s.blocks * words;
    float *delta = nullptr;
    unsigned *bits = nullptr;
    NACHO_TRY(call.scratch_n(static_cast<size_t>(rows), &delta));
    NACHO_TRY(call.scratch_n(static_cast<size_t>(all_words), &bits));
    if (rows > 0) {
        delta_kernel<T><<<static_cast<unsigned>((rows + 15) / 16), kThreads, 0, stream>>>(a, delta);
        NACHO_TRY_HIP(hipGetLastError());
        const unsigned tiles = static_cast<unsigned>(tiling(s, 64).per_head * heads);
        with_step<T>(s, [&](auto keys) {
            dq_kernel<T, DP, keys()><<<tiles, kThreads, 0, stream>>>(a, delta);
        });
        NACHO_TRY_HIP(hipGetLastError());
    }
    if (heads * static_cast<int64_t>(s.blocks) > 0) {
        if (all_words > 0) {
            clear_kernel<<<grid_for(all_words, kThreads), kThreads, 0, stream>>>(bits, all_words);
            NACHO_TRY_HIP(hipGetLastError());
            const int64_t n = rows / s.group * s.count;
            mark_kernel<<<grid_for(n, kThreads), kThreads, 0, stream>>>(s, a.lengths, a.ids, words,
                                                                        bits);
            NACHO_TRY_HIP(hipGetLastError());
        }
        if (s.block % 64 == 0) {
            const unsigned grid = static_cast<unsigned>(heads * s.blocks * (s.block / 64));
            dkv_kernel<T, DP, 4><<<grid, 4 * dev::kWave, 0, stream>>>(a, delta, words, bits);
        } else {
            const unsigned grid = static_cast<unsigned>(heads * s.blocks * (s.block / 32));
            dkv_kernel<T, DP, 2><<<grid, 2 * dev::kWave, 0, stream>>>(a, delta, words, bits);
        }
        NACHO_TRY_HIP(hipGetLastError());
    }
    return NACHO_OK;
}

template <typename T>
int run(const nacho_block_attention_args &p, const Shape &s, Call &call, bool back) {
    const Args<T> a = args_of<T>(p, s);
    if (s.dim <= 64) return back ? backward<T, 64>(call, a) : forward<T, 64>(call, a);
    return back ? backward<T, 128>(call, a) : forward<T, 128>(call, a);
}

int attention(const nacho_block_attention_args *p, void *stream, const nacho_allocator *alloc,
              bool back) {
    Shape s{};
    NACHO_TRY(check(p, back, &s));
    const bool no_rows = static_cast<int64_t>(s.batch) * s.queries == 0;
    if (no_rows && (!back || s.keys == 0 || s.batch == 0)) return NACHO_OK;
    Call call(stream, alloc);
    switch (p->dtype) {
        case NACHO_F32: return run<float>(*p, s, call, back);
        case NACHO_F16: return run<_Float16>(*p, s, call, back);
        default: return run<__bf16>(*p, s, call, back);
    }
}

}  // namespace attention
}  // namespace nacho

extern "C" int nacho_block_attention(const nacho_block_attention_args *args, void *stream,
                                     const nacho_allocator *alloc) {
    try {
        return nacho::attention::attention(args, stream, alloc, false);
    } catch (const std::bad_alloc &) {
        return NACHO_ERR_OUT_OF_MEMORY;
    }
}

extern "C" int nacho_block_attention_backward(const nacho_block_attention_args *args, void *stream,
                                              const nacho_allocator *alloc) {
    try {
        return nacho::attention::attention(args, stream, alloc, true);
    } catch (const std::bad_alloc &) {
        return NACHO_ERR_OUT_OF_MEMORY;
    }
}
