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
// O^T = V^T P^T (dense_tiles.hpp).  An operand of a product has to have the rows' type.  Where a
// sequence has few rows, bound by their keys' bytes, 16-bit types take a probability in two parts,
// so that out is what rounding it once makes it: 0.0017 of its norm off with bfloat16, 0.0002 with
// float16.  Where it has many, bound by products, one rounded part is taken: out is 0.0022 and
// 0.00026 off for three quarters of the time (kPartsRows).  The sum l is of the unrounded ones in
// float32 either way.
//
// Backward, with delta = dout . out and p from the stored lse: ds = p (dout . v - delta),
// dq = scale ds K goes tile by tile as the forward pass; dk = scale ds^T Q and dv = p^T dout go
// block by block over the tokens that selected the block, found from a bit matrix [block][token],
// the transpose of the lists; so no sum depends on an order of atomics.
//
// A key that a row does not see must not reach it, whatever its values: keys past the sequence's
// end are read as zeros, but a block's other rows are there for the tile's other tokens, and 0
// times infinity is no number.  So a tile whose result is not finite is done again with masks key
// by key and with the values that are not finite taken out (Pass); nothing else pays for that.
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
// Ids of a query: those of 128 queries, which a tile or a workgroup that marks tokens may have,
// are counted in 32 bits, kThreads at a time.
constexpr int kMostIds = (INT_MAX - kThreads) / 128;

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
struct Forward {
    Shape s;
    Heads<T> q, k, v, out;
    const int *lengths;
    const int *ids;
    float *lse;
};

template <typename T>
struct Backward : Forward<T> {
    Heads<T> dout, dq, dk, dv;
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
struct RowTile {
    int b, h, t0, head0, tokens;  // tokens: those that exist
    int length, place0;           // place of token t0

    // heads: sequences x key heads; the fastest index, so that workgroups that follow each
    // other, which go to different XCDs, read different heads' keys.
    __device__ __forceinline__ RowTile(const Shape &s, const int *lengths, int index) {
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

// The union of the tile's blocks within [first, first + kWindow): a mask of tokens by block of
// the window, and the numbers of the blocks with a token, ascending, in ids[0 .. returned).
template <int R>
struct Lists {
    static constexpr int kWords = (R + 63) / 64;
    unsigned long long mask[kWindow][kWords];
    unsigned short ids[kWindow];
    int sums[kWaves];

    __device__ __forceinline__ bool has(int nth, int token) const {
        return mask[ids[nth]][token / 64] >> (token % 64) & 1ull;
    }
};

template <int R>
__device__ int window_lists(const Shape &s, const int *__restrict__ ids, const RowTile<R> &tile,
                            int first, Lists<R> &lists) {
    constexpr int kWords = Lists<R>::kWords;
    __syncthreads();  // (the lists of the window before are done with)
    for (int i = threadIdx.x; i < kWindow * kWords; i += kThreads) (&lists.mask[0][0])[i] = 0ull;
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
            atomicOr(&lists.mask[id - first][token / 64], 1ull << (token % 64));
        }
    }
    __syncthreads();
    constexpr int kPer = kWindow / kThreads;
    auto filled = [&](int i) {
        unsigned long long any = lists.mask[i][0];
#pragma unroll
        for (int w = 1; w < kWords; ++w) any |= lists.mask[i][w];
        return any != 0ull;
    };
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) mine += filled(threadIdx.x * kPer + j);
    int total = 0;
    int at = dev::block_exclusive_sum<kThreads>(mine, lists.sums, total);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = threadIdx.x * kPer + j;
        if (filled(i)) lists.ids[at++] = static_cast<unsigned short>(i);
    }
    __syncthreads();
    return total;
}

// How a tile is worked on: as it is; where that is not finite, once more for which results see
// something that is not (these keep what they have), and once with what is not finite left out of
// the products over keys, for the others.
enum Pass { kPlain = 0, kMarks, kFinite };

// A result of a pass after kPlain's, at a place that holds those of the passes before.
template <typename T>
__device__ __forceinline__ void store_again(T *p, float v, int pass) {
    const float there = static_cast<float>(*p);
    if (pass == kMarks ? v == 0.0f : there - there == 0.0f) {
        *p = static_cast<T>(pass == kMarks ? 0.0f : v);
    }
}

// Goes over the tile's blocks BN keys at a time: use(k, v, nth, first key) with both operands'
// rows in LDS, while the next step's are on their way into the other buffer.  Rows past the
// sequence's end are zeros.  Every wavefront calls it, and every one calls `use` for every step.
//
// Loads go from memory to LDS without registers, into one of two buffers while the other is used.
template <typename T, int DP, int BN, int R>
struct KeySteps {
    using Lds = Tile<T, DP, BN, kThreads>;
    T *k[2], *v[2];
    Lists<R> &lists;

    // masked: the operand (k or v) whose products over keys the pass concerns, for passes after
    // kPlain's to mask when it has arrived; null where `use` does that.
    template <typename Use>
    __device__ __forceinline__ void run(const Forward<T> &a, const RowTile<R> &tile, int pass,
                                        T *const *masked, Use use) {
        const Shape &s = a.s;
        const T *k_base = a.k.row(tile.b, 0, tile.h), *v_base = a.v.row(tile.b, 0, tile.h);
        const int end = tile.last_key(s, tile.tokens - 1) + 1;  // keys that some row sees
        const int shift = s.block / BN == 1 ? 0 : s.block / BN == 2 ? 1 : 2;  // steps of a block
        const typename Lds::Source k_source(threadIdx.x, s.dim, a.k.row_stride);
        const typename Lds::Source v_source(threadIdx.x, s.dim, a.v.row_stride);
        for (int first = 0; first * s.block < end; first += kWindow) {  // uniform
            const int steps = window_lists(s, a.ids, tile, first, lists) << shift;
            auto first_key = [&](int step) {
                return (first + __builtin_amdgcn_readfirstlane(lists.ids[step >> shift])) *
                           s.block +
                       (step & ((1 << shift) - 1)) * BN;
            };
            auto load = [&](int step, T *to_k, T *to_v) {
                const int key = first_key(step), there = tile.length - key;
                Lds::load(to_k, threadIdx.x, k_source, k_base + key * a.k.row_stride, there);
                Lds::load(to_v, threadIdx.x, v_source, v_base + key * a.v.row_stride, there);
            };
            auto arrived = [&](int buffer) {
                rows_arrived();
                if (pass != kPlain && masked) {  // uniform
                    Lds::make_finite(masked[buffer], threadIdx.x, pass == kMarks);
                    __syncthreads();
                }
            };
            if (steps > 0) load(0, k[0], v[0]);
            arrived(0);
            for (int step = 0; step < steps; step += 2) {
                if (step + 1 < steps) load(step + 1, k[1], v[1]);
                use(k[0], v[0], step >> shift, first_key(step));
                arrived(1);
                if (step + 2 < steps) load(step + 2, k[0], v[0]);
                if (step + 1 < steps) use(k[1], v[1], (step + 1) >> shift, first_key(step + 1));
                arrived(0);
            }
        }
    }
};

// ---- forward, tiles of 64 or 128 rows -------------------------------------------------

// The factor of q . k for base-2 exponentials.  It is not negative (operands are negated for a
// negative scale), so that the largest product is the largest score, and not 0, so that a masked
// score of -inf stays one.
__device__ __forceinline__ float base2_scale(float scale) {
    return fmaxf(fabsf(scale) * kLog2e, 1.17549435e-38f);
}

// The running maximum follows a row's when it is 2^kSlack behind.  float16's probabilities in two
// parts are 2^kUp times as large, so that neither part of one of more than 2^-25 is 0.
template <typename T, bool PARTS>
constexpr int kUp = __is_same(T, _Float16) && PARTS ? 13 : 0;
template <int UP>
constexpr float kSlack = UP ? 15 - UP : 8;

// One online-softmax step for a row (a lane's column) over 16 N keys: s are the products, the
// first `limit` keys from the step's first (this lane's 4 g included) are seen.  s become the
// probabilities against the running maximum m, which may stay up to kSlack below the row's own
// (they are at most 2^(UP + kSlack) then): sums are brought to a new one only when some row of the
// wavefront needs it.  Returns whether they were, by `factor`.
//
// Most steps are seen whole or not at all: a row that sees nothing of a step takes a maximum of
// infinity there, and only steps that some row sees in part, or every one after kPlain's pass, are
// masked key by key.  With kMarks the scores are 0, so that each key that a row sees counts, the
// ones of the least probabilities too.
template <int UP, int N>
__device__ __forceinline__ bool softmax_step(f32x4 (&s)[N], float scale2, int limit, int pass,
                                             float &m, float &l, float &factor) {
    const bool none = limit <= 0;
    if (pass != kPlain || __any(!none && limit < 16 * N)) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float seen = pass == kMarks ? 0.0f : s[t][i];
                s[t][i] = 16 * t + i < limit ? seen : kNegInf;
            }
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[t][i]);
    }
    top = column_max(none ? kNegInf : top) * scale2;
    const bool moved = __any(top > m + kSlack<UP>);
    factor = 1.0f;
    if (moved) {
        const float now = fmaxf(m, top);
        factor = now == kNegInf ? 1.0f : exp2_fast(m - now);
        m = now;
        l *= factor;
    }
    const float base = none ? -kNegInf : m == kNegInf ? 0.0f : m - UP;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[t][i] = exp2_fast(__builtin_fmaf(s[t][i], scale2, -base));
            sum += s[t][i];
        }
    }
    l += sum;
    return moved;
}

// The keys of a step that a row sees, as softmax_step's limit.
__device__ __forceinline__ int step_limit(bool selected, int last_key, int first_key, int g) {
    return selected ? last_key + 1 - first_key - 4 * g : 0;
}

// What a row's sum of p v is to be multiplied by: `sum` is that of p.
template <typename T, bool PARTS>
__device__ __forceinline__ float row_factor(float sum) {
    return sum > 0.0f ? (PARTS ? kPartsScale<T> : 1.0f) / sum : sum == 0.0f ? 0.0f : sum;
}

// The log of a row's sum of exponentials, from its maximum and sum of base 2.
template <typename T, bool PARTS>
__device__ __forceinline__ float row_lse(float m, float sum) {
    return sum == 0.0f ? kNegInf : (m - kUp<T, PARTS> + log2_fast(sum)) * kLn2;
}

// A lane's rows of a tile: COLS of them, 16 apart.
template <int COLS>
struct LaneRows {
    int token[COLS], head[COLS], last_key[COLS];
    bool exists[COLS];

    __device__ __forceinline__ LaneRows(const Shape &s, const RowTile<64 * COLS> &tile, int wave,
                                        int c) {
#pragma unroll
        for (int x = 0; x < COLS; ++x) {
            exists[x] = tile.row(s, 16 * (COLS * wave + x) + c, token[x], head[x]);
            if (!exists[x]) token[x] = 0;
            last_key[x] = exists[x] ? tile.last_key(s, token[x]) : -1;
        }
    }
    // softmax_step's limits; whether some row of the wavefront sees a key
    __device__ __forceinline__ bool limits(const Lists<64 * COLS> &lists, int nth, int first_key,
                                           int g, int (&limit)[COLS]) const {
        bool any = false;
#pragma unroll
        for (int x = 0; x < COLS; ++x) {
            const bool selected = exists[x] && lists.has(nth, token[x]);
            limit[x] = step_limit(selected, last_key[x], first_key, g);
            any = any || limit[x] > 0;
        }
        return __any(any);
    }
};

// 64 COLS rows of a key head, four wavefronts.  Each has COLS column tiles of 16 rows, which share
// what it reads of LDS: with one, LDS takes as long as the matrix products and the softmax each.
//
// 8192 queries of 32 heads of 128 (8 key heads, bfloat16), 16 of 128 blocks: 306 us.  The union of
// a wavefront's rows is 27 blocks where each selects 15, so 233 GFLOP are done for 125 that are
// asked for, at 760 TFLOP/s; a large matrix product of the library reaches 1250 here.  Matrix
// products are 32% of a CU's time and the vector unit 42%, and with two wavefronts to a SIMD (254
// registers) these overlap only in part: that is the bound.  64 single tokens of caches of 16384
// keys, with the same heads and blocks: 50 us for 270 MB, 5.4 TB/s, near a large copy's 5.7.
// Three sequences of up to 777 queries of 12 heads of 80 in float32, 9 blocks of 32: 55 to 70 us
// by their lengths, half of it float32 matrix products.
template <typename T, int DP, int BN, int COLS, bool PARTS>
__global__ __launch_bounds__(kThreads, 2) void tile_kernel(Forward<T> a) {
    using Lds = Tile<T, DP, BN, kThreads>;
    constexpr int kRowsOf = 64 * COLS;
    __shared__ __align__(16) T s_k0[Lds::kElements];
    __shared__ __align__(16) T s_v0[Lds::kElements];
    __shared__ __align__(16) T s_k1[Lds::kElements];
    __shared__ __align__(16) T s_v1[Lds::kElements];
    __shared__ Lists<kRowsOf> s_lists;
    const Shape &s = a.s;
    const RowTile<kRowsOf> tile(s, a.lengths, static_cast<int>(blockIdx.x));
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
    const LaneRows<COLS> rows(s, tile, wave, c);
    Frag<T> q[COLS][DP / 32];
    f32x4 o[COLS][DP / 16];
    float m[COLS], l[COLS];
#pragma unroll
    for (int x = 0; x < COLS; ++x) {
        load_row_frags<T, DP>(
            rows.exists[x] ? a.q.row(tile.b, tile.t0 + rows.token[x], rows.head[x]) : nullptr,
            s.dim, g, q[x]);
        if (s.scale < 0.0f) negate<T, DP>(q[x]);
    }
    const float scale2 = base2_scale(s.scale);
    KeySteps<T, DP, BN, kRowsOf> steps{{s_k0, s_k1}, {s_v0, s_v1}, s_lists};
    for (int pass = kPlain; pass <= kFinite; ++pass) {  // uniform
#pragma unroll
        for (int x = 0; x < COLS; ++x) {
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) o[x][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            m[x] = kNegInf;
            l[x] = 0.0f;
        }
        T *const masked[2] = {s_v0, s_v1};
        steps.run(a, tile, pass, masked, [&](const T *s_k, const T *s_v, int nth, int first_key) {
            int limit[COLS];
            if (!rows.limits(s_lists, nth, first_key, g, limit)) return;
            f32x4 p[COLS][BN / 16];
            row_products<Lds, T, DP, COLS, BN / 16>(s_k, q, g, c, p);
#pragma unroll
            for (int x = 0; x < COLS; ++x) {
                float factor;
                if (softmax_step<kUp<T, PARTS>>(p[x], scale2, limit[x], pass, m[x], l[x], factor)) {
#pragma unroll
                    for (int i = 0; i < DP / 16; ++i) o[x][i] *= factor;
                }
            }
            column_products<Lds, T, DP, COLS, BN / 16, PARTS ? kTwo : kOne>(s_v, p, g, c, o);
        });
        float wrong = 0.0f;
#pragma unroll
        for (int x = 0; x < COLS; ++x) {
            wrong += not_finite<DP / 16>(o[x]) + l[x] * 0.0f;
            const float sum = column_sum(l[x]);
            if (!rows.exists[x]) continue;
            const float inverse = row_factor<T, PARTS>(sum);
            const int t = tile.t0 + rows.token[x], head = rows.head[x];
            T *out = a.out.row(tile.b, t, head);
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                const int col = 16 * i + 4 * g;
                if (col >= s.dim) continue;
                if (pass == kPlain) {
                    store4<T>(out + col, o[x][i] * inverse);
                    continue;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) store_again(out + col + j, o[x][i][j] * inverse, pass);
            }
            if (a.lse && g == 0) {
                a.lse[(static_cast<int64_t>(tile.b) * s.queries + t) * s.q_heads + head] =
                    row_lse<T, PARTS>(m[x], sum);
            }
        }
        if (pass == kPlain && !__syncthreads_or(wrong != wrong)) break;
    }
}

// ---- forward, few rows: tiles of 16 rows, their blocks split over wavefronts -----------

// Partial results of a split: per row its maximum and sum (base 2) and its sum of p v.
struct Partials {
    float *ml;  // [tile][split][16][2]
    float *o;   // [tile][split][16][DP]
};

constexpr int kSplitKeys = 32;  // keys of a step

// ONE: a tile is one token (of at most 64 ids): its ids are the list, and its rows see the same
// keys, so that nothing is masked but what is read as zeros.
//
// Keys go from memory into operand registers, since no other wavefront reads them; values pass
// through the wavefront's own LDS for the transposed read.  One step is on its way while the last
// is worked on; with two, which take the registers of a CU, a call is 0.7 us longer.
// Bound by the time that operands take to arrive, while there is less than one workgroup to a
// CU: one token of 16 heads of 64 over 8 blocks of 32 takes 6.0 us a call, one of 32 heads of
// 128 over 16 blocks of 64 11.5 with the launch that joins its splits (12.9 without ONE), 32
// such tokens 33 us for 134 MB.
template <typename T, int DP, bool ONE>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 ? 1 : 2) void split_kernel(
    Forward<T> a, int splits, Partials part) {
    using Stage = TileStage<T, DP, kSplitKeys>;
    constexpr int kJoin = DP + 4;  // floats of a row of o in LDS
    constexpr int kTileBytes = Stage::Lds::kElements * static_cast<int>(sizeof(T));
    constexpr int kJoinBytes = 16 * kJoin * 4;
    constexpr int kWaveBytes = kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes;
    __shared__ __align__(16) unsigned char s_wave[kWaves][kWaveBytes];
    __shared__ float s_m[kWaves][16], s_l[kWaves][16];
    __shared__ std::conditional_t<ONE, int[kWaves][dev::kWave], Lists<16>> s_lists;
    const Shape &s = a.s;
    const int split = static_cast<int>(blockIdx.x) % splits;
    const int index = static_cast<int>(blockIdx.x) / splits;
    const RowTile<16> tile(s, a.lengths, index);
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
    T *s_v = reinterpret_cast<T *>(s_wave[wave]);
    int token, head;
    const bool exists = tile.row(s, c, token, head);
    if (!exists) token = 0;
    const int last_key = exists ? tile.last_key(s, token) : -1;
    Frag<T> q[1][DP / 32];
    load_row_frags<T, DP>(exists ? a.q.row(tile.b, tile.t0 + token, head) : nullptr, s.dim, g,
                          q[0]);
    if (s.scale < 0.0f) negate<T, DP>(q[0]);
    f32x4 o[1][DP / 16];
    float m, l;
    int pass = kPlain;
    const float scale2 = base2_scale(s.scale);
    const T *k_base = a.k.row(tile.b, 0, tile.h), *v_base = a.v.row(tile.b, 0, tile.h);
    // Keys that some row sees; past them zeros are read.  (Not the sequence's end: a later
    // token's keys may lie in the last one's block, and with ONE nothing else masks values.)
    const int end = tile.last_key(s, tile.tokens - 1) + 1;
    const int shift = s.block == 32 ? 0 : s.block == 64 ? 1 : 2;  // steps of a block
    const int stride = splits * kWaves;
    Stage v_next;
    Frag<T> k_next[2][DP / 32];
    // The wavefront's own of `steps` steps; block_of(n): the n-th block, selected(n): whether
    // the lane's row selected it.
    auto work = [&](int steps, auto block_of, auto selected) {
        auto first_key = [&](int step) {
            return block_of(step >> shift) * s.block + (step & ((1 << shift) - 1)) * kSplitKeys;
        };
        auto load = [&](int step) {
            const int key = first_key(step);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int r = key + 16 * t + c;
                load_row_frags<T, DP>(r < end ? k_base + r * a.k.row_stride : nullptr, s.dim, g,
                                      k_next[t]);
            }
            v_next.load(lane, s.dim, [&](int r) -> const T * {
                return key + r < end ? v_base + (key + r) * a.v.row_stride : nullptr;
            });
        };
        const int from = split * kWaves + wave;
        if (from < steps) load(from);
        for (int step = from; step < steps; step += stride) {
            const int limit =
                step_limit(exists && selected(step >> shift), last_key, first_key(step), g);
            f32x4 p[1][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                p[0][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int kk = 0; kk < DP / 32; ++kk) {
                    p[0][t] = mma(k_next[t][kk], q[0][kk], p[0][t]);
                }
            }
            dev::wave_sync();  // the reads of the step before
            if (pass != kPlain) v_next.make_finite(pass == kMarks);
            v_next.store(lane, s_v);
            dev::wave_sync();
            if (step + stride < steps) load(step + stride);
            if (!__any(limit > 0)) continue;
            float factor;
            if (softmax_step<kUp<T, true>>(p[0], scale2, limit, pass, m, l, factor)) {
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) o[0][i] *= factor;
            }
            column_products<typename Stage::Lds, T, DP, 1, 2, kTwo>(s_v, p, g, c, o);
        }
    };
    for (;; ++pass) {  // uniform
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) o[0][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m = kNegInf;
        l = 0.0f;
        if constexpr (ONE) {
            // The valid ids, once each.  Every wavefront makes its own copy.
            const int last = tile.last_key(s, 0);
            const int64_t row =
                (static_cast<int64_t>(tile.b) * s.queries + tile.t0) * s.kv_heads + tile.h;
            const int id = lane < s.count ? a.ids[row * s.count + lane] : -1;
            bool first =
                last >= 0 && static_cast<unsigned>(id) <= static_cast<unsigned>(last / s.block);
            for (int j = 0; j + 1 < s.count; ++j) {
                const int other = __builtin_amdgcn_readlane(id, j);
                first = first && !(j < lane && other == id);
            }
            const unsigned long long listed = __ballot(first);
            int *list = s_lists[wave];
            if (first) list[__popcll(listed & ((1ull << lane) - 1ull))] = id;
            dev::wave_sync();
            work(static_cast<int>(__popcll(listed)) << shift,
                 [&](int n) { return __builtin_amdgcn_readfirstlane(list[n]); },
                 [](int) { return true; });
        } else {
            for (int first = 0; first * s.block < end; first += kWindow) {  // uniform
                const int blocks = window_lists(s, a.ids, tile, first, s_lists);
                work(blocks << shift,
                     [&](int n) {
                         return first + __builtin_amdgcn_readfirstlane(s_lists.ids[n]);
                     },
                     [&](int n) { return s_lists.has(n, token); });
            }
        }
        l = column_sum(l);
        // Join the wavefronts: each row's sums are brought to the largest maximum.
        dev::wave_sync();
        float *s_o = reinterpret_cast<float *>(s_wave[wave]);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            *reinterpret_cast<f32x4 *>(s_o + c * kJoin + 16 * i + 4 * g) = o[0][i];
        }
        if (g == 0) {
            s_m[wave][c] = m;
            s_l[wave][c] = l;
        }
        __syncthreads();
        bool wrong = false;
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
            wrong = wrong || !(v - v == 0.0f) || !(sum - sum == 0.0f);
            if (splits > 1) {
                const int64_t at = (static_cast<int64_t>(index) * splits + split) * 16 + r;
                if (pass == kPlain) {
                    part.o[at * DP + col] = v;
                } else {
                    store_again(&part.o[at * DP + col], v, pass);
                }
                if (col == 0) {
                    part.ml[2 * at] = top;
                    part.ml[2 * at + 1] = sum;
                }
                continue;
            }
            const float inverse = row_factor<T, true>(sum);
            T *out = a.out.row(tile.b, tile.t0 + t, hd) + col;
            if (col < s.dim && pass == kPlain) *out = static_cast<T>(v * inverse);
            if (col < s.dim && pass != kPlain) store_again(out, v * inverse, pass);
            if (col == 0 && a.lse) {
                a.lse[(static_cast<int64_t>(tile.b) * s.queries + tile.t0 + t) * s.q_heads + hd] =
                    row_lse<T, true>(top, sum);
            }
        }
        if (ONE || pass == kFinite) break;
        if (!__syncthreads_or(wrong) && pass == kPlain) break;
    }
}

// Joins the splits of a row: a workgroup of DP threads per row of a tile.
template <typename T, int DP>
__global__ __launch_bounds__(DP) void join_kernel(Forward<T> a, int splits, Partials part) {
    const Shape &s = a.s;
    const int index = static_cast<int>(blockIdx.x) / 16, r = static_cast<int>(blockIdx.x) % 16;
    const RowTile<16> tile(s, a.lengths, index);
    int t, hd;
    if (!tile.row(s, r, t, hd)) return;
    const int64_t at = static_cast<int64_t>(index) * splits * 16 + r;
    float top = kNegInf;
#pragma unroll 8
    for (int i = 0; i < splits; ++i) top = fmaxf(top, part.ml[2 * (at + 16 * i)]);
    const float base = top == kNegInf ? 0.0f : top;
    float sum = 0.0f, v = 0.0f;
    const int col = static_cast<int>(threadIdx.x);
#pragma unroll 8
    for (int i = 0; i < splits; ++i) {
        const int64_t x = at + 16 * i;
        const float f = exp2_fast(part.ml[2 * x] - base);
        sum += f * part.ml[2 * x + 1];
        v += f * part.o[x * DP + col];
    }
    const float inverse = row_factor<T, true>(sum);
    if (col < s.dim) a.out.row(tile.b, tile.t0 + t, hd)[col] = static_cast<T>(v * inverse);
    if (col == 0 && a.lse) {
        a.lse[(static_cast<int64_t>(tile.b) * s.queries + tile.t0 + t) * s.q_heads + hd] =
            row_lse<T, true>(top, sum);
    }
}

// ---- backward -------------------------------------------------------------------------

// bits[b][h][block][token / 32]: the tokens that see something of the block through their ids.
// A workgroup has 128 tokens of a head (four words of each block), gathered in LDS for
// kMarkWindow blocks at a time: with a word per block and tokens of 32 each, atomics on the
// words in memory took 29 us, this 6, for 2 x 4096 tokens with 12 ids of 4 heads.
constexpr int kMarkWords = 4;
constexpr int kMarkWindow = 1024;

// counts[b][h][block], 0 before, become the numbers of tokens.
__global__ __launch_bounds__(kThreads) void mark_kernel(Shape s, const int *__restrict__ lengths,
                                                        const int *__restrict__ ids, int words,
                                                        unsigned *__restrict__ bits,
                                                        int *__restrict__ counts) {
    __shared__ __align__(16) unsigned s_bits[kMarkWindow][kMarkWords];
    const int heads = s.batch * s.kv_heads;
    const int bh = static_cast<int>(blockIdx.x) % heads;
    const int w0 = static_cast<int>(blockIdx.x) / heads * kMarkWords;
    const int b = bh / s.kv_heads, h = bh % s.kv_heads;
    const int length = length_of(s, lengths, b);
    const int t0 = 32 * w0;
    const int n = min(32 * kMarkWords, s.queries - t0) * s.count;
    for (int first = 0; first < s.blocks; first += kMarkWindow) {  // uniform
        for (int i = threadIdx.x; i < kMarkWindow * kMarkWords; i += kThreads) {
            (&s_bits[0][0])[i] = 0u;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const int t = i / s.count, x = i - t * s.count;
            const int place = length - s.queries + t0 + t;
            const int last = place < 0 ? -1 : s.causal ? place : length - 1;
            const int64_t row = (static_cast<int64_t>(b) * s.queries + t0 + t) * s.kv_heads + h;
            const int id = ids[row * s.count + x];
            if (last >= 0 && static_cast<unsigned>(id) <= static_cast<unsigned>(last / s.block) &&
                id >= first && id < first + kMarkWindow) {
                atomicOr(&s_bits[id - first][t / 32], 1u << (t % 32));
            }
        }
        __syncthreads();
        const int there = min(kMarkWindow, s.blocks - first);
        for (int i = threadIdx.x; i < there; i += kThreads) {
            const int64_t row = static_cast<int64_t>(bh) * s.blocks + first + i;
            const u32x4 mine = *reinterpret_cast<const u32x4 *>(s_bits[i]);
            *reinterpret_cast<u32x4 *>(bits + row * words + w0) = mine;
            const int n = __popc(mine[0]) + __popc(mine[1]) + __popc(mine[2]) + __popc(mine[3]);
            if (n > 0) atomicAdd(&counts[row], n);
        }
        __syncthreads();
    }
}

// start[row]: the items before the row's, each of at most per_item of its tokens, one at least;
// start[rows] is their number.  One workgroup: the rows are the blocks of the key heads.
constexpr int kStartBlock = 1024;

__global__ __launch_bounds__(kStartBlock) void start_kernel(int64_t rows, int per_item,
                                                            const int *__restrict__ counts,
                                                            int *__restrict__ start) {
    __shared__ int s_sums[kStartBlock / dev::kWave];
    int carry = 0;
    for (int64_t first = 0; first < rows; first += kStartBlock) {  // uniform
        const int64_t row = first + threadIdx.x;
        const int n = row < rows && counts ? counts[row] : 0;
        const int items = row < rows ? max(1, (n + per_item - 1) / per_item) : 0;
        int total = 0;
        const int at = carry + dev::block_exclusive_sum<kStartBlock>(items, s_sums, total);
        if (row < rows) start[row] = at;
        carry += total;
    }
    if (threadIdx.x == 0) start[rows] = carry;
}

// float16 has less range than gradients take that it can hold the sums of: the scores' gradients
// of a small step fall below 2^-24, those of a scaled loss rise above 65504.  So a column of them
// is multiplied by a power of two that keeps the largest so far below 2^15, and was at least 2^12
// when it was chosen; when it has to change, the column's sums follow.  Training steps of 2 x 4096
// queries of 16 heads of 128 take 566 us instead of 527 for it, of heads of 64 304 instead of 282.
template <typename T>
struct Range {
    static constexpr bool kNeeded = __is_same(T, _Float16);
    int shift = 100;

    template <int N, int M>
    __device__ __forceinline__ void bring(f32x4 (&ds)[N], f32x4 (&sums)[M]) {
        if constexpr (kNeeded) {
            float top = 0.0f;
#pragma unroll
            for (int t = 0; t < N; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(ds[t][i]));
            }
            top = column_max(top);
            const bool over = __builtin_amdgcn_ldexpf(top, shift) > 0x1p15f;
            if (__any(over)) {
                // (2^13 is over top 2^now; the exponent of an infinity is 0)
                const int now = over ? min(shift, 13 - __builtin_amdgcn_frexp_expf(top)) : shift;
                const float factor = __builtin_amdgcn_ldexpf(1.0f, now - shift);
#pragma unroll
                for (int i = 0; i < M; ++i) sums[i] *= factor;
                shift = now;
            }
            const float factor = __builtin_amdgcn_ldexpf(1.0f, shift);
#pragma unroll
            for (int t = 0; t < N; ++t) ds[t] *= factor;
        }
    }
    // What undoes it in the sums.
    __device__ __forceinline__ float inverse() const {
        return kNeeded ? __builtin_amdgcn_ldexpf(1.0f, -shift) : 1.0f;
    }
};

// The same for probabilities, which are at most 1: for dv they are 2^kMore times as large.
template <typename T>
constexpr int kMore = Range<T>::kNeeded ? 15 : 0;

// From the products s = q . k and dp = dout . v of 16 N keys with a row: s become probabilities
// and dp the scores' gradients (without the scale); with kMarks 1 for each key that the row sees.
template <int N>
__device__ __forceinline__ void score_gradient(f32x4 (&s)[N], f32x4 (&dp)[N], float scale2,
                                               float lse2, float delta, int limit, int pass) {
    const bool none = limit <= 0;
    const float base = none ? -kNegInf : lse2;  // (as in softmax_step)
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s[t][i] = exp2_fast(__builtin_fmaf(s[t][i], scale2, -base));
            dp[t][i] = s[t][i] * (dp[t][i] - delta);
        }
    }
    if (pass != kPlain || __any(!none && limit < 16 * N)) {
#pragma unroll
        for (int t = 0; t < N; ++t) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float seen = pass == kMarks ? 1.0f : dp[t][i];
                dp[t][i] = 16 * t + i < limit ? seen : 0.0f;
            }
        }
    }
}

// dq, and delta and zeroed counts for the launches that follow.  32 keys a step where two column
// tiles of q and dout fill the registers.
//
// ds is in two parts of the operands' type for its product (16-bit types): dq then is 0.0019 of its
// norm off with bfloat16 instead of 0.0026, where its own rounding makes 0.0017 and delta, which is
// of the rounded out, 0.0006.
// 2 x 4096 queries of 16 heads of 128, 12 of 64 blocks: 200 us (172 without the second product), 68
// GFLOP that are asked for and 1.6 times that with the union's.  Matrix products 36%, vector unit
// 37% of a CU's time.
template <typename T, int DP, int BN, int COLS>
__global__ __launch_bounds__(kThreads, 2) void dq_kernel(Backward<T> a, float *__restrict__ delta,
                                                         int64_t rows_of_blocks,
                                                         int *__restrict__ counts) {
    using Lds = Tile<T, DP, BN, kThreads>;
    constexpr int kRowsOf = 64 * COLS;
    __shared__ __align__(16) T s_k0[Lds::kElements];
    __shared__ __align__(16) T s_v0[Lds::kElements];
    __shared__ __align__(16) T s_k1[Lds::kElements];
    __shared__ __align__(16) T s_v1[Lds::kElements];
    __shared__ Lists<kRowsOf> s_lists;
    const Shape &s = a.s;
    const RowTile<kRowsOf> tile(s, a.lengths, static_cast<int>(blockIdx.x));
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < rows_of_blocks;
         i += static_cast<int64_t>(gridDim.x) * kThreads) {
        counts[i] = 0;  // for the launch that counts
    }
    const LaneRows<COLS> rows(s, tile, wave, c);
    Frag<T> q[COLS][DP / 32], dout[COLS][DP / 32];
    f32x4 o[COLS][DP / 16];
    float lse2[COLS], row_delta[COLS];
#pragma unroll
    for (int x = 0; x < COLS; ++x) {
        const bool exists = rows.exists[x];
        const int t = tile.t0 + rows.token[x], head = rows.head[x];
        load_row_frags<T, DP>(exists ? a.q.row(tile.b, t, head) : nullptr, s.dim, g, q[x]);
        load_row_frags<T, DP>(exists ? a.dout.row(tile.b, t, head) : nullptr, s.dim, g, dout[x]);
        if (s.scale < 0.0f) negate<T, DP>(q[x]);
        const int64_t at = (static_cast<int64_t>(tile.b) * s.queries + t) * s.q_heads + head;
        const float lse = exists ? a.lse[at] : 0.0f;
        lse2[x] = lse == kNegInf ? 0.0f : lse * kLog2e;
        Frag<T> out[DP / 32];
        load_row_frags<T, DP>(exists ? a.out.row(tile.b, t, head) : nullptr, s.dim, g, out);
        float sum = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DP / 32; ++kk) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum = __builtin_fmaf(static_cast<float>(dout[x][kk][j]),
                                     static_cast<float>(out[kk][j]), sum);
            }
        }
        row_delta[x] = column_sum(sum);
        if (exists && g == 0) delta[at] = row_delta[x];
    }
    const float scale2 = base2_scale(s.scale);
    KeySteps<T, DP, BN, kRowsOf> steps{{s_k0, s_k1}, {s_v0, s_v1}, s_lists};
    for (int pass = kPlain; pass <= kFinite; ++pass) {  // uniform
        Range<T> range[COLS];
#pragma unroll
        for (int x = 0; x < COLS; ++x) {
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) o[x][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        steps.run(a, tile, pass, nullptr, [&](T *s_k, const T *s_v, int nth, int first_key) {
            int limit[COLS];
            // (after kPlain's pass every wavefront goes on, to the barriers below)
            if (!rows.limits(s_lists, nth, first_key, g, limit) && pass == kPlain) return;
            f32x4 p[COLS][BN / 16], dp[COLS][BN / 16];
            row_products<Lds, T, DP, COLS, BN / 16>(s_k, q, g, c, p);
            row_products<Lds, T, DP, COLS, BN / 16>(s_v, dout, g, c, dp);
#pragma unroll
            for (int x = 0; x < COLS; ++x) {
                score_gradient<BN / 16>(p[x], dp[x], scale2, lse2[x], row_delta[x], limit[x], pass);
                range[x].bring(dp[x], o[x]);
            }
            if (pass != kPlain) {  // uniform; the scores are those of the keys as they are
                __syncthreads();
                Lds::make_finite(s_k, threadIdx.x, pass == kMarks);
                __syncthreads();
            }
            column_products<Lds, T, DP, COLS, BN / 16, kTwo>(s_k, dp, g, c, o);
        });
        float wrong = 0.0f;
#pragma unroll
        for (int x = 0; x < COLS; ++x) {
            wrong += not_finite<DP / 16>(o[x]);
            if (!rows.exists[x]) continue;
            T *dq = a.dq.row(tile.b, tile.t0 + rows.token[x], rows.head[x]);
            const float undo = range[x].inverse();
            const float factor = pass == kMarks ? 1.0f : s.scale * kPartsScale<T>;
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                const int col = 16 * i + 4 * g;
                if (col >= s.dim) continue;
                const f32x4 v = o[x][i] * undo * factor;
                if (pass == kPlain) {
                    store4<T>(dq + col, v);
                    continue;
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) store_again(dq + col + j, v[j], pass);
            }
        }
        if (pass == kPlain && !__syncthreads_or(wrong != wrong)) break;
    }
}

constexpr int kItemTokens = 2048;  // tokens of an item, at most (their numbers are in LDS)
constexpr int kStepRows = 32;      // (token, head) rows of a wavefront's step
constexpr int kMaxGroup = 1024;    // heads of a group: what the division below holds for

// Work on dk and dv: the rows (blocks of heads) in items of at most per_item tokens, so that a
// block that every query selects is not one workgroup's.  start[row] are the rows' first items.
struct Items {
    const int *start;
    int64_t rows;
    int per_item, words;
    const unsigned *bits;
    float *partial;  // [item][key of the block][2][DP]: dk and dv of an item of several
};

// dk and dv of 16 COLS LANES keys of a block.  Each of LANES wavefronts has 16 COLS of the keys;
// with LANES = 2 the four wavefronts are two such sets, which take 32 rows of the item's tokens
// in turn and add their sums at the end.
//
// p and ds are in two parts of the operands' type for their products (16-bit types), so that dk
// and dv are what rounding them once makes them, 0.0017 of their norms off with bfloat16 and 0.0002
// with float16 (0.0024 and 0.0003 with one rounded part); training steps of 2 x 4096 queries of 16
// heads of 128 take 541 us instead of 504 for it.
//
// 2 x 4096 queries of 16 heads of 128, 12 of 64 blocks: 240 us for 90 GFLOP (rows that did not
// select the block take no part; with one rounded part 203, and 1146 with one workgroup per block
// instead of items).  LDS is the bound, 40% of a CU's time and waits for it, before matrix products
// with 34%: a wavefront's 16 keys use each fragment once.  Two column tiles use it twice: for heads
// of 64 training steps are 35 us of 330 shorter with them; for 128 they do not fit the registers,
// and a step takes 920 us instead of 544.  32 keys to a workgroup instead of 64: training steps 562
// us instead of 544, heads of 64 306 instead of 295.
template <typename T, int DP, int COLS, int LANES>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 ? 1 : 2) void dkv_kernel(
    Backward<T> a, const float *__restrict__ delta, Items items, unsigned group_inverse) {
    constexpr int kSets = kWaves / LANES;
    constexpr int kStep = kSets * kStepRows;
    using Lds = Tile<T, DP, kStep, kThreads>;
    constexpr int kKeys = 16 * COLS * LANES;
    // two buffers of q and dout, and later the sums of the second set
    __shared__ __align__(16) T s_q0[Lds::kElements];
    __shared__ __align__(16) T s_do0[Lds::kElements];
    __shared__ __align__(16) T s_q1[Lds::kElements];
    __shared__ __align__(16) T s_do1[Lds::kElements];
    // of the rows of four steps: where they are, and what their products need
    __shared__ int64_t s_at_q[4][kStep], s_at_do[4][kStep];
    __shared__ __align__(16) float s_lse[4][kStep], s_delta[4][kStep];
    __shared__ __align__(16) int s_last[4][kStep];
    __shared__ bool s_partial[4];
    __shared__ int s_tokens[kItemTokens];
    __shared__ int s_sums[kWaves];
    const Shape &s = a.s;
    const int parts = s.block / kKeys;
    // Workgroups go to the 8 XCDs in turn: each XCD takes a stretch of items, so that the rows
    // of few heads are in its L2.
    const int64_t all = static_cast<int64_t>(items.start[items.rows]) * parts;
    const int64_t stretch = (all + 7) / 8;
    const int64_t index = blockIdx.x % 8 * stretch + blockIdx.x / 8;
    if (blockIdx.x / 8 >= stretch || index >= all) return;
    const int64_t item = index / parts;
    const int part = static_cast<int>(index % parts);
    const int64_t row = dev::last_le(items.start, 0, items.rows - 1, item);
    const int64_t nth = item - items.start[row];
    const bool whole = items.start[row + 1] - items.start[row] == 1;
    const int bh = static_cast<int>(row / s.blocks), id = static_cast<int>(row % s.blocks);
    const int b = bh / s.kv_heads, h = bh % s.kv_heads;
    const int wave = static_cast<int>(threadIdx.x) / dev::kWave;
    const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
    const int part_of = wave % LANES, set = wave / LANES;  // of the keys, of the rows
    const int length = length_of(s, a.lengths, b);
    const int in_block = part * kKeys + 16 * COLS * part_of + c;  // + 16 x
    const int first_key = id * s.block + in_block;
    Frag<T> k[COLS][DP / 32], v[COLS][DP / 32];
    f32x4 dk[COLS][DP / 16], dv[COLS][DP / 16];
#pragma unroll
    for (int x = 0; x < COLS; ++x) {
        const int key = first_key + 16 * x;
        const bool exists = key < length;
        load_row_frags<T, DP>(exists ? a.k.row(b, key, h) : nullptr, s.dim, g, k[x]);
        load_row_frags<T, DP>(exists ? a.v.row(b, key, h) : nullptr, s.dim, g, v[x]);
        if (s.scale < 0.0f) negate<T, DP>(k[x]);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) dk[x][i] = dv[x][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const float scale2 = base2_scale(s.scale);
    const int place0 = length - s.queries;
    Range<T> range[COLS];

    // The item's tokens, ascending: those of the row's set bits from the nth * per_item-th on.
    const unsigned *row_bits = items.bits + row * items.words;
    const int64_t from = nth * items.per_item;
    int64_t seen = 0;
    for (int w0 = 0; w0 < items.words; w0 += kThreads) {  // uniform
        const int w = w0 + static_cast<int>(threadIdx.x);
        unsigned mine = w < items.words ? row_bits[w] : 0u;
        int total = 0;
        const int before = dev::block_exclusive_sum<kThreads>(static_cast<int>(__popc(mine)),
                                                              s_sums, total);
        int64_t at = seen + before - from;
        for (; mine; mine &= mine - 1u, ++at) {
            if (at >= 0 && at < items.per_item) {
                s_tokens[at] = 32 * w + __ffs(static_cast<int>(mine)) - 1;
            }
        }
        seen += total;
        if (seen >= from + items.per_item) break;
    }
    __syncthreads();
    const int64_t left = seen - from;
    const int rows = static_cast<int>(left < items.per_item ? (left < 0 ? 0 : left)
                                                            : items.per_item) * s.group;
    // x / group (exact: x < 2^11 group, and group^2 2^11 < 2^32)
    auto token_at = [&](int x) {
        return s.group == 1 ? x
                            : static_cast<int>(__umulhi(static_cast<unsigned>(x), group_inverse));
    };
    const T *q_base = a.q.row(b, 0, h * s.group), *do_base = a.dout.row(b, 0, h * s.group);
    auto load = [&](int step, T *to_q, T *to_do) {
        const int ring = step & 3;
        Lds::load(to_q, threadIdx.x, s.dim, [&](int r) { return q_base + s_at_q[ring][r]; });
        Lds::load(to_do, threadIdx.x, s.dim, [&](int r) { return do_base + s_at_do[ring][r]; });
    };
    // The first kStep threads (part of the first wavefront) work out the rows of a step: `begin`
    // two steps ahead, and `end` once lse and delta are there.  Steps past the last row repeat
    // it as one that sees no key.
    const int block_end = (id + 1) * s.block - 1;
    const bool informs = threadIdx.x < kStep;
    float next_lse = 0.0f, next_delta = 0.0f;
    int next_last = 0;
    auto begin = [&](int step) {
        const int x = min(step * kStep + static_cast<int>(threadIdx.x), rows - 1);
        const int at = token_at(x), t = s_tokens[at], head = x - at * s.group;
        s_at_q[step & 3][threadIdx.x] = t * a.q.row_stride + head * a.q.head_stride;
        s_at_do[step & 3][threadIdx.x] = t * a.dout.row_stride + head * a.dout.head_stride;
        const int64_t i =
            (static_cast<int64_t>(b) * s.queries + t) * s.q_heads + h * s.group + head;
        next_lse = a.lse[i];
        next_delta = delta[i];
        next_last = s.causal ? place0 + t : length - 1;
    };
    auto end = [&](int step) {
        const bool there = step * kStep + static_cast<int>(threadIdx.x) < rows;
        const int last = there ? next_last : -1;
        s_lse[step & 3][threadIdx.x] =
            (next_lse == kNegInf ? 0.0f : next_lse * kLog2e) - kMore<T>;
        s_delta[step & 3][threadIdx.x] = next_delta;
        s_last[step & 3][threadIdx.x] = last;
        // whether some row sees a part of the block only
        const bool partial = __any(last < block_end);
        if (threadIdx.x == 0) s_partial[step & 3] = partial;
    };
    auto use = [&](const T *s_q, const T *s_do, int step) {
        const int buffer = step & 3;
        const T *my_q = s_q + set * kStepRows * Lds::kRow,
                *my_do = s_do + set * kStepRows * Lds::kRow;
        constexpr int kN = kStepRows / 16;
        f32x4 p[COLS][kN], dp[COLS][kN];
        row_products<Lds, T, DP, COLS, kN>(my_q, k, g, c, p);
        row_products<Lds, T, DP, COLS, kN>(my_do, v, g, c, dp);
#pragma unroll
        for (int t = 0; t < kN; ++t) {
            // this lane's rows 16 t + 4 g + i, its keys in each
            const int r = set * kStepRows + 16 * t + 4 * g;
            const f32x4 lse = *reinterpret_cast<const f32x4 *>(&s_lse[buffer][r]);
            const f32x4 d = *reinterpret_cast<const f32x4 *>(&s_delta[buffer][r]);
#pragma unroll
            for (int x = 0; x < COLS; ++x) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[x][t][i] = exp2_fast(__builtin_fmaf(p[x][t][i], scale2, -lse[i]));
                    dp[x][t][i] = p[x][t][i] * (dp[x][t][i] - d[i]);
                }
            }
        }
        if (s_partial[buffer]) {
#pragma unroll
            for (int t = 0; t < kN; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int last = s_last[buffer][set * kStepRows + 16 * t + 4 * g + i];
#pragma unroll
                    for (int x = 0; x < COLS; ++x) {
                        const bool sees = first_key + 16 * x <= last;
                        p[x][t][i] = sees ? p[x][t][i] : 0.0f;
                        dp[x][t][i] = sees ? dp[x][t][i] : 0.0f;
                    }
                }
            }
        }
#pragma unroll
        for (int x = 0; x < COLS; ++x) range[x].bring(dp[x], dk[x]);
        column_products<Lds, T, DP, COLS, kN, kTwo>(my_do, p, g, c, dv);
        column_products<Lds, T, DP, COLS, kN, kTwoOrInfinite>(my_q, dp, g, c, dk);
    };
    if (rows > 0) {  // uniform
        if (informs) {
            begin(0);
            end(0);
            begin(1);
            end(1);
        }
        __syncthreads();
        load(0, s_q0, s_do0);
        rows_arrived();
        // (A last step without rows takes probabilities of 0: a branch around it costs a second
        // copy of the sums' registers.)
        const int steps = (rows + kStep - 1) / kStep;
        for (int step = 0; step < steps; step += 2) {
            load(step + 1, s_q1, s_do1);
            if (informs) begin(step + 2);
            use(s_q0, s_do0, step);
            if (informs) end(step + 2);
            rows_arrived();
            load(step + 2, s_q0, s_do0);
            if (informs) begin(step + 3);
            use(s_q1, s_do1, step + 1);
            if (informs) end(step + 3);
            rows_arrived();
        }
    }
    if constexpr (Range<T>::kNeeded) {
        constexpr float kLess = 1.0f / (1 << kMore<T>);
#pragma unroll
        for (int x = 0; x < COLS; ++x) {
            const float undo = range[x].inverse();
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                dk[x][i] = dk[x][i] * undo * kLess;
                dv[x][i] *= kLess;
            }
        }
    }
    if constexpr (kSets == 2) {
        // The second set's sums are added to the first's, dk's through the buffers of q and dv's
        // through those of dout.
        static_assert(16 * COLS * DP * 4 <= Lds::kElements * static_cast<int>(sizeof(T)),
                      "a wavefront's sums fit a buffer");
        float *sum_k = reinterpret_cast<float *>(part_of ? s_q1 : s_q0);
        float *sum_v = reinterpret_cast<float *>(part_of ? s_do1 : s_do0);
        auto each = [&](auto f) {
#pragma unroll
            for (int x = 0; x < COLS; ++x) {
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    const int at = ((x * (DP / 16) + i) * dev::kWave + lane) * 4;
                    f(*reinterpret_cast<f32x4 *>(sum_k + at), dk[x][i]);
                    f(*reinterpret_cast<f32x4 *>(sum_v + at), dv[x][i]);
                }
            }
        };
        if (set == 1) each([](f32x4 &there, const f32x4 &mine) { there = mine; });
        __syncthreads();
        if (set == 1) return;
        each([](const f32x4 &there, f32x4 &mine) { mine += there; });
    }
#pragma unroll
    for (int x = 0; x < COLS; ++x) {
        const int key = first_key + 16 * x;
        float *part_out = items.partial + (item * s.block + in_block + 16 * x) * (2 * DP);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const f32x4 sk = dk[x][i], sv = dv[x][i];
            const int col = 16 * i + 4 * g;
            if (!whole) {
                *reinterpret_cast<f32x4 *>(part_out + col) = sk;
                *reinterpret_cast<f32x4 *>(part_out + DP + col) = sv;
            } else if (key < s.keys && col < s.dim) {  // (past the length: zeros)
                store4<T>(a.dk.row(b, key, h) + col, sk * (s.scale * kPartsScale<T>));
                store4<T>(a.dv.row(b, key, h) + col, sv * kPartsScale<T>);
            }
        }
    }
}

// Adds up the items of a row that has several, in their order: a workgroup per 16 keys.  16 us
// after the items above, bound by reading them.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void dkv_join_kernel(Backward<T> a, Items items) {
    const Shape &s = a.s;
    const int parts = s.block / 16;
    const int64_t row = blockIdx.x / parts;
    const int part = static_cast<int>(blockIdx.x % parts);
    const int from = items.start[row], to = items.start[row + 1];
    if (to - from <= 1) return;
    const int bh = static_cast<int>(row / s.blocks), id = static_cast<int>(row % s.blocks);
    const int b = bh / s.kv_heads, h = bh % s.kv_heads;
    constexpr int kPieces = 2 * DP / 4;  // of a key: four columns of dk or dv
    for (int x = threadIdx.x; x < 16 * kPieces; x += kThreads) {
        const int in_block = 16 * part + x / kPieces, piece = x % kPieces;
        const int key = id * s.block + in_block;
        const bool is_v = piece >= kPieces / 2;
        const int col = 4 * (is_v ? piece - kPieces / 2 : piece);
        if (key >= s.keys || col >= s.dim) continue;
        f32x4 sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int64_t i = from; i < to; ++i) {
            sum += *reinterpret_cast<const f32x4 *>(
                items.partial + (i * s.block + in_block) * (2 * DP) + 4 * piece);
        }
        if (is_v) {
            store4<T>(a.dv.row(b, key, h) + col, sum * kPartsScale<T>);
        } else {
            store4<T>(a.dk.row(b, key, h) + col, sum * (s.scale * kPartsScale<T>));
        }
    }
}

// ---- host -----------------------------------------------------------------------------

bool aligned(const nacho_heads &h, int item, bool optional = false) {
    if (!h.data) return optional;
    const int64_t per = 16 / item;
    return reinterpret_cast<uintptr_t>(h.data) % 16 == 0 && h.batch_stride % per == 0 &&
           h.row_stride % per == 0 && h.head_stride % per == 0 && h.row_stride >= 0 &&
           h.row_stride <= NACHO_MAX_ROW_BYTES / item;
}

int check(const nacho_block_attention_args *p, bool backward, Shape *s) {
    if (!p || p->dtype < NACHO_F32 || p->dtype > NACHO_BF16) return NACHO_ERR_INVALID_ARGUMENT;
    if (p->batch < 0 || p->queries < 0 || p->keys < 0 || p->q_heads < 1 || p->kv_heads < 1 ||
        p->q_heads % p->kv_heads != 0 || p->q_heads / p->kv_heads > kMaxGroup ||
        p->head_dim < 8 || p->head_dim > 128 || p->head_dim % 8 != 0 ||
        (p->block != 32 && p->block != 64 && p->block != 128) ||
        p->count < 0 || (p->causal != 0 && p->causal != 1) || !std::isfinite(p->scale * kLog2e)) {
        return NACHO_ERR_INVALID_ARGUMENT;
    }
    const int64_t rows = static_cast<int64_t>(p->batch) * p->queries * p->q_heads;
    const int64_t blocks = (static_cast<int64_t>(p->keys) + p->block - 1) / p->block;
    const int64_t parts = blocks * (p->block / 32) * p->batch * p->kv_heads;
    if (rows > INT32_MAX / 16 || parts > INT32_MAX || p->keys > INT32_MAX - (1 << 17) ||
        p->count > kMostIds) {
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
    if (static_cast<int64_t>(tiling(*s, 64).per_head) * p->batch * p->kv_heads > kMostGroups) {
        return NACHO_ERR_INDEX_OVERFLOW;
    }
    return NACHO_OK;
}

template <typename T>
Backward<T> args_of(const nacho_block_attention_args &p, const Shape &s) {
    Backward<T> a;
    static_cast<Forward<T> &>(a) = Forward<T>{s,
                                              heads<T>(p.q),
                                              heads<T>(p.k),
                                              heads<T>(p.v),
                                              heads<T>(p.out),
                                              p.lengths,
                                              p.blocks,
                                              p.lse};
    a.dout = heads<T>(p.dout);
    a.dq = heads<T>(p.dq);
    a.dk = heads<T>(p.dk);
    a.dv = heads<T>(p.dv);
    return a;
}

constexpr int kFullGrid = 256;  // workgroups that occupy the device: one per CU

// Two column tiles per wavefront share what each reads of LDS, but are half as many workgroups
// with twice the work.  us with two and with one, by tiles of 128 rows; attention of heads of 128:
// 192: 114 72, 320: 112 112, 512: 116 123 and 107 103, 768: 171 163, 1024: 183 202, 2048: 308 361
// and 276 320; its training steps: 512: 284 264, 896: 480 472, 1024: 543 540, 2048: 1031 1075; of
// heads of 96: 512: 242 231, 1024: 473 477.  Heads of 64, whose registers leave room for more
// wavefronts with one: 512: 81 57, 1024: 127 97, 2048: 158 145; training 1024: 344 295.
constexpr int64_t kTwoColumns = 4 * kFullGrid;
template <typename T, int DP>
constexpr bool kMayShare = sizeof(T) == 2 && DP > 64;

// Tiles of 16 rows up to which their kernel is faster than that of tiles of 64; us of the one
// and the other by their number: bfloat16 heads of 128 256: 41 62, 512: 49 63, 544: 64 53, 640:
// 79 64; float16 of 64 512: 27 37, 640: 33 38; float32 of 128 256: 81 211, 512: 152 219, 768:
// 219 215, 1024: 288 226; of 64 768: 106 137. Where there are as many tiles of 64 as CUs
// (single tokens of many sequences make as many of either) these are at least as fast: 64 x 4
// tokens 93 with them, 100 with 16.
template <typename T>
constexpr int64_t kFewTiles = (sizeof(T) == 2 ? 2 : 3) * kFullGrid;

// A sequence's rows up to which a probability reaches its product in two parts of the operands'
// type: one tile then has all of a key head's rows, and its keys' bytes take longer than their
// products.
// 64 single tokens of 32 heads of 128: 51.1 us either way, 256 of them 198 and 197 (with two column
// tiles); 8192 queries: 307 us with one part, 416 with two.
constexpr int64_t kPartsRows = 64;

// Calls f with the keys of a step, 64, or 32 where the block or float32's tiles (twice as large)
// want it (attention of 8192 queries of 32 heads of 128: 308 us with 64, 398 with 32), and the
// column tiles of a wavefront (`one_column`: one, however many tiles there are).
template <typename T, int DP, typename F>
int with_tiles(const Shape &s, bool one_column, F f) {
    const int heads = s.batch * s.kv_heads;
    const int64_t large = static_cast<int64_t>(tiling(s, 128).per_head) * heads;
    auto columns = [&](auto keys) {
        if constexpr (kMayShare<T, DP>) {
            if (!one_column && large >= kTwoColumns) {
                return f(keys, std::integral_constant<int, 2>{}, static_cast<unsigned>(large));
            }
        }
        f(keys, std::integral_constant<int, 1>{},
          static_cast<unsigned>(tiling(s, 64).per_head * heads));
    };
    if constexpr (sizeof(T) == 2) {
        if (s.block % 64 == 0) {
            columns(std::integral_constant<int, 64>{});
        } else {
            columns(std::integral_constant<int, 32>{});
        }
    } else {
        columns(std::integral_constant<int, 32>{});
    }
    NACHO_TRY_HIP(hipGetLastError());
    return NACHO_OK;
}

// Training steps of 16 heads of 128, 4 key heads, in us by the target (384, 512, 768, 1024, 1536):
// 2 x 4096 queries 610 571 544 558 551; 2 x 2048 (512, 768, 1024) 278 264 253; by the least (128,
// 192, 256, 384): 2 x 1024 141 128 139 144, 1 x 1024 of half the heads 103 111 120 138.
constexpr int64_t kItemTarget = 768;
constexpr int64_t kItemLeast = 192;  // tokens

template <typename T, int DP>
int forward(Call &call, const Forward<T> &a) {
    const Shape &s = a.s;
    const hipStream_t stream = call.stream();
    const int heads = s.batch * s.kv_heads;
    const Tiling small = tiling(s, 16);
    const int64_t few = static_cast<int64_t>(small.per_head) * heads;
    const int64_t tiles = static_cast<int64_t>(tiling(s, 64).per_head) * heads;
    if (few > kFewTiles<T> || tiles >= kFullGrid) {
        const bool parts =
            sizeof(T) == 2 && static_cast<int64_t>(s.queries) * s.group <= kPartsRows;
        return with_tiles<T, DP>(s, parts, [&](auto keys, auto columns, unsigned grid) {
            if constexpr (sizeof(T) == 2 && columns() == 1) {
                if (parts) {
                    tile_kernel<T, DP, keys(), 1, true><<<grid, kThreads, 0, stream>>>(a);
                    return;
                }
            }
            tile_kernel<T, DP, keys(), columns(), false><<<grid, kThreads, 0, stream>>>(a);
        });
    }
    // Few rows: tiles of 16 of them, whose wavefronts share the steps.  What a step waits
    // for is its operands (2 to 3 us from memory that nothing read lately), so there are as many
    // workgroups as find a CU, down to less than a step for each wavefront; past 16 splits the
    // join costs more than they save, and up to 8 steps one split is done before it would begin.
    // One query of 32 heads of 128, in us by splits (1, 2, 4, 8, 16, 32): over 4 blocks of 64
    // 8.6 10.3 11.1 10.1 10.9 12.6, over 16 blocks 18 15 13 10.8 11.8 13, over 64 blocks
    // 64 40 27 18.4 16.1 16.8; 16 sequences over 16 blocks 23.2 20.8 21.4 24.7 38 66.
    const int64_t listed =
        static_cast<int64_t>(small.tokens < s.queries ? small.tokens : s.queries) * s.count;
    const int64_t steps = (listed < s.blocks ? listed : s.blocks) * (s.block / kSplitKeys);
    int64_t splits = kFullGrid / few;
    const int64_t most = steps <= 2 * kWaves ? 1 : (steps + 2) / 3;
    if (splits > most) splits = most;
    if (splits > 16) splits = 16;
    if (splits < 1) splits = 1;
    Partials part{};
    if (splits > 1) {
        const size_t rows = static_cast<size_t>(few) * static_cast<size_t>(splits) * 16;
        NACHO_TRY(call.scratch_n(rows * (DP + 2), &part.o));
        part.ml = part.o + rows * DP;
    }
    const unsigned grid = static_cast<unsigned>(few * splits);
    const int n = static_cast<int>(splits);
    if ((small.tokens == 1 || s.queries == 1) && s.count <= dev::kWave) {
        split_kernel<T, DP, true><<<grid, kThreads, 0, stream>>>(a, n, part);
    } else {
        split_kernel<T, DP, false><<<grid, kThreads, 0, stream>>>(a, n, part);
    }
    NACHO_TRY_HIP(hipGetLastError());
    if (splits > 1) {
        join_kernel<T, DP><<<static_cast<unsigned>(few * 16), DP, 0, stream>>>(a, n, part);
        NACHO_TRY_HIP(hipGetLastError());
    }
    return NACHO_OK;
}

template <typename T, int DP>
int backward(Call &call, const Backward<T> &a) {
    const Shape &s = a.s;
    const hipStream_t stream = call.stream();
    const int heads = s.batch * s.kv_heads;
    const int64_t queries = static_cast<int64_t>(s.batch) * s.queries * s.q_heads;
    Items items{};
    items.rows = static_cast<int64_t>(heads) * s.blocks;
    const int groups = (s.queries + 32 * kMarkWords - 1) / (32 * kMarkWords);
    items.words = groups * kMarkWords;
    const int64_t listed = queries / s.group * s.count;
    // About kItemTarget items of equal size, but none so short that its sums cost more to store
    // than to compute.
    const int64_t per_item = (listed + kItemTarget - 1) / kItemTarget;
    items.per_item = static_cast<int>(
        per_item < kItemLeast ? kItemLeast : per_item > kItemTokens ? kItemTokens : per_item);
    const int64_t most = items.rows + listed / items.per_item;
    const bool wide = sizeof(T) == 2 && s.block % 64 == 0;  // 64 keys to a workgroup
    const int parts = s.block / (wide ? 64 : 32);
    if (most * parts > kMostGroups - 8 || items.rows * (s.block / 16) > kMostGroups ||
        static_cast<int64_t>(groups) * heads > kMostGroups) {
        return NACHO_ERR_INDEX_OVERFLOW;
    }
    const bool several = listed > items.per_item;  // else no row has several items
    // One piece of scratch: an allocation costs about as much as a small kernel.
    const size_t sizes[] = {static_cast<size_t>(queries) * 4,
                            static_cast<size_t>(items.rows) * items.words * 4,
                            static_cast<size_t>(items.rows) * 4,
                            static_cast<size_t>(items.rows + 1) * 4,
                            several ? static_cast<size_t>(most) * s.block * 2 * DP * 4 : 0};
    size_t at[6] = {0};
    for (int i = 0; i < 5; ++i) at[i + 1] = at[i] + (sizes[i] + 255) / 256 * 256;
    unsigned char *scratch = nullptr;
    NACHO_TRY(call.scratch_n(at[5], &scratch));
    float *delta = reinterpret_cast<float *>(scratch + at[0]);
    unsigned *bits = reinterpret_cast<unsigned *>(scratch + at[1]);
    int *counts = reinterpret_cast<int *>(scratch + at[2]);
    int *start = reinterpret_cast<int *>(scratch + at[3]);
    items.partial = reinterpret_cast<float *>(scratch + at[4]);
    items.bits = bits;
    items.start = start;
    if (queries > 0) {
        auto launch = [&](auto keys, auto columns, unsigned grid) {
            // (two column tiles leave registers for 32 keys of q . k and dout . v)
            constexpr int kKeys = columns() == 2 ? 32 : keys();
            dq_kernel<T, DP, kKeys, columns()><<<grid, kThreads, 0, stream>>>(
                a, delta, items.rows, counts);
        };
        const int launched = with_tiles<T, DP>(s, false, launch);
        NACHO_TRY(launched);
    }
    if (items.rows == 0) return NACHO_OK;
    if (queries > 0) {
        mark_kernel<<<static_cast<unsigned>(groups * heads), kThreads, 0, stream>>>(
            s, a.lengths, a.ids, items.words, bits, counts);
        NACHO_TRY_HIP(hipGetLastError());
    }
    start_kernel<<<1, kStartBlock, 0, stream>>>(items.rows, items.per_item,
                                                queries > 0 ? counts : nullptr, start);
    NACHO_TRY_HIP(hipGetLastError());
    const unsigned grid = static_cast<unsigned>((most * parts + 7) / 8 * 8);
    const unsigned group = static_cast<unsigned>(s.group);
    const unsigned inverse = group == 1 ? 0u : static_cast<unsigned>((1ull << 32) / group) + 1u;
    if (!wide) {
        dkv_kernel<T, DP, 1, 2><<<grid, kThreads, 0, stream>>>(a, delta, items, inverse);
    } else if constexpr (sizeof(T) == 2) {
        // (two column tiles of 128 do not fit the registers)
        dkv_kernel<T, DP, DP == 64 ? 2 : 1, DP == 64 ? 2 : 4>
            <<<grid, kThreads, 0, stream>>>(a, delta, items, inverse);
    }
    NACHO_TRY_HIP(hipGetLastError());
    if (several) {
        dkv_join_kernel<T, DP><<<static_cast<unsigned>(items.rows * (s.block / 16)), kThreads, 0,
                                 stream>>>(a, items);
        NACHO_TRY_HIP(hipGetLastError());
    }
    return NACHO_OK;
}

template <typename T>
int run(const nacho_block_attention_args &p, const Shape &s, Call &call, bool back) {
    const Backward<T> a = args_of<T>(p, s);
    if (s.dim <= 64) return back ? backward<T, 64>(call, a) : forward<T, 64>(call, a);
    if (s.dim <= 96) return back ? backward<T, 96>(call, a) : forward<T, 96>(call, a);
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
