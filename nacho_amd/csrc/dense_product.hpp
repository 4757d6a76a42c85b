// Matrix products of dense operands in memory: tiles of C = A B on the matrix cores, A's rows (m)
// against B's columns (n), sums in float32.
//
// An operand lies in memory either with its k next to each other ("along": rows of k, one for each
// m or n) or with its m or n next to each other ("across": a row for each k).  A workgroup takes a
// tile of BM x BN and goes over k in steps of 128 bytes of k (64 16-bit elements, 32 float32).  The
// next step's tiles are on their way from memory to LDS, without registers, while the wavefronts
// multiply this one's: two buffers, one barrier a step.  Products take eight consecutive k per
// lane (lane = 16 g + c: row or column c, k = 8 g + j); operands that lie across are read with the
// transposing LDS read.
//
// Measured, bfloat16, 8028 x 131072 by 2048, matrix cores' share of the time in brackets: both operands
// along k 1.26 PFLOP/s (60%), across k 1.06 for a mix of the two (46%, 47% of it waits).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>
#include <utility>

#include "dense_tiles.hpp"
#include "device_utils.hpp"

namespace nacho {
namespace dense {

// f(0), f(1) .. f(N - 1), each number a type: arrays that f indexes by it stay in registers.
template <int... I, typename F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F f) {
    each_of(std::make_integer_sequence<int, N>{}, f);
}

// Elements of k in a step.
template <typename T>
constexpr int kStepK = 128 / static_cast<int>(sizeof(T));

// Offsets past any buffer's end, where a load gives zeros.  Buffers are described as kBufferEnd
// bytes long whatever they are: what lies in them is decided by the loads' offsets alone.
constexpr unsigned kBufferEnd = 0x80000000u, kNowhere = 0xffffff00u;

template <typename T>
__device__ __forceinline__ void load_pieces(const T *base, T *lds, unsigned offset) {
#if defined(__HIP_DEVICE_COMPILE__)  // (the host pass does not know buffer descriptors)
    using Shared = __attribute__((address_space(3))) void *;
    const auto buffer =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base), 0, kBufferEnd, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (Shared)lds, 16, static_cast<int>(offset), 0,
                                             0, 0);
#endif
}

// ROWS rows of a step's k.  In LDS a row is 128 bytes, eight pieces of 16, piece p of row r at
// place p ^ swizzle(r): the 16 rows that a fragment reads lie in different banks.
template <typename T, int ROWS, int THREADS>
struct Along {
    static constexpr int kPer = 16 / static_cast<int>(sizeof(T));
    static constexpr int kPieces = 8;
    static constexpr int kElements = ROWS * kStepK<T>;
    static constexpr int kAll = ROWS * kPieces;
    static constexpr int kLoads = (kAll + THREADS - 1) / THREADS;
    static_assert(kAll % dev::kWave == 0 && THREADS % 128 == 0, "whole wavefronts");

    unsigned offset[kLoads];
    unsigned piece;  // of every load of this thread: swizzle repeats after 16 rows

    // A 16-byte read takes 16 lanes at a time: rows 0-3 and 12-15 of one g and 4-11 of the next, and
    // the other way round.  Of the eight rows in each half of the banks those two groups have
    // numbers whose second and third bits differ, so that what g adds to a piece, its last bits,
    // keeps them apart.  (With any numbers that differ between all rows half of the LDS's cycles
    // were conflicts.)
    __device__ __forceinline__ static int swizzle(int row) {
        const int k = row >> 1;
        return ((k >> 1 ^ k >> 2) & 1) << 2 | (k >> 2 & 1) << 1 | (k & 1);
    }

    // Rows from `there` on are zeros.  stride: elements from row to row.
    __device__ __forceinline__ void start(int thread, int64_t stride, int there) {
        piece = static_cast<unsigned>(thread % kPieces ^ swizzle(thread / kPieces));
        const unsigned bytes = static_cast<unsigned>(stride * static_cast<int>(sizeof(T)));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = thread / kPieces + i * (THREADS / kPieces);
            offset[i] = r < there ? static_cast<unsigned>(r) * bytes + 16u * piece : kNowhere;
        }
    }
    __device__ __forceinline__ static int64_t advance(int64_t) { return kStepK<T>; }

    // k from `left` on are zeros (left: a multiple of a piece's elements).
    __device__ __forceinline__ void load(int thread, const T *base, int64_t left, T *tile) const {
        const int wave_first = __builtin_amdgcn_readfirstlane(thread & ~(dev::kWave - 1));
        const bool cut = left < kStepK<T> && static_cast<int>(piece) * kPer >= left;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            if (kAll % THREADS != 0 && wave_first + i * THREADS >= kAll) break;
            load_pieces(base, tile + (i * THREADS + wave_first) * kPer,
                        cut ? kNowhere : offset[i]);
        }
    }

    // k 32 kk + 8 g .. + 8 of row 16 t + c.
    __device__ __forceinline__ static Frag<T> frag(const T *tile, int t, int kk, int g, int c) {
        const T *p = tile + (16 * t + c) * kStepK<T>;
        const int x = swizzle(c);
        if constexpr (sizeof(T) == 4) {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(p + ((2 * g) ^ x) * kPer);
            const f32x4 b = *reinterpret_cast<const f32x4 *>(p + ((2 * g + 1) ^ x) * kPer);
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *reinterpret_cast<const Frag<T> *>(p + ((4 * kk + g) ^ x) * kPer);
        }
    }
};

// A step's k, COLS elements of each.
template <typename T, int COLS, int THREADS>
struct Across {
    static constexpr int kPer = 16 / static_cast<int>(sizeof(T));
    static constexpr int kPieces = COLS / kPer;
    static constexpr int kElements = COLS * kStepK<T>;
    static constexpr int kLoads = kStepK<T> * kPieces / THREADS;
    static_assert(kStepK<T> * kPieces % THREADS == 0 && kPieces * 128 / kStepK<T> >= 16,
                  "whole pieces per thread, and banks for what is read at a time");

    unsigned offset[kLoads];

    // What a fragment reads at a time lies in different banks: two neighbouring pieces of eight
    // rows (16-bit types), four of four rows.
    __device__ __forceinline__ static int swizzle(int row) {
        if constexpr (sizeof(T) == 4) {
            return (row >> 3 & 3) << 2;
        } else if constexpr (kPieces == 8) {  // (two rows in all banks)
            return ((row >> 1 & 1) | (row >> 3 & 1) << 1) << 1;
        } else {
            return ((row & 3) | (row >> 3 & 1) << 2) << 1;
        }
    }

    // Columns from `there` on, which is a multiple of a piece's elements, are zeros.
    __device__ __forceinline__ void start(int thread, int64_t stride, int there) {
        const unsigned bytes = static_cast<unsigned>(stride * static_cast<int>(sizeof(T)));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = thread + i * THREADS;
            const int r = at / kPieces, piece = (at % kPieces) ^ swizzle(r);
            offset[i] = piece * kPer < there
                            ? static_cast<unsigned>(r) * bytes + 16u * static_cast<unsigned>(piece)
                            : kNowhere;
        }
    }
    __device__ __forceinline__ static int64_t advance(int64_t stride) {
        return stride * kStepK<T>;
    }

    __device__ __forceinline__ void load(int thread, const T *base, int64_t left, T *tile) const {
        const int wave_first = __builtin_amdgcn_readfirstlane(thread & ~(dev::kWave - 1));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = (thread + i * THREADS) / kPieces;
            load_pieces(base, tile + (i * THREADS + wave_first) * kPer,
                        r < left ? offset[i] : kNowhere);
        }
    }

    // k 32 kk + 8 g .. + 8 of column 16 t + c.  16-bit types: the 16 lanes of a group name four
    // rows of 16 elements, four lanes a row, and lane c receives column c of the four rows.
    __device__ __forceinline__ static Frag<T> frag(const T *tile, int t, int kk, int g, int c) {
        if constexpr (sizeof(T) == 4) {
            Frag<T> f;
            const int piece = (4 * t + (c >> 2)) ^ swizzle(8 * g);
            const T *p = tile + 8 * g * COLS + piece * kPer + (c & 3);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = p[j * COLS];
            return f;
        } else {
            using Shared = __attribute__((address_space(3))) s16x4 *;
            const int r = 32 * kk + 8 * g + (c >> 2);
            const int at = r * COLS + ((2 * t + ((c >> 1) & 1)) ^ swizzle(r)) * kPer + 4 * (c & 1);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (Shared)(reinterpret_cast<const s16x4 *>(tile + at)));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (Shared)(reinterpret_cast<const s16x4 *>(tile + at + 4 * COLS)));
            const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(Frag<T>, both);
        }
    }
};

// The same with a product's rows in another order: the results of tiles 2 p and 2 p + 1 in a lane are
// eight consecutive rows, 32 p + 8 g .. + 8, for wider stores.  Reads take the LDS twice as long.
template <typename T, int COLS, int THREADS>
struct AcrossPairs : Across<T, COLS, THREADS> {
    using Base = Across<T, COLS, THREADS>;

    __device__ __forceinline__ static Frag<T> frag(const T *tile, int t, int kk, int g, int c) {
        if constexpr (sizeof(T) == 4) {
            Frag<T> f;
            const int piece = (8 * (t >> 1) + 2 * (c >> 2) + (t & 1)) ^ Base::swizzle(8 * g);
            const T *p = tile + 8 * g * COLS + piece * Base::kPer + (c & 3);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = p[j * COLS];
            return f;
        } else {
            using Shared = __attribute__((address_space(3))) s16x4 *;
            const int r = 32 * kk + 8 * g + (c >> 2);
            const int at = r * COLS + ((4 * (t >> 1) + (c & 3)) ^ Base::swizzle(r)) * Base::kPer +
                           4 * (t & 1);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (Shared)(reinterpret_cast<const s16x4 *>(tile + at)));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (Shared)(reinterpret_cast<const s16x4 *>(tile + at + 4 * COLS)));
            const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(Frag<T>, both);
        }
    }
};

// A tile's shape: BM x BN by WM x WN wavefronts.
template <int BM_, int BN_, int WM_, int WN_>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
    static constexpr int kThreads = WM * WN * dev::kWave;
    static constexpr int MT = BM / WM / 16, NT = BN / WN / 16;  // 16 x 16 tiles of a wavefront
};

// An operand of a tile: its first element (m or n, and k, of the tile) and the elements from a row
// to the next.
template <typename T>
struct Matrix {
    const T *data;
    int64_t stride;
};

// Eight float32 in three parts of bfloat16, each what the one before leaves, rounded: together they
// are the number (8 + 8 + 8 bits).
struct Split {
    bf16x8 part[3];
};
__device__ __forceinline__ Split split(f32x8 x) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    Split s;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        float u = x[j], v = x[j + 1];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            const b2 h{static_cast<__bf16>(u), static_cast<__bf16>(v)};
            s.part[p][j] = h[0], s.part[p][j + 1] = h[1];
            if (p < 2) {
                const unsigned bits = __builtin_bit_cast(unsigned, h);
                u -= __uint_as_float(bits << 16);
                v -= __uint_as_float(bits & 0xffff0000u);
            }
        }
    }
    return s;
}
// The products of parts that make a product, from the smallest to the largest: a's part and b's.
// Left out are those of a second and a third part and of two third ones, together at most 2^-24 of
// |a| |b|.
constexpr int kSplitProducts[6][2] = {{1, 1}, {0, 2}, {2, 0}, {0, 1}, {1, 0}, {0, 0}};

template <typename T, typename S, template <typename, int, int> class OfA,
          template <typename, int, int> class OfB>
struct Product {
    using A = OfA<T, S::BM, S::kThreads>;
    using B = OfB<T, S::BN, S::kThreads>;
    static constexpr int kLdsElements = 2 * (A::kElements + B::kElements);
    // float32: six products of bfloat16 parts take 96 cycles of the matrix cores where eight steps
    // of the float32 instruction take 256, and splitting the operands, which the rows of a fragment
    // share, runs beside them (a loss and its gradients, 2048 tokens of 1024, 16384 words:
    // 1287 us instead of 2047).  Narrow tiles are bound by memory.
    static constexpr bool kSplit = sizeof(T) == 4 && S::BN > 16;

    // sums[i][t]: rows 16 (wm MT + i) + 4 g .. + 4 of column 16 (wn NT + t) + c, over k < `depth`.
    // Every thread of the workgroup calls this; m and n: rows and columns that there are.
    __device__ __forceinline__ static void run(Matrix<T> a, int m, Matrix<T> b, int n,
                                               int64_t depth, T *lds, f32x4 (&sums)[S::MT][S::NT]) {
        run_as<kSplit>(a, m, b, n, depth, lds, sums);
        if constexpr (kSplit) {
            // The parts of an infinity are one and numbers that are none.  A tile with a sum that
            // is not finite is worked out again without parts.
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < S::MT; ++i) x += not_finite(sums[i]);
            volatile int *again = reinterpret_cast<volatile int *>(lds);
            __syncthreads();
            if (threadIdx.x == 0) *again = 0;
            __syncthreads();
            if (x != x) *again = 1;
            __syncthreads();
            const bool redo = *again != 0;
            __syncthreads();
            if (redo) run_as<false>(a, m, b, n, depth, lds, sums);
        }
    }

    template <bool SPLIT>
    __device__ __forceinline__ static void run_as(Matrix<T> a, int m, Matrix<T> b, int n,
                                               int64_t depth, T *lds, f32x4 (&sums)[S::MT][S::NT]) {
        const int thread = static_cast<int>(threadIdx.x);
        const int wave = __builtin_amdgcn_readfirstlane(thread / dev::kWave);
        const int wm = wave / S::WN, wn = wave % S::WN;
        const int lane = dev::lane(), g = lane >> 4, c = lane & 15;
        A from_a;
        B from_b;
        from_a.start(thread, a.stride, m);
        from_b.start(thread, b.stride, n);
#pragma unroll
        for (int i = 0; i < S::MT; ++i) {
#pragma unroll
            for (int t = 0; t < S::NT; ++t) sums[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        if (depth <= 0) return;
        const int64_t step_a = A::advance(a.stride), step_b = B::advance(b.stride);
        T *tile_a = lds, *tile_b = lds + A::kElements;
        T *next_a = lds + A::kElements + B::kElements, *next_b = next_a + A::kElements;
        int64_t left = depth;  // of the step that is loaded next
        auto load = [&](T *to_a, T *to_b) {
            from_a.load(thread, a.data, left, to_a);
            from_b.load(thread, b.data, left, to_b);
            a.data += step_a;
            b.data += step_b;
            left -= kStepK<T>;
        };
        auto swap = [&] {
            T *const was_a = tile_a, *const was_b = tile_b;
            tile_a = next_a, tile_b = next_b;
            next_a = was_a, next_b = was_b;
        };
        // Fragment f of a half of the step's k: B's, then A's.
        auto read = [&](auto f, int kk, Frag<T> (&fa)[S::MT], Frag<T> (&fb)[S::NT]) {
            if constexpr (f() < S::NT) {
                fb[f()] = B::frag(tile_b, wn * S::NT + f(), kk, g, c);
            } else {
                fa[f() - S::NT] = A::frag(tile_a, wm * S::MT + f() - S::NT, kk, g, c);
            }
        };
        constexpr int kFrags = S::MT + S::NT;
        auto multiply = [&](auto i, const Frag<T> (&fa)[S::MT], const Frag<T> (&fb)[S::NT]) {
            each<S::NT>([&](auto t) { sums[i()][t()] = mma(fa[i()], fb[t()], sums[i()][t()]); });
        };
        load(tile_a, tile_b);
        int64_t steps = (depth + kStepK<T> - 1) / kStepK<T>;
        if constexpr (sizeof(T) == 4) {
            for (; steps > 0; --steps) {
                rows_arrived();
                if (left > 0) load(next_a, next_b);
                Frag<T> fa[S::MT], fb[S::NT];
                constexpr int kFirst = SPLIT ? S::NT + 2 : kFrags;
                each<(kFirst < kFrags ? kFirst : kFrags)>([&](auto f) { read(f, 0, fa, fb); });
                if constexpr (SPLIT) {
                    // (a row's operand is split between the matrix instructions of the row before,
                    // and read between those of the one before that)
                    Split pb[S::NT], pa[2];
                    each<S::NT>([&](auto t) { pb[t()] = split(fb[t()]); });
                    pa[0] = split(fa[0]);
                    each<S::MT>([&](auto i) {
                        __builtin_amdgcn_sched_barrier(0);
                        if constexpr (i() + 2 < S::MT) {
                            read(std::integral_constant<int, S::NT + i() + 2>{}, 0, fa, fb);
                        }
                        if constexpr (i() + 1 < S::MT) pa[(i() + 1) % 2] = split(fa[i() + 1]);
                        each<6>([&](auto p) {
                            each<S::NT>([&](auto t) {
                                sums[i()][t()] = mma(pa[i() % 2].part[kSplitProducts[p()][0]],
                                                     pb[t()].part[kSplitProducts[p()][1]],
                                                     sums[i()][t()]);
                            });
                        });
                        each<6 * S::NT>([&](auto) {
                            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // matrix
                            __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);  // vector
                        });
                    });
                    __builtin_amdgcn_sched_barrier(0);
                } else {
                    // (a step's products by themselves: one sum of all k would be rounded for each
                    // of their instructions.  Gradients of 9 tokens of 2784 and 3931 words are
                    // 2.7e-7 of their norms off instead of 1.3e-6, in 137 us instead of 136.)
                    each<S::MT>([&](auto i) {
                        each<S::NT>([&](auto t) {
                            sums[i()][t()] +=
                                mma(fa[i()], fb[t()], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
                        });
                    });
                }
                swap();
            }
        } else {
            // A step's products are two halves of 32 k, and while one half is multiplied the next
            // one's fragments are read, a few between the matrix instructions of each row.  The
            // barrier that ends a step for its buffer stands between its halves: by then a
            // wavefront has the second half's fragments in registers, so that its matrix
            // instructions go on behind it, while the next step's first half is read and the step
            // after that is loaded.
            Frag<T> fa0[S::MT], fb0[S::NT], fa1[S::MT], fb1[S::NT];
            auto half = [&](const Frag<T> (&fa)[S::MT], const Frag<T> (&fb)[S::NT], auto reads,
                            int kk, Frag<T> (&next_fa)[S::MT], Frag<T> (&next_fb)[S::NT]) {
                each<S::MT>([&](auto i) {
                    if constexpr (reads()) {
                        constexpr int kFrom = i() * kFrags / S::MT;
                        each<(i() + 1) * kFrags / S::MT - kFrom>([&](auto f) {
                            read(std::integral_constant<int, kFrom + f()>{}, kk, next_fa, next_fb);
                        });
                    }
                    multiply(i, fa, fb);
                    __builtin_amdgcn_sched_barrier(0);
                });
            };
            constexpr std::true_type kReads{};
            constexpr std::false_type kLast{};
            rows_arrived();
            if (left > 0) load(next_a, next_b);
            each<kFrags>([&](auto f) { read(f, 0, fa0, fb0); });
            for (; steps > 1; --steps) {
                half(fa0, fb0, kReads, 1, fa1, fb1);
                rows_arrived();
                if (left > 0) load(tile_a, tile_b);
                swap();
                half(fa1, fb1, kReads, 0, fa0, fb0);
            }
            half(fa0, fb0, kReads, 1, fa1, fb1);
            half(fa1, fb1, kLast, 0, fa0, fb0);
        }
    }
};

// The order of workgroup `at` of `all`.  Workgroups go to the eight dies in turn, each with a cache
// of its own: a die gets neighbours.
__device__ __forceinline__ unsigned order_of(unsigned at, unsigned all) {
    constexpr unsigned kDies = 8;
    const unsigned die = at % kDies, per = all / kDies, more = all % kDies;
    return die * per + min(die, more) + at / kDies;
}

// Tile i of m_tiles x n_tiles, in groups of kGroup along n, so that neighbours read few different
// rows.
__device__ __forceinline__ void tile_of(unsigned i, unsigned m_tiles, unsigned n_tiles,
                                        unsigned &m, unsigned &n) {
    constexpr unsigned kGroup = 8;
    const unsigned first = i / (kGroup * m_tiles) * kGroup, wide = min(kGroup, n_tiles - first);
    i -= first * m_tiles;
    n = first + i % wide;
    m = i / wide;
}

}  // namespace dense
}  // namespace nacho
