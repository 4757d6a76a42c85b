// Building blocks of the kernels that multiply dense rows: element types, 16x16 matrix products
// with float32 sums, and the tiles in LDS that feed them.
//
// A matrix instruction takes eight consecutive k per lane (lane = 16 g + c: row or column c,
// k = 8 g + j).  All products here go over k in an order that both operands share, so a tile
// whose k is its row index can be read with any fixed permutation of rows: `column_frag` reads
// rows 4 g + j and 16 + 4 g + j, the order in which a product's result already lies in the lanes
// (column c, rows 4 g + i of each 16).  A product's result is therefore the next product's
// operand without passing through LDS.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "device_utils.hpp"

namespace nacho {
namespace dense {

// Workgroups of 256 threads that a launch can have.  A launch of 2^32 work-items or more is no
// error: it runs what is left of their number modulo 2^32.
constexpr int64_t kMostGroups = ((int64_t{1} << 32) - 1) / 256;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct FragOf;
template <>
struct FragOf<float> {
    using type = f32x8;
};
template <>
struct FragOf<_Float16> {
    using type = f16x8;
};
template <>
struct FragOf<__bf16> {
    using type = bf16x8;
};
template <typename T>
using Frag = typename FragOf<T>::type;

// c += a * b over 32 k: a's rows and b's columns are the lanes' c.  float32 operands keep their
// 32 bits (eight steps of the float32 instruction, whose k are 4).
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

template <typename T>
__device__ __forceinline__ Frag<T> zero_frag() {
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = static_cast<T>(0.0f);
    return f;
}

// Two results of a product (rows 0-15 and 16-31 of k), rounded to T, as an operand.
template <typename T>
__device__ __forceinline__ Frag<T> result_frag(f32x4 lo, f32x4 hi) {
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = static_cast<T>(lo[j]);
        f[4 + j] = static_cast<T>(hi[j]);
    }
    return f;
}

// How the results of a product become the next one's operand: one part of its type, or two; with
// kTwoOrInfinite infinities among them are that in the sums too (their rests are no numbers).
enum Parts { kOne, kTwo, kTwoOrInfinite };

// Two results of a product as an operand in two parts of T, a 16-bit type, that together hold what
// one would round away: `head` is x cut off toward 0, `rest` what is left of (1 + 2^-12) x.  The
// part of 2^-12, which kPartsScale undoes in the sums, gives the rest x's sign and keeps it from
// being 0 where x is not, so that the products of both with an infinity are the same infinity.
// (float16: for an x of 2^-12 or more; below, the rest may be 0.)
template <typename T, Parts PARTS>
__device__ __forceinline__ void parts_frag(f32x4 lo, f32x4 hi, Frag<T> &head, Frag<T> &rest) {
    typedef T t2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float x = j < 4 ? lo[j] : hi[j - 4], y = j < 4 ? lo[j + 1] : hi[j - 3];
        t2 h, r;
        f2 cut;
        if constexpr (__is_same(T, __bf16)) {
            const unsigned a = __float_as_uint(x), b = __float_as_uint(y);
            h = __builtin_bit_cast(t2, __builtin_amdgcn_perm(b, a, 0x07060302u));
            cut = f2{__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)};
        } else {
            h = __builtin_bit_cast(t2, __builtin_amdgcn_cvt_pkrtz(x, y));
            cut = f2{static_cast<float>(h[0]), static_cast<float>(h[1])};
        }
        constexpr float kMore = 1.0f + 0x1p-12f;
        float u = __builtin_fmaf(x, kMore, -cut[0]), v = __builtin_fmaf(y, kMore, -cut[1]);
        if constexpr (PARTS == kTwoOrInfinite) {  // (no number to any finite one)
            u = fmaxf(u, -0x1p100f);
            v = fmaxf(v, -0x1p100f);
        }
        if constexpr (__is_same(T, __bf16)) {
            r = t2{static_cast<T>(u), static_cast<T>(v)};
        } else {
            r = __builtin_bit_cast(t2, __builtin_amdgcn_cvt_pkrtz(u, v));
        }
        head[j] = h[0], head[j + 1] = h[1];
        rest[j] = r[0], rest[j + 1] = r[1];
    }
}
template <typename T>
constexpr float kPartsScale = sizeof(T) == 2 ? 1.0f / (1.0f + 0x1p-12f) : 1.0f;

// Eight consecutive elements in memory (16-byte aligned).
template <typename T>
__device__ __forceinline__ Frag<T> row_frag(const T *p) {
    return *reinterpret_cast<const Frag<T> *>(p);
}
template <>
__device__ __forceinline__ Frag<float> row_frag<float>(const float *p) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p);
    const f32x4 b = *reinterpret_cast<const f32x4 *>(p + 4);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Elements of a padded row of DP elements in LDS: 16 bytes more than the data, so that the 16 rows
// that a fragment's lanes read lie in different banks.
template <typename T, int DP>
constexpr int kTileRow = DP + 16 / static_cast<int>(sizeof(T));

// What a product with masked operands needs where some are not finite (0 times infinity is no
// number): each element that is not becomes 0, or with `marks` 1, and the others 0.
template <typename T>
__device__ __forceinline__ u32x4 finite_piece(u32x4 bits, bool marks) {
    constexpr int kN = 16 / static_cast<int>(sizeof(T));
    typedef T piece_t __attribute__((ext_vector_type(kN)));
    piece_t v = __builtin_bit_cast(piece_t, bits);
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const float x = static_cast<float>(v[j]);
        const bool finite = x - x == 0.0f;
        v[j] = marks ? static_cast<T>(finite ? 0.0f : 1.0f) : finite ? v[j] : static_cast<T>(0.0f);
    }
    return __builtin_bit_cast(u32x4, v);
}

// A barrier after which every wavefront's loads from memory to LDS are complete.  (Each waits for
// its own: a barrier alone orders accesses to LDS, and these loads count as memory's.)
__device__ __forceinline__ void rows_arrived() {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
}

// Rows in LDS, filled straight from memory: a wavefront's load names a source per
// lane and writes 64 consecutive 16-byte pieces.  Rows are not padded (they cannot be); instead
// piece p of row r lies at place p ^ swizzle(r), which the loads' sources take care of, so that
// the 16 rows that a fragment reads lie in different banks, and so do the rows of a column.
// Products use the first DP columns; a row in LDS has the next power of two.
template <typename T, int DP, int ROWS, int THREADS>
struct Tile {
    static constexpr int kRow = DP <= 64 ? 64 : 128;
    static constexpr int kPer = 16 / static_cast<int>(sizeof(T));  // elements of a piece
    static constexpr int kPieces = kRow / kPer;                    // pieces of a row
    static constexpr int kLoads = ROWS * kPieces / THREADS;
    static constexpr int kElements = ROWS * kRow;
    static_assert(ROWS * kPieces % THREADS == 0, "whole pieces per thread");

    // A different number for each of the 16 rows of a fragment (of 8 rows in each half of the
    // banks, where a row is half of them), and for the rows of a column read, which takes two
    // neighbouring pieces of eight rows at a time, one that differs in more than its last bit.
    __device__ __forceinline__ static int swizzle(int row) {
        if constexpr (kPieces >= 16) {
            return ((row << 1) & 14) | ((row >> 3) & 1);
        } else {
            return (row & 6) | ((row >> 3) & 1);
        }
    }

    // row_of(r): row r of the source, r < ROWS; every one has to be there (rows that are masked
    // name another's).  Pieces at or past column D repeat the row's first.  Complete after the
    // next rows_arrived.
    template <typename RowOf>
    __device__ __forceinline__ static void load(T *tile, int thread, int D, RowOf row_of) {
        using Global = const __attribute__((address_space(1))) void *;
        using Shared = __attribute__((address_space(3))) void *;
        const int wave_first = __builtin_amdgcn_readfirstlane(thread & ~(dev::kWave - 1));
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int at = thread + i * THREADS;
            const int r = at / kPieces;
            const int piece = (at % kPieces) ^ swizzle(r);
            const T *from = row_of(r) + (piece * kPer < D ? piece * kPer : 0);
            T *to = tile + (i * THREADS + wave_first) * kPer;
            __builtin_amdgcn_global_load_lds((Global)from, (Shared)to, 16, 0, 0);
        }
    }

    // The same for rows `stride` bytes apart from a step to the next: what a thread reads of the
    // step's first row on, in bytes, is worked out once.  Rows from `there` on and pieces at or
    // past column D are past the buffer's end, where loads give zeros.
    struct Source {
        unsigned offset[kLoads];
        unsigned stride, bytes;  // of a row, of its data

        __device__ __forceinline__ Source(int thread, int D, int64_t row_stride)
            : stride(static_cast<unsigned>(row_stride * static_cast<int>(sizeof(T)))),
              bytes(static_cast<unsigned>(D * static_cast<int>(sizeof(T)))) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int at = thread + i * THREADS;
                const int r = at / kPieces;
                const unsigned piece = static_cast<unsigned>((at % kPieces) ^ swizzle(r));
                offset[i] = 16u * piece < bytes ? static_cast<unsigned>(r) * stride + 16u * piece
                                                : 0xffffff00u;
            }
        }
    };

    __device__ __forceinline__ static void load(T *tile, int thread, const Source &from,
                                                const T *first, int there) {
#if defined(__HIP_DEVICE_COMPILE__)  // (the host pass does not know buffer descriptors)
        using Shared = __attribute__((address_space(3))) void *;
        const int wave_first = __builtin_amdgcn_readfirstlane(thread & ~(dev::kWave - 1));
        const unsigned end =
            there > 0 ? static_cast<unsigned>(min(there, ROWS) - 1) * from.stride + from.bytes : 0u;
        const auto buffer = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<T *>(first), 0, end, 0x00020000);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            T *to = tile + (i * THREADS + wave_first) * kPer;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (Shared)to, 16,
                                                     static_cast<int>(from.offset[i]), 0, 0, 0);
        }
#endif
    }

    __device__ static void make_finite(T *tile, int thread, bool marks) {
        for (int i = 0; i < kLoads; ++i) {
            u32x4 *p = reinterpret_cast<u32x4 *>(tile + (thread + i * THREADS) * kPer);
            *p = finite_piece<T>(*p, marks);
        }
    }

    // Columns 32 kk + 8 g .. + 8 of row 16 t + c.
    __device__ __forceinline__ static Frag<T> row(const T *tile, int t, int kk, int g, int c) {
        const T *p = tile + (16 * t + c) * kRow;
        const int x = swizzle(c);  // (of row 16 t + c as well)
        if constexpr (sizeof(T) == 4) {
            const int piece = 8 * kk + 2 * g;
            const f32x4 a = *reinterpret_cast<const f32x4 *>(p + (piece ^ x) * kPer);
            const f32x4 b = *reinterpret_cast<const f32x4 *>(p + ((piece + 1) ^ x) * kPer);
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *reinterpret_cast<const Frag<T> *>(p + ((4 * kk + g) ^ x) * kPer);
        }
    }

    // Column 16 i + c of rows 32 u + 4 g + j and 32 u + 16 + 4 g + j (j < 4).  16-bit types use
    // the transposing LDS read: the 16 lanes of a group name four rows of 16 elements, four lanes
    // a row, and lane c receives column c of the four rows.
    __device__ __forceinline__ static Frag<T> column(const T *tile, int u, int i, int g, int c) {
        if constexpr (sizeof(T) == 4) {
            Frag<T> f;
            const int piece = 4 * i + (c >> 2);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 4 * g + j;
                const T *p = tile + (32 * u + r) * kRow + (piece ^ swizzle(r)) * kPer + (c & 3);
                f[j] = p[0];
                f[4 + j] = p[16 * kRow];
            }
            return f;
        } else {
            using Shared = __attribute__((address_space(3))) s16x4 *;
            const int r = 4 * g + (c >> 2);
            const int at = r * kRow + ((2 * i + ((c >> 1) & 1)) ^ swizzle(r)) * kPer + 4 * (c & 1);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (Shared)(reinterpret_cast<const s16x4 *>(tile + (32 * u * kRow + at))));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (Shared)(reinterpret_cast<const s16x4 *>(tile + (32 * u * kRow + 16 * kRow + at))));
            const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(Frag<T>, both);
        }
    }
};

// A Tile's rows on their way through registers, for a tile that one wavefront fills and reads by
// itself: pieces at or past column D, and rows that are not there, are zeros.
template <typename T, int DP, int ROWS>
struct TileStage {
    using Lds = Tile<T, DP, ROWS, dev::kWave>;
    u32x4 piece[Lds::kLoads];

    // row_of(r): the row's first element, or null.
    template <typename RowOf>
    __device__ __forceinline__ void load(int lane, int D, RowOf row_of) {
#pragma unroll
        for (int i = 0; i < Lds::kLoads; ++i) {
            const int at = lane + i * dev::kWave;
            const int col = at % Lds::kPieces * Lds::kPer;
            const T *row = row_of(at / Lds::kPieces);
            piece[i] = u32x4{0u, 0u, 0u, 0u};
            if (row && col < D) piece[i] = *reinterpret_cast<const u32x4 *>(row + col);
        }
    }
    __device__ __forceinline__ void make_finite(bool marks) {
#pragma unroll
        for (int i = 0; i < Lds::kLoads; ++i) piece[i] = finite_piece<T>(piece[i], marks);
    }
    __device__ __forceinline__ void store(int lane, T *tile) const {
#pragma unroll
        for (int i = 0; i < Lds::kLoads; ++i) {
            const int at = lane + i * dev::kWave;
            const int r = at / Lds::kPieces, p = (at % Lds::kPieces) ^ Lds::swizzle(r);
            *reinterpret_cast<u32x4 *>(tile + r * Lds::kRow + p * Lds::kPer) = piece[i];
        }
    }
};

// products[x][t] = rows 16 t .. of the tile times column tile x of the operand.
template <typename Lds, typename T, int DP, int COLS, int N>
__device__ __forceinline__ void row_products(const T *tile, const Frag<T> (&operand)[COLS][DP / 32],
                                             int g, int c, f32x4 (&products)[COLS][N]) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
#pragma unroll
        for (int x = 0; x < COLS; ++x) products[x][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < DP / 32; ++kk) {
            const Frag<T> f = Lds::row(tile, t, kk, g, c);
#pragma unroll
            for (int x = 0; x < COLS; ++x) products[x][t] = mma(f, operand[x][kk], products[x][t]);
        }
    }
}

// sums[x] += the tile's columns times p[x], the products' rows, which 16-bit types take rounded, or
// in two parts: a second product with the same columns, and a sum that is 1 / kPartsScale times as
// large.
template <typename Lds, typename T, int DP, int COLS, int N, Parts PARTS>
__device__ __forceinline__ void column_products(const T *tile, const f32x4 (&p)[COLS][N], int g,
                                                int c, f32x4 (&sums)[COLS][DP / 16]) {
    constexpr bool kSplit = PARTS != kOne && sizeof(T) == 2;
#pragma unroll
    for (int u = 0; u < N / 2; ++u) {
        Frag<T> f[COLS], rest[COLS];
#pragma unroll
        for (int x = 0; x < COLS; ++x) {
            if constexpr (kSplit) {
                parts_frag<T, PARTS>(p[x][2 * u], p[x][2 * u + 1], f[x], rest[x]);
            } else {
                f[x] = result_frag<T>(p[x][2 * u], p[x][2 * u + 1]);
            }
        }
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const Frag<T> v = Lds::column(tile, u, i, g, c);
#pragma unroll
            for (int x = 0; x < COLS; ++x) {
                sums[x][i] = mma(v, f[x], sums[x][i]);
                if constexpr (kSplit) sums[x][i] = mma(v, rest[x], sums[x][i]);
            }
        }
    }
}

// A row of D elements as operand fragments (k = 32 kk + 8 g + j); null gives zeros.
template <typename T, int DP>
__device__ __forceinline__ void load_row_frags(const T *row, int D, int g, Frag<T> (&f)[DP / 32]) {
#pragma unroll
    for (int kk = 0; kk < DP / 32; ++kk) {
        const int col = 32 * kk + 8 * g;
        f[kk] = (row && col < D) ? row_frag<T>(row + col) : zero_frag<T>();
    }
}

template <typename T, int DP>
__device__ __forceinline__ void negate(Frag<T> (&f)[DP / 32]) {
#pragma unroll
    for (int kk = 0; kk < DP / 32; ++kk) f[kk] = -f[kk];
}

// Four consecutive results rounded to T and stored together.
template <typename T>
__device__ __forceinline__ void store4(T *p, f32x4 v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = static_cast<T>(v[i]);
    *reinterpret_cast<t4 *>(p) = o;
}

// Maximum and sum over the four lanes of a column (lanes c, 16 + c, 32 + c, 48 + c): exchanges of
// rows of 16 and of 32 lanes between two registers, which hold the same value here.
__device__ __forceinline__ float column_max(float v) {
    const unsigned x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const unsigned y = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_sum(float v) {
    const unsigned x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    const unsigned y = __float_as_uint(__uint_as_float(a[0]) + __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 0, or no number where some sum is not finite.
template <int N>
__device__ __forceinline__ float not_finite(const f32x4 (&v)[N]) {
    float x = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x = __builtin_fmaf(v[n][i], 0.0f, x);
    }
    return x;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

}  // namespace dense
}  // namespace nacho
