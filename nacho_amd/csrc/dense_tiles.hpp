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

// Elements of a row of a tile of DP columns in LDS: 16 bytes more than the data, so that the 16
// rows that a fragment's lanes read lie in different banks.
template <typename T, int DP>
constexpr int kTileRow = DP + 16 / static_cast<int>(sizeof(T));

// Eight consecutive elements (16-byte aligned).
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

// Column `col0 + c` of rows 4 g + j and 16 + 4 g + j (j < 4) of the 32 rows at `tile` (rows of
// ROW elements).  16-bit types use the transposing LDS read: the 16 lanes of a group name four
// rows of 16 elements, four lanes a row, and lane c receives column c of the four rows.
template <int ROW>
__device__ __forceinline__ f32x8 column_frag(const float *tile, int col0, int g, int c) {
    f32x8 f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = tile[(4 * g + j) * ROW + col0 + c];
        f[4 + j] = tile[(16 + 4 * g + j) * ROW + col0 + c];
    }
    return f;
}
template <int ROW, typename T>
__device__ __forceinline__ Frag<T> column_frag(const T *tile, int col0, int g, int c) {
    using Shared = __attribute__((address_space(3))) s16x4 *;
    const T *p = tile + (4 * g + (c >> 2)) * ROW + col0 + 4 * (c & 3);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (Shared)(reinterpret_cast<const s16x4 *>(p)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (Shared)(reinterpret_cast<const s16x4 *>(p + 16 * ROW)));
    const auto both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(Frag<T>, both);
}

// Rows of a [rows][D] operand on their way to a tile of ROWS x DP in LDS: each of THREADS
// threads carries N 16-byte pieces.  Pieces at or past column D are zero.
template <typename T, int DP, int ROWS, int THREADS>
struct TileLoad {
    static constexpr int kPer = 16 / sizeof(T);       // elements of a piece
    static constexpr int kPieces = DP / kPer;         // pieces of a row
    static constexpr int kN = ROWS * kPieces / THREADS;
    static_assert(ROWS * kPieces % THREADS == 0, "whole pieces per thread");
    u32x4 piece[kN];

    // row_of(r): the row's first element, or null for a row of zeros.
    template <typename RowOf>
    __device__ __forceinline__ void load(int thread, int D, RowOf row_of) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int at = thread + i * THREADS;
            const int r = at / kPieces, col = at % kPieces * kPer;
            const T *row = row_of(r);
            piece[i] = u32x4{0u, 0u, 0u, 0u};
            if (row && col < D) piece[i] = *reinterpret_cast<const u32x4 *>(row + col);
        }
    }
    __device__ __forceinline__ void store(int thread, T *tile) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int at = thread + i * THREADS;
            const int r = at / kPieces, col = at % kPieces * kPer;
            *reinterpret_cast<u32x4 *>(tile + r * kTileRow<T, DP> + col) = piece[i];
        }
    }
};

// A row of D elements as operand fragments (k = 32 kk + 8 g + j); null gives zeros.
template <typename T, int DP>
__device__ __forceinline__ void load_row_frags(const T *row, int D, int g, Frag<T> (&f)[DP / 32]) {
#pragma unroll
    for (int kk = 0; kk < DP / 32; ++kk) {
        const int col = 32 * kk + 8 * g;
        f[kk] = (row && col < D) ? row_frag<T>(row + col) : zero_frag<T>();
    }
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

// Maximum and sum over the four lanes of a column (lanes c, 16 + c, 32 + c, 48 + c).
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, dev::kWave));
    return fmaxf(v, __shfl_xor(v, 32, dev::kWave));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16, dev::kWave);
    return v + __shfl_xor(v, 32, dev::kWave);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

}  // namespace dense
}  // namespace nacho
