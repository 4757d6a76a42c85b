// Rows of elements in memory: the pieces in which kernels that move them read and write, and what
// the host checks of their addresses.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "dense_tiles.hpp"
#include "runtime.hpp"

namespace nacho {
namespace dense {

// N elements that are read or written together: 16 bytes where rows allow it, one element where
// a row starts between (odd widths and strides).  With the alignment of an element they lie wherever
// it does: loads and stores of 16 bytes take any address.
template <typename T, int N, int ALIGN = N * sizeof(T)>
struct alignas(ALIGN) Piece {
    T v[N];
};
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// Rows are too many to be read again from a cache by what comes next: they go past it.
template <typename T, int N, int ALIGN = N * sizeof(T)>
__device__ __forceinline__ Piece<T, N, ALIGN> load_piece(const T *p) {
    if constexpr (N * sizeof(T) == 16) {
        u32x4 v;
        if constexpr (ALIGN < 16) {
            v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(p));
        } else {
            v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
        }
        return __builtin_bit_cast(Piece<T, N, ALIGN>, v);
    } else {
        return *reinterpret_cast<const Piece<T, N, ALIGN> *>(p);
    }
}
template <typename T, int N, int ALIGN>
__device__ __forceinline__ void store_piece(T *p, const Piece<T, N, ALIGN> &v) {
    if constexpr (N * sizeof(T) == 16) {
        if constexpr (ALIGN < 16) {
            __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v),
                                        reinterpret_cast<u32x4_any *>(p));
        } else {
            __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4 *>(p));
        }
    } else {
        *reinterpret_cast<Piece<T, N, ALIGN> *>(p) = v;
    }
}

// Elements to zero, 16 bytes a thread; `head` of them before the first aligned ones.
constexpr int kClearThreads = 256;

template <typename T>
__global__ __launch_bounds__(kClearThreads) void clear_kernel(T *__restrict__ p, int64_t n) {
    constexpr int64_t kN = 16 / sizeof(T);
    const int64_t head = min(n, static_cast<int64_t>(
                                    (-reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T)));
    const int64_t whole = (n - head) / kN;
    const int64_t at = blockIdx.x * static_cast<int64_t>(kClearThreads) + threadIdx.x;
    const int64_t all = gridDim.x * static_cast<int64_t>(kClearThreads);
    const u32x4 zero{0u, 0u, 0u, 0u};
    for (int64_t i = at; i < whole; i += all) {
        reinterpret_cast<u32x4 *>(p + head)[i] = zero;
    }
    if (at < head) p[at] = static_cast<T>(0.0f);
    if (at < n - head - whole * kN) p[head + whole * kN + at] = static_cast<T>(0.0f);
}

// ---- host -----------------------------------------------------------------------------

inline int item_of(int32_t dtype) { return dtype == NACHO_F32 ? 4 : 2; }

// Whether rows of `width` elements at `p`, `stride` apart, are whole aligned 16-byte pieces.
inline bool pieces(const void *p, int64_t stride, int64_t width, int item) {
    const int64_t per = 16 / item;
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % per == 0 && width % per == 0;
}

inline bool element_aligned(const void *p, int item) {
    return reinterpret_cast<uintptr_t>(p) % static_cast<unsigned>(item) == 0;
}

template <typename T>
int clear(hipStream_t stream, T *p, int64_t n) {
    const int64_t bytes = n * static_cast<int64_t>(sizeof(T)), per = 16 * kClearThreads;
    const int64_t groups = (bytes + per - 1) / per;
    const unsigned grid =
        static_cast<unsigned>(groups < 1 ? 1 : groups < kMostGroups ? groups : kMostGroups);
    clear_kernel<T><<<grid, kClearThreads, 0, stream>>>(p, n);
    NACHO_TRY_HIP(hipGetLastError());
    return NACHO_OK;
}

}  // namespace dense
}  // namespace nacho
