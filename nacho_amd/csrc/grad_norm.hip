// The common norm of many tensors, and the tensors scaled so that it is at most a given one.
//
// norm = root of the sum of squares; out = x min(1, max_norm / (norm + 1e-6)).  Bound by bytes: all
// tensors are read for the norm, then read again and written.  Squares are summed in float64, which
// costs nothing beside the bytes and neither overflows nor loses small tensors next to large ones.
//
// The tensors' addresses travel in the kernels' arguments, kTensors a launch, cut into chunks of
// kChunk elements: a workgroup finds the tensor of its chunk by a search of their first chunks.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <new>

#include "dense_rows.hpp"
#include "runtime.hpp"

namespace nacho {
namespace grad_norm {

using dense::element_aligned;
using dense::item_of;
using dense::Piece;

constexpr int kThreads = 256;
constexpr int64_t kChunk = 32768;
constexpr int kTensors = 96;

// (arguments of a launch: less than 4 KB)
struct Table {
    const void *data[kTensors];
    void *out[kTensors];
    int64_t size[kTensors];
    unsigned first[kTensors + 1];  // chunk
    unsigned char dtype[kTensors], out_dtype[kTensors];
    int count;
};
static_assert(sizeof(Table) <= 3584, "a launch's arguments");

// The tensor of a chunk: the last whose first chunk is not after it.
__device__ __forceinline__ int tensor_of(const Table &t, unsigned chunk) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= chunk) {
            lo = mid;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

// Calls f with the element type of a code.
template <typename F>
__device__ __forceinline__ void typed(int dtype, F f) {
    if (dtype == NACHO_F32) {
        f(float{});
    } else if (dtype == NACHO_F16) {
        f(_Float16{});
    } else {
        f(__bf16{});
    }
}

template <typename T>
__device__ __forceinline__ double squares_of(const T *p, int64_t n) {
    constexpr int kN = 16 / sizeof(T), kStep = 4;
    double sum = 0.0;
    auto add = [&](T v) {
        const double x = static_cast<double>(static_cast<float>(v));
        sum = __builtin_fma(x, x, sum);
    };
    // (elements before the first whole piece; a chunk starts anywhere)
    const int64_t head =
        min(n, static_cast<int64_t>((-reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T)));
    const int64_t whole = (n - head) / kN;
    const Piece<T, kN> *from = reinterpret_cast<const Piece<T, kN> *>(p + head);
    for (int64_t i0 = threadIdx.x; i0 < whole; i0 += kThreads * kStep) {
        Piece<T, kN> piece[kStep];
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int64_t i = i0 + s * kThreads;
            if (i < whole) piece[s] = from[i];
        }
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            if (i0 + s * kThreads < whole) {
#pragma unroll
                for (int j = 0; j < kN; ++j) add(piece[s].v[j]);
            }
        }
    }
    if (threadIdx.x < head) add(p[threadIdx.x]);
    if (threadIdx.x < n - head - whole * kN) add(p[head + whole * kN + threadIdx.x]);
    return sum;
}

__device__ __forceinline__ double group_sum(double sum, double *s_sum, int waves) {
    sum = dev::wave_sum(sum);
    if (dev::lane() == 0) s_sum[threadIdx.x / dev::kWave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < waves; ++w) sum += s_sum[w];
    return sum;
}

__global__ __launch_bounds__(kThreads) void square_kernel(Table t, double *__restrict__ sums) {
    __shared__ double s_sum[kThreads / dev::kWave];
    const int i = tensor_of(t, blockIdx.x);
    const int64_t at = (blockIdx.x - t.first[i]) * kChunk;
    const int64_t n = min(kChunk, t.size[i] - at);
    double sum = 0.0;
    typed(t.dtype[i], [&](auto type) {
        sum = squares_of(static_cast<const decltype(type) *>(t.data[i]) + at, n);
    });
    sum = group_sum(sum, s_sum, kThreads / dev::kWave);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

__global__ __launch_bounds__(1024) void norm_kernel(const double *__restrict__ sums, int64_t n,
                                                    float max_norm, float *__restrict__ norm,
                                                    float *__restrict__ factor) {
    __shared__ double s_sum[1024 / dev::kWave];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) sum += sums[i];
    sum = group_sum(sum, s_sum, 1024 / dev::kWave);
    if (threadIdx.x != 0) return;
    const double root = sqrt(sum);
    *norm = static_cast<float>(root);
    const double f = static_cast<double>(max_norm) / (root + 1e-6);
    // (no number stays; a limit of infinity is none)
    *factor = max_norm == dense::kInf && root == root ? 1.0f
              : f >= 1.0                              ? 1.0f
                                                      : static_cast<float>(f);
}

template <typename T, typename O>
__device__ __forceinline__ void scale_of(const T *p, O *out, int64_t n, float factor) {
    constexpr int kN = 16 / sizeof(T), kStep = 4;
    auto scaled = [&](T v) { return static_cast<O>(factor * static_cast<float>(v)); };
    int64_t head =
        min(n, static_cast<int64_t>((-reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T)));
    // (both sides in whole pieces, or element by element)
    const bool both = (reinterpret_cast<uintptr_t>(out + head) & 15) == 0;
    if (!both) {
        for (int64_t i0 = threadIdx.x; i0 < n; i0 += kThreads * 2 * kStep) {
            T v[2 * kStep];
#pragma unroll
            for (int s = 0; s < 2 * kStep; ++s) {
                if (i0 + s * kThreads < n) v[s] = p[i0 + s * kThreads];
            }
#pragma unroll
            for (int s = 0; s < 2 * kStep; ++s) {
                if (i0 + s * kThreads < n) out[i0 + s * kThreads] = scaled(v[s]);
            }
        }
        return;
    }
    const int64_t whole = (n - head) / kN;
    const Piece<T, kN> *from = reinterpret_cast<const Piece<T, kN> *>(p + head);
    for (int64_t i0 = threadIdx.x; i0 < whole; i0 += kThreads * kStep) {
        Piece<T, kN> piece[kStep];
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int64_t i = i0 + s * kThreads;
            if (i < whole) piece[s] = from[i];
        }
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int64_t i = i0 + s * kThreads;
            if (i < whole) {
                // (16 or 32 bytes)
                constexpr int kM = 16 / sizeof(O);
                Piece<O, kM> *to = reinterpret_cast<Piece<O, kM> *>(out + head + i * kN);
#pragma unroll
                for (int h = 0; h < kN / kM; ++h) {
                    Piece<O, kM> o;
#pragma unroll
                    for (int j = 0; j < kM; ++j) o.v[j] = scaled(piece[s].v[h * kM + j]);
                    dense::store_piece<O, kM>(reinterpret_cast<O *>(to + h), o);
                }
            }
        }
    }
    if (threadIdx.x < head) out[threadIdx.x] = scaled(p[threadIdx.x]);
    if (threadIdx.x < n - head - whole * kN) {
        const int64_t i = head + whole * kN + threadIdx.x;
        out[i] = scaled(p[i]);
    }
}

__global__ __launch_bounds__(kThreads) void scale_kernel(Table t,
                                                         const float *__restrict__ factor) {
    const int i = tensor_of(t, blockIdx.x);
    const int64_t at = (blockIdx.x - t.first[i]) * kChunk;
    const int64_t n = min(kChunk, t.size[i] - at);
    const float f = *factor;
    if (f == 1.0f && t.data[i] == t.out[i]) return;  // (as they are)
    typed(t.dtype[i], [&](auto type) {
        using T = decltype(type);
        const T *from = static_cast<const T *>(t.data[i]) + at;
        if (t.out_dtype[i] == t.dtype[i]) {
            scale_of(from, static_cast<T *>(t.out[i]) + at, n, f);
        } else {
            scale_of(from, static_cast<float *>(t.out[i]) + at, n, f);
        }
    });
}

// ---- host -----------------------------------------------------------------------------

int check(const nacho_gradient *tensors, int64_t count, bool clip, const float *norm,
          int64_t *chunks) {
    *chunks = 0;
    if (count < 0 || (count > 0 && !tensors) || !norm) return NACHO_ERR_INVALID_ARGUMENT;
    for (int64_t i = 0; i < count; ++i) {
        const nacho_gradient &t = tensors[i];
        if (t.size < 0 || t.dtype < NACHO_F32 || t.dtype > NACHO_BF16) {
            return NACHO_ERR_INVALID_ARGUMENT;
        }
        if (t.size > 0 && (!t.data || !element_aligned(t.data, item_of(t.dtype)))) {
            return NACHO_ERR_INVALID_ARGUMENT;
        }
        if (clip && ((t.out_dtype != t.dtype && t.out_dtype != NACHO_F32) ||
                     (t.size > 0 && (!t.out || !element_aligned(t.out, item_of(t.out_dtype)))))) {
            return NACHO_ERR_INVALID_ARGUMENT;
        }
        if (t.size > int64_t{1} << 46) return NACHO_ERR_INDEX_OVERFLOW;
        *chunks += (t.size + kChunk - 1) / kChunk;
    }
    // (also the chunks of each launch)
    return *chunks > dense::kMostGroups ? NACHO_ERR_INDEX_OVERFLOW : NACHO_OK;
}

// Calls f(table, chunks, chunks before) for each launch's tensors.
template <typename F>
int each_table(const nacho_gradient *tensors, int64_t count, F f) {
    Table t;
    t.count = 0;
    t.first[0] = 0;
    int64_t before = 0;
    for (int64_t i = 0; i < count; ++i) {
        const nacho_gradient &x = tensors[i];
        if (x.size > 0) {
            const int n = t.count++;
            t.data[n] = x.data;
            t.out[n] = x.out;
            t.size[n] = x.size;
            t.dtype[n] = static_cast<unsigned char>(x.dtype);
            t.out_dtype[n] = static_cast<unsigned char>(x.out_dtype);
            t.first[n + 1] = t.first[n] + static_cast<unsigned>((x.size + kChunk - 1) / kChunk);
        }
        if (t.count > 0 && (t.count == kTensors || i + 1 == count)) {
            NACHO_TRY(f(t, t.first[t.count], before));
            before += t.first[t.count];
            t.count = 0;
        }
    }
    return NACHO_OK;
}

int run(const nacho_gradient *tensors, int64_t count, bool clip, float max_norm, float *norm,
        void *stream, const nacho_allocator *alloc) {
    int64_t chunks = 0;
    if (clip && !(max_norm >= 0.0f)) return NACHO_ERR_INVALID_ARGUMENT;
    NACHO_TRY(check(tensors, count, clip, norm, &chunks));
    Call call(stream, alloc);
    const hipStream_t s = call.stream();
    double *sums = nullptr;  // and the factor
    NACHO_TRY(call.scratch_n(static_cast<size_t>(chunks) + 1, &sums));
    float *factor = reinterpret_cast<float *>(sums + chunks);
    NACHO_TRY(each_table(tensors, count, [&](const Table &t, unsigned n, int64_t before) -> int {
        square_kernel<<<n, kThreads, 0, s>>>(t, sums + before);
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    }));
    norm_kernel<<<1, 1024, 0, s>>>(sums, chunks, max_norm, norm, factor);
    NACHO_TRY_HIP(hipGetLastError());
    if (!clip) return NACHO_OK;
    return each_table(tensors, count, [&](const Table &t, unsigned n, int64_t) -> int {
        scale_kernel<<<n, kThreads, 0, s>>>(t, factor);
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    });
}

}  // namespace grad_norm
}  // namespace nacho

extern "C" int nacho_grad_norm(const nacho_gradient *tensors, int64_t count, float *norm,
                               void *stream, const nacho_allocator *alloc) {
    try {
        return nacho::grad_norm::run(tensors, count, false, 0.0f, norm, stream, alloc);
    } catch (const std::bad_alloc &) {
        return NACHO_ERR_OUT_OF_MEMORY;
    }
}

extern "C" int nacho_clip_grad_norm(const nacho_gradient *tensors, int64_t count, float max_norm,
                                    float *norm, void *stream, const nacho_allocator *alloc) {
    try {
        return nacho::grad_norm::run(tensors, count, true, max_norm, norm, stream, alloc);
    } catch (const std::bad_alloc &) {
        return NACHO_ERR_OUT_OF_MEMORY;
    }
}
