// The common norm of many tensors, and the tensors scaled so that it is at most a given one.
//
// norm = root of the sum of squares; out = x min(1, max_norm / (norm + 1e-6)).  Bound by bytes: all
// tensors are read for the norm, then read again and written.  Squares are summed in float64, which
// costs nothing beside the bytes and neither overflows nor loses small tensors next to large ones.
//
// The tensors are cut into chunks of kChunk elements, one a workgroup, which finds the tensor of its
// chunk by a search of their first chunks.  The tensors' addresses travel in the kernels'
// arguments; those of more than kTensors are first written into memory by small launches (with
// passes of kTensors at a time instead, 611 tensors of 120 M elements took 204 us a call).
//
// Measured: 290 tensors of 2^30 bfloat16 elements scaled into float32 1585 us, 5.4 TB/s, of which the
// norm 345 (6.2 TB/s) and the scaling 1217; 611 tensors of 120 M float16 elements in place 144 us.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>
#include <new>
#include <type_traits>

#include "dense_rows.hpp"
#include "runtime.hpp"

namespace nacho {
namespace grad_norm {

using dense::element_aligned;
using dense::item_of;
using dense::Piece;

constexpr int kThreads = 256;
constexpr int64_t kChunk = 32768;
constexpr int kTensors = 96;  // (of a launch's arguments)
// Up to so many chunks, every workgroup that scales adds up the chunks' sums itself (8 KB from a
// cache), instead of a launch between: 14 small tensors 12 us a call instead of 16.
constexpr int64_t kFewChunks = 1024;

struct Tensor {
    const void *data;
    void *out;
    int64_t size;
    unsigned first;  // chunk
    unsigned char dtype, out_dtype;
};

// (arguments of a launch: less than 4 KB)
struct Table {
    Tensor tensors[kTensors];
    int count;
};
static_assert(sizeof(Table) <= 3584, "a launch's arguments");

// Where a kernel finds the tensors: in its arguments, or in memory.
struct InArguments {
    Table table;

    // The tensor of a chunk, the last whose first chunk is not after it, and that chunk's place.
    __device__ __forceinline__ const Tensor &of(unsigned chunk) const {
        int lo = 0, hi = table.count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (table.tensors[mid].first <= chunk) {
                lo = mid;
            } else {
                hi = mid - 1;
            }
        }
        return table.tensors[lo];
    }
};
struct InMemory {
    const Tensor *tensors;
    int64_t count;

    // (the lanes look at 64 tensors at a time, the same number apart)
    __device__ __forceinline__ const Tensor &of(unsigned chunk) const {
        int64_t lo = 0, hi = count - 1;
        while (lo < hi) {
            const int64_t step = (hi - lo) / dev::kWave + 1, i = lo + dev::lane() * step;
            const bool there = i <= hi && tensors[i].first <= chunk;
            lo += (__popcll(__ballot(there)) - 1) * step;
            hi = min(hi, lo + step - 1);
        }
        return tensors[lo];
    }
};

__global__ __launch_bounds__(dev::kWave) void table_kernel(Table t, Tensor *__restrict__ tensors) {
    for (int i = threadIdx.x; i < t.count; i += dev::kWave) tensors[i] = t.tensors[i];
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

// The sum of the threads' values, for all of them.
__device__ __forceinline__ double group_sum(double sum) {
    __shared__ double s_sum[kThreads / dev::kWave];
    sum = dev::wave_sum(sum);
    if (dev::lane() == 0) s_sum[threadIdx.x / dev::kWave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / dev::kWave; ++w) sum += s_sum[w];
    return sum;
}

template <typename Tensors>
__global__ __launch_bounds__(kThreads) void square_kernel(Tensors tensors,
                                                          double *__restrict__ sums) {
    const Tensor t = tensors.of(blockIdx.x);
    const int64_t at = (blockIdx.x - t.first) * kChunk;
    const int64_t n = min(kChunk, t.size - at);
    double sum = 0.0;
    typed(t.dtype, [&](auto type) {
        sum = squares_of(static_cast<const decltype(type) *>(t.data) + at, n);
    });
    sum = group_sum(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// The norm from the chunks' sums, whose order is that of a workgroup's threads wherever this runs.
__device__ __forceinline__ double norm_of(const double *__restrict__ sums, int64_t n) {
    constexpr int kStep = 16;
    double sum = 0.0;
    for (int64_t i0 = threadIdx.x; i0 < n; i0 += kThreads * kStep) {
        double x[kStep];
#pragma unroll
        for (int s = 0; s < kStep; ++s) {
            const int64_t i = i0 + s * kThreads;
            x[s] = i < n ? sums[i] : 0.0;
        }
#pragma unroll
        for (int s = 0; s < kStep; ++s) sum += x[s];
    }
    return sqrt(group_sum(sum));
}

__device__ __forceinline__ float factor_of(double norm, float max_norm) {
    const double f = static_cast<double>(max_norm) / (norm + 1e-6);
    // (no number stays; a limit of infinity is none)
    return max_norm == dense::kInf && norm == norm ? 1.0f
           : f >= 1.0                              ? 1.0f
                                                   : static_cast<float>(f);
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const double *__restrict__ sums, int64_t n,
                                                        float max_norm, float *__restrict__ norm,
                                                        float *__restrict__ factor) {
    const double x = norm_of(sums, n);
    if (threadIdx.x != 0) return;
    *norm = static_cast<float>(x);
    *factor = factor_of(x, max_norm);
}

template <typename T, typename O>
__device__ __forceinline__ void scale_of(const T *p, O *out, int64_t n, float factor) {
    // (16 bytes of the wider of the two: a wavefront's stores lie next to each other)
    constexpr int kN = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
    constexpr int kStep = sizeof(T) == sizeof(O) ? 4 : 8;
    constexpr uintptr_t kAlign = kN * sizeof(T) - 1;
    auto scaled = [&](T v) { return static_cast<O>(factor * static_cast<float>(v)); };
    const int64_t head =
        min(n, static_cast<int64_t>((-reinterpret_cast<uintptr_t>(p) & kAlign) / sizeof(T)));
    // (both sides in whole pieces, or element by element)
    const bool both = (reinterpret_cast<uintptr_t>(out + head) & (kN * sizeof(O) - 1)) == 0;
    if (!both) {
        for (int64_t i0 = threadIdx.x; i0 < n; i0 += kThreads * kStep) {
            T v[kStep];
#pragma unroll
            for (int s = 0; s < kStep; ++s) {
                if (i0 + s * kThreads < n) v[s] = p[i0 + s * kThreads];
            }
#pragma unroll
            for (int s = 0; s < kStep; ++s) {
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
                Piece<O, kN> o;
#pragma unroll
                for (int j = 0; j < kN; ++j) o.v[j] = scaled(piece[s].v[j]);
                dense::store_piece<O, kN>(out + head + i * kN, o);
            }
        }
    }
    if (threadIdx.x < head) out[threadIdx.x] = scaled(p[threadIdx.x]);
    if (threadIdx.x < n - head - whole * kN) {
        const int64_t i = head + whole * kN + threadIdx.x;
        out[i] = scaled(p[i]);
    }
}

// What the chunks are scaled by: `factor`, or where that is null, what the chunks' sums give.
struct Limit {
    const float *factor;
    const double *sums;
    int64_t chunks;
    float max_norm;
    float *norm;
};

// Chunks go from the last to the first: those that the norm has read last are still in a cache.
template <typename Tensors>
__global__ __launch_bounds__(kThreads) void scale_kernel(Tensors tensors, Limit limit) {
    float f;
    if (limit.factor) {
        f = *limit.factor;
    } else {
        const double norm = norm_of(limit.sums, limit.chunks);
        f = factor_of(norm, limit.max_norm);
        if (blockIdx.x == 0 && threadIdx.x == 0) *limit.norm = static_cast<float>(norm);
    }
    const unsigned chunk = gridDim.x - 1 - blockIdx.x;
    const Tensor t = tensors.of(chunk);
    const int64_t at = (chunk - t.first) * kChunk;
    const int64_t n = min(kChunk, t.size - at);
    if (f == 1.0f && t.data == t.out) return;  // (as they are)
    typed(t.dtype, [&](auto type) {
        using T = decltype(type);
        const T *from = static_cast<const T *>(t.data) + at;
        if (t.out_dtype == t.dtype) {
            scale_of(from, static_cast<T *>(t.out) + at, n, f);
        } else {
            scale_of(from, static_cast<float *>(t.out) + at, n, f);
        }
    });
}

// ---- host -----------------------------------------------------------------------------

int check(const nacho_gradient *tensors, int64_t count, bool clip, const float *norm,
          int64_t *held, int64_t *chunks) {
    *held = *chunks = 0;
    if (count < 0 || (count > 0 && !tensors) || !norm) return NACHO_ERR_INVALID_ARGUMENT;
    for (int64_t i = 0; i < count; ++i) {
        const nacho_gradient &t = tensors[i];
        if (t.size < 0 || t.dtype < NACHO_F32 || t.dtype > NACHO_BF16) {
            return NACHO_ERR_INVALID_ARGUMENT;
        }
        if (t.size > 0 && (!t.data || !element_aligned(t.data, item_of(t.dtype)))) {
            return NACHO_ERR_INVALID_ARGUMENT;
        }
        // (wider elements over narrower ones that are still to be read)
        if (clip && t.size > 0 && t.out == t.data && t.out_dtype != t.dtype) {
            return NACHO_ERR_INVALID_ARGUMENT;
        }
        if (clip && ((t.out_dtype != t.dtype && t.out_dtype != NACHO_F32) ||
                     (t.size > 0 && (!t.out || !element_aligned(t.out, item_of(t.out_dtype)))))) {
            return NACHO_ERR_INVALID_ARGUMENT;
        }
        *held += t.size > 0;
        *chunks += t.size / kChunk + (t.size % kChunk > 0);
        if (*chunks > dense::kMostGroups) return NACHO_ERR_INDEX_OVERFLOW;
    }
    return NACHO_OK;
}

// Calls f(table, tensors before) with the tensors that have elements, kTensors at a time.
template <typename F>
int each_table(const nacho_gradient *tensors, int64_t count, F f) {
    Table t;
    t.count = 0;
    int64_t before = 0;
    unsigned chunk = 0;
    for (int64_t i = 0; i < count; ++i) {
        const nacho_gradient &x = tensors[i];
        if (x.size > 0) {
            t.tensors[t.count++] = {x.data, x.out, x.size, chunk,
                                    static_cast<unsigned char>(x.dtype),
                                    static_cast<unsigned char>(x.out_dtype)};
            chunk += static_cast<unsigned>((x.size + kChunk - 1) / kChunk);
        }
        if (t.count == kTensors || (i + 1 == count && t.count > 0)) {
            NACHO_TRY(f(t, before));
            before += t.count;
            t.count = 0;
        }
    }
    return NACHO_OK;
}

int run(const nacho_gradient *tensors, int64_t count, bool clip, float max_norm, float *norm,
        void *stream, const nacho_allocator *alloc) {
    int64_t held = 0, chunks = 0;
    if (clip && !(max_norm >= 0.0f)) return NACHO_ERR_INVALID_ARGUMENT;
    NACHO_TRY(check(tensors, count, clip, norm, &held, &chunks));
    Call call(stream, alloc);
    const hipStream_t s = call.stream();
    double *sums = nullptr;  // and the factor
    NACHO_TRY(call.scratch_n(static_cast<size_t>(chunks) + 1, &sums));
    float *factor = reinterpret_cast<float *>(sums + chunks);
    const unsigned grid = static_cast<unsigned>(chunks);
    auto with = [&](const auto &from) -> int {
        using Tensors = std::decay_t<decltype(from)>;
        if (grid > 0) {
            square_kernel<Tensors><<<grid, kThreads, 0, s>>>(from, sums);
            NACHO_TRY_HIP(hipGetLastError());
        }
        const bool few = clip && grid > 0 && chunks <= kFewChunks;
        if (!few) {
            norm_kernel<<<1, kThreads, 0, s>>>(sums, chunks, max_norm, norm, factor);
            NACHO_TRY_HIP(hipGetLastError());
        }
        if (clip && grid > 0) {
            const Limit limit{few ? nullptr : factor, sums, chunks, max_norm, norm};
            scale_kernel<Tensors><<<grid, kThreads, 0, s>>>(from, limit);
            NACHO_TRY_HIP(hipGetLastError());
        }
        return NACHO_OK;
    };
    if (held <= kTensors) {
        InArguments from;
        from.table.count = 0;
        NACHO_TRY(each_table(tensors, count, [&](const Table &t, int64_t) -> int {
            from.table = t;
            return NACHO_OK;
        }));
        return with(from);
    }
    Tensor *list = nullptr;
    NACHO_TRY(call.scratch_n(static_cast<size_t>(held), &list));
    NACHO_TRY(each_table(tensors, count, [&](const Table &t, int64_t before) -> int {
        table_kernel<<<1, dev::kWave, 0, s>>>(t, list + before);
        NACHO_TRY_HIP(hipGetLastError());
        return NACHO_OK;
    }));
    return with(InMemory{list, held});
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
