// The call path between the Python classes and the C ABI (include/nacho_hip.h), in C++: fills
// the operands' descriptors from their torch buffers, calls the entry point without the
// interpreter lock, and hands the result buffers to torch in place (no copy, released with
// nacho_free on the stream that produced them when the last tensor over them dies), as the
// reference's generated nanobind wrapper does (src/backend/generate_bindings.cpp:288-327,
// runtime/nacho_nb.h:37-58).
//
// The same steps through ctypes and __cuda_array_interface__ cost about 11 us more per call, as
// much as the kernels of a small merge: csr_add of 200 rows 25.2 -> 14.5 us.
//
// An operand that does not pass the checks here (lengths, devices) makes invoke() return None:
// the caller (ops.py) then raises the exception that names what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>
#include <vector>

#include "../../include/nacho_hip.h"

namespace {

enum Kind { kCsr = 0, kCoo, kCoo3, kDcsr, kCsf3, kCsr64, kScalar };
constexpr int kMaxBuffers = 6;

// Number of buffers and dimensions of a kind.
constexpr int kBuffers[] = {3, 3, 4, 4, 6, 3, 1};
constexpr int kDims[] = {2, 2, 3, 2, 3, 2, 0};

// Buffers that hold offsets: one entry more than the level above.
constexpr bool kIsOffsets[][kMaxBuffers] = {{true},        {false}, {false}, {false, true},
                                            {false, true, false, true}, {true}, {false}};

union Desc {
    nacho_csr csr;
    nacho_coo coo;
    nacho_coo3 coo3;
    nacho_dcsr dcsr;
    nacho_csf3 csf3;
    nacho_csr64 csr64;
    nacho_scalar scalar;
};

using FreeFn = int (*)(void *, void *);
FreeFn g_free = nullptr;

struct Buffer {
    void *ptr;
    int64_t n;
};

// The operand's buffers and dimensions; false when a buffer is not on `device`.
bool read_operand(int kind, PyObject *buffers, PyObject *dims, int device, Buffer *out,
                  int32_t *size) {
    if (!PyTuple_CheckExact(buffers) || PyTuple_GET_SIZE(buffers) != kBuffers[kind]) return false;
    if (!PyTuple_CheckExact(dims) || PyTuple_GET_SIZE(dims) != kDims[kind]) return false;
    for (int i = 0; i < kBuffers[kind]; ++i) {
        PyObject *o = PyTuple_GET_ITEM(buffers, i);
        if (!THPVariable_Check(o)) return false;
        const at::Tensor &t = THPVariable_Unpack(o);
        if (!t.is_cuda() || t.get_device() != device) return false;
        out[i].n = t.numel();
        out[i].ptr = out[i].n > 0 ? t.data_ptr() : nullptr;
    }
    for (int i = 0; i < kDims[kind]; ++i) {
        size[i] = static_cast<int32_t>(PyLong_AsLong(PyTuple_GET_ITEM(dims, i)));
    }
    return !PyErr_Occurred();
}

template <typename T>
T *as(const Buffer &b) {
    return static_cast<T *>(b.ptr);
}

// The operand's descriptor; false when its lengths do not fit each other or 32 bits.
bool fill(int kind, const Buffer *b, const int32_t *s, Desc *d) {
    for (int i = 0; i < kBuffers[kind]; ++i) {
        if (b[i].n > INT32_MAX + int64_t{kIsOffsets[kind][i]}) {
            return false;
        }
    }
    const int32_t n0 = static_cast<int32_t>(b[0].n), n1 = static_cast<int32_t>(b[1].n);
    switch (kind) {
        case kCsr:
            if (b[0].n != static_cast<int64_t>(s[0]) + 1 || b[2].n != n1) return false;
            d->csr = nacho_csr{s[0], s[1], as<int32_t>(b[0]), n1, as<int32_t>(b[1]),
                               as<float>(b[2]), n1};
            return true;
        case kCoo:
            if (b[1].n != n0 || b[2].n != n0) return false;
            d->coo = nacho_coo{s[0], s[1], n0, as<int32_t>(b[0]), n0, as<int32_t>(b[1]),
                               as<float>(b[2]), n0};
            return true;
        case kCoo3:
            if (b[1].n != n0 || b[2].n != n0 || b[3].n != n0) return false;
            d->coo3 = nacho_coo3{s[0], s[1], s[2], n0, as<int32_t>(b[0]), n0, as<int32_t>(b[1]),
                                 n0, as<int32_t>(b[2]), as<float>(b[3]), n0};
            return true;
        case kDcsr: {
            const int32_t n2 = static_cast<int32_t>(b[2].n);
            if (b[1].n != b[0].n + 1 || b[3].n != n2) return false;
            d->dcsr = nacho_dcsr{s[0], s[1], n0, as<int32_t>(b[0]), as<int32_t>(b[1]), n2,
                                 as<int32_t>(b[2]), as<float>(b[3]), n2};
            return true;
        }
        case kCsf3: {
            const int32_t n2 = static_cast<int32_t>(b[2].n), n4 = static_cast<int32_t>(b[4].n);
            if (b[1].n != b[0].n + 1 || b[3].n != b[2].n + 1 || b[5].n != n4) return false;
            d->csf3 = nacho_csf3{s[0], s[1], s[2], n0, as<int32_t>(b[0]), as<int32_t>(b[1]), n2,
                                 as<int32_t>(b[2]), as<int32_t>(b[3]), n4, as<int32_t>(b[4]),
                                 as<float>(b[5]), n4};
            return true;
        }
        default: return false;
    }
}

PyObject *wrap(void *ptr, int64_t n, at::ScalarType type, int device, void *stream) {
    const auto options = at::TensorOptions().dtype(type).device(at::kCUDA, device);
    if (!ptr) return THPVariable_Wrap(at::empty({0}, options));
    return THPVariable_Wrap(at::from_blob(
        ptr, {n}, [stream](void *p) { (void)g_free(p, stream); }, options,
        at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device))));
}

// The result's tensors and dimensions: ((tensor, ...), (size, ...)).
PyObject *adopt(int kind, const Desc &z, int device, void *stream) {
    const auto I = at::kInt, L = at::kLong, F = at::kFloat;
    struct {
        void *p;
        int64_t n;
        at::ScalarType t;
    } b[kMaxBuffers] = {};
    int64_t s[3] = {0, 0, 0};
    auto put = [&](int i, void *p, int64_t n, at::ScalarType t) { b[i] = {p, n, t}; };
    switch (kind) {
        case kCsr:
            put(0, z.csr.dim_j_offsets, z.csr.dim_i_size + int64_t{1}, I);
            put(1, z.csr.dim_j_indices, z.csr.dim_j_length, I);
            put(2, z.csr.values, z.csr.dim_j_length, F);
            s[0] = z.csr.dim_i_size, s[1] = z.csr.dim_j_size;
            break;
        case kCsr64:
            put(0, z.csr64.dim_j_offsets, z.csr64.dim_i_size + int64_t{1}, L);
            put(1, z.csr64.dim_j_indices, z.csr64.dim_j_length, I);
            put(2, z.csr64.values, z.csr64.dim_j_length, F);
            s[0] = z.csr64.dim_i_size, s[1] = z.csr64.dim_j_size;
            break;
        case kCoo:
            put(0, z.coo.dim_i_indices, z.coo.nnz, I);
            put(1, z.coo.dim_j_indices, z.coo.nnz, I);
            put(2, z.coo.values, z.coo.nnz, F);
            s[0] = z.coo.dim_i_size, s[1] = z.coo.dim_j_size;
            break;
        case kCoo3:
            put(0, z.coo3.dim_i_indices, z.coo3.nnz, I);
            put(1, z.coo3.dim_j_indices, z.coo3.nnz, I);
            put(2, z.coo3.dim_k_indices, z.coo3.nnz, I);
            put(3, z.coo3.values, z.coo3.nnz, F);
            s[0] = z.coo3.dim_i_size, s[1] = z.coo3.dim_j_size, s[2] = z.coo3.dim_k_size;
            break;
        case kDcsr:
            put(0, z.dcsr.dim_i_indices, z.dcsr.dim_i_length, I);
            put(1, z.dcsr.dim_j_offsets, z.dcsr.dim_i_length + int64_t{1}, I);
            put(2, z.dcsr.dim_j_indices, z.dcsr.dim_j_length, I);
            put(3, z.dcsr.values, z.dcsr.dim_j_length, F);
            s[0] = z.dcsr.dim_i_size, s[1] = z.dcsr.dim_j_size;
            break;
        case kCsf3:
            put(0, z.csf3.dim_i_indices, z.csf3.dim_i_length, I);
            put(1, z.csf3.dim_j_offsets, z.csf3.dim_i_length + int64_t{1}, I);
            put(2, z.csf3.dim_j_indices, z.csf3.dim_j_length, I);
            put(3, z.csf3.dim_k_offsets, z.csf3.dim_j_length + int64_t{1}, I);
            put(4, z.csf3.dim_k_indices, z.csf3.dim_k_length, I);
            put(5, z.csf3.values, z.csf3.dim_k_length, F);
            s[0] = z.csf3.dim_i_size, s[1] = z.csf3.dim_j_size, s[2] = z.csf3.dim_k_size;
            break;
        default: put(0, z.scalar.values, 1, F); break;
    }
    PyObject *tensors = PyTuple_New(kBuffers[kind]);
    PyObject *dims = tensors ? PyTuple_New(kDims[kind]) : nullptr;
    int done = 0;
    if (dims) {
        for (; done < kBuffers[kind]; ++done) {
            PyObject *t = wrap(b[done].p, b[done].n, b[done].t, device, stream);
            if (!t) break;
            PyTuple_SET_ITEM(tensors, done, t);
        }
        for (int i = 0; i < kDims[kind] && done == kBuffers[kind]; ++i) {
            PyObject *v = PyLong_FromLongLong(s[i]);
            if (!v) break;
            PyTuple_SET_ITEM(dims, i, v);
        }
    }
    if (done != kBuffers[kind] || PyErr_Occurred()) {  // out of memory
        for (int i = done; i < kBuffers[kind]; ++i) {
            if (b[i].p) (void)g_free(b[i].p, stream);
        }
        Py_XDECREF(tensors);
        Py_XDECREF(dims);
        return nullptr;
    }
    return Py_BuildValue("NN", tensors, dims);
}

// invoke(entry, result_kind, num_blocks, threads_per_block, stream, device,
//        kind, buffers, dims, kind, buffers, dims[, kind, buffers, dims])
//   -> ((tensor, ...), (size, ...)), an int error code, or None
PyObject *invoke(PyObject *, PyObject *const *args, Py_ssize_t n) {
    const int operands = static_cast<int>((n - 6) / 3);
    if (n != 6 + 3 * operands || operands < 2 || operands > 3) {
        PyErr_SetString(PyExc_TypeError, "invoke: two or three operands");
        return nullptr;
    }
    void *entry = PyLong_AsVoidPtr(args[0]);
    const long kind = PyLong_AsLong(args[1]);
    const int32_t nb = static_cast<int32_t>(PyLong_AsUnsignedLongLongMask(args[2]));
    const int32_t tpb = static_cast<int32_t>(PyLong_AsUnsignedLongLongMask(args[3]));
    void *stream = PyLong_AsVoidPtr(args[4]);
    const int device = static_cast<int>(PyLong_AsLong(args[5]));
    if (PyErr_Occurred()) return nullptr;
    if (!entry || !g_free || kind < kCsr || kind > kScalar) {
        PyErr_SetString(PyExc_ValueError, "invoke: no such entry point or result");
        return nullptr;
    }
    try {
        Desc d[3], z;
        for (int i = 0; i < operands; ++i) {
            const long k = PyLong_AsLong(args[6 + 3 * i]);
            Buffer b[kMaxBuffers];
            int32_t s[3];
            if (k < kCsr || k > kCsf3 ||
                !read_operand(static_cast<int>(k), args[7 + 3 * i], args[8 + 3 * i], device, b, s) ||
                !fill(static_cast<int>(k), b, s, &d[i])) {
                PyErr_Clear();
                Py_RETURN_NONE;
            }
        }
        int rc = 0;
        std::string failure;  // an exception must not pass the point where the lock is taken again
        Py_BEGIN_ALLOW_THREADS
        try {
            if (operands == 2) {
                using Fn = int (*)(const void *, const void *, void *, int32_t, int32_t, void *,
                                   const nacho_allocator *);
                rc = reinterpret_cast<Fn>(entry)(&d[0], &d[1], &z, nb, tpb, stream, nullptr);
            } else {
                using Fn = int (*)(const void *, const void *, const void *, void *, int32_t,
                                   int32_t, void *, const nacho_allocator *);
                rc = reinterpret_cast<Fn>(entry)(&d[0], &d[1], &d[2], &z, nb, tpb, stream,
                                                 nullptr);
            }
        } catch (const std::exception &e) {
            failure = std::string("the entry point threw: ") + e.what();
        }
        Py_END_ALLOW_THREADS
        if (!failure.empty()) {
            PyErr_SetString(PyExc_RuntimeError, failure.c_str());
            return nullptr;
        }
        if (rc != 0) return PyLong_FromLong(rc);
        return adopt(static_cast<int>(kind), z, device, stream);
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

// ---- dense rows through computed structure ----------------------------------------------
//
// Results and scratch are torch tensors here (the sizes are known before the call, and torch's
// allocator may be used in a graph capture).  A tensor whose rows are not whole 16-byte pieces
// apart is copied into one first.

// Scratch from torch's allocator, held until the call's kernels are queued.
struct Scratch {
    std::vector<at::Tensor> held;
    at::TensorOptions options;
    nacho_allocator allocator;

    explicit Scratch(int device)
        : options(at::TensorOptions().dtype(at::kByte).device(
              at::kCUDA, static_cast<c10::DeviceIndex>(device))),
          allocator{this, &allocate, &release} {}

    static void *allocate(void *ctx, size_t bytes, void *) {
        Scratch *s = static_cast<Scratch *>(ctx);
        try {
            s->held.push_back(at::empty({static_cast<int64_t>(bytes)}, s->options));
            return s->held.back().data_ptr();
        } catch (const std::exception &) {
            return nullptr;  // the entry point reports it
        }
    }
    static void release(void *, void *, void *) {}  // with the call
};

// Thrown by a check that fails: the caller then raises the exception that names the reason.
struct Refused {};

void need(bool ok) {
    if (!ok) throw Refused();
}

int type_code(at::ScalarType t) {
    need(t == at::kFloat || t == at::kHalf || t == at::kBFloat16);
    return t == at::kFloat ? NACHO_F32 : t == at::kHalf ? NACHO_F16 : NACHO_BF16;
}

at::Tensor tensor(PyObject *o, int device, int64_t dim) {
    need(THPVariable_Check(o));
    const at::Tensor &t = THPVariable_Unpack(o);
    need(t.is_cuda() && t.get_device() == device && t.dim() == dim);
    return t;
}

at::Tensor tensor(PyObject *o, int device, int64_t dim, at::ScalarType type) {
    at::Tensor t = tensor(o, device, dim);
    need(t.scalar_type() == type);
    return t;
}

// The descriptor of a [batch, row, head, dim] tensor; `t` becomes a copy where it has to.
nacho_heads heads(at::Tensor &t) {
    const int64_t per = 16 / static_cast<int64_t>(t.element_size());
    bool ok = (t.stride(3) == 1 || t.size(3) == 1) &&
              reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) % per == 0);
    ok = ok && (t.size(1) <= 1 || t.stride(1) * t.element_size() <= NACHO_MAX_ROW_BYTES);
    if (!ok) t = t.clone(at::MemoryFormat::Contiguous);
    auto stride = [&](int i) { return t.size(i) <= 1 ? int64_t{0} : t.stride(i); };
    return nacho_heads{t.numel() > 0 ? t.data_ptr() : nullptr, stride(0), stride(1), stride(2)};
}

int32_t size32(int64_t n) {
    need(n >= 0 && n <= INT32_MAX);
    return static_cast<int32_t>(n);
}

// Contiguous int32 ids, and the sequences' lengths (None: null).
const int32_t *lengths_of(PyObject *o, int device, int64_t batch, at::Tensor &keep) {
    if (o == Py_None) return nullptr;
    keep = tensor(o, device, 1, at::kInt).contiguous();
    need(keep.size(0) == batch);
    return batch > 0 ? keep.data_ptr<int32_t>() : nullptr;
}

template <typename T>
T *data_or_null(const at::Tensor &t) {
    return t.numel() > 0 ? t.data_ptr<T>() : nullptr;
}

// Calls f(), an entry point, without the interpreter lock.  Throws what it throws.
template <typename F>
int unlocked(F f) {
    int rc = 0;
    std::exception_ptr failure;
    Py_BEGIN_ALLOW_THREADS
    try {
        rc = f();
    } catch (...) {
        failure = std::current_exception();
    }
    Py_END_ALLOW_THREADS
    if (failure) std::rethrow_exception(failure);
    return rc;
}

PyObject *tuple_of(std::initializer_list<at::Tensor> tensors) {
    PyObject *out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
    if (!out) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor &t : tensors) {
        PyObject *o = THPVariable_Wrap(t);
        if (!o) {
            Py_DECREF(out);
            return nullptr;
        }
        PyTuple_SET_ITEM(out, i++, o);
    }
    return out;
}

// Runs a call's body: a refused operand is None, an error code an int.
template <typename F>
PyObject *guarded(F body) {
    try {
        // (results have no history: autograd is the caller's)
        at::AutoDispatchBelowADInplaceOrView below;
        return body();
    } catch (const Refused &) {
        PyErr_Clear();
        Py_RETURN_NONE;
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
}

struct Where {
    void *entry, *stream;
    int device;
};

Where where(PyObject *const *args) {
    Where w{PyLong_AsVoidPtr(args[0]), PyLong_AsVoidPtr(args[1]),
            static_cast<int>(PyLong_AsLong(args[2]))};
    need(!PyErr_Occurred() && w.entry);
    return w;
}

int32_t int_of(PyObject *o) {
    const long v = PyLong_AsLong(o);
    need(!PyErr_Occurred() && v >= INT32_MIN && v <= INT32_MAX);
    return static_cast<int32_t>(v);
}

float float_of(PyObject *o) {
    const double v = PyFloat_AsDouble(o);
    need(!PyErr_Occurred());
    return static_cast<float>(v);
}

bool arguments(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return n == want;
}

// The attention's operands as tensors, kept alive, and as the C struct.
struct Attention {
    at::Tensor q, k, v, ids, lengths, out, lse, dout, dq, dk, dv;
    nacho_block_attention_args a{};

    // q, k, v, blocks, lengths, block, causal, scale
    Attention(PyObject *const *args, int device) {
        q = tensor(args[0], device, 4);
        const at::ScalarType type = q.scalar_type();
        k = tensor(args[1], device, 4, type);
        v = tensor(args[2], device, 4, type);
        ids = tensor(args[3], device, 4, at::kInt).contiguous();
        need(q.size(0) == k.size(0) && k.sizes() == v.sizes() && q.size(3) == k.size(3));
        need(ids.size(0) == q.size(0) && ids.size(1) == q.size(1) && ids.size(2) == k.size(2));
        a.dtype = type_code(type);
        a.batch = size32(q.size(0)), a.queries = size32(q.size(1)), a.keys = size32(k.size(1));
        a.q_heads = size32(q.size(2)), a.kv_heads = size32(k.size(2));
        a.head_dim = size32(q.size(3)), a.count = size32(ids.size(3));
        a.lengths = lengths_of(args[4], device, q.size(0), lengths);
        a.block = int_of(args[5]), a.causal = int_of(args[6]), a.scale = float_of(args[7]);
        a.blocks = data_or_null<int32_t>(ids);
        a.q = heads(q), a.k = heads(k), a.v = heads(v);
    }
};

using AttentionFn = int (*)(const nacho_block_attention_args *, void *, const nacho_allocator *);

// block_attention(entry, stream, device, q, k, v, blocks, lengths, block, causal, scale,
//                 want_lse) -> (out, lse) or (out,)
PyObject *block_attention(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (!arguments(n, 12)) return nullptr;
    return guarded([&]() -> PyObject * {
        const Where w = where(args);
        Attention t(args + 3, w.device);
        const bool want_lse = PyObject_IsTrue(args[11]) == 1;
        t.out = at::empty({t.a.batch, t.a.queries, t.a.q_heads, t.a.head_dim}, t.q.options());
        t.a.out = heads(t.out);
        if (want_lse) {
            t.lse = at::empty({t.a.batch, t.a.queries, t.a.q_heads},
                              t.q.options().dtype(at::kFloat));
            t.a.lse = data_or_null<float>(t.lse);
        }
        Scratch scratch(w.device);
        const int rc = unlocked([&] {
            return reinterpret_cast<AttentionFn>(w.entry)(&t.a, w.stream, &scratch.allocator);
        });
        if (rc != 0) return PyLong_FromLong(rc);
        return want_lse ? tuple_of({t.out, t.lse}) : tuple_of({t.out});
    });
}

// block_attention_backward(entry, stream, device, q, k, v, blocks, lengths, block, causal,
//                          scale, dout, out, lse) -> (dq, dk, dv)
PyObject *block_attention_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (!arguments(n, 14)) return nullptr;
    return guarded([&]() -> PyObject * {
        const Where w = where(args);
        Attention t(args + 3, w.device);
        const at::ScalarType type = t.q.scalar_type();
        t.dout = tensor(args[11], w.device, 4, type);
        t.out = tensor(args[12], w.device, 4, type);
        t.lse = tensor(args[13], w.device, 3, at::kFloat).contiguous();
        need(t.dout.sizes() == t.q.sizes() && t.out.sizes() == t.q.sizes());
        need(t.lse.size(0) == t.q.size(0) && t.lse.size(1) == t.q.size(1) &&
             t.lse.size(2) == t.q.size(2));
        t.dq = at::empty(t.q.sizes(), t.q.options(), at::MemoryFormat::Contiguous);
        t.dk = at::empty(t.k.sizes(), t.k.options(), at::MemoryFormat::Contiguous);
        t.dv = at::empty(t.v.sizes(), t.v.options(), at::MemoryFormat::Contiguous);
        t.a.out = heads(t.out), t.a.dout = heads(t.dout);
        t.a.dq = heads(t.dq), t.a.dk = heads(t.dk), t.a.dv = heads(t.dv);
        t.a.lse = data_or_null<float>(t.lse);
        Scratch scratch(w.device);
        const int rc = unlocked([&] {
            return reinterpret_cast<AttentionFn>(w.entry)(&t.a, w.stream, &scratch.allocator);
        });
        return rc != 0 ? PyLong_FromLong(rc) : tuple_of({t.dq, t.dk, t.dv});
    });
}

// block_means(entry, stream, device, k, lengths, block) -> means
PyObject *block_means(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (!arguments(n, 6)) return nullptr;
    return guarded([&]() -> PyObject * {
        const Where w = where(args);
        at::Tensor k = tensor(args[3], w.device, 4), lengths;
        const int type = type_code(k.scalar_type());
        const int32_t *len = lengths_of(args[4], w.device, k.size(0), lengths);
        const int32_t block = int_of(args[5]);
        need(block > 0);
        const int32_t batch = size32(k.size(0)), keys = size32(k.size(1));
        const int32_t count = size32(k.size(2)), dim = size32(k.size(3));
        at::Tensor out = at::empty({batch, (int64_t{keys} + block - 1) / block, count, dim},
                                   k.options().dtype(at::kFloat));
        const nacho_heads h = heads(k);
        const int rc = unlocked([&] {
            return reinterpret_cast<decltype(&nacho_block_means)>(w.entry)(
                type, batch, keys, count, dim, block, &h, len, data_or_null<float>(out), w.stream);
        });
        return rc != 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}

// block_scores(entry, stream, device, q, means, lengths, block, keys, causal, scale) -> scores
PyObject *block_scores(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (!arguments(n, 10)) return nullptr;
    return guarded([&]() -> PyObject * {
        const Where w = where(args);
        at::Tensor q = tensor(args[3], w.device, 4), lengths;
        const at::Tensor means = tensor(args[4], w.device, 4, at::kFloat).contiguous();
        const int type = type_code(q.scalar_type());
        const int32_t *len = lengths_of(args[5], w.device, q.size(0), lengths);
        const int32_t block = int_of(args[6]), keys = int_of(args[7]);
        need(block > 0 && keys >= 0 && means.size(0) == q.size(0) &&
             means.size(1) == (int64_t{keys} + block - 1) / block && means.size(3) == q.size(3));
        const int32_t batch = size32(q.size(0)), queries = size32(q.size(1));
        const int32_t kv = size32(means.size(2));
        at::Tensor out = at::empty({batch, queries, kv, means.size(1)},
                                   q.options().dtype(at::kFloat));
        const nacho_heads h = heads(q);
        const int32_t causal = int_of(args[8]);
        const float scale = float_of(args[9]);
        const int rc = unlocked([&] {
            return reinterpret_cast<decltype(&nacho_block_scores)>(w.entry)(
                type, batch, queries, keys, size32(q.size(2)), kv, size32(q.size(3)), block,
                causal, scale, &h, data_or_null<float>(means), len, data_or_null<float>(out),
                w.stream);
        });
        return rc != 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}

// block_select(entry, stream, device, scores, lengths, count, block, keys, causal, sink, local)
//   -> ids
PyObject *block_select(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (!arguments(n, 11)) return nullptr;
    return guarded([&]() -> PyObject * {
        const Where w = where(args);
        const at::Tensor scores = tensor(args[3], w.device, 4, at::kFloat).contiguous();
        at::Tensor lengths;
        const int32_t *len = lengths_of(args[4], w.device, scores.size(0), lengths);
        const int32_t count = int_of(args[5]), block = int_of(args[6]), keys = int_of(args[7]);
        need(count >= 0 && block > 0 && keys >= 0 &&
             scores.size(3) == (int64_t{keys} + block - 1) / block);
        const int32_t batch = size32(scores.size(0)), queries = size32(scores.size(1));
        const int32_t kv = size32(scores.size(2));
        at::Tensor out = at::empty({batch, queries, kv, count}, scores.options().dtype(at::kInt));
        const int32_t causal = int_of(args[8]), sink = int_of(args[9]), local = int_of(args[10]);
        const int rc = unlocked([&] {
            return reinterpret_cast<decltype(&nacho_block_select)>(w.entry)(
                batch, queries, kv, keys, block, count, sink, local, causal,
                data_or_null<float>(scores), len, data_or_null<int32_t>(out), w.stream);
        });
        return rc != 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}

// route(entry, stream, device, experts, n_experts) -> (pos, order, slot)
PyObject *route(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (!arguments(n, 5)) return nullptr;
    return guarded([&]() -> PyObject * {
        const Where w = where(args);
        const at::Tensor experts = tensor(args[3], w.device, 2).contiguous();
        const bool wide = experts.scalar_type() == at::kLong;
        need(wide || experts.scalar_type() == at::kInt);
        const int32_t n_experts = int_of(args[4]);
        need(n_experts >= 1);
        const int64_t tokens = experts.size(0);
        const int32_t per_token = size32(experts.size(1));
        const auto options = experts.options().dtype(at::kInt);
        at::Tensor pos = at::empty({int64_t{n_experts} + 1}, options);
        at::Tensor order = at::empty({experts.numel()}, options);
        at::Tensor slot = at::empty({tokens, per_token}, options);
        Scratch scratch(w.device);
        const int rc = unlocked([&] {
            return reinterpret_cast<decltype(&nacho_route)>(w.entry)(
                experts.numel() > 0 ? experts.data_ptr() : nullptr, wide ? 8 : 4, tokens,
                per_token, n_experts, pos.data_ptr<int32_t>(), data_or_null<int32_t>(order),
                data_or_null<int32_t>(slot), w.stream, &scratch.allocator);
        });
        return rc != 0 ? PyLong_FromLong(rc) : tuple_of({pos, order, slot});
    });
}

// A matrix of contiguous rows, and the elements between them.
at::Tensor rows_of(PyObject *o, int device, int64_t *stride) {
    at::Tensor t = tensor(o, device, 2);
    if (t.size(1) > 1 && t.stride(1) != 1) t = t.contiguous();
    *stride = t.size(0) > 1 ? t.stride(0) : t.size(1);
    return t;
}

void *rows_data(const at::Tensor &t) { return t.numel() > 0 ? t.data_ptr() : nullptr; }

// dispatch(entry, stream, device, x, pos, slot) -> rows
PyObject *dispatch(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (!arguments(n, 6)) return nullptr;
    return guarded([&]() -> PyObject * {
        const Where w = where(args);
        int64_t stride = 0;
        const at::Tensor x = rows_of(args[3], w.device, &stride);
        const int type = type_code(x.scalar_type());
        const at::Tensor pos = tensor(args[4], w.device, 1, at::kInt);
        const at::Tensor slot = tensor(args[5], w.device, 2, at::kInt);
        need(slot.size(0) == x.size(0));
        at::Tensor out = at::empty({slot.numel(), x.size(1)}, x.options());
        const int rc = unlocked([&] {
            return reinterpret_cast<decltype(&nacho_dispatch)>(w.entry)(
                type, x.size(0), size32(slot.size(1)), size32(pos.size(0) - 1), x.size(1),
                rows_data(x), stride, pos.data_ptr<int32_t>(), data_or_null<int32_t>(slot),
                rows_data(out), w.stream);
        });
        return rc != 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}

// combine(entry, stream, device, rows, weights or None, slot) -> out
PyObject *combine(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (!arguments(n, 6)) return nullptr;
    return guarded([&]() -> PyObject * {
        const Where w = where(args);
        int64_t stride = 0;
        const at::Tensor rows = rows_of(args[3], w.device, &stride);
        const int type = type_code(rows.scalar_type());
        const at::Tensor slot = tensor(args[5], w.device, 2, at::kInt);
        at::Tensor weights;
        if (args[4] != Py_None) {
            weights = tensor(args[4], w.device, 2, at::kFloat).contiguous();
            need(weights.sizes() == slot.sizes());
        }
        need(rows.size(0) == slot.numel());
        at::Tensor out = at::empty({slot.size(0), rows.size(1)}, rows.options());
        const int rc = unlocked([&] {
            return reinterpret_cast<decltype(&nacho_combine)>(w.entry)(
                type, slot.size(0), size32(slot.size(1)), rows.size(1), rows_data(rows), stride,
                weights.defined() ? data_or_null<float>(weights) : nullptr,
                data_or_null<int32_t>(slot), rows_data(out), w.stream);
        });
        return rc != 0 ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}

// combine_backward(entry, stream, device, rows, weights, pos, slot, dout) -> (drows, dweights)
PyObject *combine_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
    if (!arguments(n, 8)) return nullptr;
    return guarded([&]() -> PyObject * {
        const Where w = where(args);
        int64_t stride = 0, dout_stride = 0;
        const at::Tensor rows = rows_of(args[3], w.device, &stride);
        const int type = type_code(rows.scalar_type());
        const at::Tensor weights = tensor(args[4], w.device, 2, at::kFloat).contiguous();
        const at::Tensor pos = tensor(args[5], w.device, 1, at::kInt);
        const at::Tensor slot = tensor(args[6], w.device, 2, at::kInt);
        const at::Tensor dout = rows_of(args[7], w.device, &dout_stride);
        need(weights.sizes() == slot.sizes() && rows.size(0) == slot.numel() &&
             dout.size(0) == slot.size(0) && dout.size(1) == rows.size(1) &&
             dout.scalar_type() == rows.scalar_type());
        at::Tensor drows = at::empty({rows.size(0), rows.size(1)}, rows.options());
        at::Tensor dweights = at::empty({slot.size(0), slot.size(1)}, weights.options());
        const int rc = unlocked([&] {
            return reinterpret_cast<decltype(&nacho_combine_backward)>(w.entry)(
                type, slot.size(0), size32(slot.size(1)), size32(pos.size(0) - 1), rows.size(1),
                rows_data(rows), stride, data_or_null<float>(weights), pos.data_ptr<int32_t>(),
                data_or_null<int32_t>(slot), rows_data(dout), dout_stride, rows_data(drows),
                data_or_null<float>(dweights), w.stream);
        });
        return rc != 0 ? PyLong_FromLong(rc) : tuple_of({drows, dweights});
    });
}

// set_free(address of nacho_free)
PyObject *set_free(PyObject *, PyObject *arg) {
    void *p = PyLong_AsVoidPtr(arg);
    if (PyErr_Occurred()) return nullptr;
    g_free = reinterpret_cast<FreeFn>(p);
    Py_RETURN_NONE;
}

PyCFunction fast(PyObject *(*f)(PyObject *, PyObject *const *, Py_ssize_t)) {
    return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef g_methods[] = {
    {"invoke", fast(invoke), METH_FASTCALL,
     "Call a C entry point on torch buffers and adopt its result."},
    {"block_attention", fast(block_attention), METH_FASTCALL, "nacho_block_attention."},
    {"block_attention_backward", fast(block_attention_backward), METH_FASTCALL,
     "nacho_block_attention_backward."},
    {"block_means", fast(block_means), METH_FASTCALL, "nacho_block_means."},
    {"block_scores", fast(block_scores), METH_FASTCALL, "nacho_block_scores."},
    {"block_select", fast(block_select), METH_FASTCALL, "nacho_block_select."},
    {"route", fast(route), METH_FASTCALL, "nacho_route."},
    {"dispatch", fast(dispatch), METH_FASTCALL, "nacho_dispatch."},
    {"combine", fast(combine), METH_FASTCALL, "nacho_combine."},
    {"combine_backward", fast(combine_backward), METH_FASTCALL, "nacho_combine_backward."},
    {"set_free", set_free, METH_O, "Address of nacho_free."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_bridge", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bridge() { return PyModule_Create(&g_module); }
