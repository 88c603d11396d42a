// What the operators of language-model training (embedding.cu, block_norm.cu, distill.cu, recurrence.cu, logprobs.cu, adamw.cu) share: checks of their
// arguments, rows of strided tensors, workspaces, and wide accesses.
#pragma once

#include "context.h"

#include <cuda_fp16.h>

#include <initializer_list>
#include <tuple>

namespace b200 {

// Runs the body of an entry point on its context's device and turns what it throws into a status and a message.
template <typename Fn>
int guarded_operator(b200_ctx* ctx, Fn&& fn) {
    auto answer = [&](int status, const char* message) {
        if (ctx != nullptr) {
            std::lock_guard<std::mutex> lock(ctx->err_mu);
            ctx->last_error = message;
        }
        return status;
    };
    try {
        if (ctx != nullptr) {
            B200_CUDA_CHECK(cudaSetDevice(ctx->device));
            ctx->current_op = B200_OP_COUNT;  // (a profile's records of these launches belong to no node)
        }
        fn();
        return B200_OK;
    } catch (const Error& e) {
        return answer(e.status, e.message.c_str());
    } catch (const std::bad_alloc&) {
        return answer(B200_OUT_OF_MEMORY, "host allocation failed");
    } catch (const std::exception& e) {
        return answer(B200_INTERNAL_ERROR, e.what());
    }
}

// ---- arguments --------------------------------------------------------------

inline bool is_float(int dtype) { return dtype == B200_F32 || dtype == B200_F16; }
inline bool is_index(int dtype) { return dtype == B200_I32 || dtype == B200_I64; }

inline int64_t numel_of(const b200_tensor& t) {
    int64_t n = 1;
    for (int d = 0; d < t.ndim; ++d) n *= t.dims[d];
    return n;
}

// A tensor with a rank, extents and strides that can be: what every later check relies on.  The largest view reaches less than 2^62 bytes.
inline void check_tensor(const b200_tensor& t, const char* name) {
    const std::string who(name);
    const int64_t size = static_cast<int64_t>(dtype_size(t.dtype));
    if (size == 0) fail(B200_DTYPE_ERROR, who + ": unknown dtype " + std::to_string(t.dtype));
    if (t.ndim < 0 || t.ndim > kMaxDims) fail(B200_SHAPE_ERROR, who + ": rank " + std::to_string(t.ndim) + " is outside 0..4");
    double elements = 1, reach = 0;
    for (int d = 0; d < t.ndim; ++d) {
        if (t.dims[d] < 0) fail(B200_SHAPE_ERROR, who + ": negative extent");
        if (t.strides[d] % size != 0) fail(B200_NOT_IMPLEMENTED, who + ": byte stride is not a multiple of the element size");
        elements *= static_cast<double>(t.dims[d]);
        reach += static_cast<double>(t.dims[d]) * (t.strides[d] < 0 ? -static_cast<double>(t.strides[d]) : static_cast<double>(t.strides[d]));
    }
    if (elements >= 9.0e18 || reach >= 4.0e18) fail(B200_SHAPE_ERROR, who + ": extents or strides are too large");
    if (reinterpret_cast<uintptr_t>(t.data) % static_cast<uintptr_t>(size) != 0) fail(B200_INVALID_ARGUMENT, who + ": address is not aligned to its elements");
}

inline bool same_extents(const b200_tensor& a, const b200_tensor& b, int axes) {
    for (int d = 0; d < axes; ++d) {
        if (a.dims[d] != b.dims[d]) return false;
    }
    return true;
}

inline bool same_view(const b200_tensor& a, const b200_tensor& b) {
    if (a.data != b.data || a.dtype != b.dtype || a.ndim != b.ndim) return false;
    for (int d = 0; d < a.ndim; ++d) {
        if (a.dims[d] != b.dims[d] || (a.dims[d] > 1 && a.strides[d] != b.strides[d])) return false;
    }
    return true;
}

inline bool is_dense(const b200_tensor& t) {
    if (numel_of(t) == 0) return true;
    int64_t expected = static_cast<int64_t>(dtype_size(t.dtype));
    for (int d = t.ndim - 1; d >= 0; --d) {
        if (t.dims[d] != 1 && t.strides[d] != expected) return false;
        expected *= t.dims[d];
    }
    return true;
}

// Whether no element of a view lies on another: sorted by stride, each axis steps over everything below it.
inline bool elements_distinct(const b200_tensor& t) {
    if (numel_of(t) == 0) return true;
    bool used[kMaxDims] = {};
    int64_t end = static_cast<int64_t>(dtype_size(t.dtype));
    for (int k = 0; k < t.ndim; ++k) {
        int at = -1;
        for (int d = 0; d < t.ndim; ++d) {
            if (used[d] || t.dims[d] <= 1) continue;
            if (at < 0 || std::abs(t.strides[d]) < std::abs(t.strides[at])) at = d;
        }
        if (at < 0) break;
        used[at] = true;
        const int64_t step = std::abs(t.strides[at]);
        if (step < end) return false;
        end += step * (t.dims[at] - 1);
    }
    return true;
}

// Rows of a tensor of rank 1 to 3: row r starts at base + (r / inner) * outer_stride + (r % inner) * inner_stride, in bytes.
struct RowsArg {
    char* base;
    int64_t outer, step;
};

// The leading extents that every tensor of rows in a call shares.
struct RowShape {
    int64_t rows = 1, outer = 1, inner = 1;
};

inline RowShape row_shape(const b200_tensor& t, int axes) {
    RowShape s;
    if (axes >= 1) s.inner = t.dims[axes - 1];
    if (axes >= 2) s.outer = t.dims[axes - 2];
    s.rows = s.outer * s.inner;
    return s;
}

// `axes`: how many of the tensor's axes stand in front of its rows.
inline RowsArg rows_arg(const b200_tensor& t, int axes) {
    RowsArg r;
    r.base = static_cast<char*>(t.data);
    r.step = axes >= 1 && t.dims[axes - 1] > 1 ? t.strides[axes - 1] : 0;
    r.outer = axes >= 2 && t.dims[axes - 2] > 1 ? t.strides[axes - 2] : 0;
    return r;
}

// Whether rows can be read and written eight elements at a time (load8, store8), given that their width is a multiple of eight.
inline bool aligned_rows(const RowsArg& r, int dtype) {
    const int64_t bytes = 8 * static_cast<int64_t>(dtype_size(dtype));
    return r.base == nullptr || (reinterpret_cast<uintptr_t>(r.base) % static_cast<uintptr_t>(bytes) == 0 && r.outer % bytes == 0 && r.step % bytes == 0);
}

inline void check_rows(const b200_tensor& t, const char* name) {
    check_tensor(t, name);
    if (t.ndim < 1 || t.ndim > 3) fail(B200_SHAPE_ERROR, std::string(name) + ": rank " + std::to_string(t.ndim) + " is outside 1..3");
    const int64_t width = t.dims[t.ndim - 1];
    if (numel_of(t) != 0 && width > 1 && t.strides[t.ndim - 1] != static_cast<int64_t>(dtype_size(t.dtype))) {
        fail(B200_NOT_IMPLEMENTED, std::string(name) + ": the last axis has no unit stride");
    }
    if (numel_of(t) != 0 && t.data == nullptr) fail(B200_INVALID_ARGUMENT, std::string(name) + " has no storage");
    const RowShape s = row_shape(t, t.ndim - 1);
    if (s.rows >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, std::string(name) + ": more than 2^31 - 1 rows");
}

// Whether a tensor that a call can do without is not there: no storage.  (One of no elements has none either, and still says what its extents are.)
inline bool is_absent(const b200_tensor& t, const char* name) {
    if (t.data != nullptr) return false;
    if (t.ndim == 0) return true;
    check_tensor(t, name);
    return numel_of(t) != 0;
}

// Whether two views may have an element in common.  Ranges of addresses that do not meet settle it; where they do (columns of one
// buffer, say), every run of consecutive elements of a view starts at its address plus a multiple of g, the greatest common divisor of all strides
// between runs: runs whose places modulo g do not meet never meet.
inline bool may_share(const b200_tensor& x, const b200_tensor& y) {
    if (!overlap(x, y)) return false;
    auto gcd = [](int64_t a, int64_t b) {
        a = std::abs(a), b = std::abs(b);
        while (b != 0) {
            const int64_t r = a % b;
            a = b, b = r;
        }
        return a;
    };
    int64_t g = 0, run[2];
    const b200_tensor* both[2] = {&x, &y};
    for (int k = 0; k < 2; ++k) {
        const b200_tensor& t = *both[k];
        run[k] = static_cast<int64_t>(dtype_size(t.dtype));
        for (int d = t.ndim - 1; d >= 0; --d) {
            if (t.dims[d] <= 1) continue;
            if (d == t.ndim - 1 && t.strides[d] == run[k]) run[k] *= t.dims[d];
            else g = gcd(g, t.strides[d]);
        }
    }
    if (g == 0) return true;
    const int64_t apart = static_cast<const char*>(y.data) - static_cast<const char*>(x.data);
    const int64_t place = ((apart % g) + g) % g;
    return !(place >= run[0] && place + run[1] <= g);
}

// What a forward call leaves for its backward: four floats for each row.
inline void check_stats(const b200_tensor& t, int64_t rows) {
    check_tensor(t, "stats");
    if (t.dtype != B200_F32) fail(B200_DTYPE_ERROR, "stats are F32");
    if (t.ndim != 2 || t.dims[0] != rows || t.dims[1] != 4 || !is_dense(t) || reinterpret_cast<uintptr_t>(t.data) % 16 != 0) {
        fail(B200_SHAPE_ERROR, "stats: not [rows, 4], dense and 16-byte aligned");
    }
}

struct Named {
    const b200_tensor* t;
    const char* name;
};

// Every result's elements are its own, and lie on no other tensor's: on a tensor of `exact` only where the two are the same view.
inline void check_results(std::initializer_list<Named> results, std::initializer_list<Named> inputs, std::initializer_list<Named> exact) {
    for (const Named* r = results.begin(); r != results.end(); ++r) {
        if (r->t->data == nullptr) continue;
        const std::string who(r->name);
        if (!elements_distinct(*r->t)) fail(B200_INVALID_ARGUMENT, who + ": a result's elements lie on one another");
        for (const Named* o = results.begin(); o != r; ++o) {
            if (may_share(*r->t, *o->t)) fail(B200_INVALID_ARGUMENT, who + " overlaps " + o->name);
        }
        for (const Named& i : inputs) {
            if (may_share(*r->t, *i.t)) fail(B200_INVALID_ARGUMENT, who + " overlaps " + i.name);
        }
        for (const Named& i : exact) {
            if (may_share(*r->t, *i.t) && !same_view(*r->t, *i.t)) fail(B200_INVALID_ARGUMENT, who + " overlaps " + i.name + " without being the same view");
        }
    }
}

// What b200_compute does before it queues a node: the tensors' pending all-reduces come first.
inline void wait_for_tensors(b200_ctx* ctx, std::initializer_list<const b200_tensor*> tensors) {
    if (!dist_has_pending(ctx)) return;
    for (const b200_tensor* t : tensors) {
        if (t->data == nullptr || numel_of(*t) == 0) continue;
        const char* lo = static_cast<const char*>(t->data);
        const char* hi = lo + dtype_size(t->dtype);
        for (int d = 0; d < t->ndim; ++d) {
            const int64_t reach = (t->dims[d] - 1) * t->strides[d];
            (reach < 0 ? lo : hi) += reach;
        }
        dist_wait_range(ctx, lo, hi);
    }
}

// A caller's workspace, where a call needs one of `need` bytes.
inline void check_workspace(const void* workspace, size_t have, size_t need) {
    if (need == 0 || workspace == nullptr) return;
    if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) fail(B200_INVALID_ARGUMENT, "workspace is not 256-byte aligned");
    if (have < need) fail(B200_INVALID_ARGUMENT, "workspace has " + std::to_string(have) + " bytes, " + std::to_string(need) + " are needed");
}

// The caller's workspace (checked), or the context's own, grown where it has to be.  A graph of the caller's would go on writing to the context's after a later call had
// moved it, and beside whatever else uses it: a call that is captured brings its own.
inline char* operator_workspace(b200_ctx* ctx, void* workspace, size_t need) {
    if (need == 0) return nullptr;
    if (workspace != nullptr) return static_cast<char*>(workspace);
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    B200_CUDA_CHECK(cudaStreamIsCapturing(ctx->stream, &status));
    if (status != cudaStreamCaptureStatusNone) fail(B200_INVALID_ARGUMENT, "a call that is captured into a graph needs a workspace of the caller's");
    return static_cast<char*>(ctx->ensure_workspace(need));
}

// A caller's workspace as a tensor, so that results are checked against it too.
inline b200_tensor workspace_tensor(void* workspace, size_t bytes) {
    b200_tensor t{};
    t.data = bytes != 0 ? workspace : nullptr;
    t.ndim = 1;
    t.dims[0] = static_cast<int64_t>(bytes);
    t.strides[0] = 1;
    t.dtype = B200_BOOL;
    return t;
}

// What a call asks of its arguments, without a context: throws Error where it would be refused.  Nothing is asked of the device, which may not be there, or not be
// begun with yet, unless an argument that comes from one needs it: a workspace, or rows beyond 2^28.
void check_embedding_call(const b200_embedding_args& a, bool backward);
void check_block_norm(const b200_block_norm_args& a);
void check_block_norm_backward(const b200_block_norm_grad_args& a);
void check_distill_loss(const b200_distill_args& a, bool forward);
void check_gated_recurrence(const b200_recurrence_args& a);
void check_gated_recurrence_backward(const b200_recurrence_grad_args& a);
void check_token_logprobs(const b200_token_logprobs_args& a, bool forward);
void check_adamw(const b200_adamw_args& a);

// How many blocks of a kernel an SM of the current device holds at once; allows the kernel that much shared memory.
inline int blocks_at_once(const void* kernel, int threads, size_t shared) {
    struct Key {
        const void* kernel;
        int threads;
        size_t shared;
        int device;
        bool operator<(const Key& o) const { return std::tie(kernel, threads, shared, device) < std::tie(o.kernel, o.threads, o.shared, o.device); }
    };
    static std::mutex mutex;
    static std::map<Key, int> known;
    static std::map<std::pair<const void*, int>, size_t> allowed;
    int dev = 0;
    B200_CUDA_CHECK(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mutex);
    int& n = known[Key{kernel, threads, shared, dev}];
    if (n == 0) {
        size_t& most = allowed[{kernel, dev}];  // (never lowered: a call of the larger size may come again, and finds its answer here)
        if (shared > most) {
            B200_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared)));
            most = shared;
        }
        int found = 0;
        B200_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&found, kernel, threads, shared));
        if (found < 1) fail(B200_INTERNAL_ERROR, "a kernel does not fit on an SM");
        n = found;
    }
    return n;
}

// ---- device side ------------------------------------------------------------

#ifdef __CUDACC__

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// Eight elements of a row as they lie in memory: 16 bytes of F16 or 32 of F32, moved in one access of that width and alignment.
template <typename T>
struct Raw8;
template <>
struct Raw8<__half> {
    uint4 a;
};
template <>
struct Raw8<float> {
    float a[8];
};

__device__ __forceinline__ void load8(Raw8<__half>& r, const __half* p) { r.a = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void load8(Raw8<float>& r, const float* p) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(r.a[0]), "=f"(r.a[1]), "=f"(r.a[2]), "=f"(r.a[3]), "=f"(r.a[4]), "=f"(r.a[5]), "=f"(r.a[6]), "=f"(r.a[7])
                 : "l"(__cvta_generic_to_global(p))
                 : "memory");
}

__device__ __forceinline__ void unpack8(const Raw8<__half>& r, float (&x)[8]) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = r.a[i];
}

__device__ __forceinline__ void store8(__half* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(__cvta_generic_to_global(p)), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
                 "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
}

// Arithmetic on eight values, two to an instruction.
__device__ __forceinline__ void fma_pair(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ void mul_pair(float& d0, float& d1, float a0, float a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
__device__ __forceinline__ void add_pair(float& d0, float& d1, float a0, float a1, float b0, float b1) {
    asm("{\n\t.reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
// d = a * b + c, of eight; of one b; of one b and one c
__device__ __forceinline__ void fma8(float (&d)[8], const float (&a)[8], const float (&b)[8], const float (&c)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) fma_pair(d[i], d[i + 1], a[i], a[i + 1], b[i], b[i + 1], c[i], c[i + 1]);
}
__device__ __forceinline__ void fma8(float (&d)[8], const float (&a)[8], float b, const float (&c)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) fma_pair(d[i], d[i + 1], a[i], a[i + 1], b, b, c[i], c[i + 1]);
}
__device__ __forceinline__ void fma8(float (&d)[8], const float (&a)[8], float b, float c) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) fma_pair(d[i], d[i + 1], a[i], a[i + 1], b, b, c, c);
}
__device__ __forceinline__ void mul8(float (&d)[8], const float (&a)[8], const float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) mul_pair(d[i], d[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
}
__device__ __forceinline__ void mul8(float (&d)[8], const float (&a)[8], float b) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) mul_pair(d[i], d[i + 1], a[i], a[i + 1], b, b);
}
__device__ __forceinline__ void add8(float (&d)[8], const float (&a)[8], const float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) add_pair(d[i], d[i + 1], a[i], a[i + 1], b[i], b[i + 1]);
}
__device__ __forceinline__ void add8(float (&d)[8], const float (&a)[8], float b) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) add_pair(d[i], d[i + 1], a[i], a[i + 1], b, b);
}
// s += a * b, and s += a, in two sums
__device__ __forceinline__ void dot8(float2& s, const float (&a)[8], const float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) fma_pair(s.x, s.y, a[i], a[i + 1], b[i], b[i + 1], s.x, s.y);
}
__device__ __forceinline__ void sum8(float2& s, const float (&a)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) add_pair(s.x, s.y, s.x, s.y, a[i], a[i + 1]);
}

// Eight columns of a row, from `first` on, for thread t of `threads` that share the row: eight neighbours where WIDE (rows of whole pieces, aligned),
// else one of each eight stretches of `threads` neighbours.
template <bool WIDE>
__device__ __forceinline__ int piece_column(int e, int t, int threads) {
    return WIDE ? t * 8 + e : e * threads + t;
}

template <typename T, bool WIDE>
struct Piece {
    Raw8<T> raw;
    __device__ __forceinline__ void load(const char* row, int first, int t, int threads, int width) {
        raw = {};
        if (first + t * 8 < width) load8(raw, reinterpret_cast<const T*>(row) + first + t * 8);
    }
    __device__ __forceinline__ void clear() { raw = {}; }
    __device__ __forceinline__ void get(float (&x)[8]) const { unpack8(raw, x); }
};
template <typename T>
struct Piece<T, false> {
    T raw[8];
    __device__ __forceinline__ void load(const char* row, int first, int t, int threads, int width) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = first + piece_column<false>(e, t, threads);
            raw[e] = c < width ? reinterpret_cast<const T*>(row)[c] : from_float<T>(0.f);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[e] = from_float<T>(0.f);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to_float(raw[e]);
    }
};

template <typename T, bool WIDE>
__device__ __forceinline__ void store_piece(char* row, const float (&x)[8], int first, int t, int threads, int width) {
    T* p = reinterpret_cast<T*>(row) + first;
    if constexpr (WIDE) {
        if (first + t * 8 < width) store8(p + t * 8, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = piece_column<false>(e, t, threads);
            if (first + c < width) p[c] = from_float<T>(x[e]);
        }
    }
}

// Where row r of a tensor lies.
__device__ __forceinline__ char* row_at(const RowsArg& t, const FastDiv& inner, uint32_t r) {
    uint32_t b, i;
    inner.divmod(r, b, i);
    return t.base + static_cast<int64_t>(b) * t.outer + static_cast<int64_t>(i) * t.step;
}

__device__ __forceinline__ int64_t load_index(const void* p, bool wide) {
    return wide ? *static_cast<const int64_t*>(p) : static_cast<int64_t>(*static_cast<const int32_t*>(p));
}

#endif  // __CUDACC__

}  // namespace b200
