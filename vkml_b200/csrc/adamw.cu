// One AdamW step over many tensors, states in F32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2        p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound by memory: 28 bytes to an element with everything in F32, 14 to 18 with 8-bit states.  The tensors' addresses travel in the launch's parameters, some
// hundreds at a time, so that a step over all of a model's tensors is one launch and uploads nothing.  A warp takes 256 elements, which are a block of 8-bit
// states: their largest is a reduction in the warp, and a state is read, updated, scaled and written without leaving its registers.  176 M parameters in F32: 720 us, 6.8
// TB/s; 118 M with 8-bit states, F16 gradients and F16 copies: 328 to 347 us, 5.5 to 5.8 TB/s, where the instructions of a state's rounding are what is left.
//
// An 8-bit state's change in a step is mostly smaller than half a step of its byte (v moves by a thousandth, a byte's step is 6 to 12 %): rounded to the nearest,
// it would stay where it is.  Each is rounded up or down by random bits instead, whose mean is what was computed.  The root of v is what is kept: it has half
// of v's range in powers of two, and a byte covers 2^17 of them, as for m.
// (This file is compiled without joining multiplications and additions: the bytes are what the formulas give, operation by operation.)
#include "operators.cuh"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

namespace b200 {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;                // elements that share a scale: a warp's
constexpr int kRound = kThreads / 32 * kBlock;  // elements that a block of threads takes at once
constexpr int kMostRounds = 8;             // ... and how often, with 8-bit states: the next round's elements are on their way (8 a thread: 328 us in place of 369); half as often with F32
constexpr int kMostTensors = 384;          // of a launch: 32,764 bytes of parameters
constexpr int kFewTensors = 24;            // (fewer bytes go with a launch of few)

struct Tensor {
    float* param;
    const void* grad;
    void* first;
    void* second;
    float2* scales;  // null: F32 states
    __half* copy;
    int64_t n;
    float decay, lr_scale;
    uint32_t item;    // its first of the launch
    uint32_t number;  // in the caller's list
    uint32_t half_grad, wide;
};

struct Numbers {
    const float* lr_at;
    const int64_t* step_at;
    const float* scale_at;
    int64_t step;
    float lr, b1, rest1, b2, rest2, eps, scale, one;
    float log_b1, log_b2;                  // natural logarithms
    float inverse1, root_inverse2;         // 1 / (1 - b1^step), 1 / sqrt(1 - b2^step)
    uint32_t seed;
    int rounds;
};

template <int N>
struct Table {
    Numbers numbers;
    int count;
    Tensor t[N];
};

// ---- 8-bit states -----------------------------------------------------------

__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x6a09e667u;
    x = (x ^ (x >> 15)) * 0x3c6ef373u;
    return x ^ (x >> 16);
}

// The values of two bytes.
__device__ __forceinline__ float2 byte_values(uint32_t pair) {
    uint32_t h;
    asm("{\n\t.reg .b16 p;\n\tcvt.u16.u32 p, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, p;\n\t}" : "=r"(h) : "r"(pair));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// The byte of a size that is at most 448, in the upper 8 bits, up or down by 16 random bits, which lie in `noise` as 0x00rrrr80.  Times 2^-120 a float's exponent field is
// the byte's, and so are the leading bits of its fraction, subnormal ones too: adding below them carries into them.  `size`: that product, its sign aside.
__device__ __forceinline__ uint32_t byte_of(float size, uint32_t noise) { return min((__float_as_uint(size) << 4) + noise, 0x7effffffu); }
__device__ __forceinline__ uint32_t upper_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410); }
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a block's sizes are divided by, and its inverse; of a block that is zero, or not finite.
struct Scale {
    float scale, inverse;
    bool broken;
};
__device__ __forceinline__ Scale scale_of(uint32_t most_bits) {
    const float most = __uint_as_float(most_bits);
    Scale s;
    s.broken = most_bits >= 0x7f800000u;
    const bool some = most >= 0x1p-100f;
    s.scale = s.broken ? __uint_as_float(0x7fffffffu) : some ? most * (1.f / 448.f) : 0.f;
    s.inverse = some ? 1.f / most * 448.f : 0.f;
    return s;
}

// ---- the step ---------------------------------------------------------------

struct Step {
    float b1, rest1, b2, rest2, eps, scale, root_inverse2, keep, rate;
    // 1, as the launch's parameters have it: a + b is a multiply-add by it.  Products and sums of pairs are joined into multiply-adds by the assembler, whatever the
    // compiler is told (and so are those by a 1 that it sees), and the bytes would not be those of the formulas.
    float one;
    __device__ __forceinline__ void moments(const float (&grad)[8], float (&m)[8], float (&v)[8]) const {
        float g[8], t[8];
        mul8(g, grad, scale);
        mul8(t, g, rest1);
        mul8(m, m, b1);
        fma8(m, m, one, t);
        mul8(t, g, g);
        mul8(t, t, rest2);
        mul8(v, v, b2);
        fma8(v, v, one, t);
    }
    __device__ __forceinline__ void update(float (&p)[8], const float (&m)[8], const float (&root)[8]) const {
        float t[8];
        mul8(t, root, root_inverse2);
        add8(t, t, eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = fast_reciprocal(t[e]);
        mul8(t, t, m);
        mul8(t, t, -rate);
        mul8(p, p, keep);
        add8(p, p, t);
    }
};

// Eight elements of a lane: neighbours where the tensor's addresses allow it, else 32 apart.
template <bool WIDE, typename T>
__device__ __forceinline__ void load_values(float (&x)[8], const T* from, int64_t left, int lane) {
    if constexpr (WIDE) {
        Raw8<T> raw;
        load8(raw, from + lane * 8);
        unpack8(raw, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e * 32 + lane < left ? to_float(from[e * 32 + lane]) : 0.f;
    }
}
template <bool WIDE, typename T>
__device__ __forceinline__ void store_values(T* to, const float (&x)[8], int64_t left, int lane) {
    if constexpr (WIDE) {
        store8(to + lane * 8, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e * 32 + lane < left) to[e * 32 + lane] = from_float<T>(x[e]);
        }
    }
}
template <bool WIDE>
__device__ __forceinline__ void load_bytes(uint32_t (&c)[2], const uint8_t* from, int64_t left, int lane) {
    if constexpr (WIDE) {
        const uint2 w = *reinterpret_cast<const uint2*>(from + lane * 8);
        c[0] = w.x, c[1] = w.y;
    } else {
        c[0] = c[1] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e * 32 + lane < left) c[e / 4] |= static_cast<uint32_t>(from[e * 32 + lane]) << (e % 4 * 8);
        }
    }
}
template <bool WIDE>
__device__ __forceinline__ void store_bytes(uint8_t* to, const uint32_t (&c)[2], int64_t left, int lane) {
    if constexpr (WIDE) {
        *reinterpret_cast<uint2*>(to + lane * 8) = make_uint2(c[0], c[1]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e * 32 + lane < left) to[e * 32 + lane] = static_cast<uint8_t>(c[e / 4] >> (e % 4 * 8));
        }
    }
}
__device__ __forceinline__ void bytes_values(float (&x)[8], const uint32_t (&c)[2], float scale) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = byte_values(c[i / 2] >> (i % 2 * 16));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
    mul8(x, x, scale);
}

// What a lane has of 256 elements with 8-bit states, as it lies in memory.
struct RawBytes {
    Raw8<float> param, grad32;
    Raw8<__half> grad16;
    uint2 first, second;
    float2 scales;
    __device__ __forceinline__ void load(const Tensor& t, int64_t from, int lane) {
        const int64_t at = from + lane * 8;
        load8(param, t.param + at);
        if (t.half_grad) load8(grad16, static_cast<const __half*>(t.grad) + at);
        else load8(grad32, static_cast<const float*>(t.grad) + at);
        first = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.first) + at);
        second = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(t.second) + at);
        scales = t.scales[from / kBlock];
    }
};

// The step of 256 elements with 8-bit states: p, g and the bytes as they were.
template <bool WIDE>
__device__ __forceinline__ void step_bytes(const Tensor& t, const Step& s, uint32_t key, int64_t from, int lane, float (&p)[8], const float (&g)[8], uint32_t (&a)[2], uint32_t (&b)[2],
                                           float2 scales) {
    const int64_t left = t.n - from;
    float m[8], v[8];
    bytes_values(m, a, scales.x);
    bytes_values(v, b, scales.y);
    mul8(v, v, v);
    s.moments(g, m, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = sqrtf(v[e]);
    s.update(p, m, v);
    store_values<WIDE>(t.param + from, p, left, lane);
    if (t.copy != nullptr) store_values<WIDE>(t.copy + from, p, left, lane);
    float most_m = fabsf(m[0]), most_v = v[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) most_m = max_nan(most_m, fabsf(m[e])), most_v = max_nan(most_v, v[e]);
    const Scale sm = scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(most_m))), sv = scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(most_v)));
    // over the scale, times 2^-120: one product, where that factor is not subnormal (values up to 14336), else two
    float x[8], y[8];
    if (min(sm.inverse, sv.inverse) >= 0x1p-5f) {
        mul8(x, m, sm.inverse * 0x1p-120f);
        mul8(y, v, sv.inverse * 0x1p-120f);
    } else {
        mul8(x, m, sm.inverse);
        mul8(x, x, 0x1p-120f);
        mul8(y, v, sv.inverse);
        mul8(y, y, 0x1p-120f);
    }
    const uint32_t least = sv.inverse > 0.f ? 0x01000000u : 0u;
    uint32_t first[8], second[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t i = static_cast<uint32_t>(from) + static_cast<uint32_t>(WIDE ? lane * 8 + e : e * 32 + lane);
        const uint32_t bits = mix(key + i * 0x9e3779b9u);
        first[e] = byte_of(x[e], __byte_perm(bits, 0x80u, 0x7104)) | (__float_as_uint(m[e]) & 0x80000000u);
        second[e] = byte_of(y[e], __byte_perm(bits, 0x80u, 0x7324));
        if (v[e] > 0.f) second[e] = max(second[e], least);
    }
    a[0] = upper_bytes(first[0], first[1], first[2], first[3]), a[1] = upper_bytes(first[4], first[5], first[6], first[7]);
    b[0] = upper_bytes(second[0], second[1], second[2], second[3]), b[1] = upper_bytes(second[4], second[5], second[6], second[7]);
    if (sm.broken) a[0] = a[1] = 0x7f7f7f7fu;
    if (sv.broken) b[0] = b[1] = 0x7f7f7f7fu;
    store_bytes<WIDE>(static_cast<uint8_t*>(t.first) + from, a, left, lane);
    store_bytes<WIDE>(static_cast<uint8_t*>(t.second) + from, b, left, lane);
    if (lane == 0) t.scales[from / kBlock] = make_float2(sm.scale, sv.scale);
}
__device__ __forceinline__ void step_bytes(const Tensor& t, const Step& s, uint32_t key, int64_t from, int lane, const RawBytes& raw) {
    float p[8], g[8];
    unpack8(raw.param, p);
    if (t.half_grad) unpack8(raw.grad16, g);
    else unpack8(raw.grad32, g);
    uint32_t a[2] = {raw.first.x, raw.first.y}, b[2] = {raw.second.x, raw.second.y};
    step_bytes<true>(t, s, key, from, lane, p, g, a, b, raw.scales);
}

// 256 elements from element `from` on, or what is left of them.
template <bool WIDE, bool BYTES>
__device__ __forceinline__ void step_block(const Tensor& t, const Step& s, uint32_t key, int64_t from, int lane) {
    const int64_t left = t.n - from;
    float p[8], g[8], m[8], v[8];
    load_values<WIDE>(p, t.param + from, left, lane);
    if (t.half_grad) load_values<WIDE>(g, static_cast<const __half*>(t.grad) + from, left, lane);
    else load_values<WIDE>(g, static_cast<const float*>(t.grad) + from, left, lane);
    if (BYTES && t.scales != nullptr) {
        uint32_t a[2], b[2];
        load_bytes<WIDE>(a, static_cast<const uint8_t*>(t.first) + from, left, lane);
        load_bytes<WIDE>(b, static_cast<const uint8_t*>(t.second) + from, left, lane);
        step_bytes<WIDE>(t, s, key, from, lane, p, g, a, b, t.scales[from / kBlock]);
        return;
    }
    load_values<WIDE>(m, static_cast<const float*>(t.first) + from, left, lane);
    load_values<WIDE>(v, static_cast<const float*>(t.second) + from, left, lane);
    s.moments(g, m, v);
    store_values<WIDE>(static_cast<float*>(t.first) + from, m, left, lane);
    store_values<WIDE>(static_cast<float*>(t.second) + from, v, left, lane);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = sqrtf(v[e]);
    s.update(p, m, v);
    store_values<WIDE>(t.param + from, p, left, lane);
    if (t.copy != nullptr) store_values<WIDE>(t.copy + from, p, left, lane);
}

// BYTES: whether a tensor has 8-bit states.  (Without them four blocks fit on an SM: 176 M parameters 720 us, 730 with three.)
template <int N, bool BYTES>
__global__ void __launch_bounds__(kThreads, BYTES ? 3 : 4) adamw_kernel(const __grid_constant__ Table<N> k) {
    pdl_prologue();
    int lo = 0, hi = k.count;  // the tensor whose items this block's is one of
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (k.t[mid].item <= blockIdx.x) lo = mid;
        else hi = mid;
    }
    const Tensor& t = k.t[lo];
    const Numbers& n = k.numbers;
    Step s;
    s.b1 = n.b1, s.rest1 = n.rest1, s.b2 = n.b2, s.rest2 = n.rest2, s.eps = n.eps, s.scale = n.scale, s.one = n.one;
    float inverse1 = n.inverse1, lr = n.lr;
    int64_t step = n.step;
    s.root_inverse2 = n.root_inverse2;
    if (n.step_at != nullptr) {
        step = *n.step_at;
        if (step < 1) return;
        inverse1 = -1.f / expm1f(static_cast<float>(step) * n.log_b1);
        s.root_inverse2 = 1.f / sqrtf(-expm1f(static_cast<float>(step) * n.log_b2));
    }
    if (n.lr_at != nullptr) lr = *n.lr_at;
    if (n.scale_at != nullptr) {
        s.scale = s.scale * *n.scale_at;
        if (!isfinite(s.scale)) return;
    }
    lr = lr * t.lr_scale;
    s.keep = 1.f - lr * t.decay;
    s.rate = lr * inverse1;
    const uint32_t key = t.scales != nullptr ? mix(mix(mix(n.seed) + static_cast<uint32_t>(step)) + t.number) : 0u;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int64_t from = int64_t(blockIdx.x - t.item) * (n.rounds * kRound) + warp * kBlock;
    const int64_t whole = t.n / kBlock * kBlock, end = min(t.n, from - warp * kBlock + n.rounds * kRound);
    if (BYTES && t.wide && t.scales != nullptr) {  // whole blocks, the next one on its way
        const int64_t end_whole = min(whole, end);
        if (from < end_whole) {
            RawBytes raw;
            raw.load(t, from, lane);
#pragma unroll 1
            for (; from < end_whole; from += kRound) {
                const RawBytes now = raw;
                if (from + kRound < end_whole) raw.load(t, from + kRound, lane);
                step_bytes(t, s, key, from, lane, now);
            }
        }
    }
#pragma unroll 1
    for (; from < end; from += kRound) {
        if (t.wide && (!BYTES || t.scales == nullptr) && from < whole) step_block<true, false>(t, s, key, from, lane);
        else step_block<false, BYTES>(t, s, key, from, lane);
    }
}

// ---- arguments --------------------------------------------------------------

bool present(const b200_tensor& t) { return t.data != nullptr; }

void check_one(const b200_tensor& t, const char* name, int dtype) {
    if (!present(t)) return;
    check_tensor(t, name);
    if (t.dtype != dtype) fail(B200_DTYPE_ERROR, std::string(name) + " has another type");
    if (numel_of(t) != 1) fail(B200_SHAPE_ERROR, std::string(name) + ": not one element");
}

struct Range {
    const char *lo, *hi;
    bool written;
    bool operator<(const Range& o) const { return lo < o.lo; }
};

void check_numbers(const b200_adamw_args& a) {
    if (a.count < 0 || a.count >= (int64_t(1) << 31)) fail(B200_INVALID_ARGUMENT, "adamw: the number of tensors is below 0 or too large");
    if (a.count > 0 && a.tensors == nullptr) fail(B200_INVALID_ARGUMENT, "adamw: no tensors");
    check_one(a.lr_on_device, "lr_on_device", B200_F32);
    check_one(a.step_on_device, "step_on_device", B200_I64);
    check_one(a.scale_on_device, "scale_on_device", B200_F32);
    if (!(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1)) fail(B200_INVALID_ARGUMENT, "adamw: a beta is not in [0, 1)");
    if (!(a.eps >= 0x1p-126f) || std::isinf(a.eps)) fail(B200_INVALID_ARGUMENT, "adamw: eps is not a normal number above 0");
    if (!std::isfinite(a.lr) || !std::isfinite(a.grad_scale)) fail(B200_INVALID_ARGUMENT, "adamw: lr or grad_scale is not finite");
    if (a.step < 1) fail(B200_INVALID_ARGUMENT, "adamw: the step is below 1");
}

// The tensors' checks; what is written lies on nothing else of the call (sorted addresses: a neighbour shows it).
void check_tensors(const b200_adamw_args& a) {
    // Addresses are sorted kind by kind (each kind of a model's mostly lies in order) and then merged.
    std::vector<Range> kinds[7];
    auto add = [&](int kind, const b200_tensor& t, bool written) {
        const int64_t bytes = numel_of(t) * static_cast<int64_t>(dtype_size(t.dtype));
        if (present(t) && bytes != 0) kinds[kind].push_back({static_cast<const char*>(t.data), static_cast<const char*>(t.data) + bytes, written});
    };
    for (std::vector<Range>& k : kinds) k.reserve(static_cast<size_t>(a.count) + 3);
    // A tensor that is one of param's extents and strides, of its type, needs no other check than that of its address.
    auto alike = [](const b200_tensor& x, const b200_tensor& y) {
        return x.ndim == y.ndim && x.dtype == y.dtype && std::memcmp(x.dims, y.dims, sizeof(int64_t) * static_cast<size_t>(x.ndim)) == 0 &&
               std::memcmp(x.strides, y.strides, sizeof(int64_t) * static_cast<size_t>(x.ndim)) == 0 && reinterpret_cast<uintptr_t>(x.data) % 4 == 0;
    };
    for (int64_t i = 0; i < a.count; ++i) {
        const b200_adamw_tensor& t = a.tensors[i];
        auto refuse = [&](int status, const char* why) { fail(status, "adamw: tensor " + std::to_string(i) + ": " + why); };
        check_tensor(t.param, "param");
        if (t.param.dtype != B200_F32) refuse(B200_DTYPE_ERROR, "param is F32");
        const int64_t n = numel_of(t.param);
        const bool bytes = t.first.dtype == B200_I32;
        if (!is_dense(t.param)) refuse(B200_NOT_IMPLEMENTED, "a tensor is not dense");
        if (!alike(t.grad, t.param)) {
            check_tensor(t.grad, "grad");
            if (!is_float(t.grad.dtype)) refuse(B200_DTYPE_ERROR, "grad is F32 or F16");
            if (t.grad.ndim != t.param.ndim || !same_extents(t.grad, t.param, t.param.ndim)) refuse(B200_SHAPE_ERROR, "grad has not param's extents");
            if (!is_dense(t.grad)) refuse(B200_NOT_IMPLEMENTED, "a tensor is not dense");
        }
        if (t.first.dtype != t.second.dtype || (!bytes && t.first.dtype != B200_F32)) refuse(B200_DTYPE_ERROR, "first and second are both F32, or both I32 words of bytes");
        for (const b200_tensor* s : {&t.first, &t.second}) {
            if (alike(*s, t.param)) continue;
            check_tensor(*s, s == &t.first ? "first" : "second");
            if (bytes ? s->ndim != 1 || s->dims[0] != ceil_div(n, 4) : s->ndim != t.param.ndim || !same_extents(*s, t.param, t.param.ndim)) {
                refuse(B200_SHAPE_ERROR, "a state has not param's extents, or its number of bytes");
            }
            if (!is_dense(*s)) refuse(B200_NOT_IMPLEMENTED, "a tensor is not dense");
        }
        if (bytes ? n != 0 && !present(t.scales) : present(t.scales)) refuse(B200_INVALID_ARGUMENT, "scales go with 8-bit states, and only with them");
        if (present(t.scales)) {
            check_tensor(t.scales, "scales");
            if (t.scales.dtype != B200_F32) refuse(B200_DTYPE_ERROR, "scales are F32");
            if (t.scales.ndim != 2 || t.scales.dims[0] != ceil_div(n, kBlock) || t.scales.dims[1] != 2 || !is_dense(t.scales) || reinterpret_cast<uintptr_t>(t.scales.data) % 8 != 0) {
                refuse(B200_SHAPE_ERROR, "scales: not two for every 256 elements, dense and 8-byte aligned");
            }
        }
        if (present(t.copy)) {
            check_tensor(t.copy, "copy");
            if (t.copy.dtype != B200_F16) refuse(B200_DTYPE_ERROR, "copy is F16");
            if (t.copy.ndim != t.param.ndim || !same_extents(t.copy, t.param, t.param.ndim)) refuse(B200_SHAPE_ERROR, "copy has not param's extents");
            if (!is_dense(t.copy)) refuse(B200_NOT_IMPLEMENTED, "copy is not dense");
        }
        for (const b200_tensor* s : {&t.param, &t.grad, &t.first, &t.second}) {
            if (n != 0 && !present(*s)) refuse(B200_INVALID_ARGUMENT, "a tensor has no storage");
        }
        if (!(t.weight_decay >= 0.f) || std::isinf(t.weight_decay) || !std::isfinite(t.lr_scale)) refuse(B200_INVALID_ARGUMENT, "weight_decay or lr_scale is not finite, or weight_decay below 0");
        add(0, t.param, true);
        add(1, t.grad, false);
        add(2, t.first, true);
        add(3, t.second, true);
        if (present(t.scales)) add(4, t.scales, true);
        if (present(t.copy)) add(5, t.copy, true);
    }
    add(6, a.lr_on_device, false);
    add(6, a.step_on_device, false);
    add(6, a.scale_on_device, false);
    std::vector<Range> ranges, merged;
    for (std::vector<Range>& k : kinds) {
        if (!std::is_sorted(k.begin(), k.end())) std::sort(k.begin(), k.end());
        merged.resize(ranges.size() + k.size());
        std::merge(ranges.begin(), ranges.end(), k.begin(), k.end(), merged.begin());
        ranges.swap(merged);
    }
    const char* reach[2] = {nullptr, nullptr};  // the farthest end so far, of what is read and of what is written
    for (const Range& r : ranges) {
        if (r.lo < reach[1] || (r.written && r.lo < reach[0])) fail(B200_INVALID_ARGUMENT, "adamw: a tensor that is written overlaps another");
        reach[r.written] = std::max(reach[r.written], r.hi);
    }
}

template <int N, bool BYTES>
void launch_table(b200_ctx* ctx, const Numbers& numbers, const std::vector<Tensor>& tensors, size_t first, size_t count, uint32_t items) {
    static_assert(sizeof(Table<N>) <= 32764, "the launch's parameters");
    Table<N> table;
    table.numbers = numbers;
    table.count = static_cast<int>(count);
    std::copy_n(tensors.begin() + static_cast<std::ptrdiff_t>(first), count, table.t);
    launch_kernel(ctx, adamw_kernel<N, BYTES>, dim3(items), dim3(kThreads), 0, table);
    check_last_launch("adamw");
    ctx->count_launch();
}

void launch_adamw(b200_ctx* ctx, const b200_adamw_args& a) {
    check_numbers(a);
    check_tensors(a);
    Numbers k{};
    k.lr_at = static_cast<const float*>(a.lr_on_device.data);
    k.step_at = static_cast<const int64_t*>(a.step_on_device.data);
    k.scale_at = static_cast<const float*>(a.scale_on_device.data);
    k.step = a.step;
    k.lr = a.lr, k.eps = a.eps, k.scale = a.grad_scale, k.seed = a.seed, k.one = 1.f;
    k.b1 = static_cast<float>(a.beta1), k.rest1 = static_cast<float>(1 - a.beta1), k.log_b1 = static_cast<float>(std::log(a.beta1));
    k.b2 = static_cast<float>(a.beta2), k.rest2 = static_cast<float>(1 - a.beta2), k.log_b2 = static_cast<float>(std::log(a.beta2));
    k.inverse1 = static_cast<float>(1 / (1 - std::pow(a.beta1, static_cast<double>(a.step))));
    k.root_inverse2 = static_cast<float>(1 / std::sqrt(1 - std::pow(a.beta2, static_cast<double>(a.step))));
    std::vector<Tensor> tensors;
    tensors.reserve(static_cast<size_t>(a.count));
    for (int64_t i = 0; i < a.count; ++i) {
        const b200_adamw_tensor& s = a.tensors[i];
        if (numel_of(s.param) == 0) continue;
        if (dist_has_pending(ctx)) wait_for_tensors(ctx, {&s.param, &s.grad, &s.first, &s.second, &s.scales, &s.copy});
        Tensor t{};
        t.param = static_cast<float*>(s.param.data);
        t.grad = s.grad.data;
        t.first = s.first.data;
        t.second = s.second.data;
        t.scales = static_cast<float2*>(s.scales.data);
        t.copy = static_cast<__half*>(s.copy.data);
        t.n = numel_of(s.param);
        t.decay = s.weight_decay;
        t.lr_scale = s.lr_scale;
        t.number = static_cast<uint32_t>(i);
        t.half_grad = s.grad.dtype == B200_F16;
        auto on = [](const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
        const uintptr_t state = t.scales != nullptr ? 8 : 32;
        t.wide = on(t.param, 32) && on(t.grad, t.half_grad ? 16 : 32) && on(t.first, state) && on(t.second, state) && on(t.copy, 16);
        tensors.push_back(t);
    }
    wait_for_tensors(ctx, {&a.lr_on_device, &a.step_on_device, &a.scale_on_device});
    ProfScope scope(ctx, "adamw");
    // As many rounds to a block as leave 6 blocks for each SM: two waves of the three with 8-bit states that an SM holds, one and a half of the four without (until the most
    // rounds are reached: a large model has more of them); one round where there is little to do.
    int64_t all = 0;
    for (const Tensor& t : tensors) all += ceil_div(t.n, kRound);
    const bool any_bytes = std::any_of(tensors.begin(), tensors.end(), [](const Tensor& t) { return t.scales != nullptr; });
    k.rounds = static_cast<int>(std::clamp<int64_t>(all / (int64_t(sm_count()) * 6), 1, any_bytes ? kMostRounds : kMostRounds / 2));
    size_t done = 0;
    while (done < tensors.size()) {
        size_t count = 0;
        int64_t items = 0;
        while (done + count < tensors.size() && count < kMostTensors) {
            const int64_t more = ceil_div(tensors[done + count].n, int64_t(kRound) * k.rounds);
            if (items + more >= (int64_t(1) << 31)) break;
            tensors[done + count].item = static_cast<uint32_t>(items);
            items += more;
            ++count;
        }
        if (count == 0) fail(B200_SHAPE_ERROR, "adamw: a tensor is too large");
        const bool bytes = std::any_of(tensors.begin() + static_cast<std::ptrdiff_t>(done), tensors.begin() + static_cast<std::ptrdiff_t>(done + count), [](const Tensor& t) { return t.scales != nullptr; });
        auto go = [&](auto launch) { launch(ctx, k, tensors, done, count, static_cast<uint32_t>(items)); };
        if (count <= kFewTensors) go(bytes ? launch_table<kFewTensors, true> : launch_table<kFewTensors, false>);
        else go(bytes ? launch_table<kMostTensors, true> : launch_table<kMostTensors, false>);
        done += count;
    }
}

}  // namespace

void check_adamw(const b200_adamw_args& a) {
    check_numbers(a);
    check_tensors(a);
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_adamw(b200_ctx* ctx, const b200_adamw_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_adamw(ctx, *args); });
}

}  // extern "C"
