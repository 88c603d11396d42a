// Gated linear recurrences along a sequence, forward and backward.
//
//   h_t = a_t h_{t-1} + b_t,  out_t = h_t       sigmoid: a = s(gate), b = (1 - a) x       exp: a = e^gate, b = x
//   D_t = dout_t + a_{t+1} D_{t+1}              sigmoid: dx = (1 - a) D, dgate = a (1 - a) (h_{t-1} - x) D       exp: dx = D, dgate = a h_{t-1} D
//
// Each channel is by itself.  Bound by memory: gates, inputs and results once each (backward: three streams read, two written; h is computed again from the
// states that the forward pass leaves every 16 steps).
//
// A step is h + (b - d h) with d = 1 - a where a is above a half, and a h + b where it is not: a channel that remembers for thousands of steps multiplies as
// many decays just below 1, whose digits a product of rounded a's would lose (3e-5 of the result at a memory of 3000 steps), and one that forgets keeps none
// of a large state's rounding.
#include "operators.cuh"

#include <algorithm>
#include <cmath>

namespace b200 {
namespace {

constexpr int kSteps = B200_RECURRENCE_CHUNK;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float fast_reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A step's decay: -d where a = 1 - d is above a half (the sign bit says so, also of zero), else a.
__device__ __forceinline__ bool keeps(float c) { return __float_as_int(c) < 0; }
__device__ __forceinline__ float apply(float c, float h, float b) {
    const float t = fmaf(c, h, b);
    return keeps(c) ? h + t : t;
}
constexpr float kHold = -0.f;  // h stays

// c, and b / x, of a gate.
template <int KIND>
__device__ __forceinline__ float decay(float gate, float& input) {
    if constexpr (KIND == B200_GATES_SIGMOID) {
        const float z = fast_exp2(fabsf(gate) * -kLog2e);
        const float r = fast_reciprocal(1.f + z), s = z * r;  // s(|gate|) and s(-|gate|)
        const bool keep = gate > 0.f;
        input = keep ? s : r;
        return keep ? -s : s;
    } else {
        input = 1.f;
        // e^x - 1 by its series (the term left out is 2e-8 of it at |x| = 0.69), e^x itself beyond
        float e = fmaf(gate, 1.f / 362880.f, 1.f / 40320.f);
        e = fmaf(gate, e, 1.f / 5040.f);
        e = fmaf(gate, e, 1.f / 720.f);
        e = fmaf(gate, e, 1.f / 120.f);
        e = fmaf(gate, e, 1.f / 24.f);
        e = fmaf(gate, e, 1.f / 6.f);
        e = fmaf(gate, e, 0.5f);
        e = fmaf(gate * gate, e, gate);
        const bool near = fabsf(gate) < 0.6931f;
        // (a growing state keeps its digits in the same form, with a positive e: the sign bit tells the forms apart, so such a decay is given as a)
        return near && gate <= 0.f ? -fabsf(e) : near ? 1.f + e : fast_exp2(gate * kLog2e);
    }
}
// What dgate is (h_{t-1} - x) D times, or h_{t-1} D times; and dx is D times.
template <int KIND>
__device__ __forceinline__ void slopes(float c, float& gate, float& input) {
    if constexpr (KIND == B200_GATES_SIGMOID) {
        const float s = fabsf(c), r = 1.f - s;
        gate = s * r;
        input = keeps(c) ? s : r;
    } else {
        gate = keeps(c) ? 1.f + c : c;
        input = 1.f;
    }
}

struct Stream {
    char* base;
    int64_t batch, step;  // bytes
};

struct Args {
    Stream x, gate, out, dout, dx, dgate;  // (out: forward; the d's: backward)
    RowsArg initial, final_state;          // forward: read, written; backward: written (initial's gradient), read (final's)
    float* states;
    const char* lengths;
    int64_t lengths_step;
    bool wide_lengths;
    int64_t length;
    int batch, width, chunks;
    uint32_t* status;
};

template <typename T>
__device__ __forceinline__ T* at(const Stream& s, int b, int64_t t, int ch) {
    return reinterpret_cast<T*>(s.base + b * s.batch + t * s.step) + ch;
}

// Steps of sequence b.
__device__ __forceinline__ int64_t steps_of(const Args& k, int b) {
    if (k.lengths == nullptr) return k.length;
    const int64_t n = load_index(k.lengths + b * k.lengths_step, k.wide_lengths);
    if (n < 0 || n > k.length) atomicOr(k.status, kStatusIndexOutOfRange);
    return n < 0 ? 0 : n > k.length ? k.length : n;
}

// ---- a thread to a channel, step by step ------------------------------------

constexpr int kThreads = 128;

template <typename T, typename G, int KIND>
__global__ void __launch_bounds__(kThreads) serial_kernel(const Args k) {
    pdl_prologue();
    const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= int64_t(k.batch) * k.width) return;
    const int b = static_cast<int>(i / k.width), ch = static_cast<int>(i % k.width);
    const int64_t n = steps_of(k, b);
    float h = k.initial.base != nullptr ? reinterpret_cast<const float*>(k.initial.base + b * k.initial.step)[ch] : 0.f;
    float* state = k.states != nullptr ? k.states + int64_t(b) * k.chunks * k.width + ch : nullptr;
    for (int64_t t0 = 0; t0 < k.length; t0 += kSteps) {
        if (state != nullptr) {
            *state = h;
            state += k.width;
        }
        float x[kSteps], g[kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            const bool in = t0 + j < n;
            x[j] = in ? to_float(*at<const T>(k.x, b, t0 + j, ch)) : 0.f;
            g[j] = in ? to_float(*at<const G>(k.gate, b, t0 + j, ch)) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            float input;
            const float c = decay<KIND>(g[j], input);
            const bool in = t0 + j < n;
            if (in) h = apply(c, h, input * x[j]);
            if (t0 + j < k.length) *at<T>(k.out, b, t0 + j, ch) = from_float<T>(in ? h : 0.f);
        }
    }
    if (k.final_state.base != nullptr) reinterpret_cast<float*>(k.final_state.base + b * k.final_state.step)[ch] = h;
}

template <typename T, typename G, int KIND>
__global__ void __launch_bounds__(kThreads) serial_backward_kernel(const Args k) {
    pdl_prologue();
    const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
    if (i >= int64_t(k.batch) * k.width) return;
    const int b = static_cast<int>(i / k.width), ch = static_cast<int>(i % k.width);
    const int64_t n = steps_of(k, b);
    float e = k.final_state.base != nullptr ? reinterpret_cast<const float*>(k.final_state.base + b * k.final_state.step)[ch] : 0.f;
    for (int chunk = k.chunks - 1; chunk >= 0; --chunk) {
        const int64_t t0 = int64_t(chunk) * kSteps;
        float h = k.states[(int64_t(b) * k.chunks + chunk) * k.width + ch];
        float c[kSteps], w[kSteps], d[kSteps];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            const bool in = t0 + j < n;
            w[j] = in ? to_float(*at<const T>(k.x, b, t0 + j, ch)) : 0.f;
            c[j] = in ? to_float(*at<const G>(k.gate, b, t0 + j, ch)) : 0.f;
            d[j] = in && k.dout.base != nullptr ? to_float(*at<const T>(k.dout, b, t0 + j, ch)) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            const bool in = t0 + j < n;
            const float x = w[j];
            float input;
            c[j] = decay<KIND>(c[j], input);
            w[j] = KIND == B200_GATES_SIGMOID ? h - x : h;
            if (in) h = apply(c[j], h, input * x);
            else c[j] = kHold;
        }
#pragma unroll
        for (int j = kSteps - 1; j >= 0; --j) {
            const bool in = t0 + j < n;
            const float D = d[j] + e;
            e = apply(c[j], D, 0.f);
            float gate, input;
            slopes<KIND>(c[j], gate, input);
            if (t0 + j < k.length) {
                if (k.dx.base != nullptr) *at<T>(k.dx, b, t0 + j, ch) = from_float<T>(in ? input * D : 0.f);
                if (k.dgate.base != nullptr) *at<G>(k.dgate, b, t0 + j, ch) = from_float<G>(in ? gate * w[j] * D : 0.f);
            }
        }
    }
    if (k.initial.base != nullptr) reinterpret_cast<float*>(k.initial.base + b * k.initial.step)[ch] = e;
}

// ---- arguments --------------------------------------------------------------

bool present(const b200_tensor& t) { return t.data != nullptr; }

struct Shape {
    int axes;  // of x in front of the rows
    int64_t batch, length, width, chunks;
};

Shape check_streams(const b200_tensor& x, const b200_tensor& gate, const b200_tensor& lengths, const b200_tensor& states, int kind, uint32_t flags, const char* who) {
    check_rows(x, "x");
    check_rows(gate, "gate");
    if (x.ndim < 2) fail(B200_SHAPE_ERROR, "x: rank " + std::to_string(x.ndim) + " is outside 2..3");
    if (gate.ndim != x.ndim || !same_extents(gate, x, x.ndim)) fail(B200_SHAPE_ERROR, "gate has not x's extents");
    if (!is_float(x.dtype) || !is_float(gate.dtype) || (x.dtype == B200_F32 && gate.dtype == B200_F16)) {
        fail(B200_DTYPE_ERROR, std::string(who) + ": (x, gate) are (F32, F32), (F16, F16) or (F16, F32)");
    }
    if (kind != B200_GATES_SIGMOID && kind != B200_GATES_EXP) fail(B200_INVALID_ARGUMENT, std::string(who) + ": unknown kind of gates");
    if (flags != 0) fail(B200_INVALID_ARGUMENT, std::string(who) + ": unknown flags");
    Shape s{};
    s.axes = x.ndim - 1;
    s.width = x.dims[s.axes];
    s.length = x.dims[s.axes - 1];
    s.batch = x.ndim == 3 ? x.dims[0] : 1;
    s.chunks = ceil_div(s.length, kSteps);
    if (s.width >= (int64_t(1) << 31) || s.batch >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "x: 2^31 or more channels or sequences");
    if (present(lengths)) {
        check_tensor(lengths, "lengths");
        if (!is_index(lengths.dtype)) fail(B200_DTYPE_ERROR, "lengths are I32 or I64");
        if (lengths.ndim != x.ndim - 2 || (lengths.ndim == 1 && lengths.dims[0] != s.batch)) fail(B200_SHAPE_ERROR, "lengths: not one for each sequence");
    }
    if (present(states)) {
        check_tensor(states, "states");
        if (states.dtype != B200_F32) fail(B200_DTYPE_ERROR, "states are F32");
        if (states.ndim != x.ndim || states.dims[s.axes] != s.width || states.dims[s.axes - 1] != s.chunks || (x.ndim == 3 && states.dims[0] != s.batch) || !is_dense(states)) {
            fail(B200_SHAPE_ERROR, "states: not one for every 16 steps, dense");
        }
    }
    return s;
}

// h in front of a sequence or behind it, or a gradient of one.
void check_end(const b200_tensor& t, const char* name, const Shape& s) {
    if (!present(t)) return;
    check_rows(t, name);
    if (t.dtype != B200_F32) fail(B200_DTYPE_ERROR, std::string(name) + " is F32");
    if (t.ndim != s.axes || t.dims[t.ndim - 1] != s.width || (t.ndim == 2 && t.dims[0] != s.batch)) fail(B200_SHAPE_ERROR, std::string(name) + ": not a row for each sequence");
}

void check_stream_like(const b200_tensor& t, const char* name, const b200_tensor& like, int dtype) {
    check_rows(t, name);
    if (t.ndim != like.ndim || !same_extents(t, like, like.ndim)) fail(B200_SHAPE_ERROR, std::string(name) + " has not x's extents");
    if (t.dtype != dtype) fail(B200_DTYPE_ERROR, std::string(name) + " has another type");
}

Shape check_forward(const b200_recurrence_args& a) {
    const Shape s = check_streams(a.x, a.gate, a.lengths, a.states, a.kind, a.flags, "gated_recurrence");
    check_end(a.initial, "initial", s);
    check_end(a.final_state, "final_state", s);
    check_stream_like(a.out, "out", a.x, a.x.dtype);
    check_results({{&a.out, "out"}}, {{&a.initial, "initial"}, {&a.lengths, "lengths"}, {&a.final_state, "final_state"}, {&a.states, "states"}}, {{&a.x, "x"}, {&a.gate, "gate"}});
    check_results({{&a.final_state, "final_state"}, {&a.states, "states"}}, {{&a.x, "x"}, {&a.gate, "gate"}, {&a.lengths, "lengths"}}, {});
    check_results({{&a.states, "states"}}, {{&a.initial, "initial"}}, {});
    check_results({{&a.final_state, "final_state"}}, {}, {{&a.initial, "initial"}});
    return s;
}

Shape check_backward(const b200_recurrence_grad_args& a) {
    const Shape s = check_streams(a.x, a.gate, a.lengths, a.states, a.kind, a.flags, "gated_recurrence_backward");
    check_end(a.final_grad, "final_grad", s);
    check_end(a.initial_grad, "initial_grad", s);
    if (present(a.out_grad)) check_stream_like(a.out_grad, "out_grad", a.x, a.x.dtype);
    if (present(a.x_grad)) check_stream_like(a.x_grad, "x_grad", a.x, a.x.dtype);
    if (present(a.gate_grad)) check_stream_like(a.gate_grad, "gate_grad", a.x, a.gate.dtype);
    const std::initializer_list<Named> apart = {{&a.lengths, "lengths"}, {&a.states, "states"}, {&a.final_grad, "final_grad"}};
    const std::initializer_list<Named> exact = {{&a.x, "x"}, {&a.gate, "gate"}, {&a.out_grad, "out_grad"}};
    check_results({{&a.x_grad, "x_grad"}, {&a.gate_grad, "gate_grad"}, {&a.initial_grad, "initial_grad"}}, {}, {});
    check_results({{&a.x_grad, "x_grad"}}, apart, exact);
    check_results({{&a.gate_grad, "gate_grad"}}, apart, exact);
    check_results({{&a.initial_grad, "initial_grad"}}, {{&a.lengths, "lengths"}, {&a.states, "states"}, {&a.x, "x"}, {&a.gate, "gate"}, {&a.out_grad, "out_grad"}}, {{&a.final_grad, "final_grad"}});
    if (s.batch * s.width == 0) return s;
    if (s.length > 0 && !present(a.states)) fail(B200_INVALID_ARGUMENT, "gated_recurrence_backward: the forward call's states are needed");
    if (s.length > 0 && !present(a.x_grad) && !present(a.gate_grad) && !present(a.initial_grad)) fail(B200_INVALID_ARGUMENT, "gated_recurrence_backward: no result is asked for");
    return s;
}

Stream stream_of(const b200_tensor& t) {
    Stream s{};
    s.base = static_cast<char*>(t.data);
    if (s.base == nullptr) return s;
    s.step = t.dims[t.ndim - 2] > 1 ? t.strides[t.ndim - 2] : 0;
    s.batch = t.ndim == 3 && t.dims[0] > 1 ? t.strides[0] : 0;
    return s;
}

Args common_args(b200_ctx* ctx, const Shape& s, const b200_tensor& x, const b200_tensor& gate, const b200_tensor& lengths, const b200_tensor& states) {
    Args k{};
    k.x = stream_of(x);
    k.gate = stream_of(gate);
    k.states = static_cast<float*>(states.data);
    k.lengths = static_cast<const char*>(lengths.data);
    k.lengths_step = lengths.ndim == 1 && lengths.dims[0] > 1 ? lengths.strides[0] : 0;
    k.wide_lengths = lengths.dtype == B200_I64;
    k.length = s.length;
    k.batch = static_cast<int>(s.batch);
    k.width = static_cast<int>(s.width);
    k.chunks = static_cast<int>(s.chunks);
    k.status = ctx->d_status;
    return k;
}

RowsArg end_of(const b200_tensor& t) { return present(t) ? rows_arg(t, t.ndim - 1) : RowsArg{}; }

// Calls go(T, G, kind) with the types of a call.
template <typename Fn>
void by_type(const b200_tensor& x, const b200_tensor& gate, int kind, Fn&& go) {
    auto with = [&](auto t, auto g) {
        if (kind == B200_GATES_SIGMOID) go(t, g, std::integral_constant<int, B200_GATES_SIGMOID>{});
        else go(t, g, std::integral_constant<int, B200_GATES_EXP>{});
    };
    if (x.dtype == B200_F32) with(float{}, float{});
    else if (gate.dtype == B200_F32) with(__half{}, float{});
    else with(__half{}, __half{});
}

void launch_forward(b200_ctx* ctx, const b200_recurrence_args& a) {
    const Shape s = check_forward(a);
    if (s.batch * s.width == 0 || (s.length == 0 && !present(a.final_state))) return;
    wait_for_tensors(ctx, {&a.x, &a.gate, &a.initial, &a.lengths, &a.out, &a.final_state, &a.states});
    Args k = common_args(ctx, s, a.x, a.gate, a.lengths, a.states);
    k.out = stream_of(a.out);
    k.initial = end_of(a.initial);
    k.final_state = end_of(a.final_state);
    ProfScope scope(ctx, "gated_recurrence");
    by_type(a.x, a.gate, a.kind, [&](auto t, auto g, auto kind) {
        launch_kernel(ctx, serial_kernel<decltype(t), decltype(g), decltype(kind)::value>, dim3(static_cast<unsigned>(ceil_div(s.batch * s.width, kThreads))), dim3(kThreads), 0, k);
    });
    check_last_launch("gated_recurrence");
    ctx->count_launch();
}

void launch_backward(b200_ctx* ctx, const b200_recurrence_grad_args& a) {
    const Shape s = check_backward(a);
    if (s.batch * s.width == 0 || (s.length == 0 && !present(a.initial_grad))) return;
    wait_for_tensors(ctx, {&a.x, &a.gate, &a.lengths, &a.states, &a.out_grad, &a.final_grad, &a.x_grad, &a.gate_grad, &a.initial_grad});
    Args k = common_args(ctx, s, a.x, a.gate, a.lengths, a.states);
    k.dout = stream_of(a.out_grad);
    k.dx = stream_of(a.x_grad);
    k.dgate = stream_of(a.gate_grad);
    k.initial = end_of(a.initial_grad);
    k.final_state = end_of(a.final_grad);
    ProfScope scope(ctx, "gated_recurrence_backward");
    by_type(a.x, a.gate, a.kind, [&](auto t, auto g, auto kind) {
        launch_kernel(ctx, serial_backward_kernel<decltype(t), decltype(g), decltype(kind)::value>, dim3(static_cast<unsigned>(ceil_div(s.batch * s.width, kThreads))), dim3(kThreads), 0, k);
    });
    check_last_launch("gated_recurrence_backward");
    ctx->count_launch();
}

}  // namespace

void check_gated_recurrence(const b200_recurrence_args& a) { (void)check_forward(a); }
void check_gated_recurrence_backward(const b200_recurrence_grad_args& a) { (void)check_backward(a); }

}  // namespace b200

using namespace b200;

extern "C" {

int b200_gated_recurrence(b200_ctx* ctx, const b200_recurrence_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_forward(ctx, *args); });
}

int b200_gated_recurrence_backward(b200_ctx* ctx, const b200_recurrence_grad_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_backward(ctx, *args); });
}

}  // extern "C"
