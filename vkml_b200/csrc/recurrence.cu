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

__device__ __forceinline__ float fast_root(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A step's decay: -d where a = 1 - d is above a half (never 0: the sign tells), else a.
constexpr float kHold = -0x1p-126f;  // h stays
__device__ __forceinline__ bool keeps(float c) { return c < 0.f; }
// Arithmetic on a lane's channels, two to an instruction.
template <int V>
__device__ __forceinline__ void fma_v(float (&d)[V], const float (&a)[V], const float (&b)[V], const float (&c)[V]) {
    if constexpr (V == 2) fma_pair(d[0], d[1], a[0], a[1], b[0], b[1], c[0], c[1]);
    else d[0] = fmaf(a[0], b[0], c[0]);
}
template <int V>
__device__ __forceinline__ void mul_v(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
    if constexpr (V == 2) mul_pair(d[0], d[1], a[0], a[1], b[0], b[1]);
    else d[0] = a[0] * b[0];
}
template <int V>
__device__ __forceinline__ void add_v(float (&d)[V], const float (&a)[V], const float (&b)[V]) {
    if constexpr (V == 2) add_pair(d[0], d[1], a[0], a[1], b[0], b[1]);
    else d[0] = a[0] + b[0];
}
template <int V>
__device__ __forceinline__ void apply_v(float (&h)[V], const float (&c)[V], const float (&b)[V]) {
    float t[V], more[V];
    fma_v(t, c, h, b);
    add_v(more, h, t);
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = keeps(c[e]) ? more[e] : t[e];
}

// e^x - 1 by its series, for x of (-0.69, 0.17) (the term left out is 2e-8 of it at the lower end); never 0 where x is not above 0, which is where steps use it.
__device__ __forceinline__ bool in_series(float x) { return x <= 0.f && x > -0.6931f; }
template <int V>
__device__ __forceinline__ void series_of(const float (&x)[V], float (&s)[V]) {
    float q[V], k[V];
    auto constant = [&](float value) {
#pragma unroll
        for (int e = 0; e < V; ++e) k[e] = value;
    };
    auto next = [&](float value) {
        constant(value);
        fma_v(s, x, s, k);
    };
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] = 1.f / 362880.f;
    next(1.f / 40320.f);
    next(1.f / 5040.f);
    next(1.f / 720.f);
    next(1.f / 120.f);
    next(1.f / 24.f);
    next(1.f / 6.f);
    next(0.5f);
    mul_v(q, x, x);
    constant(-0x1p-126f);
    add_v(k, x, k);
    fma_v(s, q, s, k);
}

// What gates do to a step: its decay c (as above), a, d = 1 - a, and b / x.
template <int KIND, int V>
__device__ __forceinline__ void gates_of(const float (&gate)[V], float (&c)[V], float (&a)[V], float (&d)[V], float (&input)[V]) {
    if constexpr (KIND == B200_GATES_SIGMOID) {
        // a = 1 / (1 + z), 1 - a = z a, z = e^-gate up to 2^126, where a is 2^-126: that is taken off, so that a gate of -inf has a = 0 (and added to the
        // other, so that it is never 0).  Nothing else is as small.
        float z[V], one[V], tiny[V], least[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            one[e] = -kLog2e, tiny[e] = 0x1p-126f, least[e] = -0x1p-126f;
        }
        mul_v(z, gate, one);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            asm("min.NaN.f32 %0, %1, %2;" : "=f"(z[e]) : "f"(z[e]), "f"(126.f));
            z[e] = fast_exp2(z[e]);
            one[e] = 1.f;
        }
        add_v(one, one, z);
#pragma unroll
        for (int e = 0; e < V; ++e) a[e] = fast_reciprocal(one[e]);
        fma_v(d, z, a, tiny);
        add_v(a, a, least);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            c[e] = gate[e] > 0.f ? -d[e] : a[e];
            input[e] = d[e];
        }
    } else {
        float s[V];
        series_of(gate, s);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const bool near = in_series(gate[e]);
            const float far = fast_exp2(gate[e] * kLog2e);
            c[e] = near ? s[e] : far;  // (a growing state: a itself, as below a half)
            a[e] = near ? 1.f + s[e] : far;
            d[e] = near ? -s[e] : 1.f - far;
            input[e] = 1.f;
        }
    }
}
// What dgate is (h_{t-1} - x) D times, or h_{t-1} D times; what dx is D times; and a.
template <int KIND>
__device__ __forceinline__ void slopes(float c, float& gate, float& input, float& a) {
    if constexpr (KIND == B200_GATES_SIGMOID) {
        const float s = fabsf(c), r = 1.f - s;
        gate = s * r;
        input = keeps(c) ? s : r;
        a = keeps(c) ? r : s;
    } else {
        gate = a = keeps(c) ? 1.f + c : c;
        input = 1.f;
    }
}

// What a run of steps does to the state in front of it: h becomes a h + sum, as h + (sum - d h) where a is above a half.  The product of the a's is kept as such and as
// d = 1 - a: either has digits that the other loses.  A run tells its decay as a step does.
//
// Kind exp: states may grow, and a product of growing decays leaves F32's range long before the state that it multiplies has to (128 steps of gates of 0.8 make 1e-30
// to 3e14 by a product of 3e44).  What a run tells is -d where a is above a half and not above 1, -a up to 1.19, and beyond these a's root, which is in F32's range for every
// product that takes one number of normal size to another.  (Where decays fall and then rise d has no digits left: sixteen runs that grow by 1.19 at most multiply its rounding by 16 at most.)
constexpr float kMild = 0.19f;
__device__ __forceinline__ bool is_root(float c) { return !(c < 0.f); }
__device__ __forceinline__ bool grows(float c) { return c < -0.75f; }
template <int KIND, int V>
struct Run {
    static constexpr bool kRoot = KIND == B200_GATES_EXP;
    float a[V], d[V], sum[V];   // (kRoot: a is the root, but for `near`; d is no number where a part tells a root)
    float near[kRoot ? V : 1];  // the product of the parts that do not
    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int e = 0; e < V; ++e) a[e] = 1.f, d[e] = 0.f, sum[e] = 0.f, near[kRoot ? e : 0] = 1.f;
    }
    // A step behind this one.  (a's rounding counts within the run only.)
    __device__ __forceinline__ void decays(const float (&a1)[V], const float (&d1)[V]) {
        mul_v(a, a, a1);
        fma_v(d, a1, d, d1);
    }
    __device__ __forceinline__ void adds(const float (&a1)[V], const float (&b)[V]) { fma_v(sum, a1, sum, b); }
    // Steps of the kind exp have the product of their a's by the sum of their gates: that of one step.
    __device__ __forceinline__ void decays_of_sum(const float (&gate)[V]) {
        float s[V];
        series_of(gate, s);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            d[e] = gate[e] < 0.17f && gate[e] > -0.6931f ? -s[e] : NAN;  // (up to kMild)
            a[e] = fast_exp2(gate[e] * (0.5f * kLog2e));
        }
        stay_finite();
    }
    // Another run behind this one, by its decay and sum.
    __device__ __forceinline__ void then(const float (&c)[V], const float (&s)[V]) {
        float a1[V], d1[V];
        if constexpr (kRoot) {
            // (What does not depend on what is in front comes first: of the sums a product and a multiply-add follow one another.)
            float first[V], second[V], factor[V], kept[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const bool root = is_root(c[e]);
                a1[e] = grows(c[e]) ? -c[e] : 1.f + c[e];
                d1[e] = grows(c[e]) ? 1.f + c[e] : -c[e];
                first[e] = root ? c[e] : 1.f;
                second[e] = root ? c[e] : a1[e];
                factor[e] = root ? 1.f : a1[e];
                kept[e] = root ? NAN : a1[e];
            }
            mul_v(a, a, first);
            mul_v(first, first, sum);
            fma_v(sum, second, first, s);
            mul_v(near, near, factor);
            fma_v(d, kept, d, d1);
            stay_finite();
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                a1[e] = keeps(c[e]) ? 1.f + c[e] : c[e];
                d1[e] = keeps(c[e]) ? -c[e] : 1.f - c[e];
            }
            adds(a1, s);
            decays(a1, d1);
        }
    }
    // (A product beyond even that has no state to grow but zero: not a number would come of an infinite one.)
    __device__ __forceinline__ void stay_finite() {
#pragma unroll
        for (int e = 0; e < V; ++e) asm("min.NaN.f32 %0, %1, %2;" : "=f"(a[e]) : "f"(a[e]), "f"(3.4e38f));
    }
    // What the run tells.
    __device__ __forceinline__ float decay(int e) const {
        if constexpr (kRoot) {
            const float mild = d[e] >= 0.f ? fminf(-d[e], kHold) : d[e] - 1.f;
            return d[e] > -kMild && d[e] < 0.5f ? mild : a[e] * fast_root(near[e]);
        } else {
            return d[e] >= 0.f && d[e] < 0.5f ? fminf(-d[e], kHold) : a[e];
        }
    }
};
// h behind a run, by what it tells and its sum.
template <int KIND, int V>
__device__ __forceinline__ void apply_run(float (&h)[V], const float (&c)[V], const float (&sum)[V]) {
    if constexpr (KIND == B200_GATES_EXP) {
        float t[V], less[V], far[V], more[V];
        mul_v(t, c, h);
#pragma unroll
        for (int e = 0; e < V; ++e) t[e] = is_root(c[e]) ? t[e] : -h[e];
        fma_v(far, t, c, sum);
        fma_v(less, c, h, sum);
        add_v(more, h, less);
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = is_root(c[e]) || grows(c[e]) ? far[e] : more[e];
    } else {
        apply_v(h, c, sum);
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

// Steps of sequence b.
__device__ __forceinline__ int64_t steps_of(const Args& k, int b) {
    if (k.lengths == nullptr) return k.length;
    const int64_t n = load_index(k.lengths + b * k.lengths_step, k.wide_lengths);
    if (n < 0 || n > k.length) atomicOr(k.status, kStatusIndexOutOfRange);
    return n < 0 ? 0 : n > k.length ? k.length : n;
}

// VEC neighbouring channels of a lane as they lie in memory, and as floats.
template <typename T, int VEC>
struct Raw {
    T a;
    __device__ __forceinline__ void load(const char* p) { a = *reinterpret_cast<const T*>(p); }
    __device__ __forceinline__ void clear() { a = from_float<T>(0.f); }
    __device__ __forceinline__ void get(float (&x)[1]) const { x[0] = to_float(a); }
    static __device__ __forceinline__ void store(char* p, const float (&x)[1]) { *reinterpret_cast<T*>(p) = from_float<T>(x[0]); }
};
template <>
struct Raw<__half, 2> {
    uint32_t a;
    __device__ __forceinline__ void load(const char* p) { a = *reinterpret_cast<const uint32_t*>(p); }
    __device__ __forceinline__ void clear() { a = 0; }
    __device__ __forceinline__ void get(float (&x)[2]) const {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
        x[0] = f.x, x[1] = f.y;
    }
    static __device__ __forceinline__ void store(char* p, const float (&x)[2]) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x[0], x[1]); }
};
template <>
struct Raw<float, 2> {
    float2 a;
    __device__ __forceinline__ void load(const char* p) { a = *reinterpret_cast<const float2*>(p); }
    __device__ __forceinline__ void clear() { a = make_float2(0.f, 0.f); }
    __device__ __forceinline__ void get(float (&x)[2]) const { x[0] = a.x, x[1] = a.y; }
    static __device__ __forceinline__ void store(char* p, const float (&x)[2]) { *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]); }
};

template <int VEC>
__device__ __forceinline__ void load_end(float (&h)[VEC], const RowsArg& end, int b, int ch, bool in) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[e] = end.base != nullptr && in ? reinterpret_cast<const float*>(end.base + b * end.step)[ch + e] : 0.f;
}
template <int VEC>
__device__ __forceinline__ void store_end(const RowsArg& end, int b, int ch, const float (&h)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) reinterpret_cast<float*>(end.base + b * end.step)[ch + e] = h[e];
}

// ---- a thread to its channels, step by step ----------------------------------
//
// Few steps: the next token of many sequences, say, where the launch is what takes the time (64 sequences of 2048 channels, F16, one step: 4.9 us; 17 steps 8.1 us, 6.8 by
// the walk below; 32 steps 13.6 and 7.0).  Every step is exact to its own rounding, so that a state that is carried on a token at a time drifts no more than one that a
// long call carries.

constexpr int kThreads = 128;

// The steps of one sequence and VEC channels, N at a time.
template <typename T, typename G, int KIND, int VEC, int N>
__global__ void __launch_bounds__(kThreads) serial_kernel(const Args k) {
    pdl_prologue();
    const int ch = (blockIdx.x * kThreads + threadIdx.x) * VEC;
    if (ch >= k.width) return;
    const int length = static_cast<int>(k.length);
    for (uint32_t i = blockIdx.y; i < static_cast<uint32_t>(k.batch); i += gridDim.y) {  // (what is behind the last of 2^31 - 1 sequences has 32 bits)
        const int b = static_cast<int>(i);
        const int n = static_cast<int>(steps_of(k, b));
        const char *x = k.x.base + b * k.x.batch + ch * int64_t(sizeof(T)), *gate = k.gate.base + b * k.gate.batch + ch * int64_t(sizeof(G));
        char* out = k.out.base + b * k.out.batch + ch * int64_t(sizeof(T));
        float* state = k.states != nullptr ? k.states + int64_t(b) * k.chunks * k.width + ch : nullptr;
        float h[VEC];
        load_end<VEC>(h, k.initial, b, ch, true);
        for (int t = 0; t < length; t += N) {
            if (state != nullptr && t % kSteps == 0) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) state[e] = h[e];
                state += k.width;
            }
            Raw<T, VEC> rx[N];
            Raw<G, VEC> rg[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                rx[j].clear(), rg[j].clear();
                if (t + j < n) rx[j].load(x + (t + j) * k.x.step), rg[j].load(gate + (t + j) * k.gate.step);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (t + j >= length) break;
                float y[VEC] = {};
                if (t + j < n) {
                    float xs[VEC], gs[VEC], c[VEC], a[VEC], d[VEC], input[VEC], add[VEC];
                    rx[j].get(xs);
                    rg[j].get(gs);
                    gates_of<KIND>(gs, c, a, d, input);
                    mul_v(add, input, xs);
                    apply_v(h, c, add);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) y[e] = h[e];
                }
                Raw<T, VEC>::store(out + (t + j) * k.out.step, y);
            }
        }
        if (k.final_state.base != nullptr) store_end<VEC>(k.final_state, b, ch, h);
    }
}

// One chunk of steps at most.
template <typename T, typename G, int KIND, int VEC, int N>
__global__ void __launch_bounds__(kThreads) serial_backward_kernel(const Args k) {
    pdl_prologue();
    const int ch = (blockIdx.x * kThreads + threadIdx.x) * VEC;
    if (ch >= k.width) return;
    const int length = static_cast<int>(k.length);
    for (uint32_t i = blockIdx.y; i < static_cast<uint32_t>(k.batch); i += gridDim.y) {  // (what is behind the last of 2^31 - 1 sequences has 32 bits)
        const int b = static_cast<int>(i);
        const int n = static_cast<int>(steps_of(k, b));
        const char *x = k.x.base + b * k.x.batch + ch * int64_t(sizeof(T)), *gate = k.gate.base + b * k.gate.batch + ch * int64_t(sizeof(G));
        const char* dout = k.dout.base != nullptr ? k.dout.base + b * k.dout.batch + ch * int64_t(sizeof(T)) : nullptr;
        char* dx = k.dx.base != nullptr ? k.dx.base + b * k.dx.batch + ch * int64_t(sizeof(T)) : nullptr;
        char* dgate = k.dgate.base != nullptr ? k.dgate.base + b * k.dgate.batch + ch * int64_t(sizeof(G)) : nullptr;
        float later[VEC], h[VEC];
        load_end<VEC>(later, k.final_state, b, ch, true);
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[e] = length > 0 ? k.states[int64_t(b) * k.width + ch + e] : 0.f;
        Raw<T, VEC> rx[N], rd[N];
        Raw<G, VEC> rg[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            rx[j].clear(), rg[j].clear(), rd[j].clear();
            if (j < n) {
                rx[j].load(x + j * k.x.step), rg[j].load(gate + j * k.gate.step);
                if (dout != nullptr) rd[j].load(dout + j * k.dout.step);
            }
        }
        float c[N][VEC], u[N][VEC];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float xs[VEC], gs[VEC], a[VEC], d[VEC], input[VEC], add[VEC];
            rx[j].get(xs);
            rg[j].get(gs);
            gates_of<KIND>(gs, c[j], a, d, input);
            mul_v(add, input, xs);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (j >= n) c[j][e] = kHold, add[e] = 0.f;
                u[j][e] = KIND == B200_GATES_SIGMOID ? h[e] - xs[e] : h[e];
            }
            apply_v(h, c[j], add);
        }
#pragma unroll
        for (int j = N - 1; j >= 0; --j) {
            if (j >= length) continue;
            float D[VEC], px[VEC] = {}, pg[VEC] = {}, zero[VEC] = {};
            rd[j].get(D);
            add_v(D, D, later);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                later[e] = D[e];
                float slope, input, a;
                slopes<KIND>(c[j][e], slope, input, a);
                if (j < n) px[e] = input * D[e], pg[e] = slope * u[j][e] * D[e];
            }
            apply_v(later, c[j], zero);
            if (dx != nullptr) Raw<T, VEC>::store(dx + j * k.dx.step, px);
            if (dgate != nullptr) Raw<G, VEC>::store(dgate + j * k.dgate.step, pg);
        }
        if (k.initial.base != nullptr) store_end<VEC>(k.initial, b, ch, later);
    }
}

// ---- blocks that walk along a sequence --------------------------------------
//
// A block, or a cluster of blocks, has 32 lanes' channels of a sequence and walks along it window by window; a warp has 16 steps of a window.  A thread computes what
// its steps do to a state that comes in (a decay and a sum: a step like any other), the warps tell each other by shared memory, the cluster's blocks by each
// other's, and every thread goes through its steps again from the state that does come in.  All of it stays in registers: gates and inputs are read once, and the
// next window's are under way while this one is computed.
//
// 8 sequences of 4096 steps, 2048 channels, F16: 82 to 86 us (5.0 TB/s), gradient 141 to 147 us (4.8 TB/s).  Neither memory nor the issue slots are full (56 and 65 % of them where an SM has
// work, at the 16 warps that its registers hold): steps follow one another in both walks, results wait for gates' functions, warps for the block's meeting in each window; and 256 blocks on 296 places
// leave 40 SMs with one block where the others have two.  The same in F32: 143 to 146 us (5.7 TB/s), gradient 240 to 257.  50000 steps of 1000 channels, F32, kind exp: 152 to 154 us (4.0 TB/s), a cluster's
// meeting in each of 49 windows.

constexpr int kWarps = 8;        // of a block, two of which an SM holds
constexpr int kMostWarps = 16;   // of one that has an SM to itself
constexpr int kMostCluster = 8;
constexpr int kAheadSlots = 4;   // (walk_ahead_kernel)

// What the segments of a block, and the blocks of a cluster, do to a state: a decay and a sum, for every channel; and the state in front of the window.  Two of each: a
// window's are read while the next one's are written.  (A block that is told of the window after next has told the next one itself, behind its reading of
// this one.)
template <int VEC>
struct Told {
    static constexpr int kRow = 32 * VEC;
    float* at;  // in dynamic shared memory, behind the windows
    int warps;
    uint64_t* bars;  // one for each place to be told at: counts the bytes that the cluster's blocks tell this one
    int* given_up;
    static __host__ __device__ constexpr size_t bytes(int warps, int slots) { return size_t(2 * (2 * warps + 1) + 2 * slots * kMostCluster) * kRow * 4; }
    __device__ __forceinline__ float* front(uint32_t parity) const { return at + parity * kRow; }
    __device__ __forceinline__ float* segment(uint32_t parity, int i) const { return at + (2 + (parity * warps + i) * 2) * kRow; }
    __device__ __forceinline__ float* block(uint32_t slot, uint32_t i) const { return at + (2 + 4 * warps + (slot * kMostCluster + i) * 2) * kRow; }
};
template <int VEC>
__device__ __forceinline__ void get_row(float (&x)[VEC], const float* from, int lane) {
    Raw<float, VEC> r;
    r.load(reinterpret_cast<const char*>(from + lane * VEC));
    r.get(x);
}
template <int VEC>
__device__ __forceinline__ void put_row(float* to, int lane, const float (&x)[VEC]) { Raw<float, VEC>::store(reinterpret_cast<char*>(to + lane * VEC), x); }
// h behind a segment or a block.
template <int KIND, int VEC>
__device__ __forceinline__ void pass(float (&h)[VEC], const float* run, int lane) {
    float c[VEC], sum[VEC];
    get_row<VEC>(c, run, lane);
    get_row<VEC>(sum, run + 32 * VEC, lane);
    apply_run<KIND>(h, c, sum);
}

// h behind a cluster's blocks, and the state in front of the one that has `ahead` of them in front of it.  Kind exp: each is asked for while the one before it is passed, which takes longer
// there (gradient of 4 sequences of 4096 steps, 2048 channels, F16: 92 us, 98 without; kind sigmoid, 50000 steps of 1000 channels, F32: 143 and 137).
template <int KIND, int VEC, bool BACK>
__device__ __forceinline__ void pass_blocks(const Told<VEC>& told, uint32_t slot, int lane, uint32_t cluster, uint32_t ahead, float (&h)[VEC], float (&in)[VEC]) {
    constexpr bool kAsk = KIND == B200_GATES_EXP;
    float c[2][VEC], sum[2][VEC];
    auto ask = [&](uint32_t j) {
        const float* const run = told.block(slot, BACK ? cluster - 1 - j : j);
        get_row<VEC>(c[j % 2], run, lane);
        get_row<VEC>(sum[j % 2], run + 32 * VEC, lane);
    };
    if (kAsk) ask(0);
#pragma unroll
    for (uint32_t j = 0; j < kMostCluster; ++j) {
        if (kAsk && j >= cluster) break;
        if (j == ahead) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) in[e] = h[e];
        }
        if (j < cluster) {
            if (!kAsk) ask(j);
            else if (j + 1 < cluster) ask(j + 1);
            apply_run<KIND>(h, c[j % 2], sum[j % 2]);
        }
    }
}

// Stores to another block of the cluster that its barrier counts.  (A cluster barrier would order them too, but waits for every store of the block before it.)
template <int VEC>
__device__ __forceinline__ void tell(uint32_t to, uint32_t bar, const float (&x)[VEC]) {
    if constexpr (VEC == 2) {
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(to), "f"(x[0]), "f"(x[1]), "r"(bar) : "memory");
    } else {
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(to), "f"(x[0]), "r"(bar) : "memory");
    }
}
__device__ __forceinline__ uint32_t in_block(uint32_t address, uint32_t rank) {
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(address), "r"(rank));
    return to;
}
__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// Waits for a phase of a barrier, four seconds at most; whoever gives up says so, and goes on with what is there.
__device__ __noinline__ void wait_for(uint32_t bar, uint32_t phase, int* given_up, uint32_t* status) {
    uint64_t start = 0;
    for (uint32_t spins = 0;; ++spins) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, 2000;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(done) : "r"(bar), "r"(phase) : "memory");
        if (done || *static_cast<volatile int*>(given_up) != 0) return;
        if (spins % 64 == 63) {
            uint64_t now;
            asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
            if (start == 0) start = now;
            else if (now - start > 4000000000ull) {
                *static_cast<volatile int*>(given_up) = 1;
                atomicOr(status, kStatusWaitTimedOut);
                return;
            }
        }
    }
}

// Before a cluster's blocks tell each other anything, and before one of them ends.
template <int VEC>
__device__ __forceinline__ void begin_cluster(const Told<VEC>& told, int slots) {
    if (threadIdx.x == 0) {
        *told.given_up = 0;
        for (int i = 0; i < slots; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&told.bars[i])) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    cluster_sync();
}
__device__ __forceinline__ void end_cluster() {
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    asm volatile("barrier.cluster.wait;" ::: "memory");
}

// The state that comes into this warp's steps.  Segments come one after another, in the order of their warps and blocks, or (BACK) the other way round.  `window` counts from 0.
// In front of window 0 the first warp has put the state to told.front[0]; behind the last one the last warp's `next` is the state there (of a cluster: everyone's).
template <int KIND, int VEC, bool BACK>
__device__ __forceinline__ void join(const Told<VEC>& told, uint32_t window, int warp, int lane, uint32_t rank, uint32_t cluster, uint32_t* status, const Run<KIND, VEC>& own, float (&in)[VEC],
                                     float (&next)[VEC]) {
    const uint32_t parity = window & 1;
    const int warps = told.warps;
    float decay[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) decay[e] = own.decay(e);
    put_row<VEC>(told.segment(parity, warp), lane, decay);
    put_row<VEC>(told.segment(parity, warp) + 32 * VEC, lane, own.sum);
    __syncthreads();
    const int mine = BACK ? warps - 1 - warp : warp;  // segments in front of this one
    if (cluster == 1) {
        get_row<VEC>(in, told.front(parity), lane);
    } else {
        const uint32_t bar = shared_address(&told.bars[parity]);
        // What the segments in front of this one do, while the cluster's blocks tell each other; and what all do, by the last one.
        Run<KIND, VEC> before;
        before.begin();
        float c_next[VEC], sum_next[VEC];  // (asked for one segment ahead)
        auto ask = [&](int i) {
            const float* const segment = told.segment(parity, BACK ? warps - 1 - i : i);
            get_row<VEC>(c_next, segment, lane);
            get_row<VEC>(sum_next, segment + 32 * VEC, lane);
        };
        ask(0);
        for (int i = 0; i < mine; ++i) {
            float c[VEC], sum[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) c[e] = c_next[e], sum[e] = sum_next[e];
            ask(i + 1);
            before.then(c, sum);
        }
        if (mine == warps - 1) {
            if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(cluster * 32u * VEC * 8u) : "memory");
            Run<KIND, VEC> all = before;
            all.then(decay, own.sum);
            float c[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) c[e] = all.decay(e);
            for (uint32_t to = 0; to < cluster; ++to) {
                const uint32_t there = in_block(shared_address(told.block(parity, rank) + lane * VEC), to), bar_there = in_block(bar, to);
                tell<VEC>(there, bar_there, c);
                tell<VEC>(there + 128 * VEC, bar_there, all.sum);
            }
        }
        wait_for(bar, window >> 1 & 1, told.given_up, status);
        const uint32_t ahead = BACK ? cluster - 1 - rank : rank;
        pass_blocks<KIND, VEC, BACK>(told, parity, lane, cluster, ahead, next, in);
        float c[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) c[e] = before.decay(e);
        apply_run<KIND>(in, c, before.sum);
        return;
    }
    for (int i = 0; i < mine; ++i) pass<KIND, VEC>(in, told.segment(parity, BACK ? warps - 1 - i : i), lane);
    if (mine == warps - 1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) next[e] = in[e];
        apply_run<KIND>(next, decay, own.sum);
        put_row<VEC>(told.front(parity ^ 1), lane, next);
    }
}

// What a block's segments do to a state, told to the cluster: this warp's, and beside it (decay, sum) what those in front of it do.  Segments come in the order of their
// warps and blocks, or (BACK) the other way round.
template <int KIND, bool BACK>
__device__ __forceinline__ void tell_ahead(const Told<1>& told, uint32_t parity, uint32_t slot, int warp, int lane, uint32_t rank, uint32_t cluster, const Run<KIND, 1>& own, float (&decay)[1], float (&sum)[1]) {
    const int warps = told.warps;
    const float mine[1] = {own.decay(0)};
    put_row<1>(told.segment(parity, warp), lane, mine);
    put_row<1>(told.segment(parity, warp) + 32, lane, own.sum);
    __syncthreads();
    const int in_front = BACK ? warps - 1 - warp : warp;
    Run<KIND, 1> before;
    before.begin();
    float c_next[1], sum_next[1];  // (asked for one segment ahead)
    auto ask = [&](int i) {
        const float* const segment = told.segment(parity, BACK ? warps - 1 - i : i);
        get_row<1>(c_next, segment, lane);
        get_row<1>(sum_next, segment + 32, lane);
    };
    ask(0);
    for (int i = 0; i < in_front; ++i) {
        const float c[1] = {c_next[0]}, s[1] = {sum_next[0]};
        ask(i + 1);
        before.then(c, s);
    }
    decay[0] = before.decay(0), sum[0] = before.sum[0];
    if (in_front != warps - 1) return;
    const uint32_t bar = shared_address(&told.bars[slot]);
    if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(cluster * 32u * 8u) : "memory");
    before.then(mine, own.sum);
    const float c[1] = {before.decay(0)};
    for (uint32_t to = 0; to < cluster; ++to) {
        const uint32_t there = in_block(shared_address(told.block(slot, rank) + lane), to), bar_there = in_block(bar, to);
        tell<1>(there, bar_there, c);
        tell<1>(there + 128, bar_there, before.sum);
    }
}
// The state that comes into this warp's steps of window w, and `carry`, the state behind the window before it and then behind this one.
template <int KIND, bool BACK>
__device__ __forceinline__ void hear_ahead(const Told<1>& told, uint32_t w, int lane, uint32_t rank, uint32_t cluster, uint32_t* status, const float (&decay)[1], const float (&sum)[1], float (&carry)[1],
                                           float (&in)[1]) {
    const uint32_t slot = w % kAheadSlots, ahead = BACK ? cluster - 1 - rank : rank;
    wait_for(shared_address(&told.bars[slot]), w / kAheadSlots & 1, told.given_up, status);
    pass_blocks<KIND, 1, BACK>(told, slot, lane, cluster, ahead, carry, in);
    apply_run<KIND>(in, decay, sum);
}

// Where a thread works: its sequence, channels, and place in a window.
template <int VEC>
struct Place {
    int b, ch, warp, lane, warps;
    uint32_t rank, cluster;
    bool in;
    __device__ __forceinline__ Place(const Args& k, uint32_t strips, uint32_t blocks) {
        cluster = blocks;
        rank = blockIdx.x % blocks;
        const uint32_t i = blockIdx.x / blocks;
        b = static_cast<int>(i / strips);
        warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
        ch = static_cast<int>(i % strips) * (32 * VEC) + lane * VEC;
        in = ch < k.width;
    }
    __device__ __forceinline__ uint32_t span() const { return warps * kSteps * cluster; }
    __device__ __forceinline__ uint32_t first() const { return (rank * warps + warp) * kSteps; }
    // Bytes of the warp's channels that there are, from its first on; and where that, or this lane's first, lies at step 0.
    __device__ __forceinline__ int valid(int width, size_t size) const { return min(width - (ch - lane * VEC), 32 * VEC) * static_cast<int>(size); }
    template <typename T>
    __device__ __forceinline__ const char* strip(const Stream& s) const { return s.base != nullptr ? s.base + b * s.batch + int64_t(ch - lane * VEC) * int64_t(sizeof(T)) : nullptr; }
    template <typename T>
    __device__ __forceinline__ char* base(const Stream& s) const { return s.base != nullptr ? s.base + b * s.batch + int64_t(ch) * int64_t(sizeof(T)) : nullptr; }
};

// A warp's steps of a stream come through shared memory, by asynchronous copies some windows ahead, into places of the warp's own, so that no warp waits for
// another one's.  CHUNK: bytes of a copy, where every row's part lies on so many; 2: rows of halves at odd addresses, by the words of four bytes that hold them.
template <typename T, int VEC, int CHUNK>
struct Steps {
    static constexpr bool kAround = CHUNK == 2 && sizeof(T) == 2;
    static constexpr int kCopy = CHUNK == 2 ? 4 : CHUNK;
    static constexpr int kBytes = 32 * VEC * int(sizeof(T)) + (kAround ? 4 : 0), kPlace = kSteps * kBytes;
    static constexpr int kPieces = kBytes / kCopy;  // of a row
    const char* from;     // this lane's first piece of the window that is copied next (kAround: the warp's row)
    int64_t step, jump;   // bytes to the next step's, to the next window's
    int valid;            // bytes of the row that there are
    const char* place;    // the window that is looked at
    uint32_t low;         // (kAround) of its first address

    // `base`: of the warp's first channel at step 0; windows from step t on, `span` steps apart (or back).
    __device__ __forceinline__ void begin(const char* base, int64_t bytes, uint32_t t, int64_t span, int row_bytes, int lane) {
        step = bytes, jump = span * bytes, valid = row_bytes;
        from = base + t * bytes;
        if constexpr (!kAround) {
            if constexpr (kPieces <= 32) from += lane / kPieces * bytes + lane % kPieces * kCopy;
            else from += lane * kCopy;
        }
    }
    static __device__ __forceinline__ void copy(uint32_t to, const char* p, int size) {
        if constexpr (kCopy == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(__cvta_generic_to_global(p)), "r"(size) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(__cvta_generic_to_global(p)), "r"(size) : "memory");
    }
    // The window's first `rows` steps to `to`, zeros behind them.  (Where nothing is read the address is one that could be.)
    __device__ __forceinline__ void load(char* to, int rows, int lane) {
        const uint32_t place = shared_address(to);
        if constexpr (kAround) {
            static_assert(kPieces < 32 && 2 * kPieces > 32);
            asm volatile("" : "+r"(lane));  // (nine pieces' rows and offsets are counted for every window: kept, they would leave the steps too few registers)
            int row = lane >= kPieces, off = (lane - row * kPieces) * kCopy;
            const char *p = from + row * step, *const none = reinterpret_cast<const char*>(reinterpret_cast<uintptr_t>(from) & ~uintptr_t(3));
#pragma unroll
            for (int i = 0; i < (kSteps * kPieces + 31) / 32; ++i) {
                if (row < kSteps) {
                    const int behind = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 2);  // bytes in front of the row's in its first word
                    const bool in = row < rows && off < valid + behind;
                    copy(place + (i * 32 + lane) * kCopy, in ? p - behind + off : none, in ? kCopy : 0);
                }
                off += (32 - kPieces) * kCopy, ++row, p += step;
                if (off >= kPieces * kCopy) off -= kPieces * kCopy, ++row, p += step;
            }
        } else if constexpr (kPieces <= 32) {
            constexpr int kRows = 32 / kPieces;  // of one copy of the warp's
            const int row = lane / kPieces;
            const bool in = lane % kPieces * kCopy < valid;
            const uint32_t mine = place + lane * kCopy;
            const char* p = in ? from : from - lane % kPieces * kCopy;
            const int64_t more = step * kRows;
            if (rows == kSteps) {
#pragma unroll
                for (int i = 0; i < kSteps / kRows; ++i, p += more) copy(mine + i * 32 * kCopy, p, in ? kCopy : 0);
            } else {
                const char* const first = p - row * step;
#pragma unroll
                for (int i = 0; i < kSteps / kRows; ++i, p += more) {
                    const bool here = i * kRows + row < rows;
                    copy(mine + i * 32 * kCopy, here ? p : first, in && here ? kCopy : 0);
                }
            }
        } else {
            constexpr int kTimes = kPieces / 32;
            const char* p = from;
#pragma unroll
            for (int i = 0; i < kSteps; ++i, p += step) {
#pragma unroll
                for (int m = 0; m < kTimes; ++m) {
                    const bool in = (m * 32 + lane) * kCopy < valid && i < rows;
                    copy(place + ((i * kTimes + m) * 32 + lane) * kCopy, in ? p + m * 32 * kCopy : from - lane * kCopy, in ? kCopy : 0);
                }
            }
        }
    }
    __device__ __forceinline__ void next() { from += jump; }

    // What a step's channels became, in the place that they came by; and (store) from there to `to`, this lane's first piece of the window: whole pieces of rows.  Pieces
    // of 4 bytes and less go to memory one by one, at `one`.
    static constexpr bool kPieced = CHUNK == 16;
    __device__ __forceinline__ void put(int j, int lane, char* one, const float (&y)[VEC], bool in) const {
        if constexpr (kPieced) Raw<T, VEC>::store(const_cast<char*>(place) + j * kBytes + lane * VEC * int(sizeof(T)), y);
        else if (in) Raw<T, VEC>::store(one, y);
    }
    __device__ __forceinline__ void store(char* to, int64_t bytes, int rows, int lane) const {
        if constexpr (kPieced) {
            __syncwarp();
            constexpr int kRows = 32 / kPieces;
            const int row = lane / kPieces;
            if (lane % kPieces * kCopy >= valid) return;
            const uint4* mine = reinterpret_cast<const uint4*>(place) + lane;
            char* p = to;
#pragma unroll
            for (int i = 0; i < kSteps / kRows; ++i, p += bytes * kRows) {
                if (i * kRows + row < rows) *reinterpret_cast<uint4*>(p) = mine[i * 32];
            }
        }
    }
    // This lane's first piece of a result's window, or (other pieces) its channels at the window's first step.
    static __device__ __forceinline__ char* first_piece(char* strip, int64_t bytes, uint32_t t, int lane) {
        if constexpr (kPieced) return strip + (t + lane / kPieces) * bytes + lane % kPieces * kCopy;
        else return strip + t * bytes + lane * VEC * int(sizeof(T));
    }
    // The window that begins at `base` lies at `at`.
    __device__ __forceinline__ void look(const char* at, const char* base) {
        place = at;
        if constexpr (kAround) low = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(base));
    }
    __device__ __forceinline__ Raw<T, VEC> get(int j, int lane) const {
        Raw<T, VEC> x;
        const char* p = place + j * kBytes + lane * VEC * int(sizeof(T));
        if constexpr (kAround) p += (low + j * static_cast<uint32_t>(step)) & 2;
        x.load(p);
        return x;
    }
};
// Windows in shared memory of a warp's `bytes` each: two or three, and two blocks of 8 warps on an SM (or one of 16) where they fit.
constexpr int kFewBytes = 101376;
__host__ __device__ constexpr int stages_of(int bytes) { return kWarps * bytes * 3 <= kFewBytes ? 3 : kWarps * bytes * 2 <= kFewBytes ? 2 : kWarps * bytes * 3 <= 2 * kFewBytes ? 3 : 2; }
__host__ __device__ constexpr int blocks_of(int bytes) { return kWarps * bytes * stages_of(bytes) <= kFewBytes ? 2 : 1; }
template <typename T, typename G, int VEC, int CHUNK, bool BACK>
constexpr int kWindowBytes = (BACK ? 2 : 1) * Steps<T, VEC, CHUNK>::kPlace + Steps<G, VEC, CHUNK>::kPlace;
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// The first walk through a window's steps, of which `left` are the sequence's: what they do to a state, by themselves and all together.
template <int KIND, int VEC, typename X, typename Y>
__device__ __forceinline__ void take_steps(const X& x, const Y& gate, int lane, int left, float (&a)[kSteps][VEC], float (&b)[kSteps][VEC], Run<KIND, VEC>& own) {
    own.begin();
    float gate_sum[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) gate_sum[e] = 0.f;
    auto take = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            float xs[VEC], gs[VEC], c[VEC], d[VEC], input[VEC];
            x.get(j, lane).get(xs);
            gate.get(j, lane).get(gs);
            if (!whole.value && j >= left) {  // the state stays
#pragma unroll
                for (int e = 0; e < VEC; ++e) gs[e] = KIND == B200_GATES_SIGMOID ? INFINITY : 0.f, xs[e] = 0.f;
            }
            gates_of<KIND>(gs, c, a[j], d, input);
            mul_v(b[j], input, xs);
            if constexpr (KIND == B200_GATES_SIGMOID) own.decays(a[j], d);
            else add_v(gate_sum, gate_sum, gs);
            own.adds(a[j], b[j]);
        }
    };
    if (left == kSteps) take(std::true_type{});
    else take(std::false_type{});
    if constexpr (KIND == B200_GATES_EXP) own.decays_of_sum(gate_sum);
}
// The second one, from the state h in front of them, to `rows` rows of the result.
template <int VEC, typename X>
__device__ __forceinline__ void put_steps(const X& x, int lane, bool in, int left, int rows, char* out, int64_t step, const float (&a)[kSteps][VEC], const float (&b)[kSteps][VEC], float (&h)[VEC]) {
    auto put = [&](auto whole) {
        char* p = out;
#pragma unroll
        for (int j = 0; j < kSteps; ++j, p += step) {
            fma_v(h, a[j], h, b[j]);  // (a's rounding counts within these steps only)
            float y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) y[e] = whole.value || j < left ? h[e] : 0.f;
            x.put(j, lane, p, y, in && (whole.value || j < rows));
        }
    };
    if (left == kSteps) put(std::true_type{});
    else put(std::false_type{});
    x.store(out, step, rows, lane);
}

// CLUSTER: whether `blocks` of them may be a cluster.
template <typename T, typename G, int KIND, int VEC, int CHUNK, bool CLUSTER>
__global__ void __launch_bounds__(32 * (blocks_of(kWindowBytes<T, G, VEC, CHUNK, false>) == 2 ? kMostWarps : kWarps), 1) walk_kernel(const Args k, uint32_t strips, uint32_t blocks) {
    const uint32_t cluster = CLUSTER ? blocks : 1;
    constexpr int kBytes = kWindowBytes<T, G, VEC, CHUNK, false>, kStages = stages_of(kBytes);
    using X = Steps<T, VEC, CHUNK>;
    using Y = Steps<G, VEC, CHUNK>;
    extern __shared__ __align__(16) char ring[];
    __shared__ uint64_t bars[2];
    __shared__ int given_up;
    const Told<VEC> told{reinterpret_cast<float*>(ring + blockDim.x / 32 * kStages * kBytes), static_cast<int>(blockDim.x / 32), bars, &given_up};
    pdl_prologue();
    if (cluster > 1) begin_cluster(told, 2);
    const Place<VEC> at(k, strips, cluster);
    const uint32_t length = static_cast<uint32_t>(k.length), n = static_cast<uint32_t>(steps_of(k, at.b)), span = at.span();
    const uint32_t windows = (length + span - 1) / span;
    X x;
    Y gate;
    x.begin(at.template strip<T>(k.x), k.x.step, at.first(), span, at.valid(k.width, sizeof(T)), at.lane);
    gate.begin(at.template strip<G>(k.gate), k.gate.step, at.first(), span, at.valid(k.width, sizeof(G)), at.lane);
    char* out = X::first_piece(const_cast<char*>(at.template strip<T>(k.out)), k.out.step, at.first(), at.lane);
    const int64_t out_jump = span * k.out.step;
    const char* x_at = at.template strip<T>(k.x) + at.first() * k.x.step;  // (of the window that is computed: X::kAround asks)
    const char* gate_at = at.template strip<G>(k.gate) + at.first() * k.gate.step;
    char *const places = ring + at.warp * kBytes, *const end = places + kStages * at.warps * kBytes, *read = places, *write = places;
    const int apart = at.warps * kBytes;
    uint32_t t = at.first(), t_load = t, w_load = 0;
    auto load = [&]() {
        if (w_load < windows && t_load < length) {
            const int rows = t_load < n ? static_cast<int>(min(n - t_load, uint32_t(kSteps))) : 0;
            x.load(write, rows, at.lane);
            gate.load(write + X::kPlace, rows, at.lane);
        }
        copies_commit();
        x.next(), gate.next();
        ++w_load, t_load += span;
        write += apart;
        if (write == end) write = places;
    };
    for (int i = 0; i < kStages - 1; ++i) load();
    float carry[VEC];
    load_end<VEC>(carry, k.initial, at.b, at.ch, at.in);
    if (at.warp == 0) put_row<VEC>(told.front(0), at.lane, carry);
    for (uint32_t w = 0; w < windows; ++w, t += span, out += out_jump) {
        copies_wait<kStages - 2>();
        __syncwarp();
        x.look(read, x_at);
        gate.look(read + X::kPlace, gate_at);
        if constexpr (X::kAround) x_at += x.jump;
        if constexpr (Y::kAround) gate_at += gate.jump;
        read += apart;
        if (read == end) read = places;
        load();  // (where the window before lay)
        float a[kSteps][VEC], b[kSteps][VEC];
        Run<KIND, VEC> own;
        const int left = t < n ? static_cast<int>(min(n - t, uint32_t(kSteps))) : 0;  // steps of the sequence
        take_steps<KIND, VEC>(x, gate, at.lane, left, a, b, own);
        float h[VEC];
        join<KIND, VEC, false>(told, w, at.warp, at.lane, at.rank, at.cluster, k.status, own, h, carry);
        if (t >= length) continue;
        if (k.states != nullptr && at.in) Raw<float, VEC>::store(reinterpret_cast<char*>(k.states + (int64_t(at.b) * k.chunks + t / kSteps) * k.width + at.ch), h);
        const int rows = static_cast<int>(min(length - t, uint32_t(kSteps)));
        put_steps<VEC>(x, at.lane, at.in, left, rows, out, k.out.step, a, b, h);
    }
    if (k.final_state.base != nullptr && at.rank == 0 && at.warp == at.warps - 1 && at.in) store_end<VEC>(k.final_state, at.b, at.ch, carry);
    if (cluster > 1) end_cluster();
}

// Clusters whose lanes have a channel each: what a window's segments do to a state is told a window ahead, so that the wait for the other blocks is one for what was sent
// while this window was gone through the first time.  (Two windows' steps in registers, and four places to be told at: a block that is told of the fourth window from here has
// told this one's cluster of the second, behind its reading of this one.)  For halves: 32768 steps of 1024 channels 78 us (kind exp 92 to 94), 103 with a wait in every window.  In F32 its
// second window in registers costs what it saves (50000 steps of 1000 channels 160 us where it was 150 without).
template <typename T, typename G, int KIND, int CHUNK>
__global__ void __launch_bounds__(32 * (blocks_of(kWindowBytes<T, G, 1, CHUNK, false>) == 2 ? kMostWarps : kWarps), 1) walk_ahead_kernel(const Args k, uint32_t strips, uint32_t cluster) {
    constexpr int kBytes = kWindowBytes<T, G, 1, CHUNK, false>, kStages = stages_of(kBytes);
    static_assert(kStages == 3);  // (one is loaded, one gone through the first time, one the second time)
    using X = Steps<T, 1, CHUNK>;
    using Y = Steps<G, 1, CHUNK>;
    extern __shared__ __align__(16) char ring[];
    __shared__ uint64_t bars[kAheadSlots];
    __shared__ int given_up;
    const Told<1> told{reinterpret_cast<float*>(ring + blockDim.x / 32 * kStages * kBytes), static_cast<int>(blockDim.x / 32), bars, &given_up};
    pdl_prologue();
    begin_cluster(told, kAheadSlots);
    const Place<1> at(k, strips, cluster);
    const uint32_t length = static_cast<uint32_t>(k.length), n = static_cast<uint32_t>(steps_of(k, at.b)), span = at.span();
    const uint32_t windows = (length + span - 1) / span;
    X x;
    Y gate;
    x.begin(at.template strip<T>(k.x), k.x.step, at.first(), span, at.valid(k.width, sizeof(T)), at.lane);
    gate.begin(at.template strip<G>(k.gate), k.gate.step, at.first(), span, at.valid(k.width, sizeof(G)), at.lane);
    char* out = X::first_piece(const_cast<char*>(at.template strip<T>(k.out)), k.out.step, at.first(), at.lane);
    const int64_t out_jump = span * k.out.step;
    // (a window is 32 steps or more: what X::kAround asks of its address is the same for all)
    const char *const x_at = at.template strip<T>(k.x) + at.first() * k.x.step, *const gate_at = at.template strip<G>(k.gate) + at.first() * k.gate.step;
    char *const places = ring + at.warp * kBytes, *const end = places + kStages * at.warps * kBytes, *read = places, *write = places;
    const int apart = at.warps * kBytes;
    uint32_t t_load = at.first(), w_load = 0;
    auto load = [&]() {
        if (w_load < windows && t_load < length) {
            const int rows = t_load < n ? static_cast<int>(min(n - t_load, uint32_t(kSteps))) : 0;
            x.load(write, rows, at.lane);
            gate.load(write + X::kPlace, rows, at.lane);
        }
        copies_commit();
        x.next(), gate.next();
        ++w_load, t_load += span;
        write += apart;
        if (write == end) write = places;
    };
    load();
    float carry[1];
    load_end<1>(carry, k.initial, at.b, at.ch, at.in);
    struct Window {
        float a[kSteps][1], b[kSteps][1], decay[1], sum[1];  // (decay, sum: of the segments in front of this one, in this block)
        int left;
        const char* place;
    } next;
    uint32_t t_first = at.first();
    auto first = [&](uint32_t w) {
        __syncwarp();
        load();  // (where the window before the last one lay)
        copies_wait<1>();
        __syncwarp();
        x.look(read, x_at);
        gate.look(read + X::kPlace, gate_at);
        next.place = read;
        read += apart;
        if (read == end) read = places;
        next.left = t_first < n ? static_cast<int>(min(n - t_first, uint32_t(kSteps))) : 0;
        t_first += span;
        Run<KIND, 1> own;
        take_steps<KIND, 1>(x, gate, at.lane, next.left, next.a, next.b, own);
        tell_ahead<KIND, false>(told, w & 1, w % kAheadSlots, at.warp, at.lane, at.rank, cluster, own, next.decay, next.sum);
    };
    first(0);
    uint32_t t = at.first();
    for (uint32_t w = 0; w < windows; ++w, t += span, out += out_jump) {
        const Window now = next;
        if (w + 1 < windows) first(w + 1);
        float h[1];
        hear_ahead<KIND, false>(told, w, at.lane, at.rank, cluster, k.status, now.decay, now.sum, carry, h);
        if (t >= length) continue;
        if (k.states != nullptr && at.in) Raw<float, 1>::store(reinterpret_cast<char*>(k.states + (int64_t(at.b) * k.chunks + t / kSteps) * k.width + at.ch), h);
        x.place = now.place;
        put_steps<1>(x, at.lane, at.in, now.left, static_cast<int>(min(length - t, uint32_t(kSteps))), out, k.out.step, now.a, now.b, h);
    }
    if (k.final_state.base != nullptr && at.rank == 0 && at.warp == at.warps - 1 && at.in) store_end<1>(k.final_state, at.b, at.ch, carry);
    end_cluster();
}

// The gradient of a step's result, of `left` steps that are the sequence's.
template <int VEC, typename X>
__device__ __forceinline__ void step_gradient(const X& dout, bool with_dout, int lane, int left, int j, float (&d)[VEC]) {
    if (with_dout && j < left) {
        dout.get(j, lane).get(d);
        return;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) d[e] = 0.f;
}
// The first walk through a window's steps, from the state h in front of them: their decays, what dgate takes of them, and what they do to a gradient that comes from behind.
template <int KIND, int VEC, typename X, typename Y>
__device__ __forceinline__ void take_back_steps(const X& x, const Y& gate, const X& dout, bool with_dout, int lane, int left, float (&h)[VEC], float (&c)[kSteps][VEC], float (&u)[kSteps][VEC],
                                                Run<KIND, VEC>& own) {
    own.begin();
    float gate_sum[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) gate_sum[e] = 0.f;
    auto take = [&](auto whole) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            float xs[VEC], gs[VEC], a[VEC], d[VEC], input[VEC], b[VEC];
            x.get(j, lane).get(xs);
            gate.get(j, lane).get(gs);
            if (!whole.value && j >= left) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) gs[e] = KIND == B200_GATES_SIGMOID ? INFINITY : 0.f, xs[e] = 0.f;
            }
            gates_of<KIND>(gs, c[j], a, d, input);
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[j][e] = KIND == B200_GATES_SIGMOID ? h[e] - xs[e] : h[e];
            mul_v(b, input, xs);
            if constexpr (KIND == B200_GATES_SIGMOID) {  // what the steps' gradients make of the state in front of them: each times the a's up to it
                float ds[VEC];
                own.decays(a, d);
                step_gradient<VEC>(dout, with_dout, lane, left, j, ds);
                fma_v(own.sum, own.a, ds, own.sum);
            } else {
                add_v(gate_sum, gate_sum, gs);
            }
            fma_v(h, a, h, b);  // (a's rounding counts within these steps only, here and below)
        }
    };
    if (left == kSteps) take(std::true_type{});
    else take(std::false_type{});
    if constexpr (KIND == B200_GATES_EXP) {  // (a product of the a's up to a step may be beyond F32, that step's gradient times it not)
        own.decays_of_sum(gate_sum);
#pragma unroll
        for (int j = kSteps - 1; j >= 0; --j) {
            float ds[VEC], a[VEC], unused[2];
            step_gradient<VEC>(dout, with_dout, lane, left, j, ds);
#pragma unroll
            for (int e = 0; e < VEC; ++e) slopes<KIND>(c[j][e], unused[0], unused[1], a[e]);
            add_v(own.sum, own.sum, ds);
            mul_v(own.sum, a, own.sum);
        }
    }
}
// The second one, from the gradient `later` behind them, to `rows` rows of the results.
template <int KIND, int VEC, typename X, typename Y>
__device__ __forceinline__ void put_back_steps(const X& x, const Y& gate, const X& dout, bool with_dout, int lane, bool there, int left, int rows, char* dx, char* dgate, int64_t dx_step, int64_t dgate_step, bool with_dx, bool with_dgate,
                                               const float (&c)[kSteps][VEC], const float (&u)[kSteps][VEC], float (&later)[VEC]) {
    auto put = [&](auto whole) {
        char *to_x = dx + (kSteps - 1) * dx_step, *to_gate = dgate + (kSteps - 1) * dgate_step;
#pragma unroll
        for (int j = kSteps - 1; j >= 0; --j, to_x -= dx_step, to_gate -= dgate_step) {
            float D[VEC], px[VEC], pg[VEC], slope[VEC], input[VEC], a[VEC];
            step_gradient<VEC>(dout, with_dout, lane, left, j, D);
            add_v(D, D, later);
#pragma unroll
            for (int e = 0; e < VEC; ++e) slopes<KIND>(c[j][e], slope[e], input[e], a[e]);
            mul_v(later, a, D);
            mul_v(px, input, D);
            mul_v(pg, slope, u[j]);
            mul_v(pg, pg, D);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (!whole.value && j >= left) px[e] = pg[e] = 0.f;
            }
            const bool in = there && (whole.value || j < rows);
            if (with_dx) x.put(j, lane, to_x, px, in);
            if (with_dgate) gate.put(j, lane, to_gate, pg, in);
        }
    };
    if (left == kSteps) put(std::true_type{});
    else put(std::false_type{});
    if (with_dx) x.store(dx, dx_step, rows, lane);
    if (with_dgate) gate.store(dgate, dgate_step, rows, lane);
}

// CLUSTER: whether `blocks` of them may be a cluster.
template <typename T, typename G, int KIND, int VEC, int CHUNK, bool CLUSTER>
__global__ void __launch_bounds__(32 * (blocks_of(kWindowBytes<T, G, VEC, CHUNK, true>) == 2 ? kMostWarps : kWarps), 1) walk_backward_kernel(const Args k, uint32_t strips, uint32_t blocks) {
    const uint32_t cluster = CLUSTER ? blocks : 1;
    constexpr int kBytes = kWindowBytes<T, G, VEC, CHUNK, true>, kStages = stages_of(kBytes);
    using X = Steps<T, VEC, CHUNK>;
    using Y = Steps<G, VEC, CHUNK>;
    extern __shared__ __align__(16) char ring[];
    __shared__ uint64_t bars[2];
    __shared__ int given_up;
    const Told<VEC> told{reinterpret_cast<float*>(ring + blockDim.x / 32 * kStages * kBytes), static_cast<int>(blockDim.x / 32), bars, &given_up};
    pdl_prologue();
    if (cluster > 1) begin_cluster(told, 2);
    const Place<VEC> at(k, strips, cluster);
    const uint32_t length = static_cast<uint32_t>(k.length), n = static_cast<uint32_t>(steps_of(k, at.b)), span = at.span();
    const uint32_t windows = (length + span - 1) / span;
    // windows from the last on
    uint32_t t = (windows - 1) * span + at.first(), t_load = t, w_load = 0;
    X x, dout;
    Y gate;
    const bool with_dout = k.dout.base != nullptr;
    x.begin(at.template strip<T>(k.x), k.x.step, t, -int64_t(span), at.valid(k.width, sizeof(T)), at.lane);
    gate.begin(at.template strip<G>(k.gate), k.gate.step, t, -int64_t(span), at.valid(k.width, sizeof(G)), at.lane);
    if (with_dout) dout.begin(at.template strip<T>(k.dout), k.dout.step, t, -int64_t(span), at.valid(k.width, sizeof(T)), at.lane);
    const bool with_dx = k.dx.base != nullptr, with_dgate = k.dgate.base != nullptr;
    char* dx = with_dx ? X::first_piece(const_cast<char*>(at.template strip<T>(k.dx)), k.dx.step, t, at.lane) : nullptr;
    char* dgate = with_dgate ? Y::first_piece(const_cast<char*>(at.template strip<G>(k.dgate)), k.dgate.step, t, at.lane) : nullptr;
    const char *x_at = at.template strip<T>(k.x) + t * k.x.step, *gate_at = at.template strip<G>(k.gate) + t * k.gate.step, *dout_at = nullptr;
    if (with_dout) dout_at = at.template strip<T>(k.dout) + t * k.dout.step;
    char *const places = ring + at.warp * kBytes, *const end = places + kStages * at.warps * kBytes, *read = places, *write = places;
    const int apart = at.warps * kBytes;
    auto load = [&]() {
        if (w_load < windows && t_load < length) {
            const int rows = t_load < n ? static_cast<int>(min(n - t_load, uint32_t(kSteps))) : 0;
            x.load(write, rows, at.lane);
            gate.load(write + X::kPlace, rows, at.lane);
            if (with_dout) dout.load(write + X::kPlace + Y::kPlace, rows, at.lane);
        }
        copies_commit();
        x.next(), gate.next();
        if (with_dout) dout.next();
        ++w_load, t_load -= span;
        write += apart;
        if (write == end) write = places;
    };
    for (int i = 0; i < kStages - 1; ++i) load();
    const float* const states = k.states + int64_t(at.b) * k.chunks * k.width + at.ch;
    Raw<float, VEC> rh;  // the state in front of the next window's steps
    auto load_state = [&](uint32_t t) {
        rh.clear();
        if (at.in && t < n) rh.load(reinterpret_cast<const char*>(states + int64_t(t / kSteps) * k.width));
    };
    load_state(t);
    float carry[VEC];
    load_end<VEC>(carry, k.final_state, at.b, at.ch, at.in);
    if (at.warp == 0) put_row<VEC>(told.front(0), at.lane, carry);
    for (uint32_t w = 0; w < windows; ++w, t -= span) {
        float c[kSteps][VEC], u[kSteps][VEC], h[VEC];
        rh.get(h);
        copies_wait<kStages - 2>();
        __syncwarp();
        x.look(read, x_at);
        gate.look(read + X::kPlace, gate_at);
        dout.look(read + X::kPlace + Y::kPlace, dout_at);
        if constexpr (X::kAround) {
            x_at += x.jump;
            if (with_dout) dout_at += dout.jump;
        }
        if constexpr (Y::kAround) gate_at += gate.jump;
        read += apart;
        if (read == end) read = places;
        load();  // (where the window before lay)
        if (w + 1 < windows) load_state(t - span);
        Run<KIND, VEC> own;
        const int left = t < n ? static_cast<int>(min(n - t, uint32_t(kSteps))) : 0;  // steps of the sequence
        take_back_steps<KIND, VEC>(x, gate, dout, with_dout, at.lane, left, h, c, u, own);
        float later[VEC];
        join<KIND, VEC, true>(told, w, at.warp, at.lane, at.rank, at.cluster, k.status, own, later, carry);
        if (t < length) {
            const int rows = static_cast<int>(min(length - t, uint32_t(kSteps)));
            put_back_steps<KIND, VEC>(x, gate, dout, with_dout, at.lane, at.in, left, rows, dx, dgate, k.dx.step, k.dgate.step, with_dx, with_dgate, c, u, later);
        }
        dx -= int64_t(span) * k.dx.step, dgate -= int64_t(span) * k.dgate.step;
    }
    if (k.initial.base != nullptr && at.rank == 0 && at.warp == 0 && at.in) store_end<VEC>(k.initial, at.b, at.ch, carry);
    if (cluster > 1) end_cluster();
}

// As walk_ahead_kernel.
template <typename T, typename G, int KIND, int CHUNK>
__global__ void __launch_bounds__(32 * (blocks_of(kWindowBytes<T, G, 1, CHUNK, true>) == 2 ? kMostWarps : kWarps), 1) walk_backward_ahead_kernel(const Args k, uint32_t strips, uint32_t cluster) {
    constexpr int kBytes = kWindowBytes<T, G, 1, CHUNK, true>, kStages = stages_of(kBytes);
    static_assert(kStages == 3);
    using X = Steps<T, 1, CHUNK>;
    using Y = Steps<G, 1, CHUNK>;
    extern __shared__ __align__(16) char ring[];
    __shared__ uint64_t bars[kAheadSlots];
    __shared__ int given_up;
    const Told<1> told{reinterpret_cast<float*>(ring + blockDim.x / 32 * kStages * kBytes), static_cast<int>(blockDim.x / 32), bars, &given_up};
    pdl_prologue();
    begin_cluster(told, kAheadSlots);
    const Place<1> at(k, strips, cluster);
    const uint32_t length = static_cast<uint32_t>(k.length), n = static_cast<uint32_t>(steps_of(k, at.b)), span = at.span();
    const uint32_t windows = (length + span - 1) / span;
    // windows from the last on
    uint32_t t = (windows - 1) * span + at.first(), t_load = t, t_first = t, w_load = 0;
    X x, dout;
    Y gate;
    const bool with_dout = k.dout.base != nullptr;
    x.begin(at.template strip<T>(k.x), k.x.step, t, -int64_t(span), at.valid(k.width, sizeof(T)), at.lane);
    gate.begin(at.template strip<G>(k.gate), k.gate.step, t, -int64_t(span), at.valid(k.width, sizeof(G)), at.lane);
    if (with_dout) dout.begin(at.template strip<T>(k.dout), k.dout.step, t, -int64_t(span), at.valid(k.width, sizeof(T)), at.lane);
    const bool with_dx = k.dx.base != nullptr, with_dgate = k.dgate.base != nullptr;
    char* dx = with_dx ? X::first_piece(const_cast<char*>(at.template strip<T>(k.dx)), k.dx.step, t, at.lane) : nullptr;
    char* dgate = with_dgate ? Y::first_piece(const_cast<char*>(at.template strip<G>(k.dgate)), k.dgate.step, t, at.lane) : nullptr;
    // (a window is 32 steps or more: what X::kAround asks of its address is the same for all)
    const char *const x_at = at.template strip<T>(k.x) + t * k.x.step, *const gate_at = at.template strip<G>(k.gate) + t * k.gate.step;
    const char* const dout_at = with_dout ? at.template strip<T>(k.dout) + t * k.dout.step : nullptr;
    char *const places = ring + at.warp * kBytes, *const end = places + kStages * at.warps * kBytes, *read = places, *write = places;
    const int apart = at.warps * kBytes;
    auto look = [&](const char* place) {
        x.look(place, x_at);
        gate.look(place + X::kPlace, gate_at);
        dout.look(place + X::kPlace + Y::kPlace, dout_at);
    };
    auto load = [&]() {
        if (w_load < windows && t_load < length) {
            const int rows = t_load < n ? static_cast<int>(min(n - t_load, uint32_t(kSteps))) : 0;
            x.load(write, rows, at.lane);
            gate.load(write + X::kPlace, rows, at.lane);
            if (with_dout) dout.load(write + X::kPlace + Y::kPlace, rows, at.lane);
        }
        copies_commit();
        x.next(), gate.next();
        if (with_dout) dout.next();
        ++w_load, t_load -= span;
        write += apart;
        if (write == end) write = places;
    };
    load();
    const float* const states = k.states + int64_t(at.b) * k.chunks * k.width + at.ch;
    Raw<float, 1> rh;  // the state in front of the next window's steps
    auto load_state = [&](uint32_t t) {
        rh.clear();
        if (at.in && t < n) rh.load(reinterpret_cast<const char*>(states + int64_t(t / kSteps) * k.width));
    };
    load_state(t);
    float carry[1];
    load_end<1>(carry, k.final_state, at.b, at.ch, at.in);
    struct Window {
        float c[kSteps][1], u[kSteps][1], decay[1], sum[1];  // (decay, sum: of the segments behind this one, in this block)
        int left;
        const char* place;
    } next;
    auto first = [&](uint32_t w) {
        float h[1];
        rh.get(h);
        __syncwarp();
        load();  // (where the window before the last one lay)
        copies_wait<1>();
        __syncwarp();
        look(read);
        next.place = read;
        read += apart;
        if (read == end) read = places;
        next.left = t_first < n ? static_cast<int>(min(n - t_first, uint32_t(kSteps))) : 0;
        t_first -= span;
        if (w + 1 < windows) load_state(t_first);
        Run<KIND, 1> own;
        take_back_steps<KIND, 1>(x, gate, dout, with_dout, at.lane, next.left, h, next.c, next.u, own);
        tell_ahead<KIND, true>(told, w & 1, w % kAheadSlots, at.warp, at.lane, at.rank, cluster, own, next.decay, next.sum);
    };
    first(0);
    for (uint32_t w = 0; w < windows; ++w, t -= span) {
        const Window now = next;
        if (w + 1 < windows) first(w + 1);
        float later[1];
        hear_ahead<KIND, true>(told, w, at.lane, at.rank, cluster, k.status, now.decay, now.sum, carry, later);
        if (t < length) {
            look(now.place);
            put_back_steps<KIND, 1>(x, gate, dout, with_dout, at.lane, at.in, now.left, static_cast<int>(min(length - t, uint32_t(kSteps))), dx, dgate, k.dx.step, k.dgate.step, with_dx, with_dgate, now.c,
                                    now.u, later);
        }
        dx -= int64_t(span) * k.dx.step, dgate -= int64_t(span) * k.dgate.step;
    }
    if (k.initial.base != nullptr && at.rank == 0 && at.warp == 0 && at.in) store_end<1>(k.initial, at.b, at.ch, carry);
    end_cluster();
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
    if (s.width >= (int64_t(1) << 30) || s.batch >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "x: 2^30 or more channels, or 2^31 or more sequences");
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

// How a call's blocks walk.
struct Walk {
    int warps = 0;   // of a block; 0: a thread to a channel
    int vec = 1;     // channels of a lane
    int chunk = 2;   // of Steps
    int cluster = 1;
    bool alone = false;  // a cluster's blocks have SMs to themselves, and there is room for them in every part of the device: twice the warps, where they fit
    int64_t strips = 0, blocks = 0;
};
struct Typed {
    Stream s;
    int dtype;
};
Walk walk_of(const Shape& s, const Args& k, std::initializer_list<Typed> streams) {
    Walk w;
    // Copies of 16 or of 4 bytes where every row lies on so many; two channels to a lane where every row has them side by side on an address for both.
    bool pairs = s.width % 2 == 0 && reinterpret_cast<uintptr_t>(k.states) % 8 == 0, halves = false;
    int chunk = 16;
    for (const Typed& t : streams) {
        if (t.s.base == nullptr) continue;
        const int64_t size = static_cast<int64_t>(dtype_size(t.dtype));
        auto on = [&](int64_t bytes) { return reinterpret_cast<uintptr_t>(t.s.base) % static_cast<uintptr_t>(bytes) == 0 && t.s.step % bytes == 0 && t.s.batch % bytes == 0; };
        halves |= t.dtype == B200_F16;
        pairs = pairs && on(2 * size);
        if (chunk == 16 && !(on(16) && s.width * size % 16 == 0)) chunk = 4;
        if (chunk == 4 && !(on(4) && s.width * size % 4 == 0)) chunk = 2;
    }
    w.vec = pairs && halves ? 2 : 1;
    w.chunk = halves && !pairs ? 2 : chunk;
    if (s.length <= kSteps) return w;
    w.warps = static_cast<int>(std::min<int64_t>(kWarps, ceil_div(s.length, kSteps)));
    // Blocks that leave half of the device's places (two to an SM) empty share their sequences' windows with another one each: 50000 steps of 1000 channels, F32, 423 us with
    // blocks by themselves, 313, 188 and 151 by clusters of 2, 4 and 8 (152 to 154 since products of growing decays are kept); 4 sequences of 4096 steps, 2048 channels, F16, 74 and, by two, 56.  Further apart than that a
    // cluster costs more than it gives: 8 such sequences 84 us by themselves, 106 by two, 111 by four.
    auto spread = [&]() {
        w.strips = ceil_div(s.width, 32 * w.vec);
        w.cluster = 1;
        while (w.cluster < kMostCluster && s.batch * w.strips * w.cluster * 2 <= int64_t(sm_count()) * 2 && s.length > int64_t(w.cluster) * w.warps * kSteps) w.cluster *= 2;
    };
    spread();
    // Half empty still: a channel to a lane, twice the blocks (1 sequence of 32768 steps, 1024 channels, F16: 78 us, 113 with two; its gradient 124 and 184).  Where two to a lane
    // leave less empty they are the faster ones (1 and 2 of 4096 steps, 2048 channels: 20.6 and 33 us, 22.6 and 41 with one).
    if (w.vec == 2 && w.cluster == kMostCluster && s.batch * w.strips * w.cluster * 2 <= int64_t(sm_count()) * 2) {
        w.vec = 1;
        spread();
    }
    w.alone = w.cluster == kMostCluster && s.batch * w.strips * w.cluster * 2 <= sm_count() && s.length > int64_t(w.cluster) * w.warps * kSteps;
    w.blocks = s.batch * w.strips * w.cluster;
    return w;
}

// Calls go(VEC, CHUNK) with what a walk has.
template <typename T, typename Fn>
void by_walk(const Walk& w, Fn&& go) {
    constexpr int kVec = sizeof(T) == 2 ? 2 : 1;
    if (w.chunk == 16) go(std::integral_constant<int, kVec>{}, std::integral_constant<int, 16>{});
    else if (w.chunk == 4) go(std::integral_constant<int, kVec>{}, std::integral_constant<int, 4>{});
    else if constexpr (kVec == 2) go(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
}

// ... and go(CHUNK), of halves.
template <typename Fn>
void by_chunk(const Walk& w, Fn&& go) {
    if (w.chunk == 16) go(std::integral_constant<int, 16>{});
    else if (w.chunk == 4) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 2>{});
}

template <int BYTES, int VEC, typename Kernel>
void launch_walk(b200_ctx* ctx, Kernel kernel, const Walk& w, const Args& k, int slots = 2) {
    const int warps = w.alone && blocks_of(BYTES) == 2 ? kMostWarps : w.warps;
    const size_t shared = static_cast<size_t>(warps) * stages_of(BYTES) * BYTES + Told<VEC>::bytes(warps, w.cluster > 1 ? slots : 0);
    const dim3 grid(static_cast<unsigned>(w.blocks)), threads(static_cast<unsigned>(32 * warps));
    (void)blocks_at_once(reinterpret_cast<const void*>(kernel), 32 * warps, shared);  // (allows that much shared memory)
    if (w.cluster == 1) launch_kernel(ctx, kernel, grid, threads, shared, k, static_cast<uint32_t>(w.strips), 1u);
    else launch_kernel_clustered(ctx, kernel, grid, threads, shared, w.cluster, false, k, static_cast<uint32_t>(w.strips), static_cast<uint32_t>(w.cluster));
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
    const Walk w = walk_of(s, k, {{k.x, a.x.dtype}, {k.gate, a.gate.dtype}, {k.out, a.out.dtype}});
    by_type(a.x, a.gate, a.kind, [&](auto t, auto g, auto kind) {
        using T = decltype(t);
        using G = decltype(g);
        constexpr int KIND = decltype(kind)::value;
        if (w.warps == 0) {
            auto go = [&](auto kernel, int vec) {
                launch_kernel(ctx, kernel, dim3(static_cast<unsigned>(ceil_div(s.width, kThreads * vec)), static_cast<unsigned>(std::min<int64_t>(s.batch, 65535))), dim3(kThreads), 0, k);
            };
            if (w.vec == 1) go(s.length <= 1 ? serial_kernel<T, G, KIND, 1, 1> : serial_kernel<T, G, KIND, 1, kSteps>, 1);
            else go(s.length <= 1 ? serial_kernel<T, G, KIND, 2, 1> : serial_kernel<T, G, KIND, 2, kSteps>, 2);
            return;
        }
        if constexpr (sizeof(T) == 2) {
            if (w.cluster > 1 && w.vec == 1) {
                by_chunk(w, [&](auto chunk) {
                    constexpr int CHUNK = decltype(chunk)::value;
                    launch_walk<kWindowBytes<T, G, 1, CHUNK, false>, 1>(ctx, walk_ahead_kernel<T, G, KIND, CHUNK>, w, k, kAheadSlots);
                });
                return;
            }
        }
        by_walk<T>(w, [&](auto vec, auto chunk) {
            constexpr int VEC = decltype(vec)::value, CHUNK = decltype(chunk)::value;
            constexpr int kBytes = kWindowBytes<T, G, VEC, CHUNK, false>;
            if constexpr (sizeof(T) == 2 && VEC == 1) launch_walk<kBytes, VEC>(ctx, walk_kernel<T, G, KIND, VEC, CHUNK, false>, w, k);
            else launch_walk<kBytes, VEC>(ctx, CHUNK == 16 && w.cluster == 1 ? walk_kernel<T, G, KIND, VEC, CHUNK, CHUNK != 16> : walk_kernel<T, G, KIND, VEC, CHUNK, true>, w, k);
        });
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
    const Walk w = walk_of(s, k, {{k.x, a.x.dtype}, {k.gate, a.gate.dtype}, {k.dout, a.x.dtype}, {k.dx, a.x.dtype}, {k.dgate, a.gate.dtype}});
    by_type(a.x, a.gate, a.kind, [&](auto t, auto g, auto kind) {
        using T = decltype(t);
        using G = decltype(g);
        constexpr int KIND = decltype(kind)::value;
        if (w.warps == 0) {
            auto go = [&](auto kernel, int vec) {
                launch_kernel(ctx, kernel, dim3(static_cast<unsigned>(ceil_div(s.width, kThreads * vec)), static_cast<unsigned>(std::min<int64_t>(s.batch, 65535))), dim3(kThreads), 0, k);
            };
            if (w.vec == 1) go(s.length <= 1 ? serial_backward_kernel<T, G, KIND, 1, 1> : serial_backward_kernel<T, G, KIND, 1, kSteps>, 1);
            else go(s.length <= 1 ? serial_backward_kernel<T, G, KIND, 2, 1> : serial_backward_kernel<T, G, KIND, 2, kSteps>, 2);
            return;
        }
        if constexpr (sizeof(T) == 2) {
            if (w.cluster > 1 && w.vec == 1) {
                by_chunk(w, [&](auto chunk) {
                    constexpr int CHUNK = decltype(chunk)::value;
                    launch_walk<kWindowBytes<T, G, 1, CHUNK, true>, 1>(ctx, walk_backward_ahead_kernel<T, G, KIND, CHUNK>, w, k, kAheadSlots);
                });
                return;
            }
        }
        by_walk<T>(w, [&](auto vec, auto chunk) {
            constexpr int VEC = decltype(vec)::value, CHUNK = decltype(chunk)::value;
            constexpr int kBytes = kWindowBytes<T, G, VEC, CHUNK, true>;
            if constexpr (sizeof(T) == 2 && VEC == 1) launch_walk<kBytes, VEC>(ctx, walk_backward_kernel<T, G, KIND, VEC, CHUNK, false>, w, k);
            else launch_walk<kBytes, VEC>(ctx, CHUNK == 16 && w.cluster == 1 ? walk_backward_kernel<T, G, KIND, VEC, CHUNK, CHUNK != 16> : walk_backward_kernel<T, G, KIND, VEC, CHUNK, true>, w, k);
        });
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
