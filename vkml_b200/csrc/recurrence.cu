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

// ---- blocks that walk along a sequence --------------------------------------
//
// A block, or a cluster of blocks, has 32 lanes' channels of a sequence and walks along it window by window; a warp has 16 steps of a window.  A thread computes what
// its steps do to a state that comes in (a decay and a sum: a step like any other), the warps tell each other by shared memory, the cluster's blocks by each
// other's, and every thread goes through its steps again from the state that does come in.  All of it stays in registers: gates and inputs are read once, and the
// next window's are under way while this one is computed.

constexpr int kMostWarps = 8;
constexpr int kMostCluster = 8;

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

// What a run of steps does to the state in front of it: their decays' product, as such and less 1 (either keeps digits that the other loses).
struct Product {
    float a = 1.f, less = 0.f;
    __device__ __forceinline__ void then(float c) {
        const float a1 = keeps(c) ? 1.f + c : c, less1 = keeps(c) ? c : c - 1.f;
        a *= a1;
        less = fmaf(less, less1, less) + less1;
    }
    __device__ __forceinline__ float decay() const { return less <= 0.f && less > -0.5f ? -fabsf(less) : a; }
};
// The decay of two runs, one behind the other.
__device__ __forceinline__ float both(float c, float d) {
    const float less = fmaf(c, d, c) + d;
    const float product = (keeps(c) ? 1.f + c : c) * (keeps(d) ? 1.f + d : d);
    return keeps(c) && keeps(d) ? (less > -0.5f ? -fabsf(less) : 1.f + less) : product;
}

// What the segments of a block, and the blocks of a cluster, do to a state: decay and sum, for every channel.  Two of each: a window's are read while the next one's
// are written.
template <int VEC>
struct Told {
    float2 segments[2][kMostWarps][32 * VEC];
    float2 blocks[2][kMostCluster][32 * VEC];
};

__device__ __forceinline__ void tell(float2* mine, uint32_t rank, float2 value) {
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(value.x), "f"(value.y) : "memory");
}

// The state that comes into this warp's steps, from `carry` in front of the window (which becomes that behind it), by every segment's decay and sum.  Segments
// come one after another, in the order of their warps and blocks, or (BACK) the other way round.
template <int VEC, bool BACK>
__device__ __forceinline__ void join(Told<VEC>& told, int parity, int warp, int lane, int warps, uint32_t rank, uint32_t cluster, const float2 (&own)[VEC], float (&carry)[VEC], float (&in)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) told.segments[parity][warp][e * 32 + lane] = own[e];
    __syncthreads();
    float begin[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) begin[e] = carry[e];
    if (cluster > 1) {
        float2 block[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) block[e] = make_float2(kHold, 0.f);
        for (int i = 0; i < warps; ++i) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 s = told.segments[parity][BACK ? warps - 1 - i : i][e * 32 + lane];
                block[e] = make_float2(both(block[e].x, s.x), apply(s.x, block[e].y, s.y));
            }
        }
        for (uint32_t to = warp; to < cluster; to += warps) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) tell(&told.blocks[parity][rank][e * 32 + lane], to, block[e]);
        }
        cluster_sync();
        for (uint32_t i = 0; i < cluster; ++i) {
            const uint32_t of = BACK ? cluster - 1 - i : i;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if (of == rank) begin[e] = carry[e];
                const float2 s = told.blocks[parity][of][e * 32 + lane];
                carry[e] = apply(s.x, carry[e], s.y);
            }
        }
    }
    for (int i = 0; i < warps; ++i) {
        const int of = BACK ? warps - 1 - i : i;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if (of == warp) in[e] = begin[e];
            const float2 s = told.segments[parity][of][e * 32 + lane];
            begin[e] = apply(s.x, begin[e], s.y);
        }
    }
    if (cluster == 1) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) carry[e] = begin[e];
    }
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
    __device__ __forceinline__ int64_t span() const { return int64_t(warps) * kSteps * cluster; }
    __device__ __forceinline__ int64_t first() const { return int64_t(rank * warps + warp) * kSteps; }
    template <typename T>
    __device__ __forceinline__ char* base(const Stream& s) const { return s.base != nullptr ? s.base + b * s.batch + int64_t(ch) * int64_t(sizeof(T)) : nullptr; }
};

// Sixteen steps of a stream, from step t on, where they are before n.
template <typename T, int VEC>
__device__ __forceinline__ void load_steps(Raw<T, VEC> (&r)[kSteps], const char* base, int64_t step, int64_t t, int64_t n, bool in) {
    const char* p = base + t * step;
    if (in && t + kSteps <= n) {
#pragma unroll
        for (int j = 0; j < kSteps; ++j) r[j].load(p + j * step);
    } else {
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            r[j].clear();
            if (in && t + j < n) r[j].load(p + j * step);
        }
    }
}

template <int VEC>
__device__ __forceinline__ void load_end(float (&h)[VEC], const RowsArg& end, int b, int ch, bool in) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[e] = end.base != nullptr && in ? reinterpret_cast<const float*>(end.base + b * end.step)[ch + e] : 0.f;
}

template <typename T, typename G, int KIND, int VEC>
__global__ void __launch_bounds__(32 * kMostWarps, 2) walk_kernel(const Args k, uint32_t strips, uint32_t cluster) {
    __shared__ Told<VEC> told;
    pdl_prologue();
    if (cluster > 1) cluster_sync();  // (every block is there before another writes to it)
    const Place<VEC> at(k, strips, cluster);
    const int64_t n = steps_of(k, at.b), span = at.span();
    const char *const x = at.template base<T>(k.x), *const gate = at.template base<G>(k.gate);
    char* const out = at.template base<T>(k.out);
    Raw<T, VEC> rx[kSteps];
    Raw<G, VEC> rg[kSteps];
    int64_t t = at.first();
    load_steps(rx, x, k.x.step, t, n, at.in);
    load_steps(rg, gate, k.gate.step, t, n, at.in);
    float carry[VEC];
    load_end<VEC>(carry, k.initial, at.b, at.ch, at.in);
    int parity = 0;
    for (int64_t begin = 0; begin < k.length; begin += span, t += span, parity ^= 1) {
        float c[kSteps][VEC], b[kSteps][VEC];
        Product product[VEC];
        float sum[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            float xs[VEC], gs[VEC];
            rx[j].get(xs);
            rg[j].get(gs);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float input;
                c[j][e] = decay<KIND>(gs[e], input);
                b[j][e] = input * xs[e];
                if (t + j >= n) c[j][e] = kHold, b[j][e] = 0.f;
                product[e].then(c[j][e]);
                sum[e] = apply(c[j][e], sum[e], b[j][e]);
            }
        }
        if (begin + span < k.length) {
            load_steps(rx, x, k.x.step, t + span, n, at.in);
            load_steps(rg, gate, k.gate.step, t + span, n, at.in);
        }
        float2 own[VEC];
        float h[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) own[e] = make_float2(product[e].decay(), sum[e]);
        join<VEC, false>(told, parity, at.warp, at.lane, at.warps, at.rank, at.cluster, own, carry, h);
        if (!at.in || t >= k.length) continue;
        if (k.states != nullptr) Raw<float, VEC>::store(reinterpret_cast<char*>(k.states + (int64_t(at.b) * k.chunks + t / kSteps) * k.width + at.ch), h);
        char* p = out + t * k.out.step;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            float y[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                h[e] = apply(c[j][e], h[e], b[j][e]);
                y[e] = t + j < n ? h[e] : 0.f;
            }
            if (t + j < k.length) Raw<T, VEC>::store(p + j * k.out.step, y);
        }
    }
    if (k.final_state.base != nullptr && at.rank == 0 && at.warp == 0 && at.in) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) reinterpret_cast<float*>(k.final_state.base + at.b * k.final_state.step)[at.ch + e] = carry[e];
    }
}

constexpr int kBackWarps = 4;

template <typename T, typename G, int KIND, int VEC>
__global__ void __launch_bounds__(32 * kBackWarps, 3) walk_backward_kernel(const Args k, uint32_t strips, uint32_t cluster) {
    __shared__ Told<VEC> told;
    pdl_prologue();
    if (cluster > 1) cluster_sync();  // (every block is there before another writes to it)
    const Place<VEC> at(k, strips, cluster);
    const int64_t n = steps_of(k, at.b), span = at.span();
    const char *const x = at.template base<T>(k.x), *const gate = at.template base<G>(k.gate), *const dout = at.template base<T>(k.dout);
    char *const dx = at.template base<T>(k.dx), *const dgate = at.template base<G>(k.dgate);
    const float* const states = k.states + int64_t(at.b) * k.chunks * k.width + at.ch;
    Raw<T, VEC> rx[kSteps], rd[kSteps];
    Raw<G, VEC> rg[kSteps];
    Raw<float, VEC> rh;
    const int64_t windows = (k.length + span - 1) / span;
    int64_t t = (windows - 1) * span + at.first();
    auto load = [&](int64_t t) {
        load_steps(rx, x, k.x.step, t, n, at.in);
        load_steps(rg, gate, k.gate.step, t, n, at.in);
        load_steps(rd, dout, k.dout.step, t, dout != nullptr ? n : 0, at.in);
        rh.clear();
        if (at.in && t < n) rh.load(reinterpret_cast<const char*>(states + t / kSteps * k.width));
    };
    load(t);
    float carry[VEC];
    load_end<VEC>(carry, k.final_state, at.b, at.ch, at.in);
    int parity = 0;
    for (int64_t w = windows - 1; w >= 0; --w, t -= span, parity ^= 1) {
        float c[kSteps][VEC], u[kSteps][VEC], d[kSteps][VEC], h[VEC];
        rh.get(h);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            float xs[VEC], gs[VEC];
            rx[j].get(xs);
            rg[j].get(gs);
            rd[j].get(d[j]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float input;
                c[j][e] = decay<KIND>(gs[e], input);
                u[j][e] = KIND == B200_GATES_SIGMOID ? h[e] - xs[e] : h[e];
                h[e] = apply(c[j][e], h[e], input * xs[e]);
                if (t + j >= n) c[j][e] = kHold;
            }
        }
        if (w > 0) load(t - span);
        Product product[VEC];
        float2 own[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            float sum = 0.f;
#pragma unroll
            for (int j = kSteps - 1; j >= 0; --j) {
                product[e].then(c[j][e]);
                sum = apply(c[j][e], d[j][e] + sum, 0.f);
            }
            own[e] = make_float2(product[e].decay(), sum);
        }
        float later[VEC];
        join<VEC, true>(told, parity, at.warp, at.lane, at.warps, at.rank, at.cluster, own, carry, later);
        if (!at.in || t >= k.length) continue;
#pragma unroll
        for (int j = kSteps - 1; j >= 0; --j) {
            float px[VEC], pg[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float D = d[j][e] + later[e];
                later[e] = apply(c[j][e], D, 0.f);
                float slope, input;
                slopes<KIND>(c[j][e], slope, input);
                const bool on = t + j < n;
                px[e] = on ? input * D : 0.f;
                pg[e] = on ? slope * u[j][e] * D : 0.f;
            }
            if (t + j < k.length) {
                if (dx != nullptr) Raw<T, VEC>::store(dx + (t + j) * k.dx.step, px);
                if (dgate != nullptr) Raw<G, VEC>::store(dgate + (t + j) * k.dgate.step, pg);
            }
        }
    }
    if (k.initial.base != nullptr && at.rank == 0 && at.warp == 0 && at.in) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) reinterpret_cast<float*>(k.initial.base + at.b * k.initial.step)[at.ch + e] = carry[e];
    }
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

// How a call's blocks walk.
struct Walk {
    int warps = 0;  // of a block; 0: a thread to a channel
    int vec = 1, cluster = 1;
    int64_t strips = 0, blocks = 0;
};
struct Typed {
    Stream s;
    int dtype;
};
Walk walk_of(const Shape& s, const Args& k, std::initializer_list<Typed> streams, int most_warps, int blocks_at_once) {
    Walk w;
    if (s.length <= kSteps) return w;
    // two channels to a lane where every row of halves has them side by side on an address for both
    bool pairs = s.width % 2 == 0 && reinterpret_cast<uintptr_t>(k.states) % 8 == 0, halves = false;
    for (const Typed& t : streams) {
        if (t.s.base == nullptr) continue;
        const int64_t bytes = 2 * static_cast<int64_t>(dtype_size(t.dtype));
        halves |= t.dtype == B200_F16;
        pairs = pairs && reinterpret_cast<uintptr_t>(t.s.base) % static_cast<uintptr_t>(bytes) == 0 && t.s.step % bytes == 0 && t.s.batch % bytes == 0;
    }
    w.vec = pairs && halves ? 2 : 1;
    w.strips = ceil_div(s.width, 32 * w.vec);
    w.warps = static_cast<int>(std::min<int64_t>(most_warps, ceil_div(s.length, kSteps)));
    while (w.cluster < kMostCluster && s.batch * w.strips * w.cluster < int64_t(sm_count()) * blocks_at_once && s.length > int64_t(w.cluster) * w.warps * kSteps) w.cluster *= 2;
    w.blocks = s.batch * w.strips * w.cluster;
    return w;
}

template <typename Kernel>
void launch_walk(b200_ctx* ctx, Kernel kernel, const Walk& w, const Args& k) {
    const dim3 grid(static_cast<unsigned>(w.blocks)), threads(static_cast<unsigned>(32 * w.warps));
    if (w.cluster == 1) launch_kernel(ctx, kernel, grid, threads, 0, k, static_cast<uint32_t>(w.strips), 1u);
    else launch_kernel_clustered(ctx, kernel, grid, threads, 0, w.cluster, false, k, static_cast<uint32_t>(w.strips), static_cast<uint32_t>(w.cluster));
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
    const Walk w = walk_of(s, k, {{k.x, a.x.dtype}, {k.gate, a.gate.dtype}, {k.out, a.out.dtype}}, kMostWarps, 2);
    by_type(a.x, a.gate, a.kind, [&](auto t, auto g, auto kind) {
        using T = decltype(t);
        using G = decltype(g);
        constexpr int KIND = decltype(kind)::value;
        if (w.warps == 0) {
            launch_kernel(ctx, serial_kernel<T, G, KIND>, dim3(static_cast<unsigned>(ceil_div(s.batch * s.width, kThreads))), dim3(kThreads), 0, k);
        } else if (w.vec == 1) {
            launch_walk(ctx, walk_kernel<T, G, KIND, 1>, w, k);
        } else if constexpr (sizeof(T) == 2) {
            launch_walk(ctx, walk_kernel<T, G, KIND, 2>, w, k);
        }
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
    const Walk w = walk_of(s, k, {{k.x, a.x.dtype}, {k.gate, a.gate.dtype}, {k.dout, a.x.dtype}, {k.dx, a.x.dtype}, {k.dgate, a.gate.dtype}}, kBackWarps, 3);
    by_type(a.x, a.gate, a.kind, [&](auto t, auto g, auto kind) {
        using T = decltype(t);
        using G = decltype(g);
        constexpr int KIND = decltype(kind)::value;
        if (w.warps == 0) {
            launch_kernel(ctx, serial_backward_kernel<T, G, KIND>, dim3(static_cast<unsigned>(ceil_div(s.batch * s.width, kThreads))), dim3(kThreads), 0, k);
        } else if (w.vec == 1) {
            launch_walk(ctx, walk_backward_kernel<T, G, KIND, 1>, w, k);
        } else if constexpr (sizeof(T) == 2) {
            launch_walk(ctx, walk_backward_kernel<T, G, KIND, 2>, w, k);
        }
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
