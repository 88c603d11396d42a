// Distillation from a teacher's top logits, with a share of cross-entropy on labels, forward and backward.
//
// For a row z of V logits, the teacher's logits t at K columns k_j, temperature T and hard weight c:
//
//   p = softmax(t / T)        q = softmax(z / T)        h = softmax(z)
//   loss = (1 - c) T^2 sum_j p_j (log p_j - log q_{k_j}) + c (log sum exp z - z_label)
//   grad = w [ (1 - c) T (q - p at k) + c (h - 1 at the label) ]
//
// Bound by memory: z read once and, with a gradient, as much written.  A row is a block's, or a cluster's whose blocks take a stretch of it each: up to
// kVectors vectors of 16 bytes to a thread, all under way at once and held in registers from the reading to the gradient, so that z is read once.  (Rows
// too long for a cluster of 8 are taken in batches and read again for the gradient.)  A thread finds the maximum of what it holds and the sums of
// exp((z - max) / T) and exp(z - max) beside it; the block, and then the cluster, joins these threes in one round.  The gradient's pass writes q and h in every
// column, and the K + 1 columns that the teacher or the label adds to are written again afterwards.
// Where both parts have a weight and T is not 1, an element takes two exponentials in each pass.
#include "operators.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace b200 {
namespace {

constexpr int kMostThreads = 512;
constexpr int kVectors = 8;
constexpr int kMostTop = 1024;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
    RowsArg logits, ids, teacher, labels, weights, grad;
    float* losses;
    float4* stats;
    FastDiv inner;
    uint32_t* status;
    int64_t vocab;
    int top;
    int slots;            // of a row's table of columns; 0: none
    int blocks;           // of a row's cluster
    bool wide_ids, wide_labels, half_teacher;
    bool soft, hard;      // which parts have a weight
    float temperature, inverse, hard_weight, grad_scale;
};

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A maximum of -inf (nothing but -inf so far) has sums of 0: differences to 0 keep them so.
__device__ __forceinline__ float shift_of(float top) { return top == -INFINITY ? 0.f : top; }

// Maximum, and the sums of exp((z - max) / T) and exp(z - max), of a part of a row.
struct Part {
    float top, soft, hard;
};

// Over the lanes of a warp, in each of them.
__device__ __forceinline__ Part warp_part(Part x, float c_soft, bool soft, bool hard) {
    float top = x.top;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float apart = x.top - shift_of(top);
    x.top = top;
    if (soft) {
        x.soft *= fast_exp2(apart * c_soft);
#pragma unroll
        for (int d = 16; d > 0; d /= 2) x.soft += __shfl_xor_sync(0xffffffffu, x.soft, d);
    }
    if (hard) {
        x.hard *= fast_exp2(apart * kLog2e);
#pragma unroll
        for (int d = 16; d > 0; d /= 2) x.hard += __shfl_xor_sync(0xffffffffu, x.hard, d);
    }
    return x;
}

// Elements of a row that lie before its first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int64_t head_of(const T* row, int64_t n) {
    const int64_t head = (16 - (reinterpret_cast<uintptr_t>(row) & 15)) % 16 / int64_t(sizeof(T));
    return head < n ? head : n;
}

template <typename T>
constexpr uint32_t kNothing = sizeof(T) == 2 ? 0xfc00fc00u : 0xff800000u;  // -inf

// The elements of a vector.  (Plain arithmetic on them: pairs in 64-bit registers, two to an instruction, cost more moves than they saved here.)
template <typename T>
__device__ __forceinline__ void unpack(const uint4& raw, float (&x)[16 / sizeof(T)]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store_vector(T* to, const float (&x)[16 / sizeof(T)], bool aligned) {
    if (aligned) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2) {
                const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                w[i] = __float_as_uint(x[i]);
            }
        }
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 16 / int(sizeof(T)); ++e) to[e] = from_float<T>(x[e]);
    }
}

// The largest element of NV vectors (halves compare as halves, two at a time).
template <typename T, int NV>
__device__ __forceinline__ float largest(const uint4 (&raw)[NV]) {
    if constexpr (sizeof(T) == 2) {
        const __half2* h = reinterpret_cast<const __half2*>(&raw[0]);
        __half2 m[2] = {__hmax2(h[0], h[1]), __hmax2(h[2], h[3])};
#pragma unroll
        for (int i = 1; i < NV; ++i) {
            const __half2* g = reinterpret_cast<const __half2*>(&raw[i]);
            m[0] = __hmax2(m[0], __hmax2(g[0], g[1]));
            m[1] = __hmax2(m[1], __hmax2(g[2], g[3]));
        }
        m[0] = __hmax2(m[0], m[1]);
        return fmaxf(__low2float(m[0]), __high2float(m[0]));
    } else {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(raw[i].x), __uint_as_float(raw[i].y)), fmaxf(__uint_as_float(raw[i].z), __uint_as_float(raw[i].w))));
        }
        return m;
    }
}

// Powers of two of (x - at) * c + plus as one multiply-add each, x * c + offset, where at * c is of a size that leaves the offset its digits: what its rounding
// took away is given back by the factor.  Where it is not (logits of the type's lowest value), the difference comes first.  The factor's terms are rounded one by
// one, as written: joined into multiply-adds they count the product's rounding twice (1e-4 of a row's sums at a maximum of 1400).
struct Exponent {
    float c, at, offset, factor;
    bool direct;
};
__device__ __forceinline__ bool is_direct(float at, float c) { return fabsf(at * c) < 4096.f; }
__device__ __forceinline__ Exponent exponent_of(float at, float c, float plus, bool direct) {
    Exponent x;
    const float p = __fmul_rn(at, c);
    x.c = c, x.at = at;
    x.direct = direct;
    x.offset = x.direct ? __fsub_rn(plus, p) : plus;
    x.factor = 1.f;
    if (x.direct) {  // plus - at c, without the offset that stands for it: the difference's rounding and the product's
        const float b = __fsub_rn(plus, x.offset), a = __fadd_rn(x.offset, b);
        const float lost = __fsub_rn(__fadd_rn(__fsub_rn(plus, a), __fsub_rn(b, p)), fmaf(at, c, -p));
        x.factor = fmaf(lost, 0.6931471805599453f, 1.f);
    }
    return x;
}
// Without the factor.
template <bool DIRECT>
__device__ __forceinline__ float power(const Exponent& x, float z) {
    if constexpr (!DIRECT) z -= x.at;
    return fast_exp2(fmaf(z, x.c, x.offset));
}

// Adds the elements of NV vectors to a part of a row.
template <typename T, bool DIRECT, int NV>
__device__ __forceinline__ float sum_powers(const Exponent& x, const uint4 (&raw)[NV]) {
    constexpr int E = 16 / sizeof(T);
    float sum[4] = {};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float z[E];
        unpack<T>(raw[i], z);
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e % 4] += power<DIRECT>(x, z[e]);
    }
    return ((sum[0] + sum[1]) + (sum[2] + sum[3])) * x.factor;
}
// A part of a row while its vectors come by: the maximum so far, the sums beside it, and what they are computed by.
struct Running {
    Part part;
    Exponent soft, hard;
    float c_soft;
    bool with_soft, with_hard;

    __device__ __forceinline__ void begin(float z, float c, bool use_soft, bool use_hard) {  // with one element, or -inf for none
        const float one = z == -INFINITY ? 0.f : 1.f + (z - z);  // (not a number where z is none or +inf, as it is in a vector)
        part = Part{z, one, one};
        c_soft = c, with_soft = use_soft, with_hard = use_hard;
        aim();
    }
    __device__ __forceinline__ void aim() {
        const float at = shift_of(part.top);
        soft = exponent_of(at, c_soft, 0.f, is_direct(at, c_soft));
        hard = exponent_of(at, kLog2e, 0.f, is_direct(at, kLog2e));
    }
    template <typename T, int NV>
    __device__ __forceinline__ void take(const uint4 (&raw)[NV]) {
        const float top = largest<T, NV>(raw);
        if (top > part.top) {
            part.soft *= fast_exp2((part.top - top) * c_soft);
            part.hard *= fast_exp2((part.top - top) * kLog2e);
            part.top = top;
            aim();
        }
        if (with_soft) part.soft += soft.direct ? sum_powers<T, true>(soft, raw) : sum_powers<T, false>(soft, raw);
        if (with_hard) part.hard += hard.direct ? sum_powers<T, true>(hard, raw) : sum_powers<T, false>(hard, raw);
    }
};

// What a row's gradient is made of: ws q + wh h, q = exp2((z - at) c_soft + soft2), h = exp2((z - at) log2 e + hard2).
struct RowGrad {
    float ws, wh, at, soft2, hard2;
};
struct GradPowers {
    Exponent soft, hard;
    float ws, wh;  // the exponents' factors included
    bool direct;   // both of them: a vector's elements take one form.  One whose weight is 0 is not asked
};
__device__ __forceinline__ GradPowers grad_powers(const RowGrad& g, float c_soft) {
    GradPowers x;
    x.direct = (g.ws == 0.f || is_direct(g.at, c_soft)) && (g.wh == 0.f || is_direct(g.at, kLog2e));
    x.soft = exponent_of(g.at, c_soft, g.soft2, x.direct);
    x.hard = exponent_of(g.at, kLog2e, g.hard2, x.direct);
    x.ws = g.ws != 0.f ? g.ws * x.soft.factor : 0.f;  // (a row that does not count may hold anything)
    x.wh = g.wh != 0.f ? g.wh * x.hard.factor : 0.f;
    return x;
}
__device__ __forceinline__ float grad_value(const GradPowers& x, float z) {
    float y = 0.f;
    if (x.ws != 0.f) y += x.ws * (x.direct ? power<true>(x.soft, z) : power<false>(x.soft, z));
    if (x.wh != 0.f) y += x.wh * (x.direct ? power<true>(x.hard, z) : power<false>(x.hard, z));
    return y;
}
template <typename T, bool DIRECT, int NV>
__device__ __forceinline__ void grad_vectors(const GradPowers& g, const uint4 (&raw)[NV], T* to, int apart_by, int count, bool aligned) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (i >= count) break;
        float z[E], y[E];
        unpack<T>(raw[i], z);
        if (g.ws != 0.f) {
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = power<DIRECT>(g.soft, z[e]) * g.ws;
            if (g.wh != 0.f) {
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] = fmaf(power<DIRECT>(g.hard, z[e]), g.wh, y[e]);
            }
        } else if (g.wh != 0.f) {
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = power<DIRECT>(g.hard, z[e]) * g.wh;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = 0.f;
        }
        store_vector<T>(to + i * apart_by, y, aligned);
    }
}
// The gradient in `count` vectors of a thread, `apart_by` elements from one to the next.
template <typename T, int NV>
__device__ __forceinline__ void put_grad(const GradPowers& g, const uint4 (&raw)[NV], T* to, int apart_by, int count, bool aligned) {
    if (g.direct) grad_vectors<T, true>(g, raw, to, apart_by, count, aligned);
    else grad_vectors<T, false>(g, raw, to, apart_by, count, aligned);
}

// A table of a row's columns in shared memory, which shows whether an entry is the only one of its column: open addressing, the sign of a slot set where
// more than one entry came.  At most a third of it is taken.  Rows of few entries compare each with all instead, which is as fast for 64 of them and takes twice as
// long for 256 (33554 x 1000 F32 with gradient: 706 us, 313 with the table).
constexpr int kMostCompared = 64;
constexpr int kEmptySlot = 0x7fffffff;  // (no column: rows have fewer than 2^31)
int table_slots(int top) {
    int slots = 256;
    while (slots < top * 3) slots *= 2;
    return top <= kMostCompared ? 0 : slots;
}
__device__ __forceinline__ void clear_table(int* table, int slots, int t, int threads) {
    for (int i = t * 4; i < slots; i += threads * 4) *reinterpret_cast<int4*>(table + i) = make_int4(kEmptySlot, kEmptySlot, kEmptySlot, kEmptySlot);
}
__device__ __forceinline__ uint32_t first_slot(int c, int slots) { return (static_cast<uint32_t>(c) * 0x9e3779b1u) >> 16 & (slots - 1); }
__device__ __forceinline__ void enter_column(int* table, int slots, int c) {
    for (uint32_t at = first_slot(c, slots);; at = (at + 1) & (slots - 1)) {
        const int seen = atomicCAS(&table[at], kEmptySlot, c);
        if (seen == kEmptySlot) return;
        if ((seen & 0x7fffffff) == c) {
            atomicOr(&table[at], static_cast<int>(0x80000000u));
            return;
        }
    }
}
__device__ __forceinline__ bool column_alone(const int* table, int slots, int c) {
    for (uint32_t at = first_slot(c, slots);; at = (at + 1) & (slots - 1)) {
        if ((table[at] & 0x7fffffff) == c) return table[at] >= 0;
    }
}

// What p and the label take off the gradient's column col[j], if entry j is the first that names it.  The columns lie on a 16-byte boundary, `top` + 1 of
// them and none (-1) up to the next multiple of four.  Almost always an entry is alone.
__device__ __forceinline__ bool entry_takes(const RowGrad& row, const int* col, const float* p, const int* table, int slots, int top, bool soft, int j, float& minus) {
    const int c = col[j];
    bool alone;
    if (slots > 0) {
        alone = column_alone(table, slots, c);
    } else {
        int equal = 0;
#pragma unroll 4
        for (int m = 0; m <= top; m += 4) {
            const int4 four = *reinterpret_cast<const int4*>(col + m);
            equal += (four.x == c) + (four.y == c) + (four.z == c) + (four.w == c);
        }
        alone = equal == 1;
    }
    minus = 0.f;
    if (alone) {
        if (j == top) minus = row.wh;
        else if (row.ws != 0.f) minus = row.ws * p[j];
        return true;
    }
    for (int m = 0; m < top && soft; m += 4) {
        const int4 four = *reinterpret_cast<const int4*>(col + m);
        if (four.x != c && four.y != c && four.z != c && four.w != c) continue;
        for (int e = m; e < m + 4 && e < top; ++e) {
            if (col[e] != c) continue;
            if (e < j) return false;
            if (row.ws != 0.f) minus += row.ws * p[e];
        }
    }
    if (col[top] == c) minus += row.wh;
    return true;
}
// Arrays of a row's entries in shared memory: the columns [top + 1 and up to 3 of none], probabilities [top], logits there [top + 1]; the table comes behind.
__host__ __device__ __forceinline__ int entry_words(int top) { return (top / 4 + 1) * 4 + (top + 3) / 4 * 4 + (top / 4 + 1) * 4; }

// Few rows, or short ones: a block or a cluster to a row.  Its warps meet as seldom as can be, since that is what a row of few vectors takes its time for: when
// the teacher's entries are there, when the warps' sums are, and before the entries' columns are written.  Each warp finds the teacher's maximum and sum by itself.
template <typename T, bool FORWARD, bool GRAD>
__global__ void __launch_bounds__(kMostThreads, 2)
distill_kernel(const Args k) {
    constexpr int E = 16 / sizeof(T);
    extern __shared__ __align__(16) char shared[];
    int* const col = reinterpret_cast<int*>(shared);                         // the columns, -1: none
    float* const p = reinterpret_cast<float*>(col + (k.top / 4 + 1) * 4);    // the teacher's probabilities
    float* const zk = p + (k.top + 3) / 4 * 4;                               // the logits at the teacher's columns, and at the label's
    int* const table = col + entry_words(k.top);
    __shared__ Part parts[32];
    __shared__ Part block_part;  // read by the other blocks of the cluster
    pdl_prologue();
    const int tid = threadIdx.x, threads = blockDim.x;
    const uint32_t r = blockIdx.x / k.blocks, rank = blockIdx.x % k.blocks;
    const T* const z = reinterpret_cast<const T*>(row_at(k.logits, k.inner, r));
    T* const g = GRAD ? reinterpret_cast<T*>(row_at(k.grad, k.inner, r)) : nullptr;

    // This block's vectors, kVectors * threads at a time; and an element of the row's ends for some threads of the first and the last block.
    const int64_t head = head_of(z, k.vocab), all_vectors = (k.vocab - head) / E, tail = head + all_vectors * E;
    const int64_t v0 = all_vectors * rank / k.blocks, v1 = all_vectors * (rank + 1) / k.blocks;
    int64_t end = -1;
    if (rank == 0 && tid < head) end = tid;
    if (rank + 1 == k.blocks && tid >= 8 && tail + (tid - 8) < k.vocab) end = tail + (tid - 8);
    const uint4* const zv = reinterpret_cast<const uint4*>(z + head);
    uint4 raw[kVectors];
    float end_z = -INFINITY;
    auto load = [&](int64_t from) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
            const int64_t v = from + i * threads + tid;
            raw[i] = v < v1 ? zv[v] : make_uint4(kNothing<T>, kNothing<T>, kNothing<T>, kNothing<T>);
        }
    };
    load(v0);
    if (GRAD) clear_table(table, k.slots, tid, threads);
    if (end >= 0) end_z = to_float(z[end]);

    // the teacher's distribution and the logits at its columns
    if (k.soft) {
        const char* ids = row_at(k.ids, k.inner, r);
        const char* t = row_at(k.teacher, k.inner, r);
        for (int j = tid; j < k.top; j += threads) {
            const int64_t id = load_index(ids + int64_t(j) * (k.wide_ids ? 8 : 4), k.wide_ids);
            const bool in = id >= 0 && id < k.vocab;
            if (id >= k.vocab) atomicOr(k.status, kStatusIndexOutOfRange);
            col[j] = in ? static_cast<int>(id) : -1;
            p[j] = in ? (k.half_teacher ? __half2float(reinterpret_cast<const __half*>(t)[j]) : reinterpret_cast<const float*>(t)[j]) : -INFINITY;
            zk[j] = in ? to_float(z[id]) : 0.f;
        }
    } else {
        for (int j = tid; j < k.top; j += threads) col[j] = -1;
    }
    if (tid > 0 && tid < 4 && k.top + tid < (k.top / 4 + 1) * 4) col[k.top + tid] = -1;
    if (tid == 0) {
        int64_t id = -1;
        if (k.hard) id = load_index(row_at(k.labels, k.inner, r), k.wide_labels);
        if (id >= k.vocab) {
            atomicOr(k.status, kStatusIndexOutOfRange);
            id = -1;
        }
        col[k.top] = static_cast<int>(id < 0 ? -1 : id);
        zk[k.top] = id < 0 ? 0.f : to_float(z[id]);
    }
    __syncthreads();
    if (GRAD && k.slots > 0) {
        for (int j = tid; j <= k.top; j += threads) {
            if (col[j] >= 0) enter_column(table, k.slots, col[j]);
        }
    }
    const float c_soft = k.inverse * kLog2e;
    bool taught = false;  // whether the row has a teacher's entry
    float top_t = -INFINITY, log_sum = 0.f;
    if (k.soft) {
        float sum = 0.f;
        for (int j = tid % 32; j < k.top; j += 32) top_t = fmaxf(top_t, p[j]);
#pragma unroll
        for (int d = 16; d > 0; d /= 2) top_t = fmaxf(top_t, __shfl_xor_sync(0xffffffffu, top_t, d));
        for (int j = tid % 32; j < k.top; j += 32) sum += fast_exp2((p[j] - shift_of(top_t)) * c_soft);  // (no entry: -inf)
#pragma unroll
        for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        taught = !(sum == 0.f);
        log_sum = logf(sum);
        if constexpr (!FORWARD) {
            __syncthreads();  // (every warp has read what the teacher says)
            for (int j = tid; j < k.top; j += threads) p[j] = taught && col[j] >= 0 ? expf((p[j] - shift_of(top_t)) * k.inverse - log_sum) : 0.f;
        }
    }

    // The row's maximum and log sums of exponentials: q = exp((z - at) / T - log_soft), h = exp(z - at - log_hard).  The maximum and the logarithms stay
    // apart: their sum would lose the logarithm in a row whose logits are all the type's lowest value.
    float at = 0.f, log_soft = 0.f, log_hard = 0.f;
    if constexpr (FORWARD) {
        Running running;
        running.begin(end_z, c_soft, k.soft, k.hard);
        for (int64_t from = v0;;) {
            const int64_t left = v1 - from;  // (what lies behind the end costs exponentials too)
            if (left <= threads) running.take<T>(reinterpret_cast<const uint4 (&)[1]>(raw));
            else if (left <= 2 * threads) running.take<T>(reinterpret_cast<const uint4 (&)[2]>(raw));
            else if (left <= 4 * threads) running.take<T>(reinterpret_cast<const uint4 (&)[4]>(raw));
            else running.take<T>(raw);
            from += kVectors * threads;
            if (from >= v1) break;
            load(from);
        }
        Part run = warp_part(running.part, c_soft, k.soft, k.hard);
        if (tid % 32 == 0) parts[tid / 32] = run;
        __syncthreads();
        run = tid % 32 < threads / 32 ? parts[tid % 32] : Part{-INFINITY, 0.f, 0.f};
        run = warp_part(run, c_soft, k.soft, k.hard);
        if (k.blocks > 1) {
            if (tid == 0) block_part = run;
            cluster_sync();
            run = Part{-INFINITY, 0.f, 0.f};
            if (tid % 32 < k.blocks) {
                uint32_t there;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(&block_part))), "r"(tid % 32));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(run.top) : "r"(there) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(run.soft) : "r"(there + 4) : "memory");
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(run.hard) : "r"(there + 8) : "memory");
            }
            run = warp_part(run, c_soft, k.soft, k.hard);
            asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // this block has read the others' parts
        }
        at = shift_of(run.top);
        if (k.soft) log_soft = logf(run.soft);
        if (k.hard) log_hard = logf(run.hard);
        if (rank == 0 && tid == 0 && k.stats != nullptr) k.stats[r] = make_float4(run.top, log_soft, log_hard, 0.f);
        // a row of nothing but -inf: the sums are 0 and their logarithms -inf, which stay out of the differences so that q = 0, log q = -inf
        log_soft = shift_of(log_soft), log_hard = shift_of(log_hard);
        float kl = 0.f;
        if (k.soft && tid < 32 && (GRAD || rank == 0)) {  // the first warp's, while the others go on
            for (int j = tid; j < k.top; j += 32) {
                const float lp = (p[j] - shift_of(top_t)) * k.inverse - log_sum;
                const float pj = taught && col[j] >= 0 ? expf(lp) : 0.f;
                p[j] = pj;
                if (pj != 0.f) kl += pj * (lp - ((zk[j] - at) * k.inverse - log_soft));
            }
#pragma unroll
            for (int d = 16; d > 0; d /= 2) kl += __shfl_xor_sync(0xffffffffu, kl, d);
        }
        if (rank == 0 && tid == 0 && k.losses != nullptr) {
            float loss = 0.f;
            if (taught) loss += (1.f - k.hard_weight) * k.temperature * k.temperature * kl;
            if (k.hard && col[k.top] >= 0) loss += k.hard_weight * (log_hard - (zk[k.top] - at));
            k.losses[r] = loss;
        }
    } else {
        const float4 s = k.stats[r];
        at = shift_of(s.x), log_soft = shift_of(s.y), log_hard = shift_of(s.z);
    }

    if constexpr (GRAD) {
        // Where the gradient lies on the logits: the other blocks' reading of them.  (This block's ended before its warps met.)
        if (FORWARD && k.blocks > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        const float w = k.grad_scale * (k.weights.base != nullptr ? *reinterpret_cast<const float*>(row_at(k.weights, k.inner, r)) : 1.f);
        const bool labelled = k.hard && col[k.top] >= 0;
        RowGrad row;
        row.ws = taught ? w * (1.f - k.hard_weight) * k.temperature : 0.f;
        row.wh = labelled ? w * k.hard_weight : 0.f;
        row.at = at, row.soft2 = -log_soft * kLog2e, row.hard2 = -log_hard * kLog2e;
        const GradPowers powers = grad_powers(row, c_soft);
        if (end >= 0) g[end] = from_float<T>(grad_value(powers, end_z));
        const bool aligned = (reinterpret_cast<uintptr_t>(g + head) & 15) == 0;
        const bool again = v1 - v0 > int64_t(kVectors) * threads && FORWARD;  // not held any more
        for (int64_t from = v0; from < v1; from += kVectors * threads) {
            if (again || from != v0) load(from);
            const int64_t v = from + tid;
            put_grad<T>(powers, raw, g + head + v * E, threads * E, static_cast<int>(min(int64_t(kVectors), (v1 - v + threads - 1) / threads)), aligned);
        }
        __syncthreads();
        // the columns of this block that p or the label adds to, each by the first entry that names it
        const int64_t c0 = rank == 0 ? 0 : head + v0 * E, c1 = rank + 1 == k.blocks ? k.vocab : head + v1 * E;
        for (int j = tid; j <= k.top; j += threads) {
            const int c = col[j];
            float minus;
            if (c < 0 || c < c0 || c >= c1 || !entry_takes(row, col, p, table, k.slots, k.top, k.soft, j, minus)) continue;
            g[c] = from_float<T>(grad_value(powers, zk[j]) - minus);
        }
    } else {
        if (FORWARD && k.blocks > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");  // (no block leaves before its part is read)
    }
}

// ---- many rows ----------------------------------------------------------------

// Two blocks to an SM take one row after another each, so that one computes while the other meets.  kRowWarps warps work on the logits, which come through shared memory: each thread copies its own vectors
// (cp.async, 16 bytes) some visits ahead, and copies the next one into a place as soon as it has used what lay there, so that the memory is never idle.
// A visit is a chunk of a row, or, where the losses and the gradient are computed at once and the row fits, the whole row, which then stays until its
// gradient is written.  Three more warps do what the teacher and the label ask for, each for every third row, up to two rows ahead: ids, the
// logits at them, softmax, the loss once the row's sums are there, and the columns written again once the gradient is.  They meet by named barriers
// at which neither side waits for what it does not need: told (the teacher's part of row i is there), summed (the warps' sums are) and written.
// (A block or a cluster to each row waited for ids, logits, sums and its successor's start one after another: 4096 x 32000 took 157 us and 189 us.)
constexpr int kRowWarps = 8, kRowThreads = kRowWarps * 32, kTeachers = 3, kRowBlocks = 2;
constexpr int kBatch = 4;            // vectors that a thread works on at once
constexpr int kRowShared = 112 << 10;  // of a block: the ring and the teachers' arrays

template <int ID>
__device__ __forceinline__ void barrier_sync(int parity, int threads) {
    asm volatile("barrier.sync %0, %1;" ::"r"(ID + parity), "r"(threads) : "memory");
}
template <int ID>
__device__ __forceinline__ void barrier_arrive(int parity, int threads) {
    asm volatile("barrier.arrive %0, %1;" ::"r"(ID + parity), "r"(threads) : "memory");
}
constexpr int kRowBarrier = 1, kTold = 2, kSummed = kTold + kTeachers, kWritten = kSummed + kTeachers;
constexpr int kMeeting = kRowThreads + 32;

// What a teacher's warp says of its row (forward: at, soft2 and hard2 are not known yet).  On 32 bytes, which the rows' warps read in wide accesses (4096 x 32000 F16,
// losses and gradient: 130.3 us, 133.5 without).
struct __align__(32) Told {
    RowGrad grad;
};

struct RingArgs {
    int chunk;   // vectors of a thread in a visit
    int slots;   // visits in shared memory: 1 to 3
    int chunks;  // of a row
    bool held;   // the row stays for its gradient: one chunk
};

__device__ __forceinline__ void copy_vector(uint32_t to, const uint4* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(__cvta_generic_to_global(from)) : "memory"); }
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest `pending` groups of this thread's copies are there.
__device__ __forceinline__ void copies_wait(int pending) {
    switch (pending) {
        case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
        case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
        case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
        case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
        case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
        default: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;  // (more are waited for than need be)
    }
}

template <typename T, bool FORWARD, bool GRAD>
__global__ void __launch_bounds__(kRowThreads + kTeachers * 32, kRowBlocks)
distill_rows_kernel(const Args k, const RingArgs ring, uint32_t rows) {
    constexpr int E = 16 / sizeof(T);
    extern __shared__ __align__(16) char shared[];
    uint4* const held = reinterpret_cast<uint4*>(shared);  // [slots][chunk][kRowThreads]
    int* const entries = reinterpret_cast<int*>(held + ring.slots * ring.chunk * kRowThreads);
    __shared__ Part parts[kTeachers][kRowWarps];
    __shared__ Told told[kTeachers];
    pdl_prologue();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const uint32_t n = (rows - blockIdx.x + gridDim.x - 1) / gridDim.x;  // rows of this block: blockIdx.x + i * gridDim.x
    const float c_soft = k.inverse * kLog2e;
    auto logits_of = [&](uint32_t i) { return reinterpret_cast<const T*>(row_at(k.logits, k.inner, blockIdx.x + i * gridDim.x)); };
    auto grad_of = [&](uint32_t i) { return reinterpret_cast<T*>(row_at(k.grad, k.inner, blockIdx.x + i * gridDim.x)); };

    if (warp >= kRowWarps) {
        const int parity = warp - kRowWarps;
        int* const col = entries + parity * (entry_words(k.top) + k.slots);
        float* const p = reinterpret_cast<float*>(col + (k.top / 4 + 1) * 4);
        float* const zk = p + (k.top + 3) / 4 * 4;
        int* const table = col + entry_words(k.top);
        if (!k.soft) {
            for (int j = lane; j < k.top; j += 32) col[j] = -1;
        }
        if (lane > 0 && lane < 4 && k.top + lane < (k.top / 4 + 1) * 4) col[k.top + lane] = -1;
        for (uint32_t i = parity; i < n; i += kTeachers) {
            const uint32_t r = blockIdx.x + i * gridDim.x;
            const T* const z = logits_of(i);
            // what hangs on nothing else is asked for first
            const int64_t label_id = k.hard ? load_index(row_at(k.labels, k.inner, r), k.wide_labels) : -1;
            const float weight = GRAD && k.weights.base != nullptr ? *reinterpret_cast<const float*>(row_at(k.weights, k.inner, r)) : 1.f;
            const float4 stats = FORWARD ? make_float4(0.f, 0.f, 0.f, 0.f) : k.stats[r];
            const int label = label_id >= 0 && label_id < k.vocab ? static_cast<int>(label_id) : -1;
            if (label_id >= k.vocab && lane == 0) atomicOr(k.status, kStatusIndexOutOfRange);
            float top_t = -INFINITY, sum = 0.f;
            if (k.soft) {
                const char* ids = row_at(k.ids, k.inner, r);
                const char* t = row_at(k.teacher, k.inner, r);
                bool outside = false;
                for (int j0 = lane; j0 < k.top; j0 += 128) {  // four entries of a lane at once: their ids, then the logits there
                    int c[4];
                    float tj[4], zj[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int j = j0 + u * 32;
                        c[u] = -1, tj[u] = -INFINITY;
                        if (j < k.top) {
                            const int64_t id = load_index(ids + int64_t(j) * (k.wide_ids ? 8 : 4), k.wide_ids);
                            tj[u] = k.half_teacher ? __half2float(reinterpret_cast<const __half*>(t)[j]) : reinterpret_cast<const float*>(t)[j];
                            outside |= id >= k.vocab;
                            if (id >= 0 && id < k.vocab) c[u] = static_cast<int>(id);
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u) zj[u] = c[u] >= 0 ? to_float(z[c[u]]) : 0.f;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int j = j0 + u * 32;
                        if (c[u] < 0) tj[u] = -INFINITY;
                        if (j < k.top) col[j] = c[u], p[j] = tj[u], zk[j] = zj[u];
                        top_t = fmaxf(top_t, tj[u]);
                    }
                }
                if (outside) atomicOr(k.status, kStatusIndexOutOfRange);
            }
            const float label_z = label >= 0 ? to_float(z[label]) : 0.f;
            if (lane == 0) col[k.top] = label, zk[k.top] = label_z;
            if (k.soft) {
#pragma unroll
                for (int d = 16; d > 0; d /= 2) top_t = fmaxf(top_t, __shfl_xor_sync(0xffffffffu, top_t, d));
#pragma unroll 4
                for (int j = lane; j < k.top; j += 32) sum += fast_exp2((p[j] - shift_of(top_t)) * c_soft);  // (no entry: -inf)
#pragma unroll
                for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            }
            const bool taught = k.soft && !(sum == 0.f);
            const float log_sum = logf(sum);
            RowGrad row = {};
            if constexpr (GRAD) {
                const float w = k.grad_scale * weight;
                row.ws = taught ? w * (1.f - k.hard_weight) * k.temperature : 0.f;
                row.wh = label >= 0 ? w * k.hard_weight : 0.f;
            }
            if constexpr (!FORWARD) row.at = shift_of(stats.x), row.soft2 = -shift_of(stats.y) * kLog2e, row.hard2 = -shift_of(stats.z) * kLog2e;
            if (lane == 0) told[parity].grad = row;
            __syncwarp();
            barrier_arrive<kTold>(parity, kMeeting);
            if constexpr (FORWARD) {
                barrier_sync<kSummed>(parity, kMeeting);
                Part run = lane < kRowWarps ? parts[parity][lane] : Part{-INFINITY, 0.f, 0.f};
                run = warp_part(run, c_soft, k.soft, k.hard);
                const float at = shift_of(run.top);
                float log_soft = k.soft ? logf(run.soft) : 0.f, log_hard = k.hard ? logf(run.hard) : 0.f;
                if (lane == 0 && k.stats != nullptr) k.stats[r] = make_float4(run.top, log_soft, log_hard, 0.f);
                log_soft = shift_of(log_soft), log_hard = shift_of(log_hard);
                row.at = at, row.soft2 = -log_soft * kLog2e, row.hard2 = -log_hard * kLog2e;
                float kl = 0.f;
#pragma unroll 4
                for (int j = lane; j < (k.soft ? k.top : 0); j += 32) {
                    const float lp = (p[j] - shift_of(top_t)) * k.inverse - log_sum;
                    const float pj = taught ? fast_exp2(lp * kLog2e) : 0.f;  // (no entry: exp of -inf)
                    p[j] = pj;
                    if (pj != 0.f) kl += pj * (lp - ((zk[j] - at) * k.inverse - log_soft));
                }
#pragma unroll
                for (int d = 16; d > 0; d /= 2) kl += __shfl_xor_sync(0xffffffffu, kl, d);
                if (lane == 0 && k.losses != nullptr) {
                    float loss = 0.f;
                    if (taught) loss += (1.f - k.hard_weight) * k.temperature * k.temperature * kl;
                    if (label >= 0) loss += k.hard_weight * (log_hard - (label_z - at));
                    k.losses[r] = loss;
                }
            } else {
#pragma unroll 4
                for (int j = lane; j < (k.soft ? k.top : 0); j += 32) p[j] = taught ? fast_exp2(((p[j] - shift_of(top_t)) * k.inverse - log_sum) * kLog2e) : 0.f;
            }
            if (GRAD && k.slots > 0) {
                clear_table(table, k.slots, lane, 32);
                __syncwarp();
                for (int j = lane; j <= k.top; j += 32) {
                    if (col[j] >= 0) enter_column(table, k.slots, col[j]);
                }
            }
            __syncwarp();
            if constexpr (GRAD) {
                barrier_sync<kWritten>(parity, kMeeting);
                T* const g = grad_of(i);
                const GradPowers powers = grad_powers(row, c_soft);
                for (int j = lane; j <= k.top; j += 32) {
                    float minus;
                    if (col[j] < 0 || !entry_takes(row, col, p, table, k.slots, k.top, k.soft, j, minus)) continue;
                    g[col[j]] = from_float<T>(grad_value(powers, zk[j]) - minus);
                }
                __syncwarp();
            }
        }
        return;
    }

    // the rows' warps
    const int tid = threadIdx.x;
    const int chunks = ring.chunks, chunk = ring.chunk, slots = ring.slots;
    const bool keep = FORWARD && GRAD && ring.held;               // the row stays
    const int sweeps = FORWARD && GRAD && !keep ? 2 : 1;          // visits of a chunk of a row
    constexpr uint32_t kApart = kRowThreads * 16;                 // bytes from a thread's vector to its next
    const uint32_t my_place = static_cast<uint32_t>(__cvta_generic_to_shared(held)) + tid * 16, slot_bytes = chunk * kApart;
    // A row: where its vectors begin, how many they are, and the element at its ends that is this thread's (behind the last vector for those from 8 on; -1: none).
    struct Row {
        const T* z;
        int head, vectors;
    };
    auto row_of = [&](uint32_t i) {
        Row row;
        row.z = logits_of(i);
        row.head = static_cast<int>(head_of(row.z, k.vocab));
        row.vectors = (static_cast<int>(k.vocab) - row.head) / E;
        return row;
    };
    auto end_of = [&](const Row& row) {
        const int behind = row.head + row.vectors * E + tid - 8;
        return tid < row.head ? tid : tid >= 8 && tid < 16 && behind < static_cast<int>(k.vocab) ? behind : -1;
    };
    // how many of this thread's vectors of a row lie in the chunk that begins with its vector v
    auto count_of = [&](int vectors, int v) { return max(0, min(chunk, (vectors - tid + kRowThreads - 1) / kRowThreads - v)); };
    // the visit whose copies are issued next
    Row ahead = row_of(0);
    uint32_t ahead_row = 0;
    int ahead_chunk = 0, ahead_sweep = 0, limit = 0;
    const uint4* source = nullptr;
    auto aim = [&] {
        limit = 0;
        if (ahead_row >= n) return;
        source = reinterpret_cast<const uint4*>(ahead.z + ahead.head) + ahead_chunk * chunk * kRowThreads + tid;
        limit = count_of(ahead.vectors, ahead_chunk * chunk);
        if (++ahead_chunk == chunks) {
            ahead_chunk = 0;
            if (++ahead_sweep == sweeps) {
                ahead_sweep = 0;
                if (++ahead_row < n) ahead = row_of(ahead_row);
            }
        }
    };
    uint32_t slot = 0;  // in bytes
    // kBatch copies of the next visit into this one's places, from its vector v on
    auto copy = [&](int v) {
        const uint32_t to = my_place + slot + v * kApart;
        const uint4* const from = source + v * kRowThreads;
        if (v + kBatch <= limit) {
#pragma unroll
            for (int h = 0; h < kBatch; ++h) copy_vector(to + h * kApart, from + h * kRowThreads);
        } else {
            for (int h = 0; v + h < limit; ++h) copy_vector(to + h * kApart, from + h * kRowThreads);
        }
        if (keep) copies_commit();  // (a group to each batch, so that a row can be begun before its end is there)
    };
    auto next = [&] {
        if (!keep) copies_commit();
        slot = slot + slot_bytes == slots * slot_bytes ? 0 : slot + slot_bytes;
    };
    const int batches = (chunk + kBatch - 1) / kBatch, newest = keep ? slots * batches - 1 : slots - 1;
    // A visit with `count` vectors for this thread: f(vectors, the first one's number), kBatch at a time as far as that goes.  WAIT: the copies are waited for; FREE: the next
    // visit's take their places, which have been read: their values are used.
    auto visit = [&](int count, auto wait, auto free, auto&& f) {
        auto get = [&](uint4& x, uint32_t at) { asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory"); };
        if (decltype(free)::value) aim();
        if (decltype(wait)::value && !keep) copies_wait(newest);
        uint32_t from = my_place + slot;
        for (int v = 0, batch = 0; v < chunk; v += kBatch, ++batch, from += kBatch * kApart) {
            if (decltype(wait)::value && keep) copies_wait(newest - batch);
            if (v + kBatch <= count) {
                uint4 raw[kBatch];
#pragma unroll
                for (int h = 0; h < kBatch; ++h) get(raw[h], from + h * kApart);
                f(raw, v);
            } else {
                int h = 0;
                if (v + 2 <= count) {
                    uint4 raw[2];
                    get(raw[0], from);
                    get(raw[1], from + kApart);
                    f(raw, v);
                    h = 2;
                }
                if (v + h < count) {
                    uint4 raw[1];
                    get(raw[0], from + h * kApart);
                    f(raw, v + h);
                }
            }
            if (decltype(free)::value) copy(v);
        }
        if (decltype(free)::value) next();
    };
    using Yes = std::true_type;
    using No = std::false_type;
    for (int s = 0; s < slots; ++s) {
        aim();
        for (int v = 0; v < chunk; v += kBatch) copy(v);
        next();
    }
    Row row = row_of(0);
    int end = end_of(row);
    float end_z = end >= 0 ? to_float(row.z[end]) : -INFINITY;
    for (uint32_t i = 0; i < n; ++i) {
        const int parity = i % kTeachers;
        Row next_row = row;
        int next_end = -1;
        float next_end_z = -INFINITY;
        if (i + 1 < n) {
            next_row = row_of(i + 1);
            next_end = end_of(next_row);
            if (next_end >= 0) next_end_z = to_float(next_row.z[next_end]);
        }
        if constexpr (FORWARD) {
            Running running;
            running.begin(end_z, c_soft, k.soft, k.hard);
            auto take = [&](const auto& raw, int) { running.take<T>(raw); };
            if (keep) {
                visit(count_of(row.vectors, 0), Yes{}, No{}, take);
            } else {
                for (int c = 0; c < chunks; ++c) visit(count_of(row.vectors, c * chunk), Yes{}, Yes{}, take);
            }
            Part run = warp_part(running.part, c_soft, k.soft, k.hard);
            __syncwarp();
            barrier_sync<kTold>(parity, kMeeting);  // (so the teacher is done with the sums of its last row, too)
            if (lane == 0) parts[parity][warp] = run;
            __syncwarp();
            if constexpr (GRAD) barrier_sync<kRowBarrier>(0, kRowThreads);
            barrier_arrive<kSummed>(parity, kMeeting);
        } else {
            __syncwarp();
            barrier_sync<kTold>(parity, kMeeting);
        }
        if constexpr (GRAD) {
            RowGrad grad = told[parity].grad;
            if constexpr (FORWARD) {
                Part run = lane < kRowWarps ? parts[parity][lane] : Part{-INFINITY, 0.f, 0.f};
                run = warp_part(run, c_soft, k.soft, k.hard);
                grad.at = shift_of(run.top);
                grad.soft2 = k.soft ? -shift_of(logf(run.soft)) * kLog2e : 0.f;
                grad.hard2 = k.hard ? -shift_of(logf(run.hard)) * kLog2e : 0.f;
            }
            const GradPowers powers = grad_powers(grad, c_soft);
            T* const g = grad_of(i);
            const bool aligned = (reinterpret_cast<uintptr_t>(g + row.head) & 15) == 0;
            if (end >= 0) g[end] = from_float<T>(grad_value(powers, end_z));
            T* to = g + row.head + tid * E;
            auto put = [&](const auto& raw, int v) {
                constexpr int M = std::extent<std::remove_reference_t<decltype(raw)>>::value;
                put_grad<T, M>(powers, raw, to + v * kRowThreads * E, kRowThreads * E, M, aligned);
            };
            if (keep) {
                visit(count_of(row.vectors, 0), No{}, Yes{}, put);
            } else {
                for (int c = 0; c < chunks; ++c, to += chunk * kRowThreads * E) visit(count_of(row.vectors, c * chunk), Yes{}, Yes{}, put);
            }
            __syncwarp();
            barrier_arrive<kWritten>(parity, kMeeting);
        }
        row = next_row;
        end = next_end;
        end_z = next_end_z;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- arguments --------------------------------------------------------------

bool present(const b200_tensor& t) { return t.data != nullptr; }

void check_scalar_rows(const b200_tensor& t, const char* name, const b200_tensor& logits) {
    check_tensor(t, name);
    if (t.ndim != logits.ndim - 1 || !same_extents(t, logits, t.ndim)) fail(B200_SHAPE_ERROR, std::string(name) + ": not one for each row of logits");
}

struct Plan {
    int axes;
    int64_t vocab, top;
    RowShape s;
    bool labelled;
    int64_t row_vectors;
    bool many_rows;       // blocks that stay take one row after another
    int threads, blocks;  // else: of a block, and blocks to a row
};

// How a call's rows are divided.
void divide(Plan& plan, bool forward, bool grad, bool half) {
    // Many rows of at least 16 KB each: blocks that stay take one row after another.  (Below, a block's warps have little to do between a row's meetings.)  Not where
    // a row's entries take a teacher's warp longer than its logits take the others: 2048 x 16384 F16, gradient: 64 entries 39 us and 45 by a block to a row, 256
    // entries 86 and 61; losses and gradient: 256 entries 94 and 88, 1000 276 and 174; losses alone: 256 entries 36 and 36, 1000 92 and 61.
    const int64_t vectors = plan.row_vectors = ceil_div(plan.vocab, half ? 8 : 4);
    plan.many_rows = plan.s.rows >= int64_t(sm_count()) * kRowBlocks && vectors >= std::max<int64_t>(kRowThreads * 4, plan.top * (!forward ? 16 : grad ? 6 : 4));
    if (plan.many_rows) return;
    // 256 threads and a cluster of up to 4, so that an SM has four blocks in different states; longer rows 512 threads and a cluster of up to 8.  Where there
    // are fewer rows than SMs, a cluster as large as leaves a thread a vector.
    int threads = 256, blocks = 1;
    while (blocks < 4 && vectors > int64_t(blocks) * threads * kVectors) blocks *= 2;
    if (vectors > int64_t(blocks) * threads * kVectors) threads = kMostThreads;
    while (blocks < 8 && vectors > int64_t(blocks) * threads * kVectors) blocks *= 2;
    while (blocks < 8 && plan.s.rows * blocks * 2 <= sm_count() && vectors > int64_t(blocks) * threads) blocks *= 2;
    while (threads > 64 && plan.s.rows * blocks > sm_count() && int64_t(blocks) * (threads / 2) * 4 >= vectors) threads /= 2;
    plan.threads = threads;
    plan.blocks = blocks;
    if (plan.s.rows * blocks >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "distill_loss: too many rows of this length");
}

Plan check_distill(const b200_distill_args& a, bool forward) {
    check_rows(a.logits, "logits");
    check_rows(a.teacher_ids, "teacher_ids");
    check_rows(a.teacher_logits, "teacher_logits");
    if (!is_float(a.logits.dtype) || !is_float(a.teacher_logits.dtype)) fail(B200_DTYPE_ERROR, "logits and teacher_logits are F32 or F16");
    if (!is_index(a.teacher_ids.dtype)) fail(B200_DTYPE_ERROR, "teacher_ids are I32 or I64");
    const int axes = a.logits.ndim - 1;
    const int64_t vocab = a.logits.dims[axes];
    for (const Named& n : {Named{&a.teacher_ids, "teacher_ids"}, Named{&a.teacher_logits, "teacher_logits"}}) {
        if (n.t->ndim != a.logits.ndim || !same_extents(*n.t, a.logits, axes)) fail(B200_SHAPE_ERROR, std::string(n.name) + ": rows of other extents than logits");
    }
    const int64_t top = a.teacher_ids.dims[axes];
    if (a.teacher_logits.dims[axes] != top) fail(B200_SHAPE_ERROR, "teacher_ids and teacher_logits have different widths");
    if (top > kMostTop) fail(B200_NOT_IMPLEMENTED, "distill_loss: more than 1024 of the teacher's logits");
    if (vocab < 1 || vocab >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "logits: rows of no element, or of 2^31 or more");
    const RowShape s = row_shape(a.logits, axes);
    if (!(a.temperature > 0.f) || std::isinf(a.temperature) || std::isinf(1.f / a.temperature * kLog2e)) {
        fail(B200_INVALID_ARGUMENT, "distill_loss: the temperature is not above 0 and finite, or its inverse times log2 e is not");
    }
    if (!(a.hard_weight >= 0.f && a.hard_weight <= 1.f)) fail(B200_INVALID_ARGUMENT, "distill_loss: the hard weight is not in 0..1");
    const bool labelled = !is_absent(a.labels, "labels");
    if (labelled) {
        check_scalar_rows(a.labels, "labels", a.logits);
        if (!is_index(a.labels.dtype)) fail(B200_DTYPE_ERROR, "labels are I32 or I64");
    }
    if (a.losses_grad.data != nullptr) {
        check_scalar_rows(a.losses_grad, "losses_grad", a.logits);
        if (a.losses_grad.dtype != B200_F32) fail(B200_DTYPE_ERROR, "losses_grad is F32");
    }
    if (present(a.losses)) {
        check_scalar_rows(a.losses, "losses", a.logits);
        if (a.losses.dtype != B200_F32) fail(B200_DTYPE_ERROR, "losses are F32");
        if (!is_dense(a.losses)) fail(B200_NOT_IMPLEMENTED, "losses are not dense");
    }
    if (present(a.stats)) check_stats(a.stats, s.rows);
    if (present(a.grad)) {
        check_rows(a.grad, "grad");
        if (a.grad.ndim != a.logits.ndim || !same_extents(a.grad, a.logits, a.logits.ndim)) fail(B200_SHAPE_ERROR, "grad has not the logits' extents");
        if (a.grad.dtype != a.logits.dtype) fail(B200_DTYPE_ERROR, "grad has not the logits' type");
    }
    if (!forward && present(a.losses)) fail(B200_INVALID_ARGUMENT, "distill_loss_backward computes no losses");
    const std::initializer_list<Named> read = {{&a.teacher_ids, "teacher_ids"}, {&a.teacher_logits, "teacher_logits"}, {&a.labels, "labels"}, {&a.losses_grad, "losses_grad"}};
    if (forward) {
        check_results({{&a.losses, "losses"}, {&a.stats, "stats"}}, {{&a.logits, "logits"}, {&a.teacher_ids, "teacher_ids"}, {&a.teacher_logits, "teacher_logits"},
                                                                 {&a.labels, "labels"}, {&a.losses_grad, "losses_grad"}, {&a.grad, "grad"}}, {});
        check_results({{&a.grad, "grad"}}, read, {{&a.logits, "logits"}});
    } else {
        check_results({{&a.grad, "grad"}}, {{&a.teacher_ids, "teacher_ids"}, {&a.teacher_logits, "teacher_logits"}, {&a.labels, "labels"}, {&a.losses_grad, "losses_grad"},
                                            {&a.stats, "stats"}}, {{&a.logits, "logits"}});
    }
    const Plan plan{axes, vocab, top, s, labelled, 0, false, 0, 0};
    if (s.rows == 0) return plan;
    if (forward && !present(a.losses) && !present(a.stats) && !present(a.grad)) fail(B200_INVALID_ARGUMENT, "distill_loss: no result is asked for");
    if (!forward && (!present(a.grad) || !present(a.stats))) fail(B200_INVALID_ARGUMENT, "distill_loss_backward: grad and the forward call's stats are needed");
    if (a.hard_weight > 0.f && !labelled) fail(B200_INVALID_ARGUMENT, "distill_loss: a hard weight without labels");
    return plan;
}

void launch_distill(b200_ctx* ctx, const b200_distill_args& a, bool forward) {
    Plan plan = check_distill(a, forward);
    divide(plan, forward, present(a.grad), a.logits.dtype == B200_F16);
    const int axes = plan.axes;
    const int64_t vocab = plan.vocab, top = plan.top;
    const RowShape s = plan.s;
    const bool labelled = plan.labelled;
    if (s.rows == 0) return;
    wait_for_tensors(ctx, {&a.logits, &a.teacher_ids, &a.teacher_logits, &a.labels, &a.losses, &a.stats, &a.losses_grad, &a.grad});
    Args k{};
    k.logits = rows_arg(a.logits, axes);
    k.ids = rows_arg(a.teacher_ids, axes);
    k.teacher = rows_arg(a.teacher_logits, axes);
    if (labelled) k.labels = rows_arg(a.labels, axes);
    if (present(a.losses_grad)) k.weights = rows_arg(a.losses_grad, axes);
    if (present(a.grad)) k.grad = rows_arg(a.grad, axes);
    k.losses = static_cast<float*>(a.losses.data);
    k.stats = static_cast<float4*>(a.stats.data);
    k.inner = FastDiv(static_cast<uint32_t>(s.inner));
    k.status = ctx->d_status;
    k.vocab = vocab;
    k.top = static_cast<int>(top);
    k.wide_ids = a.teacher_ids.dtype == B200_I64;
    k.wide_labels = a.labels.dtype == B200_I64;
    k.half_teacher = a.teacher_logits.dtype == B200_F16;
    k.soft = a.hard_weight < 1.f;
    k.hard = a.hard_weight > 0.f;
    k.temperature = a.temperature;
    k.inverse = 1.f / a.temperature;
    k.hard_weight = a.hard_weight;
    k.grad_scale = a.grad_scale;
    ProfScope scope(ctx, forward ? "distill_loss" : "distill_loss_backward");
    k.slots = present(a.grad) ? table_slots(static_cast<int>(top)) : 0;
    const size_t shared = static_cast<size_t>(entry_words(static_cast<int>(top)) + k.slots) * 4;
    const bool half = a.logits.dtype == B200_F16;
    if (plan.many_rows) {
        RingArgs ring{};
        const int64_t whole = ceil_div(plan.row_vectors, kRowThreads);
        const int most = static_cast<int>((kRowShared - kTeachers * shared) / (kRowThreads * 16));  // vectors of a thread
        ring.held = forward && present(a.grad) && whole <= most;
        ring.chunk = ring.held ? static_cast<int>(whole) : most >= 4 * kBatch ? 2 * kBatch : kBatch;
        ring.chunks = static_cast<int>(ceil_div(whole, ring.chunk));
        ring.slots = std::min(3, most / ring.chunk);
        const size_t bytes = static_cast<size_t>(ring.slots) * ring.chunk * kRowThreads * 16 + kTeachers * shared;
        auto go = [&](auto kernel) {
            (void)blocks_at_once(reinterpret_cast<const void*>(kernel), kRowThreads + kTeachers * 32, bytes);  // (allows that much shared memory)
            launch_kernel(ctx, kernel, dim3(static_cast<unsigned>(sm_count() * kRowBlocks)), dim3(kRowThreads + kTeachers * 32), bytes, k, ring, static_cast<uint32_t>(s.rows));
        };
        if (!forward) go(half ? distill_rows_kernel<__half, false, true> : distill_rows_kernel<float, false, true>);
        else if (present(a.grad)) go(half ? distill_rows_kernel<__half, true, true> : distill_rows_kernel<float, true, true>);
        else go(half ? distill_rows_kernel<__half, true, false> : distill_rows_kernel<float, true, false>);
        check_last_launch("distill_loss");
        ctx->count_launch();
        return;
    }
    const int blocks = k.blocks = plan.blocks, threads = plan.threads;
    const int64_t grid = s.rows * blocks;
    auto go = [&](auto kernel) {
        if (blocks == 1 || !forward) launch_kernel(ctx, kernel, dim3(static_cast<unsigned>(grid)), dim3(threads), shared, k);
        else launch_kernel_clustered(ctx, kernel, dim3(static_cast<unsigned>(grid)), dim3(threads), shared, blocks, false, k);
    };
    if (!forward) go(half ? distill_kernel<__half, false, true> : distill_kernel<float, false, true>);
    else if (present(a.grad)) go(half ? distill_kernel<__half, true, true> : distill_kernel<float, true, true>);
    else go(half ? distill_kernel<__half, true, false> : distill_kernel<float, true, false>);
    check_last_launch("distill_loss");
    ctx->count_launch();
}

}  // namespace

void check_distill_loss(const b200_distill_args& a, bool forward) {
    Plan plan = check_distill(a, forward);
    if (plan.s.rows >= int64_t(1) << 28) divide(plan, forward, present(a.grad), a.logits.dtype == B200_F16);  // (fewer rows, of up to 8 blocks each, always fit)
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_distill_loss(b200_ctx* ctx, const b200_distill_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_distill(ctx, *args, true); });
}

int b200_distill_loss_backward(b200_ctx* ctx, const b200_distill_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_distill(ctx, *args, false); });
}

}  // extern "C"
