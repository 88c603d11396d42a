// Log probabilities of given tokens, the entropy of their distribution and its likeliest tokens, and the gradient of the first two.
//
// For a row z of V logits and temperature T, with u = (z - max) / T, s = sum e^u and q = e^u / s:
//
//   log q_j = u_j - log s        H = log s - (sum e^u u) / s
//   grad = k [ a (one at token - q) - w q (log q + H) ] / T,  a and w the gradients of the token's log q and of H
//
// Bound by memory: z read once, and backward as much written.  A block takes a row after another: each thread keeps the maximum of what it has read and the sums of
// e^u and e^u u beside it, and the block joins these threes.  What comes next, of this row or the next one, is on its way into registers all the while, so that a
// row's end holds up nothing that is read.  (Through shared memory, by asynchronous copies, a row's end cost more than the registers do: 4096 x 32000 F16 95 us in place
// of 53.)  Few long rows are a cluster's each, whose blocks take a part of it.  2047 x 128000 F32: 151 to 159 us, 6.6 to 6.9 TB/s; 4096 x 32000 F16: 53 to 55 us, 4.8 to 4.9 TB/s, bound by the
// exponential, the two sums and the conversion of each element.
//
// The K largest cost no second pass.  Some K threads' maxima are K elements, so that the K-th largest of all threads' maxima is a bound that K elements at least
// reach; it is found by halving the range between the maxima, by one warp.  Each thread has kept the maxima of up to sixteen stretches of what it had, too (with four,
// the 20 largest of 2048 x 128000 F32 take 210 us in place of 179): only stretches whose maximum reaches the bound (little more than K) are read again, and what reaches
// it goes into shared memory, where an entry's rank is the number of larger ones.  Where more entries reach it than there is room for (a row of few different values: most
// of its columns forbidden, say) the bound is made exact by counting over the row, and equal ones are taken in the order of their columns.
#include "operators.cuh"

#include <algorithm>
#include <cmath>

namespace b200 {
namespace {

constexpr int kMostTop = B200_MOST_TOP;
constexpr int kMostThreads = 512;
__host__ __device__ constexpr int threads_on_sm(int threads) { return threads < 256 ? 896 : 768; }  // by their registers, in blocks of so many
constexpr int kBatch = 4;    // vectors that a thread takes at once
constexpr int kMostBlocks = 8;  // of a cluster
constexpr int kStretches = 16;   // of a thread's batches
// Entries that there is room for: where fewer threads have elements than are wanted, all of a row's are entries (8 to each of them, and the ends).
__host__ __device__ constexpr int room_for(int top) { return top * 8 + 16; }
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Args {
    RowsArg logits, tokens, ids, tops, logprobs_grad, entropies_grad, grad;
    float* logprobs;
    float* entropies;
    float4* stats;
    FastDiv inner;
    uint32_t* status;
    int64_t vocab;
    uint32_t rows;
    int top;
    bool wide_tokens, wide_ids;
    float inverse, scale;  // 1 / T; backward: grad_scale / T
};

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The larger one; no number where one of them is none.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float shift_of(float top) { return top == -INFINITY ? 0.f : top; }

// Elements of a row that lie before its first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int head_of(const T* row, int64_t n) {
    const uint32_t head = (0u - static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row))) % 16 / uint32_t(sizeof(T));
    return static_cast<int>(head < n ? head : n);
}

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

// Whole numbers in the order of the logits: equal ones (0 and -0) alike, what is no number above all.
__device__ __forceinline__ uint32_t order_of(float z) {
    if (z != z) return 0xffffffffu;
    const uint32_t b = __float_as_uint(z + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) { return __uint_as_float(order >> 31 ? order & 0x7fffffffu : ~order); }

// A number that no element is far above, and beside it the sums of e^u and of e^u u in powers of two: 2^v and 2^v v, v = (z - top) log2 e / T.
struct Part {
    float top, sum, turned;
};

__device__ __forceinline__ void shift_part(Part& x, float top, float c) {
    const float apart = (x.top - shift_of(top)) * c;
    if (x.sum != 0.f) {  // (nothing so far: a maximum of -inf)
        const float f = fast_exp2(apart);
        x.turned = f * fmaf(apart, x.sum, x.turned);
        x.sum *= f;
        if (f == 0.f) x.turned = 0.f;  // (far below: no infinity times zero)
    }
    x.top = top;
}

// The lanes' parts joined beside the largest element, of which `top` is each lane's own.
__device__ __forceinline__ Part warp_part(Part x, float top, float c) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
    shift_part(x, top, c);
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        x.sum += __shfl_xor_sync(0xffffffffu, x.sum, d);
        x.turned += __shfl_xor_sync(0xffffffffu, x.turned, d);
    }
    return x;
}

template <typename T>
constexpr uint32_t kNothing = sizeof(T) == 2 ? 0xfc00fc00u : 0xff800000u;  // -inf

// Adds vectors' powers to a part.  Elements of -inf count as far below, as powers of two of -150, which are 0.
//
// CLAMP: halves are raised to the lowest finite one instead, two to an instruction, where that is as far below.  v is one multiply-add then, z c - at c: at c's rounding
// is the same for all and at most 2^-8, and what it made of the sums is given back at the end.
template <typename T, bool CLAMP, int N>
__device__ __forceinline__ void take_powers(Part& part, uint4 (&raw)[N], float at, float c) {
    constexpr int E = 16 / sizeof(T);
    float sum[2] = {0.f, 0.f}, turned[2] = {0.f, 0.f};
    const float off = -at * c;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float z[E];
        if constexpr (CLAMP) {
            const __half2 lowest = __half2half2(__ushort_as_half(0xfbff));
            __half2* h = reinterpret_cast<__half2*>(&raw[i]);
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = __hmax2_nan(h[e], lowest);
        }
        unpack<T>(raw[i], z);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            float v[2], p[2];
            if constexpr (CLAMP) {
                fma_pair(v[0], v[1], z[e], z[e + 1], c, c, off, off);
            } else {
                add_pair(v[0], v[1], z[e], z[e + 1], -at, -at);
                mul_pair(v[0], v[1], v[0], v[1], c, c);
                v[0] = max_nan(v[0], -150.f), v[1] = max_nan(v[1], -150.f);
            }
            p[0] = fast_exp2(v[0]), p[1] = fast_exp2(v[1]);
            add_pair(sum[0], sum[1], sum[0], sum[1], p[0], p[1]);
            fma_pair(turned[0], turned[1], p[0], p[1], v[0], v[1], turned[0], turned[1]);
        }
    }
    sum[0] += sum[1], turned[0] += turned[1];
    if constexpr (CLAMP) {
        const float less = fmaf(-at, c, -off);  // what every v lacks
        const float f = fast_exp2(less);
        sum[0] *= f;
        turned[0] = fmaf(turned[0], f, less * sum[0]);
    }
    part.sum += sum[0];
    part.turned += turned[0];
}
// The largest element of N vectors (halves compare as halves, two at a time); no number where one is none.
template <typename T, int N>
__device__ __forceinline__ float largest(const uint4 (&raw)[N]) {
    float top;
    if constexpr (sizeof(T) == 2) {
        const __half2* h = reinterpret_cast<const __half2*>(&raw[0]);
        __half2 m[2] = {__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])};
#pragma unroll
        for (int i = 1; i < N; ++i) {
            m[0] = __hmax2_nan(m[0], __hmax2_nan(h[4 * i], h[4 * i + 1]));
            m[1] = __hmax2_nan(m[1], __hmax2_nan(h[4 * i + 2], h[4 * i + 3]));
        }
        m[0] = __hmax2_nan(m[0], m[1]);
        top = max_nan(__low2float(m[0]), __high2float(m[0]));
    } else {
        const float* z = reinterpret_cast<const float*>(&raw[0]);
        top = z[0];
#pragma unroll
        for (int i = 1; i < 4 * N; ++i) top = max_nan(top, z[i]);
    }
    return top;
}
// Vectors whose largest element is `most`.  The number that the sums are beside of moves when an element is above it, to two powers of two above that one: it moves a few
// times in a row.
template <typename T, int N>
__device__ __forceinline__ void take(Part& part, uint4 (&raw)[N], float most, float c, float above) {
    if (!(most <= part.top)) shift_part(part, most + above, c);
    const float at = shift_of(part.top);
    if (sizeof(T) == 2 && (at + 65504.f) * c > 160.f && fabsf(at * c) < 0x1p17f) take_powers<T, sizeof(T) == 2>(part, raw, at, c);
    else take_powers<T, false>(part, raw, at, c);
}

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t in_block(uint32_t address, uint32_t rank) {
    uint32_t to;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(address), "r"(rank));
    return to;
}

// A row, or the part of it that is a block's: its vectors [first, last), and the elements in front of its first vector and behind its last one.
template <typename T>
struct Row {
    const T* z;
    int head, first, last, tail;
    __device__ __forceinline__ Row(const Args& k, uint32_t r, uint32_t rank, uint32_t blocks) {
        z = reinterpret_cast<const T*>(row_at(k.logits, k.inner, r));
        head = head_of(z, k.vocab);
        const uint32_t vectors = static_cast<uint32_t>(k.vocab - head) / uint32_t(16 / sizeof(T));
        tail = head + static_cast<int>(vectors) * int(16 / sizeof(T));
        const int bits = 31 - __clz(blocks);  // (a power of two)
        first = static_cast<int>(uint64_t(vectors) * rank >> bits), last = static_cast<int>(uint64_t(vectors) * (rank + 1) >> bits);
    }
    __device__ __forceinline__ const uint4* vectors() const { return reinterpret_cast<const uint4*>(z + head); }
};

// A row's log sum of exponentials and entropy, from its part.
struct Totals {
    float at, log_sum, entropy;
    __device__ __forceinline__ explicit Totals(const Part& all) {
        const bool some = all.sum != 0.f;  // (or no number)
        at = shift_of(all.top);
        log_sum = some ? logf(all.sum) : 0.f;
        entropy = some ? log_sum - all.turned / all.sum * kLn2 : 0.f;
    }
};
__device__ __forceinline__ void write_row(const Args& k, uint32_t r, const Part& all, bool token, float token_z) {
    const Totals x(all);
    if (k.logprobs != nullptr) k.logprobs[r] = token ? (token_z - x.at) * k.inverse - x.log_sum : 0.f;
    if (k.entropies != nullptr) k.entropies[r] = x.entropy;
    if (k.stats != nullptr) k.stats[r] = make_float4(all.top, x.log_sum, x.entropy, 0.f);
}
// Each of n entries to the place of its rank, if it is one of the first: as a result, or, where `to` is given, as an entry in another block's shared memory.
__device__ __forceinline__ void rank_entries(const Args& k, uint32_t r, const Part& all, const uint64_t* entries, int n, const uint32_t* to) {
    if (static_cast<int>(threadIdx.x) >= n) return;
    char* const ids = k.ids.base != nullptr ? row_at(k.ids, k.inner, r) : nullptr;
    float* const tops = k.tops.base != nullptr ? reinterpret_cast<float*>(row_at(k.tops, k.inner, r)) : nullptr;
    const Totals x(all);
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const uint64_t entry = entries[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) rank += entries[j] > entry;
        if (rank >= k.top || entry == 0) continue;
        if (to != nullptr) {
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(*to + rank * 8), "l"(entry) : "memory");
            continue;
        }
        const uint32_t column = 0xffffffffu - static_cast<uint32_t>(entry);
        if (ids != nullptr) {
            if (k.wide_ids) reinterpret_cast<int64_t*>(ids)[rank] = column;
            else reinterpret_cast<int32_t*>(ids)[rank] = static_cast<int32_t>(column);
        }
        if (tops != nullptr) tops[rank] = (value_of(static_cast<uint32_t>(entry >> 32)) - x.at) * k.inverse - x.log_sum;
    }
}

// `blocks`: of a row's cluster (1: the blocks take row after row).
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, threads_on_sm(THREADS) / THREADS) logprobs_kernel(const Args k, uint32_t blocks) {
    constexpr int E = 16 / sizeof(T), kWarps = THREADS / 32, kChunk = THREADS * kBatch;  // (vectors of a chunk)
    extern __shared__ __align__(16) char shared[];
    __shared__ Part parts[2][kWarps];
    __shared__ Part cluster_parts[kMostBlocks];
    __shared__ int count, found;
    __shared__ uint32_t least;  // what an entry has to reach
    __shared__ int before[kWarps];
    pdl_prologue();
    const int tid = threadIdx.x, room = room_for(k.top);
    const uint32_t rank = blockIdx.x % blocks, stride = gridDim.x / blocks;
    uint64_t* const entries = reinterpret_cast<uint64_t*>(shared);
    uint64_t* const merged = entries + room;  // (of a cluster's first block)
    // where entries are wanted: every thread's maximum, its stretches', and the stretches that are read again
    uint32_t* const tops = reinterpret_cast<uint32_t*>(merged + (blocks > 1 ? blocks * k.top : 0));
    float* const stretch_tops = reinterpret_cast<float*>(tops + THREADS);
    uint16_t* const stretch_list = reinterpret_cast<uint16_t*>(stretch_tops + kStretches * THREADS);
    const float c = k.inverse * kLog2e, above = fminf(2.f / c, 1e30f);
    if (blocks > 1) cluster_sync();  // (every block is there before another writes to it)

    // What is on its way: this thread's vectors of the next chunk, of this row or of the one behind it; what is asked for after it, and the vectors left from there on.
    uint32_t row_next = blockIdx.x / blocks;
    const uint4* from;
    int left;
    auto begin = [&]() {
        const Row<T> row(k, row_next, rank, blocks);
        from = row.vectors() + row.first + tid;
        left = row.last - row.first;
    };
    begin();
    uint4 next[kBatch];
    auto ask = [&]() {
        while (left <= 0 && row_next < k.rows) {
            row_next += stride;
            if (row_next < k.rows) begin();
        }
        if (left >= kChunk) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) next[i] = __ldcs(from + i * THREADS);
        } else {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                next[i] = make_uint4(kNothing<T>, kNothing<T>, kNothing<T>, kNothing<T>);
                if (i * THREADS + tid < left) next[i] = __ldcs(from + i * THREADS);
            }
        }
        from += kChunk;
        left -= kChunk;
    };
    ask();

    auto token_of = [&](uint32_t r) { return tid == 0 && rank == 0 && r < k.rows && k.tokens.base != nullptr ? load_index(row_at(k.tokens, k.inner, r), k.wide_tokens) : int64_t(-1); };
    int64_t id = token_of(blockIdx.x / blocks);  // (asked for a row ahead)
    uint32_t parity = 0;
    for (uint32_t r = blockIdx.x / blocks; r < k.rows; r += stride, parity ^= 1) {
        const Row<T> row(k, r, rank, blocks);
        // an element of the row's ends for some threads
        int end = -1;
        if (rank == 0 && tid < row.head) end = tid;
        else if (rank + 1 == blocks && tid >= 8 && tid - 8 < k.vocab - row.tail) end = row.tail + (tid - 8);
        const T end_element = end >= 0 ? row.z[end] : from_float<T>(0.f);
        float token_z = 0.f;
        bool token = false;
        if (tid == 0) {
            if (id >= k.vocab) atomicOr(k.status, kStatusIndexOutOfRange);
            token = id >= 0 && id < k.vocab;
            if (token) token_z = to_float(row.z[id]);
            id = token_of(r + stride);
        }
        Part part{-INFINITY, 0.f, 0.f};
        // (two to the power of `shift` batches make a stretch)
        int shift = 0, batch = 0, stretch = 0;
        while ((row.last - row.first + kChunk - 1) / kChunk > kStretches << shift) ++shift;
        float most = -INFINITY, stretch_top = -INFINITY;
        for (int rest = row.last - row.first; rest > 0; rest -= kChunk) {
            uint4 raw[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) raw[i] = next[i];
            ask();
            const float top = largest<T>(raw);
            most = max_nan(most, top);
            if (rest == row.last - row.first) part.top = value_of(__reduce_max_sync(0xffffffffu, order_of(top))) + above;  // (the warp's, so that few lanes meet a larger one)
            take<T>(part, raw, top, c, above);
            if (k.top > 0) {
                stretch_top = max_nan(stretch_top, top);
                if ((++batch & ((1 << shift) - 1)) == 0 || rest <= kChunk) {
                    stretch_tops[stretch++ * THREADS + tid] = stretch_top;
                    stretch_top = -INFINITY;
                }
            }
        }
        const float end_z = to_float(end_element);
        if (end >= 0) {
            uint4 one[1] = {make_uint4(kNothing<T>, kNothing<T>, kNothing<T>, kNothing<T>)};
            if constexpr (sizeof(T) == 2) one[0].x = 0xfc000000u | __half_as_ushort(end_element);
            else one[0].x = __float_as_uint(end_element);
            take<T>(part, one, end_z, c, above);
            most = max_nan(most, end_z);
        }
        const uint32_t own = end >= 0 || row.first + tid < row.last ? order_of(most) : 0u;  // (0: this thread has no element)
        if (k.top > 0) tops[tid] = own;
        Part all = warp_part(part, most, c);
        if constexpr (kWarps > 1) {
            if (tid % 32 == 0) parts[parity][tid / 32] = all;
            __syncthreads();
            all = tid % 32 < kWarps ? parts[parity][tid % 32] : Part{-INFINITY, 0.f, 0.f};
            all = warp_part(all, all.top, c);
        } else {
            __syncwarp();
        }
        const float block_top = all.top;
        if (k.top == 0 && blocks == 1) {
            if (tid == 0) write_row(k, r, all, token, token_z);
            continue;
        }
        int n = 0;
        if (k.top > 0) {
            if (tid == 0) {
                count = 0, found = 0;
                if (blocks == 1) write_row(k, r, all, token, token_z);
            }
            if (tid >= THREADS - 32) {  // (the last warp:) a bound that at least `top` elements reach, if there are as many threads that have any
                uint32_t x[kWarps];
#pragma unroll
                for (int i = 0; i < kWarps; ++i) x[i] = tops[i * 32 + tid % 32];
                auto reaching = [&](uint32_t bound) {
                    int some = 0;
#pragma unroll
                    for (int i = 0; i < kWarps; ++i) some += x[i] >= bound;
                    return static_cast<int>(__reduce_add_sync(0xffffffffu, some));
                };
                uint32_t low = 0, high = order_of(block_top);
                if (k.top <= 32) {  // (what every lane's largest reaches, 32 do)
                    uint32_t lane_top = x[0];
#pragma unroll
                    for (int i = 1; i < kWarps; ++i) lane_top = max(lane_top, x[i]);
                    low = __reduce_min_sync(0xffffffffu, lane_top);
                }
                if (reaching(high) >= k.top) low = high;
                while (high - low > (sizeof(T) == 2 ? 8192u : 1u)) {
                    const uint32_t mid = low + (high - low) / 2;
                    const int reach = reaching(mid);
                    if (reach >= k.top) low = mid;
                    else high = mid;
                    if (reach >= k.top && reach <= k.top + k.top / 8) break;
                }
                if (tid == THREADS - 1) least = low;
            }
            __syncthreads();
            uint32_t lo = least;
            // (order, column) of a vector's elements that reach the bound, and, of one that is no number, others.
            auto each = [&](int v, uint32_t bound, auto&& visit) {
                const uint4 raw[1] = {row.vectors()[v]};
                const float at_least = value_of(bound);
                if (largest<T>(raw) < at_least) return;
                float x[E];
                unpack<T>(raw[0], x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (!(x[e] < at_least)) visit(order_of(x[e]), static_cast<uint32_t>(row.head + v * E + e));
                }
            };
            auto counted = [&](uint32_t bound) {  // how many of the elements reach a bound
                int some = 0;
                for (int v = row.first + tid; v < row.last && own >= bound; v += THREADS) each(v, bound, [&](uint32_t o, uint32_t) { some += o >= bound; });
                if (end >= 0) some += order_of(end_z) >= bound;
                some = __reduce_add_sync(0xffffffffu, some);
                __syncthreads();
                if (tid % 32 == 0) before[tid / 32] = some;
                __syncthreads();
                some = tid % 32 < kWarps ? before[tid % 32] : 0;
                return static_cast<int>(__reduce_add_sync(0xffffffffu, some));
            };
            auto collect = [&](uint32_t bound) {
                auto put = [&](uint32_t o, uint32_t column) {
                    if (o < bound) return;
                    const int i = atomicAdd(&count, 1);
                    if (i < room) entries[i] = uint64_t(o) << 32 | (0xffffffffu - column);
                };
                for (int s = 0; s < stretch && own >= bound; ++s) {
                    if (!(stretch_tops[s * THREADS + tid] < value_of(bound))) stretch_list[atomicAdd(&found, 1)] = static_cast<uint16_t>(s * THREADS + tid);
                }
                if (end >= 0) put(order_of(end_z), static_cast<uint32_t>(end));
                __syncthreads();
                const int all_found = found, bits = shift + 2;  // (a stretch's vectors)
                static_assert(kBatch == 4);
                for (int m = tid; m < all_found << bits; m += THREADS) {
                    const int at = stretch_list[m >> bits], v = row.first + ((at / THREADS << bits) + (m & ((1 << bits) - 1))) * THREADS + at % THREADS;
                    if (v < row.last) each(v, bound, put);
                }
                __syncthreads();
            };
            collect(lo);
            n = count;
            if (n > room) {
                uint32_t top = 0xffffffffu;
                if (counted(top) >= k.top) lo = top;
                else {
                    while (top - lo > 1) {
                        const uint32_t mid = lo + (top - lo) / 2;
                        const int reach = counted(mid);
                        if (reach >= k.top) {
                            lo = mid;
                            if (reach <= room) break;
                        } else {
                            top = mid;
                        }
                    }
                }
                const int equal_too = counted(lo);
                __syncthreads();
                if (tid == 0) count = 0, found = 0;
                __syncthreads();
                if (equal_too <= room) {
                    collect(lo);
                    n = count;
                } else {
                    // fewer than K are larger; of the equal ones those of the lowest columns
                    if (lo != 0xffffffffu) collect(lo + 1);
                    int have = count;
                    const int64_t from_column = rank == 0 ? 0 : row.head + int64_t(row.first) * E, to_column = rank + 1 == blocks ? k.vocab : row.head + int64_t(row.last) * E;
                    for (int64_t at = from_column; at < to_column && have < k.top; at += THREADS) {
                        const int64_t column = at + tid;
                        const bool hit = column < to_column && order_of(to_float(row.z[column])) == lo;
                        const uint32_t ballot = __ballot_sync(0xffffffffu, hit);
                        __syncthreads();
                        if (tid % 32 == 0) before[tid / 32] = __popc(ballot);
                        __syncthreads();
                        int at_most = have, in_front = have;
                        for (int w = 0; w < kWarps; ++w) {
                            if (w < tid / 32) in_front += before[w];
                            at_most += before[w];
                        }
                        const int i = in_front + __popc(ballot & ((1u << tid % 32) - 1));
                        if (hit && i < k.top) entries[i] = uint64_t(lo) << 32 | (0xffffffffu - static_cast<uint32_t>(column));
                        have = min(at_most, k.top);
                    }
                    __syncthreads();
                    n = have;
                }
            }
        }
        if (blocks == 1) {
            rank_entries(k, r, all, entries, n, nullptr);
        } else {
            // the first block takes what the others found: their parts, and as many entries as are wanted of each
            if (tid == 0) {
                const uint32_t to = in_block(shared_address(&cluster_parts[rank]), 0);
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(all.top) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(all.sum) : "memory");
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(all.turned) : "memory");
            }
            const uint32_t to = in_block(shared_address(merged + rank * k.top), 0);
            for (int i = tid + n; i < k.top; i += THREADS) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + i * 8), "l"(uint64_t(0)) : "memory");
            rank_entries(k, r, all, entries, n, &to);
            cluster_sync();
            if (rank == 0) {
                all = tid % 32 < static_cast<int>(blocks) ? cluster_parts[tid % 32] : Part{-INFINITY, 0.f, 0.f};
                all = warp_part(all, all.top, c);
                if (tid == 0) write_row(k, r, all, token, token_z);
                rank_entries(k, r, all, merged, static_cast<int>(blocks) * k.top, nullptr);
            }
        }
    }
}

// ---- the gradient -----------------------------------------------------------
//
// A thread takes four vectors, all of them asked for before the first is worked on; a row is as many threads' of a block, or blocks', as that makes.  2048 x 50001 F16:
// 75 us (5.5 TB/s; one exponential to an element); 4096 x 32000 F16 88 us (6.0 TB/s); 100000 x 256 F16 46 us, 226 by a block for each row.

constexpr int kGradThreads = 256;
constexpr int kGradVectors = 4;

// What a row's gradient is made of: q (plain + turned log q), and `given` at the token.
struct RowGrad {
    float at, log_sum, plain, turned, given;
    int64_t token;
};

__device__ __forceinline__ float grad_of(const RowGrad& g, float inverse, float z) {
    const float log_q = max_nan(fmaf(z - g.at, inverse, -g.log_sum), -200.f);
    return fast_exp2(log_q * kLog2e) * fmaf(g.turned, log_q, g.plain);
}

// SHORT: a block is several rows', 2^bits threads each.
template <typename T, bool SHORT>
__global__ void __launch_bounds__(kGradThreads) logprobs_grad_kernel(const Args k, uint32_t pieces, int bits) {
    constexpr int E = 16 / sizeof(T);
    pdl_prologue();
    const int threads = SHORT ? 1 << bits : kGradThreads, tid = static_cast<int>(threadIdx.x) & (threads - 1);
    const uint32_t r = SHORT ? blockIdx.x * (kGradThreads >> bits) + (threadIdx.x >> bits) : blockIdx.x / pieces, piece = SHORT ? 0 : blockIdx.x % pieces;
    if (SHORT && r >= k.rows) return;
    const T* const z = reinterpret_cast<const T*>(row_at(k.logits, k.inner, r));
    T* const to = reinterpret_cast<T*>(row_at(k.grad, k.inner, r));
    const int head = head_of(z, k.vocab);
    const int64_t vectors = (k.vocab - head) / E;
    const int64_t tail = head + vectors * E;
    RowGrad g{};
    g.token = -1;
    if (k.tokens.base != nullptr) {
        g.token = load_index(row_at(k.tokens, k.inner, r), k.wide_tokens);
        if (g.token >= k.vocab) {
            if (tid == 0) atomicOr(k.status, kStatusIndexOutOfRange);
            g.token = -1;
        }
    }
    const float4 stats = k.stats[r];
    const float a = k.logprobs_grad.base != nullptr && g.token >= 0 ? *reinterpret_cast<const float*>(row_at(k.logprobs_grad, k.inner, r)) : 0.f;
    const float w = k.entropies_grad.base != nullptr ? *reinterpret_cast<const float*>(row_at(k.entropies_grad, k.inner, r)) : 0.f;
    const bool zero = (a == 0.f && w == 0.f) || stats.x == -INFINITY;
    g.at = stats.x;
    g.log_sum = stats.y;
    g.given = a * k.scale;
    g.turned = -w * k.scale;
    g.plain = -(a + w * stats.z) * k.scale;
    if (zero) g.given = 0.f;
    const bool aligned = reinterpret_cast<uintptr_t>(to + head) % 16 == 0;
    auto value = [&](float x, int64_t column) { return (zero ? 0.f : grad_of(g, k.inverse, x)) + (column == g.token ? g.given : 0.f); };
    if (piece == 0) {
        if (tid < head) to[tid] = from_float<T>(value(zero ? 0.f : to_float(z[tid]), tid));
        const int64_t column = tail + (tid - 8);
        if (tid >= 8 && column < k.vocab) to[column] = from_float<T>(value(zero ? 0.f : to_float(z[column]), column));
    }
    const uint4* const zv = reinterpret_cast<const uint4*>(z + head);
    const int64_t first = int64_t(piece) * (threads * kGradVectors) + tid;
    uint4 raw[kGradVectors];
#pragma unroll
    for (int i = 0; i < kGradVectors; ++i) {
        const int64_t v = first + i * threads;
        raw[i] = !zero && v < vectors ? zv[v] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kGradVectors; ++i) {
        const int64_t v = first + i * threads;
        if (v >= vectors) break;
        float x[E];
        unpack<T>(raw[i], x);
        const int64_t column = head + v * E;
        if (zero) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = 0.f;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = grad_of(g, k.inverse, x[e]);
            if (g.token >= column && g.token < column + E) {
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] += g.token == column + e ? g.given : 0.f;
            }
        }
        T* const p = to + column;
        if (aligned) {
            uint32_t out[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 2) {
                    const __half2 h = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
                    out[j] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                    out[j] = __float_as_uint(x[j]);
                }
            }
            *reinterpret_cast<uint4*>(p) = make_uint4(out[0], out[1], out[2], out[3]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) p[e] = from_float<T>(x[e]);
        }
    }
}

// ---- arguments --------------------------------------------------------------

bool present(const b200_tensor& t) { return t.data != nullptr; }

struct Plan {
    int axes;
    int64_t vocab, top;
    RowShape s;
    bool told;  // tokens are given
};

void check_one_each(const b200_tensor& t, const char* name, const b200_tensor& logits, bool dense) {
    check_tensor(t, name);
    if (t.ndim != logits.ndim - 1 || !same_extents(t, logits, t.ndim)) fail(B200_SHAPE_ERROR, std::string(name) + ": not one for each row of logits");
    if (t.dtype != B200_F32) fail(B200_DTYPE_ERROR, std::string(name) + " is F32");
    if (dense && !is_dense(t)) fail(B200_NOT_IMPLEMENTED, std::string(name) + " is not dense");
}

Plan check_logprobs(const b200_token_logprobs_args& a, bool forward) {
    check_rows(a.logits, "logits");
    if (!is_float(a.logits.dtype)) fail(B200_DTYPE_ERROR, "logits are F32 or F16");
    const int axes = a.logits.ndim - 1;
    Plan plan{axes, a.logits.dims[axes], 0, row_shape(a.logits, axes), false};
    if (plan.vocab < 1 || plan.vocab >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "logits: rows of no element, or of 2^31 or more");
    if (!(a.temperature > 0.f) || std::isinf(a.temperature) || std::isinf(1.f / a.temperature * kLog2e)) {
        fail(B200_INVALID_ARGUMENT, "token_logprobs: the temperature is not above 0 and finite, or its inverse times log2 e is not");
    }
    plan.told = !is_absent(a.tokens, "tokens");
    if (plan.told) {
        check_tensor(a.tokens, "tokens");
        if (a.tokens.ndim != axes || !same_extents(a.tokens, a.logits, axes)) fail(B200_SHAPE_ERROR, "tokens: not one for each row of logits");
        if (!is_index(a.tokens.dtype)) fail(B200_DTYPE_ERROR, "tokens are I32 or I64");
    }
    for (const Named& t : {Named{&a.logprobs, "logprobs"}, Named{&a.entropies, "entropies"}}) {
        if (present(*t.t)) check_one_each(*t.t, t.name, a.logits, true);
    }
    for (const Named& t : {Named{&a.logprobs_grad, "logprobs_grad"}, Named{&a.entropies_grad, "entropies_grad"}}) {
        if (present(*t.t)) check_one_each(*t.t, t.name, a.logits, false);
    }
    if (present(a.stats)) check_stats(a.stats, plan.s.rows);
    for (const Named& t : {Named{&a.top_ids, "top_ids"}, Named{&a.top_logprobs, "top_logprobs"}}) {
        if (!present(*t.t)) continue;
        check_rows(*t.t, t.name);
        if (t.t->ndim != a.logits.ndim || !same_extents(*t.t, a.logits, axes)) fail(B200_SHAPE_ERROR, std::string(t.name) + ": rows of other extents than logits");
        plan.top = t.t->dims[axes];
    }
    if (present(a.top_ids) && !is_index(a.top_ids.dtype)) fail(B200_DTYPE_ERROR, "top_ids are I32 or I64");
    if (present(a.top_logprobs) && a.top_logprobs.dtype != B200_F32) fail(B200_DTYPE_ERROR, "top_logprobs are F32");
    if (present(a.top_ids) && present(a.top_logprobs) && a.top_ids.dims[axes] != a.top_logprobs.dims[axes]) fail(B200_SHAPE_ERROR, "top_ids and top_logprobs have different widths");
    if (plan.top > plan.vocab) fail(B200_SHAPE_ERROR, "token_logprobs: more of the largest logits than a row has");
    if (plan.top > kMostTop) fail(B200_NOT_IMPLEMENTED, "token_logprobs: more than 128 of the largest logits");
    if (present(a.grad)) {
        check_rows(a.grad, "grad");
        if (a.grad.ndim != a.logits.ndim || !same_extents(a.grad, a.logits, a.logits.ndim)) fail(B200_SHAPE_ERROR, "grad has not the logits' extents");
        if (a.grad.dtype != a.logits.dtype) fail(B200_DTYPE_ERROR, "grad has not the logits' type");
    }
    if (forward) {
        if (present(a.grad) || present(a.logprobs_grad) || present(a.entropies_grad)) fail(B200_INVALID_ARGUMENT, "token_logprobs computes no gradient");
        check_results({{&a.logprobs, "logprobs"}, {&a.entropies, "entropies"}, {&a.stats, "stats"}, {&a.top_ids, "top_ids"}, {&a.top_logprobs, "top_logprobs"}},
                      {{&a.logits, "logits"}, {&a.tokens, "tokens"}}, {});
    } else {
        if (present(a.logprobs) || present(a.entropies) || present(a.top_ids) || present(a.top_logprobs)) fail(B200_INVALID_ARGUMENT, "token_logprobs_backward computes the gradient alone");
        check_results({{&a.grad, "grad"}}, {{&a.tokens, "tokens"}, {&a.logprobs_grad, "logprobs_grad"}, {&a.entropies_grad, "entropies_grad"}, {&a.stats, "stats"}}, {{&a.logits, "logits"}});
    }
    if (plan.s.rows == 0) return plan;
    if (forward) {
        if (!present(a.logprobs) && !present(a.entropies) && !present(a.stats) && plan.top == 0) fail(B200_INVALID_ARGUMENT, "token_logprobs: no result is asked for");
        if (present(a.logprobs) && !plan.told) fail(B200_INVALID_ARGUMENT, "token_logprobs: log probabilities of no tokens");
    } else {
        if (!present(a.grad) || !present(a.stats)) fail(B200_INVALID_ARGUMENT, "token_logprobs_backward: grad and the forward call's stats are needed");
        if (present(a.logprobs_grad) && !plan.told) fail(B200_INVALID_ARGUMENT, "token_logprobs_backward: gradients of no tokens");
    }
    return plan;
}

// Pieces of a row's gradient, and the threads of one: a warp's at least, a block's at most.
int64_t grad_pieces(int64_t vocab, bool half) {
    const int64_t vectors = vocab / (half ? 8 : 4);
    return std::max<int64_t>(1, ceil_div(vectors, kGradThreads * kGradVectors));
}
int grad_bits(int64_t vocab, bool half) {
    const int64_t vectors = vocab / (half ? 8 : 4);
    int bits = 5;
    while (1 << bits < kGradThreads && vectors > int64_t(kGradVectors) << bits) ++bits;
    return bits;
}

Args common_args(b200_ctx* ctx, const b200_token_logprobs_args& a, const Plan& plan) {
    Args k{};
    k.logits = rows_arg(a.logits, plan.axes);
    if (plan.told) k.tokens = rows_arg(a.tokens, plan.axes);
    k.stats = static_cast<float4*>(a.stats.data);
    k.inner = FastDiv(static_cast<uint32_t>(plan.s.inner));
    k.status = ctx->d_status;
    k.vocab = plan.vocab;
    k.rows = static_cast<uint32_t>(plan.s.rows);
    k.wide_tokens = a.tokens.dtype == B200_I64;
    k.inverse = 1.f / a.temperature;
    return k;
}

void launch_logprobs(b200_ctx* ctx, const b200_token_logprobs_args& a) {
    const Plan plan = check_logprobs(a, true);
    if (plan.s.rows == 0) return;
    wait_for_tensors(ctx, {&a.logits, &a.tokens, &a.logprobs, &a.entropies, &a.stats, &a.top_ids, &a.top_logprobs});
    Args k = common_args(ctx, a, plan);
    k.logprobs = static_cast<float*>(a.logprobs.data);
    k.entropies = static_cast<float*>(a.entropies.data);
    if (present(a.top_ids)) k.ids = rows_arg(a.top_ids, plan.axes);
    if (present(a.top_logprobs)) k.tops = rows_arg(a.top_logprobs, plan.axes);
    k.top = static_cast<int>(plan.top);
    k.wide_ids = a.top_ids.dtype == B200_I64;
    ProfScope scope(ctx, "token_logprobs");
    const bool half = a.logits.dtype == B200_F16;
    const int64_t vectors = ceil_div(plan.vocab, half ? 8 : 4);
    // Threads of a block: as many as the rows leave room for on the device, of four vectors or more, up to 256 (300 x 128000 F32: 31 us, 98 with 64; 1024 x 128000 83 and
    // 95), or 512 where each row has an SM.  Many rows: 32 vectors to a thread, as a row's end costs it as much as 4 of them or more, up to 64 threads (2047 x 128000 F32:
    // 156 us, 161 with 128, 171 with 256), or 128 where entries are wanted and a thread's stretch would be more than one batch (the 20 largest of 2048 x 128000 F32: 188 us
    // with 64, 179 with 128, 195 with 256; of 4096 x 32000 F16 68 and 72).  And more threads than entries.  Few long rows are a cluster's each (1 x 128000 F32 6.2 us, 8.7 by one block; 16 x 128000 F16 with
    // the 20 largest 11.7 and 12.8).
    const int64_t rows = plan.s.rows, sms = sm_count();
    int threads = 32, blocks = 1;
    while (threads < (rows <= sms ? kMostThreads : kMostThreads / 2) && vectors > int64_t(threads) * 4 && rows * threads * 2 <= sms * threads_on_sm(threads * 2)) threads *= 2;
    while (threads < 64 && vectors > int64_t(threads) * 32) threads *= 2;
    if (plan.top > 0 && threads == 64 && vectors > int64_t(threads) * kBatch * kStretches) threads = 128;
    while (plan.top * 2 > threads) threads *= 2;
    while (blocks < kMostBlocks && rows * blocks * 2 <= sms && vectors >= int64_t(threads) * blocks * 8) blocks *= 2;
    auto go = [&](auto kernel) {
        size_t shared = 0;
        if (k.top > 0) shared += (static_cast<size_t>(room_for(k.top)) + (blocks > 1 ? static_cast<size_t>(blocks) * k.top : 0)) * 8 + static_cast<size_t>(threads) * (4 + 6 * kStretches);
        const int most = blocks_at_once(reinterpret_cast<const void*>(kernel), threads, shared);
        if (blocks > 1) {
            launch_kernel_clustered(ctx, kernel, dim3(static_cast<unsigned>(rows * blocks)), dim3(threads), shared, blocks, false, k, static_cast<uint32_t>(blocks));
            return;
        }
        // Blocks that stay: as many on an SM as leave the fewest without a last row, down to three quarters.
        auto rounds = [&](int on_sm) { return ceil_div(rows, sms * on_sm) * on_sm; };
        int on_sm = most;
        for (int n = most - 1; n * 4 >= most * 3; --n) {
            if (rounds(n) < rounds(on_sm)) on_sm = n;
        }
        launch_kernel(ctx, kernel, dim3(static_cast<unsigned>(std::min<int64_t>(rows, sms * on_sm))), dim3(threads), shared, k, 1u);
    };
    auto with = [&](auto element) {
        using T = decltype(element);
        switch (threads) {
            case 32: go(logprobs_kernel<T, 32>); break;
            case 64: go(logprobs_kernel<T, 64>); break;
            case 128: go(logprobs_kernel<T, 128>); break;
            case 256: go(logprobs_kernel<T, 256>); break;
            default: go(logprobs_kernel<T, 512>); break;
        }
    };
    if (half) with(__half{});
    else with(float{});
    check_last_launch("token_logprobs");
    ctx->count_launch();
}

void launch_logprobs_backward(b200_ctx* ctx, const b200_token_logprobs_args& a) {
    const Plan plan = check_logprobs(a, false);
    if (plan.s.rows == 0) return;
    const bool half = a.logits.dtype == B200_F16;
    const int64_t pieces = grad_pieces(plan.vocab, half);
    const int bits = grad_bits(plan.vocab, half);
    if (plan.s.rows * pieces >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "token_logprobs_backward: too many rows of this length");
    wait_for_tensors(ctx, {&a.logits, &a.tokens, &a.stats, &a.logprobs_grad, &a.entropies_grad, &a.grad});
    Args k = common_args(ctx, a, plan);
    if (present(a.logprobs_grad)) k.logprobs_grad = rows_arg(a.logprobs_grad, plan.axes);
    if (present(a.entropies_grad)) k.entropies_grad = rows_arg(a.entropies_grad, plan.axes);
    k.grad = rows_arg(a.grad, plan.axes);
    k.scale = a.grad_scale / a.temperature;
    ProfScope scope(ctx, "token_logprobs_backward");
    auto go = [&](auto kernel) {
        launch_kernel(ctx, kernel, dim3(static_cast<unsigned>(ceil_div(plan.s.rows * pieces, kGradThreads >> bits))), dim3(kGradThreads), 0, k, static_cast<uint32_t>(pieces), bits);
    };
    const bool shorts = 1 << bits < kGradThreads;
    if (half) go(shorts ? logprobs_grad_kernel<__half, true> : logprobs_grad_kernel<__half, false>);
    else go(shorts ? logprobs_grad_kernel<float, true> : logprobs_grad_kernel<float, false>);
    check_last_launch("token_logprobs_backward");
    ctx->count_launch();
}

}  // namespace

void check_token_logprobs(const b200_token_logprobs_args& a, bool forward) {
    const Plan plan = check_logprobs(a, forward);
    if (!forward && plan.s.rows * grad_pieces(plan.vocab, a.logits.dtype == B200_F16) >= (int64_t(1) << 31)) fail(B200_SHAPE_ERROR, "token_logprobs_backward: too many rows of this length");
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_token_logprobs(b200_ctx* ctx, const b200_token_logprobs_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_logprobs(ctx, *args); });
}

int b200_token_logprobs_backward(b200_ctx* ctx, const b200_token_logprobs_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_logprobs_backward(ctx, *args); });
}

}  // extern "C"
