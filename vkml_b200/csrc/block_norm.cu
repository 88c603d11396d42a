// Norms in front of and behind a block of a residual network, with its gate and the residual's scale, and their gradients.
//
//   u   = N(y) * w2 + b2            s = a * h + b * gate * u            n = N(s) * w1 + b1
//
// N(x) = (x - mean) * r with r = 1 / sqrt(var + eps) (layer norm), or x * r with r = 1 / sqrt(mean(x^2) + eps) (RMS norm).  With x^ = N(x)
// and g = dn * w1 the gradient through a norm is r * (g - mean(g) - x^ * mean(g * x^)), without mean(g) for the RMS norm; so
//
//   ds  = dout + r1 * (g - mean(g) - s^ * mean(g * s^))        dh = a * ds        dgate = sum over its rows of b * ds * u
//   du  = b * gate * ds       dw2 = sum du * y^      db2 = sum du       dw1 = sum dn * s^       db1 = sum dn
//   dy  = r2 * (q - mean(q) - y^ * mean(q * y^))  with q = du * w2
//
// Bound by memory: forward reads h and y and writes s and n, backward reads dout, dn, s and y and writes dh and dy.  A row is read once: it stays
// in the registers of the threads that share it, 8 elements of each tensor to a thread for each of its NV pieces.  Blocks stay on their SM and take
// one row after another, with the next row's loads under way while they work on one: a block that waits for its row, for the row's sums and then for
// the next block's start left the memory idle for a third (forward) and three quarters (backward) of the time.  What is summed over the row goes
// through shuffles and shared memory.
#include "operators.cuh"

#include <algorithm>
#include <type_traits>

namespace b200 {
namespace {

constexpr int64_t kMostWidth = 16384;
constexpr int kWarpRows = 8;  // warps of a block where a row is a warp's

// Sums of N values (1, 4 or 8) over the threads of a row, the same bits in each of them.  Lanes halve the values among each other before they halve the
// lanes: 6 shuffles for 4 values and 9 for 8, where one value after another takes 20 and 40.  `slot` alternates between calls, so that one
// barrier is enough.
template <bool WARP, int N>
__device__ __forceinline__ void row_sums(float (&x)[N], float* part, int& slot) {
    const int lane = threadIdx.x % 32;
    int d = 16;
#pragma unroll
    for (int half = N / 2; half >= 1; half /= 2, d /= 2) {
        const bool upper = (lane & d) != 0;
#pragma unroll
        for (int i = 0; i < half; ++i) {
            const float give = upper ? x[i] : x[i + half];
            x[i] = (upper ? x[i + half] : x[i]) + __shfl_xor_sync(0xffffffffu, give, d);
        }
    }
#pragma unroll
    for (; d > 0; d /= 2) x[0] += __shfl_xor_sync(0xffffffffu, x[0], d);
    constexpr int kLanes = 32 / N;  // lane v * kLanes has value v
    float total = x[0];
    int from = kLanes;
    if constexpr (!WARP) {
        const int values = blockDim.x / 32 * N;
        float* const here = part + slot * (N * 32);
        if (lane % kLanes == 0) here[threadIdx.x / 32 * N + lane / kLanes] = total;
        __syncthreads();
        total = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {  // lane l has values l % N of some warps
            if (i * 32 < values && i * 32 + lane < values) total += here[i * 32 + lane];
        }
#pragma unroll
        for (int e = N; e < 32; e *= 2) total += __shfl_xor_sync(0xffffffffu, total, e);
        slot ^= 1;
        from = 1;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = N == 1 ? total : __shfl_sync(0xffffffffu, total, i * from);
}

// Eight values to a thread in memory that no other thread touches: 16 bytes of the block's threads side by side.
__device__ __forceinline__ void own_store(float* p, int which, const float (&x)[8]) {
    float4* to = reinterpret_cast<float4*>(p) + (which * 2) * blockDim.x + threadIdx.x;
    to[0] = make_float4(x[0], x[1], x[2], x[3]);
    to[blockDim.x] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void own_load(const float* p, int which, float (&x)[8]) {
    const float4* from = reinterpret_cast<const float4*>(p) + (which * 2) * blockDim.x + threadIdx.x;
    const float4 a = from[0], b = from[blockDim.x];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// A piece of a vector over the columns (a weight, a bias, the gate), F32 or F16; `absent` where there is none.
template <bool WIDE>
__device__ __forceinline__ void read_columns(float (&x)[8], const void* p, bool half, float absent, int first, int t, int threads, int width) {
    if (p == nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = absent;
    } else if (half) {
        Piece<__half, WIDE> piece;
        piece.load(static_cast<const char*>(p), first, t, threads, width);
        piece.get(x);
    } else {
        Piece<float, WIDE> piece;
        piece.load(static_cast<const char*>(p), first, t, threads, width);
        piece.get(x);
    }
}

// A piece of sums over rows, in a row that may start anywhere.
template <typename T, bool WIDE>
__device__ __forceinline__ void store_columns(T* row, const float (&x)[8], int first, int t, int threads, int width) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int c = first + piece_column<WIDE>(e, t, threads);
        if (c < width) row[c] = from_float<T>(x[e]);
    }
}

// The rows of worker w of n: a stretch of them.
__device__ __forceinline__ uint32_t stretch(uint32_t rows, uint32_t w, uint32_t n) { return static_cast<uint32_t>(uint64_t(rows) * w / n); }

struct ForwardArgs {
    RowsArg residual, branch, out, normed;
    float4* stats;
    const void *post_weight, *post_bias, *pre_weight, *pre_bias, *gate;
    int64_t gate_pitch;  // bytes
    FastDiv inner, gate_rows;
    uint32_t rows;
    int width;
    float a, b, eps, share;  // share: 1 / width
    bool layer, post, half_columns;
};

// Mean and 1 / sqrt of a row's norm.  The variance is that of the differences to the mean, which the registers still hold: no cancellation.
template <bool WARP, bool WIDE, int NV>
__device__ __forceinline__ float2 norm_of(const float (&x)[NV][8], bool layer, float eps, float share, int t, int threads, int width, float* part, int& slot) {
    float mean[1] = {0.f}, square[1] = {0.f};
    if (layer) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) mean[0] += x[v][e];
        row_sums<WARP, 1>(mean, part, slot);
        mean[0] *= share;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = v * threads * 8 + piece_column<WIDE>(e, t, threads) < width ? x[v][e] - mean[0] : 0.f;
            square[0] += d * d;
        }
    row_sums<WARP, 1>(square, part, slot);
    return make_float2(mean[0], 1.f / sqrtf(square[0] * share + eps));
}

// AHEAD: the next row's loads are under way while a row is worked on (which takes registers that blocks of 1024 threads do not have).
template <typename TH, typename TY, int NV, bool WIDE, bool WARP, bool AHEAD>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : AHEAD ? 512 : 1024)
norm_kernel(const ForwardArgs k) {
    extern __shared__ __align__(16) float own[];  // the columns' factors: of the branch, of the norm in front; and their biases
    __shared__ float part[2 * 32];
    pdl_prologue();
    int slot = 0;
    const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x % 32 : threadIdx.x;
    const uint32_t workers = WARP ? gridDim.x * kWarpRows : gridDim.x, worker = WARP ? blockIdx.x * kWarpRows + threadIdx.x / 32 : blockIdx.x;
    const uint32_t r0 = stretch(k.rows, worker, workers), r1 = stretch(k.rows, worker + 1, workers);
    const bool has_residual = k.residual.base != nullptr, has_branch = k.branch.base != nullptr;
    const bool post_bias = k.post_bias != nullptr, pre_bias = k.pre_bias != nullptr;
    Piece<TH, WIDE> h_piece[NV];
    Piece<TY, WIDE> y_piece[NV];
    auto load = [&](uint32_t r) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (has_residual) h_piece[v].load(row_at(k.residual, k.inner, r), v * threads * 8, t, threads, k.width);
            else h_piece[v].clear();
            if (has_branch) y_piece[v].load(row_at(k.branch, k.inner, r), v * threads * 8, t, threads, k.width);
            else y_piece[v].clear();
        }
    };
    // The columns' factors and biases: b gate w2, w1, b gate b2, b1.  Kept in the thread's own shared memory (AHEAD; not for 1024 threads of 16 columns), else made
    // where they are needed.
    enum { kW2, kW1, kB2, kB1 };
    const char* gate = nullptr;
    auto read_factor = [&](int which, int v, float (&x)[8]) {
        const void* from = which == kW2 ? k.post_weight : which == kW1 ? k.pre_weight : which == kB2 ? k.post_bias : k.pre_bias;
        read_columns<WIDE>(x, from, k.half_columns, which == kW2 || which == kW1 ? 1.f : 0.f, v * threads * 8, t, threads, k.width);
        if (which == kW2 || which == kB2) {
            float g[8];
            read_columns<WIDE>(g, gate, k.half_columns, 1.f, v * threads * 8, t, threads, k.width);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= g[e] * k.b;
        }
    };
    auto place = [&](int which) { return which == kB1 && !post_bias ? 2 : which; };
    auto factor = [&](int which, int v, float (&x)[8]) {
        if constexpr (AHEAD) own_load(own, place(which) * NV + v, x);
        else read_factor(which, v, x);
    };
    auto keep_factor = [&](int which) {
        if constexpr (AHEAD) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float x[8];
                read_factor(which, v, x);
                own_store(own, place(which) * NV + v, x);
            }
        }
    };
    auto set_branch = [&](uint32_t group) {
        gate = static_cast<const char*>(k.gate);
        if (gate != nullptr) gate += int64_t(group) * k.gate_pitch;
        keep_factor(kW2);
        if (post_bias) keep_factor(kB2);
    };
    if (r0 < r1) load(r0);
    uint32_t group = r0 < r1 ? k.gate_rows.div(r0) : 0;
    if (r0 < r1 && has_branch) set_branch(group);
    if (r0 < r1 && k.normed.base != nullptr) {
        keep_factor(kW1);
        if (pre_bias) keep_factor(kB1);
    }
    for (uint32_t r = r0; r < r1; ++r) {
        float h[NV][8], y[NV][8];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            h_piece[v].get(h[v]);
            y_piece[v].get(y[v]);
        }
        if (AHEAD && r + 1 < r1) load(r + 1);
        float2 post = make_float2(0.f, 0.f), pre = make_float2(0.f, 0.f);
        if (k.post) post = norm_of<WARP, WIDE, NV>(y, k.layer, k.eps, k.share, t, threads, k.width, part, slot);
        const uint32_t now = k.gate_rows.div(r);
        if (now != group) {
            group = now;
            if (k.gate != nullptr) set_branch(group);
        }
        const float scale = k.post ? post.y : 1.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (has_branch) {
                float w[8];
                factor(kW2, v, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[v][e] = k.a * h[v][e] + (y[v][e] - post.x) * scale * w[e];
                if (post_bias) {
                    factor(kB2, v, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) h[v][e] += w[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) h[v][e] *= k.a;
            }
            if (k.out.base != nullptr) store_piece<TH, WIDE>(row_at(k.out, k.inner, r), h[v], v * threads * 8, t, threads, k.width);
            if (k.layer) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (v * threads * 8 + piece_column<WIDE>(e, t, threads) >= k.width) h[v][e] = 0.f;
                }
            }
        }
        if (k.normed.base != nullptr) {
            pre = norm_of<WARP, WIDE, NV>(h, k.layer, k.eps, k.share, t, threads, k.width, part, slot);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float w[8];
                factor(kW1, v, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[v][e] = (h[v][e] - pre.x) * pre.y * w[e];
                if (pre_bias) {
                    factor(kB1, v, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) h[v][e] += w[e];
                }
                store_piece<TY, WIDE>(row_at(k.normed, k.inner, r), h[v], v * threads * 8, t, threads, k.width);
            }
        }
        if (k.stats != nullptr && t == 0) k.stats[r] = make_float4(post.x, post.y, pre.x, pre.y);
        if (!AHEAD && r + 1 < r1) load(r + 1);
    }
}

// ---- backward ---------------------------------------------------------------

// Sums over rows: of the gate for each of its groups, of the weights and biases over all rows.
enum Sum { kGate, kPostWeight, kPostBias, kPreWeight, kPreBias, kSums };

struct BackwardArgs {
    RowsArg out, branch, out_grad, normed_grad, residual_grad, branch_grad;
    const float4* stats;
    const void *post_weight, *post_bias, *pre_weight, *gate;
    int64_t gate_pitch;          // bytes
    float* partial[kSums];       // [blocks][width], the gate's [items][width]; null: not wanted
    void* gate_grad;             // where a gate's rows are one item: its gradient itself, in place of partial[kGate]
    float* own;                  // the sums where registers do not hold them: [blocks][kOwnSums * NV * 8 * threads]; null: in shared memory
    FastDiv inner;
    uint32_t group_rows, pieces;  // rows to a gate, and how many items they are divided into
    uint32_t items;
    int width;
    float a, b, share;
    bool layer, post, half_columns, half_gate_grad;
    bool warp_items;  // WARP: an item is a warp's; else a block's, whose warps take its rows in turn
};

// In a gate's rows the gate and the weights are the same, so that two sums hold the gradients of three vectors: E = sum ds * y^ and F = sum ds, with
// dgate = b (w2 E + b2 F), dw2 += b gate E, db2 += b gate F at the end of the rows.  Both row sums of the two norms come from one reduction: with c = b gate w2
// and t = dout + r1 g, where ds = t - r1 (m0 + s^ m1),
//   mean(c y^ ds) = mean(c y^ t) - r1 (m0 mean(c y^) + m1 mean(c y^ s^))      mean(c ds) = mean(c t) - r1 (m0 mean(c) + m1 mean(c s^))
// A block takes items one after another: item i is piece i % pieces of the rows of gate i / pieces.  The gate's sums are left behind after each item, the others
// once, in the block's row of the partial sums; fold_kernel adds those up in order, so that no result depends on timing.
// FULL: layer norms and biases too; without it RMS norms alone.  REGS: the sums over rows stay in registers, else in the thread's own memory.
// HOLD: a row stays in registers between the reduction and the results, else it is read again.  AHEAD: the next row's loads are under way meanwhile.
enum OwnSum { kE, kPreW, kF, kPreB, kPostW, kPostB, kOwnSums };
constexpr int kOwnRms = 3;  // without FULL: kE, kPreW and kPostW, which come first in memory
__host__ __device__ constexpr int own_place(int which) { return which == kE ? 0 : which == kPreW ? 1 : which == kPostW ? 2 : which == kF ? 3 : which == kPreB ? 4 : 5; }

template <typename TH, typename TY, int NV, bool WIDE, bool WARP, bool FULL, bool REGS, bool HOLD, bool AHEAD>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : AHEAD ? 512 : 1024, WARP ? 2 : 1)
norm_backward_kernel(const BackwardArgs k) {
    constexpr int N = FULL ? 8 : 4;
    extern __shared__ __align__(16) float shared_own[];
    __shared__ float part[2 * N * 32];
    __shared__ float meet[WARP ? kWarpRows : 1][WARP ? 256 : 1];
    pdl_prologue();
    int slot = 0;
    const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x % 32 : threadIdx.x, warp = threadIdx.x / 32;
    float* const own = k.own != nullptr ? k.own + int64_t(blockIdx.x) * ((FULL ? kOwnSums : kOwnRms) * NV * 8) * blockDim.x : shared_own;
    constexpr bool KEEP = REGS || (HOLD && !FULL);                          // the columns' factors in shared memory, behind the sums there
    float* const factors = shared_own + (REGS ? 2 : kOwnRms) * NV * 8 * blockDim.x;  // (REGS: kPostW and kPostB lie in front)
    const bool pre = k.normed_grad.base != nullptr, branch = k.branch.base != nullptr || k.branch_grad.base != nullptr;
    // running sums: in registers, or in `own`
    float sum[REGS ? 4 : 1][REGS ? NV : 1][8];
    auto clear = [&](int which) {
        const float zero[8] = {};
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if constexpr (REGS) {
                if (which < 4) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum[which][v][e] = 0.f;
                } else {
                    own_store(shared_own, (which - kPostW) * NV + v, zero);
                }
            } else {
                own_store(own, own_place(which) * NV + v, zero);
            }
        }
    };
    auto get_sum = [&](int which, int v, float (&x)[8]) {
        if constexpr (REGS) {
            if (which < 4) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = sum[which][v][e];
            } else {
                own_load(shared_own, (which - kPostW) * NV + v, x);
            }
        } else {
            own_load(own, own_place(which) * NV + v, x);
        }
    };
    auto add = [&](int which, int v, const float (&x)[8]) {
        if constexpr (REGS) {
            if (which < 4) {
                add8(sum[which][v], sum[which][v], x);
                return;
            }
        }
        float y[8];
        get_sum(which, v, y);
        add8(y, y, x);
        if constexpr (REGS) own_store(shared_own, (which - kPostW) * NV + v, y);
        else own_store(own, own_place(which) * NV + v, y);
    };
    auto add_product = [&](int which, int v, const float (&a)[8], const float (&b)[8]) {
        if constexpr (REGS) {
            fma8(sum[which][v], a, b, sum[which][v]);
        } else {
            float y[8];
            get_sum(which, v, y);
            fma8(y, a, b, y);
            own_store(own, own_place(which) * NV + v, y);
        }
    };
    // WARP: a value summed over the block's warps, in the first one
    auto over_warps = [&](float (&x)[8]) {
        if constexpr (WARP) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) meet[warp][e * 32 + t] = x[e];
            __syncthreads();
            if (warp == 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    for (int w = 1; w < kWarpRows; ++w) x[e] += meet[w][e * 32 + t];
                }
            }
        }
    };
    // the columns' factors: w1 and c = b gate w2 in every row, b gate, w2 and b2 at an item's end; w1 and c from the thread's own memory where there is room (KEEP)
    enum { kW1, kC, kW2, kG, kB2 };
    const char* gate = nullptr;
    auto read_factor = [&](int which, int v, float (&x)[8]) {
        const int first = v * threads * 8;
        const void* from = which == kW1 ? k.pre_weight : which == kB2 ? k.post_bias : which == kG ? static_cast<const void*>(gate) : k.post_weight;
        read_columns<WIDE>(x, from, k.half_columns, which == kB2 ? 0.f : 1.f, first, t, threads, k.width);
        if (which == kG) mul8(x, x, k.b);
        if (which == kC) {
            float g[8];
            read_columns<WIDE>(g, gate, k.half_columns, 1.f, first, t, threads, k.width);
            mul8(g, g, k.b);
            mul8(x, x, g);
            if constexpr (!WIDE || FULL) {  // y^ is not 0 behind the row's end
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (first + piece_column<WIDE>(e, t, threads) >= k.width) x[e] = 0.f;
                }
            }
        }
    };
    auto factor = [&](int which, int v, float (&x)[8]) {
        if constexpr (KEEP) own_load(factors, which * NV + v, x);
        else read_factor(which, v, x);
    };
    auto keep_factor = [&](int which) {
        if constexpr (KEEP) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float x[8];
                read_factor(which, v, x);
                own_store(factors, which * NV + v, x);
            }
        }
    };
    Piece<TH, WIDE> s_piece[NV], o_piece[NV], s_next[AHEAD ? NV : 1], o_next[AHEAD ? NV : 1];
    Piece<TY, WIDE> n_piece[NV], y_piece[NV], n_next[AHEAD ? NV : 1], y_next[AHEAD ? NV : 1];
    float4 st = make_float4(0.f, 1.f, 0.f, 1.f), st_next = st;
    auto load_piece = [&](uint32_t r, int v, Piece<TH, WIDE>& s, Piece<TY, WIDE>& n, Piece<TH, WIDE>& o, Piece<TY, WIDE>& y) {
        const int first = v * threads * 8;
        if (pre) s.load(row_at(k.out, k.inner, r), first, t, threads, k.width);
        else s.clear();
        if (pre) n.load(row_at(k.normed_grad, k.inner, r), first, t, threads, k.width);
        else n.clear();
        if (k.out_grad.base != nullptr) o.load(row_at(k.out_grad, k.inner, r), first, t, threads, k.width);
        else o.clear();
        if (k.branch.base != nullptr) y.load(row_at(k.branch, k.inner, r), first, t, threads, k.width);
        else y.clear();
    };
#pragma unroll
    for (int s = 0; s < kOwnSums; ++s) {
        if (FULL || own_place(s) < kOwnRms) clear(s);
    }
    bool first_item = true;
    const bool by_warp = WARP && k.warp_items;
    const uint32_t step = WARP && !by_warp ? kWarpRows : 1, workers = by_warp ? gridDim.x * kWarpRows : gridDim.x;
    for (uint32_t item = by_warp ? blockIdx.x * kWarpRows + warp : blockIdx.x; item < k.items; item += workers) {
        const uint32_t group = item / k.pieces, piece = item % k.pieces;
        const uint32_t r0 = group * k.group_rows + stretch(k.group_rows, piece, k.pieces) + (step > 1 ? warp : 0);
        const uint32_t r1 = group * k.group_rows + stretch(k.group_rows, piece + 1, k.pieces);
        gate = static_cast<const char*>(k.gate);
        if (gate != nullptr) gate += int64_t(group) * k.gate_pitch;
        auto load_ahead = [&](uint32_t r) {
            if constexpr (AHEAD) {
#pragma unroll
                for (int v = 0; v < NV; ++v) load_piece(r, v, s_next[v], n_next[v], o_next[v], y_next[v]);
                if (k.stats != nullptr) st_next = k.stats[r];
            }
        };
        if (WIDE && r0 < r1) load_ahead(r0);  // (element by element it costs: 4096 x 3000 F16 took 75 us, 62 this way)
        if (first_item) keep_factor(kW1);
        first_item = false;
        keep_factor(kC);
        if (!WIDE && r0 < r1) load_ahead(r0);
        float mean_c = 0.f;  // FULL: of c
        if (FULL && k.layer && k.post) {
            float x[1] = {0.f};
            if (!WARP) __syncthreads();  // (the reductions before and after lay their values out otherwise)
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float c[8];
                factor(kC, v, c);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[0] += c[e];
            }
            row_sums<WARP, 1>(x, part, slot);
            if (!WARP) __syncthreads();
            mean_c = x[0] * k.share;
        }
        for (uint32_t r = r0; r < r1; r += step) {
            if constexpr (AHEAD) {
#pragma unroll
                for (int v = 0; v < NV; ++v) s_piece[v] = s_next[v], n_piece[v] = n_next[v], o_piece[v] = o_next[v], y_piece[v] = y_next[v];
                st = st_next;
                if (r + step < r1) load_ahead(r + step);
            } else {
                if constexpr (HOLD) {
#pragma unroll
                    for (int v = 0; v < NV; ++v) load_piece(r, v, s_piece[v], n_piece[v], o_piece[v], y_piece[v]);
                }
                if (k.stats != nullptr) st = k.stats[r];
            }
            const float y_scale = k.post ? st.y : 1.f, y_shift = FULL && k.post ? -st.x : 0.f;
            const float s_scale = pre ? st.w : 0.f, s_shift = FULL && pre ? -st.z : 0.f;
            float s[HOLD ? NV : 1][8], n[HOLD ? NV : 1][8], o[HOLD ? NV : 1][8], y[HOLD ? NV : 1][8];
            // s^, dn, t and y^ of a piece; adds g s^ and g
            float2 sum_gs = {}, sum_g = {};
            auto terms = [&](int v, bool sums) {
                const int h = HOLD ? v : 0;
                if constexpr (!HOLD) load_piece(r, v, s_piece[0], n_piece[0], o_piece[0], y_piece[0]);
                s_piece[h].get(s[h]);
                n_piece[h].get(n[h]);
                o_piece[h].get(o[h]);
                y_piece[h].get(y[h]);
                if constexpr (FULL) {  // (the difference first: what lies near the mean keeps its digits)
                    add8(s[h], s[h], s_shift);
                    add8(y[h], y[h], y_shift);
                }
                mul8(s[h], s[h], s_scale);
                mul8(y[h], y[h], y_scale);
                if (pre) {
                    float g[8];
                    factor(kW1, v, g);
                    mul8(g, g, n[h]);
                    fma8(o[h], g, st.w, o[h]);
                    if (sums) {
                        dot8(sum_gs, g, s[h]);
                        if (FULL) sum8(sum_g, g);
                    }
                }
            };
            float2 sum_cyt = {}, sum_cys = {}, sum_ct = {}, sum_cs = {}, sum_cy = {};
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int h = HOLD ? v : 0;
                terms(v, true);
                if (k.post) {
                    float c[8], cy[8];
                    factor(kC, v, c);
                    mul8(cy, c, y[h]);
                    dot8(sum_cyt, cy, o[h]);
                    dot8(sum_cys, cy, s[h]);
                    if (FULL && k.layer) {
                        dot8(sum_ct, c, o[h]);
                        dot8(sum_cs, c, s[h]);
                        sum8(sum_cy, cy);
                    }
                }
            }
            float x[N] = {};
            x[0] = sum_gs.x + sum_gs.y, x[1] = sum_cyt.x + sum_cyt.y, x[2] = sum_cys.x + sum_cys.y;
            if constexpr (FULL) {
                x[3] = sum_g.x + sum_g.y, x[4] = sum_ct.x + sum_ct.y, x[5] = sum_cs.x + sum_cs.y, x[6] = sum_cy.x + sum_cy.y;
            }
            row_sums<WARP, N>(x, part, slot);
            const float m1 = x[0] * k.share * s_scale;  // r1 m1, r1 m0
            const float m0 = FULL && k.layer ? x[3] * k.share * s_scale : 0.f;
            float k1 = 0.f, k0 = 0.f;
            if (k.post) {
                k1 = x[1] * k.share - m1 * (x[2] * k.share);
                if constexpr (FULL) {
                    if (k.layer) {
                        k1 -= m0 * (x[6] * k.share);
                        k0 = x[4] * k.share - m0 * mean_c - m1 * (x[5] * k.share);
                    }
                }
            }
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int h = HOLD ? v : 0;
                if constexpr (!HOLD) terms(v, false);
                if (pre) {
                    add_product(kPreW, v, n[h], s[h]);
                    if (FULL) add(kPreB, v, n[h]);
                    fma8(o[h], s[h], -m1, o[h]);  // ds
                    if constexpr (FULL) {
                        add8(o[h], o[h], -m0);
                    }
                }
                if (k.residual_grad.base != nullptr) {
                    float q[8];
                    mul8(q, o[h], k.a);
                    store_piece<TH, WIDE>(row_at(k.residual_grad, k.inner, r), q, v * threads * 8, t, threads, k.width);
                }
                if (branch) {
                    add_product(kE, v, o[h], y[h]);
                    if (FULL) add(kF, v, o[h]);
                    if (k.branch_grad.base != nullptr) {
                        float q[8];
                        factor(kC, v, q);
                        mul8(q, q, o[h]);
                        fma8(q, y[h], -k1, q);
                        if constexpr (FULL) fma8(q, q, y_scale, -k0 * y_scale);
                        else mul8(q, q, y_scale);
                        store_piece<TY, WIDE>(row_at(k.branch_grad, k.inner, r), q, v * threads * 8, t, threads, k.width);
                    }
                }
            }
        }
        // the item's sums
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float e_sum[8], f_sum[8] = {}, w[8], b[8] = {}, q[8];
            get_sum(kE, v, e_sum);
            if (FULL) get_sum(kF, v, f_sum);
            if (WARP && !by_warp) {
                over_warps(e_sum);
                if (FULL) over_warps(f_sum);
            }
            if (WARP && !by_warp && warp != 0) continue;
            if (k.partial[kGate] != nullptr || k.gate_grad != nullptr) {
                read_factor(kW2, v, w);
                if (FULL) read_factor(kB2, v, b);
#pragma unroll
                for (int e = 0; e < 8; ++e) q[e] = k.b * (w[e] * e_sum[e] + b[e] * f_sum[e]);
                // (the partial sums and a gate's gradient are dense, and may start anywhere)
                const int64_t at = int64_t(k.gate_grad != nullptr ? group : item) * k.width;
                if (k.gate_grad != nullptr && k.half_gate_grad) store_columns<__half, WIDE>(static_cast<__half*>(k.gate_grad) + at, q, v * threads * 8, t, threads, k.width);
                else store_columns<float, WIDE>((k.gate_grad != nullptr ? static_cast<float*>(k.gate_grad) : k.partial[kGate]) + at, q, v * threads * 8, t, threads, k.width);
            }
            read_factor(kG, v, w);
            mul8(e_sum, e_sum, w);
            if (FULL) mul8(f_sum, f_sum, w);
            add(kPostW, v, e_sum);
            if (FULL) add(kPostB, v, f_sum);
        }
        clear(kE);
        if (FULL) clear(kF);
    }
    const int own_of[kSums] = {kE, kPostW, kPostB, kPreW, kPreB};
#pragma unroll
    for (int s = kPostWeight; s < kSums; ++s) {
        if (k.partial[s] == nullptr || (!FULL && own_place(own_of[s]) >= kOwnRms)) continue;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float x[8];
            get_sum(own_of[s], v, x);
            over_warps(x);
            if (WARP && warp != 0) continue;
            store_columns<float, WIDE>(k.partial[s] + int64_t(blockIdx.x) * k.width, x, v * threads * 8, t, threads, k.width);
        }
    }
}

struct Fold {
    const float* from;   // [groups * parts][width]
    void* to;            // [groups][width], dense
    uint32_t groups, parts;
};
struct FoldArgs {
    Fold f[kSums];
    uint32_t vectors;  // folds of one group; one of several, the gate's, comes behind them
    int width;
    bool half;
};

// to[g][c] = sum over p of from[g * parts + p][c]: 32 columns to a block, kFoldShares threads to a column, each with its share of the parts in order, kFoldAtOnce of
// them under way.  (Eight threads to a column, eight parts under way: 10 us for 592 blocks' sums of 1024 columns, as long as their rows' reading waits.)
constexpr int kFoldShares = 16, kFoldAtOnce = 20;
__global__ void __launch_bounds__(32 * kFoldShares) fold_kernel(const FoldArgs k) {
    __shared__ float part[kFoldShares][33];
    pdl_prologue();
    const bool one = blockIdx.y < k.vectors;
    const Fold& f = k.f[one ? blockIdx.y : k.vectors];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32, c = blockIdx.x * 32 + x;
    const uint32_t step = one ? 1 : gridDim.y - k.vectors;  // (at least 1: this block is one of them)
    for (uint32_t g = one ? 0 : blockIdx.y - k.vectors; g < f.groups; g += step) {
        const uint32_t p0 = stretch(f.parts, y, kFoldShares), p1 = stretch(f.parts, y + 1, kFoldShares);
        const float* from = f.from + (int64_t(g) * f.parts + p0) * k.width + c;
        float sum = 0.f;
        for (uint32_t p = p0; p < p1; p += kFoldAtOnce, from += int64_t(kFoldAtOnce) * k.width) {
            float v[kFoldAtOnce];
#pragma unroll
            for (int i = 0; i < kFoldAtOnce; ++i) v[i] = p + i < p1 && c < k.width ? from[int64_t(i) * k.width] : 0.f;
#pragma unroll
            for (int i = 0; i < kFoldAtOnce; ++i) sum += v[i];
        }
        part[y][x] = sum;
        __syncthreads();
        if (y == 0 && c < k.width) {
            float total = part[0][x];
#pragma unroll
            for (int i = 1; i < kFoldShares; ++i) total += part[i][x];
            const int64_t at = int64_t(g) * k.width + c;
            if (k.half) static_cast<__half*>(f.to)[at] = __float2half_rn(total);
            else static_cast<float*>(f.to)[at] = total;
        }
        __syncthreads();
    }
}

// ---- arguments --------------------------------------------------------------

struct Shape {
    RowShape s;
    int axes = 0;
    int64_t width = 0, gates = 1;
    int residual_type = B200_F32, branch_type = B200_F32;
};

// The rows that a call has, all of the same extents, and the types of its two sides.
Shape check_sides(std::initializer_list<Named> residual_side, std::initializer_list<Named> branch_side, int32_t kind, uint32_t flags) {
    Shape p;
    const b200_tensor* like = nullptr;
    int types[2] = {-1, -1};
    int side = 0;
    for (const auto& list : {residual_side, branch_side}) {
        for (const Named& n : list) {
            if (is_absent(*n.t, n.name)) continue;
            check_rows(*n.t, n.name);
            if (like == nullptr) like = n.t;
            if (n.t->ndim != like->ndim || !same_extents(*n.t, *like, like->ndim)) fail(B200_SHAPE_ERROR, std::string(n.name) + ": rows of other extents");
            if (types[side] < 0) types[side] = n.t->dtype;
            if (!is_float(n.t->dtype) || types[side] != n.t->dtype) fail(B200_DTYPE_ERROR, std::string(n.name) + ": the rows of a side have one type, F32 or F16");
        }
        ++side;
    }
    if (like == nullptr) fail(B200_INVALID_ARGUMENT, "block_norm: no rows are given");
    if (types[0] < 0) types[0] = types[1];
    if (types[1] < 0) types[1] = types[0];
    if (types[0] == B200_F16 && types[1] == B200_F32) fail(B200_DTYPE_ERROR, "block_norm: a residual in F16 beside a branch in F32");
    if (kind != B200_NORM_RMS && kind != B200_NORM_LAYER) fail(B200_INVALID_ARGUMENT, "block_norm: unknown kind of norm");
    if ((flags & ~B200_NORM_POST) != 0) fail(B200_INVALID_ARGUMENT, "block_norm: unknown flags");
    p.axes = like->ndim - 1;
    p.s = row_shape(*like, p.axes);
    p.width = like->dims[p.axes];
    if (p.width > kMostWidth) fail(B200_NOT_IMPLEMENTED, "block_norm: rows of more than 16384 elements");
    p.residual_type = types[0];
    p.branch_type = types[1];
    return p;
}

bool present(const b200_tensor& t) { return t.data != nullptr; }
// Rows of no element have no storage, and are there all the same.  (For tensors that check_sides has looked at.)
bool given(const b200_tensor& t) { return present(t) || (t.ndim != 0 && numel_of(t) == 0); }

// Weights, biases and gate, or their gradients: one type, dense, of the rows' width.  The gate has a row for each of its groups.
int check_columns(std::initializer_list<Named> vectors, const Named& gate, Shape& p) {
    int type = -1;
    auto typed = [&](const Named& n) {
        check_tensor(*n.t, n.name);
        if (type < 0) type = n.t->dtype;
        if (!is_float(n.t->dtype) || type != n.t->dtype) fail(B200_DTYPE_ERROR, std::string(n.name) + ": weights, biases and gate have one type, F32 or F16");
        if (!is_dense(*n.t)) fail(B200_NOT_IMPLEMENTED, std::string(n.name) + " is not dense");
    };
    for (const Named& n : vectors) {
        if (!present(*n.t)) continue;
        typed(n);
        if (n.t->ndim != 1 || n.t->dims[0] != p.width) fail(B200_SHAPE_ERROR, std::string(n.name) + ": not a vector of the rows' width");
    }
    if (present(*gate.t)) {
        typed(gate);
        const b200_tensor& g = *gate.t;
        if (g.ndim < 1 || g.ndim > 2 || g.dims[g.ndim - 1] != p.width) fail(B200_SHAPE_ERROR, std::string(gate.name) + ": not [width] or [groups, width]");
        p.gates = g.ndim == 2 ? g.dims[0] : 1;
        if (p.gates < 1 || p.s.rows % p.gates != 0) fail(B200_SHAPE_ERROR, std::string(gate.name) + ": the rows do not divide into its groups");
    }
    return type;
}

template <typename Fn>
void with_types(const Shape& p, Fn&& fn) {
    if (p.residual_type == B200_F16) fn(__half{}, __half{});
    else if (p.branch_type == B200_F16) fn(float{}, __half{});
    else fn(float{}, float{});
}

bool aligned_columns(const void* p) { return reinterpret_cast<uintptr_t>(p) % 32 == 0; }

Shape check_forward(const b200_block_norm_args& a, int& columns) {
    Shape p = check_sides({{&a.residual, "residual"}, {&a.out, "out"}}, {{&a.branch, "branch"}, {&a.normed, "normed"}}, a.kind, a.flags);
    columns = check_columns({{&a.post_weight, "post_weight"}, {&a.post_bias, "post_bias"}, {&a.pre_weight, "pre_weight"}, {&a.pre_bias, "pre_bias"}}, {&a.gate, "gate"}, p);
    if (!given(a.branch) && (present(a.gate) || (a.flags & B200_NORM_POST) != 0)) fail(B200_INVALID_ARGUMENT, "block_norm: a gate or a norm of an absent branch");
    if ((a.flags & B200_NORM_POST) == 0 && (present(a.post_weight) || present(a.post_bias))) fail(B200_INVALID_ARGUMENT, "block_norm: weights of a norm that is not applied");
    if (!given(a.normed) && (present(a.pre_weight) || present(a.pre_bias))) fail(B200_INVALID_ARGUMENT, "block_norm: weights of a norm that is not applied");
    if (present(a.stats)) check_stats(a.stats, p.s.rows);
    check_results({{&a.out, "out"}, {&a.normed, "normed"}, {&a.stats, "stats"}},
                  {{&a.post_weight, "post_weight"}, {&a.post_bias, "post_bias"}, {&a.pre_weight, "pre_weight"}, {&a.pre_bias, "pre_bias"}, {&a.gate, "gate"}},
                  {{&a.residual, "residual"}, {&a.branch, "branch"}});
    if (p.s.rows == 0 || p.width == 0) return p;
    if (!present(a.residual) && !present(a.branch)) fail(B200_INVALID_ARGUMENT, "block_norm: neither residual nor branch is given");
    if (!present(a.out) && !present(a.normed)) fail(B200_INVALID_ARGUMENT, "block_norm: no result is asked for");
    return p;
}

void launch_forward(b200_ctx* ctx, const b200_block_norm_args& a) {
    int columns = -1;
    const Shape p = check_forward(a, columns);
    if (p.s.rows == 0 || p.width == 0) return;
    wait_for_tensors(ctx, {&a.residual, &a.branch, &a.out, &a.normed, &a.stats, &a.post_weight, &a.post_bias, &a.pre_weight, &a.pre_bias, &a.gate});
    ForwardArgs k{};
    k.residual = rows_arg(a.residual, present(a.residual) ? p.axes : 0);
    k.branch = rows_arg(a.branch, present(a.branch) ? p.axes : 0);
    k.out = rows_arg(a.out, present(a.out) ? p.axes : 0);
    k.normed = rows_arg(a.normed, present(a.normed) ? p.axes : 0);
    k.stats = static_cast<float4*>(a.stats.data);
    k.post_weight = a.post_weight.data;
    k.post_bias = a.post_bias.data;
    k.pre_weight = a.pre_weight.data;
    k.pre_bias = a.pre_bias.data;
    k.gate = a.gate.data;
    k.half_columns = columns == B200_F16;
    k.gate_pitch = p.width * (k.half_columns ? 2 : 4);
    k.inner = FastDiv(static_cast<uint32_t>(p.s.inner));
    k.gate_rows = FastDiv(static_cast<uint32_t>(p.s.rows / p.gates));
    k.rows = static_cast<uint32_t>(p.s.rows);
    k.width = static_cast<int>(p.width);
    k.a = a.residual_scale;
    k.b = a.branch_scale;
    k.eps = a.eps;
    k.share = 1.f / static_cast<float>(p.width);
    k.layer = a.kind == B200_NORM_LAYER;
    k.post = (a.flags & B200_NORM_POST) != 0;
    const bool wide = p.width % 8 == 0 && aligned_rows(k.residual, p.residual_type) && aligned_rows(k.branch, p.branch_type) && aligned_rows(k.out, p.residual_type) && aligned_rows(k.normed, p.branch_type) &&
                      aligned_columns(k.post_weight) && aligned_columns(k.post_bias) && aligned_columns(k.pre_weight) && aligned_columns(k.pre_bias) && aligned_columns(k.gate);
    // narrow rows are a warp's, eight of them to a block; wider ones a block's with one piece to a thread, two above 2048 columns
    const bool warp = p.width <= 256;
    const int pieces = p.width <= 2048 ? 1 : 2;
    const int threads = warp ? kWarpRows * 32 : static_cast<int>(ceil_div(p.width, int64_t(8) * pieces * 32)) * 32;
    const size_t shared = threads > 512 ? 0 : static_cast<size_t>(2 + (k.post_bias != nullptr) + (k.pre_bias != nullptr)) * pieces * 32 * threads;
    ProfScope scope(ctx, "block_norm");
    with_types(p, [&](auto th, auto ty) {
        using TH = decltype(th);
        using TY = decltype(ty);
        auto go = [&](auto kernel) {
            const int64_t most = int64_t(sm_count()) * blocks_at_once(reinterpret_cast<const void*>(kernel), threads, shared);
            const int64_t blocks = std::min<int64_t>(most, warp ? ceil_div(p.s.rows, kWarpRows) : p.s.rows);
            launch_kernel(ctx, kernel, dim3(static_cast<unsigned>(blocks)), dim3(static_cast<unsigned>(threads)), shared, k);
        };
        auto of_width = [&](auto is_wide) {
            constexpr bool W = decltype(is_wide)::value;
            if (warp) go(norm_kernel<TH, TY, 1, W, true, true>);
            else if (pieces == 1) go(norm_kernel<TH, TY, 1, W, false, true>);
            else if (threads <= 512) go(norm_kernel<TH, TY, 2, W, false, true>);
            else go(norm_kernel<TH, TY, 2, W, false, false>);
        };
        if (wide) of_width(std::true_type{});
        else of_width(std::false_type{});
    });
    check_last_launch("block_norm");
    ctx->count_launch();
}

// How a backward call is divided.  Rows of up to 256 elements are a warp's; up to 4096 a block's of up to 512 threads that keep the sums over rows in
// registers; up to 8192 a block's of up to 1024 threads that keep them in shared memory; wider ones are read twice by 1024 threads.
struct Division {
    uint32_t blocks, threads, pieces, items;
    bool warp, regs, hold, full, warp_items, direct_gate;
    int nv;
    size_t shared;
    int64_t partial_floats[kSums], own_floats;
    size_t bytes;
};

constexpr size_t kMostShared = 220 << 10;

Division divide(const b200_block_norm_grad_args& a, const Shape& p, int sms) {
    Division d{};
    d.warp = p.width <= 256;
    d.regs = p.width <= 4096;
    d.hold = p.width <= 8192;
    d.nv = d.hold ? 1 : 2;
    d.threads = d.warp ? kWarpRows * 32 : static_cast<uint32_t>(ceil_div(p.width, int64_t(8) * d.nv * 32)) * 32;
    d.full = a.kind == B200_NORM_LAYER || present(a.post_bias) || present(a.post_bias_grad) || present(a.pre_bias_grad);
    const size_t own = static_cast<size_t>(d.nv) * 32 * d.threads;  // bytes of one vector of the threads' columns
    d.shared = d.regs ? own * 4 : d.full ? own * kOwnSums : own * (kOwnRms + (d.hold ? 2 : 0));
    const bool own_shared = d.shared <= kMostShared;
    if (!own_shared) d.shared = 0;
    const int64_t group_rows = p.s.rows / p.gates;
    // as many blocks as the registers of an SM hold at once
    const int64_t resident = int64_t(sms) * std::max<int64_t>(1, std::min<int64_t>((d.regs ? 512 : 1024) / d.threads, static_cast<int64_t>(kMostShared / (d.shared + 4096))));
    // warps share a block's rows, unless a gate has too few of them
    d.warp_items = d.warp && p.gates > 1 && group_rows < 8 * kWarpRows;
    const int64_t workers = d.warp_items ? resident * kWarpRows : resident;
    const int64_t unit = d.warp && !d.warp_items ? kWarpRows : 1;  // rows that a worker takes at once
    // a gate's rows in as many pieces as leave the longest worker the least to do
    int64_t best = INT64_MAX;
    d.pieces = 1;
    for (int64_t n = 1; n <= std::min(ceil_div(group_rows, unit), workers) && (n == 1 || p.gates * n < 2 * workers + p.gates); ++n) {
        const int64_t longest = ceil_div(p.gates * n, workers) * ceil_div(ceil_div(group_rows, n), unit);
        if (longest < best) best = longest, d.pieces = static_cast<uint32_t>(n);
    }
    d.items = static_cast<uint32_t>(p.gates * d.pieces);
    const int64_t needed = std::min<int64_t>(workers, d.items);
    d.blocks = static_cast<uint32_t>(d.warp_items ? ceil_div(needed, kWarpRows) : needed);
    d.direct_gate = d.pieces == 1;
    const b200_tensor* wanted[kSums] = {&a.gate_grad, &a.post_weight_grad, &a.post_bias_grad, &a.pre_weight_grad, &a.pre_bias_grad};
    auto whole = [](int64_t floats) { return (static_cast<size_t>(floats) * sizeof(float) + 255) / 256 * 256; };
    for (int s = 0; s < kSums; ++s) {
        if (!present(*wanted[s]) || (s == kGate && d.direct_gate)) continue;
        d.partial_floats[s] = int64_t(s == kGate ? d.items : d.blocks) * p.width;
        d.bytes += whole(d.partial_floats[s]);
    }
    if (!own_shared) {
        d.own_floats = int64_t(d.blocks) * (d.full ? kOwnSums : kOwnRms) * d.nv * 8 * d.threads;
        d.bytes += whole(d.own_floats);
    }
    return d;
}

Shape check_backward(const b200_block_norm_grad_args& a) {
    Shape p = check_sides({{&a.out, "out"}, {&a.out_grad, "out_grad"}, {&a.residual_grad, "residual_grad"}},
                          {{&a.branch, "branch"}, {&a.normed_grad, "normed_grad"}, {&a.branch_grad, "branch_grad"}}, a.kind, a.flags);
    check_columns({{&a.post_weight, "post_weight"}, {&a.post_bias, "post_bias"}, {&a.pre_weight, "pre_weight"}}, {&a.gate, "gate"}, p);
    const int64_t gates = p.gates;
    check_columns({{&a.post_weight_grad, "post_weight_grad"}, {&a.post_bias_grad, "post_bias_grad"}, {&a.pre_weight_grad, "pre_weight_grad"},
                   {&a.pre_bias_grad, "pre_bias_grad"}}, {&a.gate_grad, "gate_grad"}, p);
    if (present(a.gate) && present(a.gate_grad) && gates != p.gates) fail(B200_SHAPE_ERROR, "gate_grad has not the gate's extents");
    if (present(a.gate)) p.gates = gates;
    const bool post = (a.flags & B200_NORM_POST) != 0, pre = given(a.normed_grad);
    if (!post && (present(a.post_weight) || present(a.post_bias) || present(a.post_weight_grad) || present(a.post_bias_grad))) {
        fail(B200_INVALID_ARGUMENT, "block_norm_backward: weights of a norm that is not applied");
    }
    if (p.s.rows != 0 && p.width != 0) {
        if (!pre && !present(a.out_grad)) fail(B200_INVALID_ARGUMENT, "block_norm_backward: neither out_grad nor normed_grad is given");
        if (pre && !present(a.out)) fail(B200_INVALID_ARGUMENT, "block_norm_backward: the gradient through a norm needs out");
        if (!present(a.branch) && ((post && present(a.branch_grad)) || present(a.gate_grad) || present(a.post_weight_grad) || present(a.post_bias_grad))) {
            fail(B200_INVALID_ARGUMENT, "block_norm_backward: the branch is needed");
        }
        if ((pre || post) && !present(a.stats)) fail(B200_INVALID_ARGUMENT, "block_norm_backward: the forward call's stats are needed");
    }
    if (!pre && (present(a.pre_weight) || present(a.pre_weight_grad) || present(a.pre_bias_grad))) {
        fail(B200_INVALID_ARGUMENT, "block_norm_backward: gradients of a norm whose result has none");
    }
    if (present(a.stats)) check_stats(a.stats, p.s.rows);
    const b200_tensor scratch = workspace_tensor(a.workspace, a.workspace_bytes);
    check_results({{&a.residual_grad, "residual_grad"}, {&a.branch_grad, "branch_grad"}, {&a.post_weight_grad, "post_weight_grad"}, {&a.post_bias_grad, "post_bias_grad"},
                   {&a.pre_weight_grad, "pre_weight_grad"}, {&a.pre_bias_grad, "pre_bias_grad"}, {&a.gate_grad, "gate_grad"}, {&scratch, "workspace"}},
                  {{&a.post_weight, "post_weight"}, {&a.post_bias, "post_bias"}, {&a.pre_weight, "pre_weight"}, {&a.gate, "gate"}, {&a.stats, "stats"}},
                  {{&a.out, "out"}, {&a.branch, "branch"}, {&a.out_grad, "out_grad"}, {&a.normed_grad, "normed_grad"}});
    return p;
}

void launch_backward(b200_ctx* ctx, const b200_block_norm_grad_args& a) {
    const Shape p = check_backward(a);
    const Division d = p.s.rows != 0 && p.width != 0 ? divide(a, p, sm_count()) : Division{};
    check_workspace(a.workspace, a.workspace_bytes, d.bytes);
    const b200_tensor* vectors[kSums] = {&a.gate_grad, &a.post_weight_grad, &a.post_bias_grad, &a.pre_weight_grad, &a.pre_bias_grad};
    if (p.width == 0) return;
    char* scratch = operator_workspace(ctx, a.workspace, d.bytes);  // (refuses, too, before anything is queued)
    wait_for_tensors(ctx, {&a.out, &a.branch, &a.stats, &a.out_grad, &a.normed_grad, &a.post_weight, &a.post_bias, &a.gate, &a.pre_weight, &a.residual_grad, &a.branch_grad,
                           &a.post_weight_grad, &a.post_bias_grad, &a.pre_weight_grad, &a.pre_bias_grad, &a.gate_grad});
    if (p.s.rows == 0) {  // sums of nothing
        for (const b200_tensor* t : vectors) {
            if (present(*t)) B200_CUDA_CHECK(cudaMemsetAsync(t->data, 0, static_cast<size_t>(numel_of(*t)) * dtype_size(t->dtype), ctx->stream));
        }
        return;
    }
    BackwardArgs k{};
    auto rows = [&](const b200_tensor& t) { return rows_arg(t, present(t) ? p.axes : 0); };
    k.out = rows(a.out);
    k.branch = rows(a.branch);
    k.out_grad = rows(a.out_grad);
    k.normed_grad = rows(a.normed_grad);
    k.residual_grad = rows(a.residual_grad);
    k.branch_grad = rows(a.branch_grad);
    k.stats = static_cast<const float4*>(a.stats.data);
    k.post_weight = a.post_weight.data;
    k.post_bias = a.post_bias.data;
    k.pre_weight = a.pre_weight.data;
    k.gate = a.gate.data;
    int columns = -1;
    for (const b200_tensor* t : {&a.post_weight, &a.post_bias, &a.pre_weight, &a.gate}) {
        if (present(*t)) columns = t->dtype;
    }
    k.half_columns = columns == B200_F16;
    k.gate_pitch = p.width * (k.half_columns ? 2 : 4);
    FoldArgs fold{};
    fold.width = static_cast<int>(p.width);
    unsigned folds = 0, groups = 0;
    auto take = [&](int64_t floats) {
        float* at = reinterpret_cast<float*>(scratch);
        scratch += (static_cast<size_t>(floats) * sizeof(float) + 255) / 256 * 256;
        return at;
    };
    if (d.own_floats > 0) k.own = take(d.own_floats);
    for (int s : {kPostWeight, kPostBias, kPreWeight, kPreBias, kGate}) {
        if (!present(*vectors[s])) continue;
        if (s == kGate && d.direct_gate) {
            k.gate_grad = vectors[s]->data;
            k.half_gate_grad = vectors[s]->dtype == B200_F16;
            continue;
        }
        k.partial[s] = take(d.partial_floats[s]);
        const bool several = s == kGate && p.gates > 1;
        fold.f[folds++] = Fold{k.partial[s], vectors[s]->data, static_cast<uint32_t>(several ? p.gates : 1), s == kGate ? d.pieces : d.blocks};
        if (several) groups = static_cast<unsigned>(std::min<int64_t>(p.gates, 4096));
        else ++fold.vectors;
        fold.half = vectors[s]->dtype == B200_F16;
    }
    k.inner = FastDiv(static_cast<uint32_t>(p.s.inner));
    k.group_rows = static_cast<uint32_t>(p.s.rows / p.gates);
    k.pieces = d.pieces;
    k.items = d.items;
    k.warp_items = d.warp_items;
    k.width = static_cast<int>(p.width);
    k.a = a.residual_scale;
    k.b = a.branch_scale;
    k.share = 1.f / static_cast<float>(p.width);
    k.layer = a.kind == B200_NORM_LAYER;
    k.post = (a.flags & B200_NORM_POST) != 0;
    const bool wide = p.width % 8 == 0 && aligned_rows(k.out, p.residual_type) && aligned_rows(k.branch, p.branch_type) && aligned_rows(k.out_grad, p.residual_type) && aligned_rows(k.normed_grad, p.branch_type) &&
                      aligned_rows(k.residual_grad, p.residual_type) && aligned_rows(k.branch_grad, p.branch_type) && aligned_columns(k.post_weight) && aligned_columns(k.post_bias) &&
                      aligned_columns(k.pre_weight) && aligned_columns(k.gate);
    ProfScope scope(ctx, "block_norm_backward");
    with_types(p, [&](auto th, auto ty) {
        using TH = decltype(th);
        using TY = decltype(ty);
        auto go = [&](auto kernel) {
            (void)blocks_at_once(reinterpret_cast<const void*>(kernel), static_cast<int>(d.threads), d.shared);  // (allows that much shared memory)
            launch_kernel(ctx, kernel, dim3(d.blocks), dim3(d.threads), d.shared, k);
        };
        auto of_kind = [&](auto is_wide, auto is_full) {
            constexpr bool W = decltype(is_wide)::value, F = decltype(is_full)::value;
            if (d.warp) go(norm_backward_kernel<TH, TY, 1, W, true, F, true, true, true>);
            else if (d.regs) go(norm_backward_kernel<TH, TY, 1, W, false, F, true, true, true>);
            else if (d.hold) go(norm_backward_kernel<TH, TY, 1, W, false, F, false, true, false>);
            else go(norm_backward_kernel<TH, TY, 2, W, false, F, false, false, false>);
        };
        if (wide && d.full) of_kind(std::true_type{}, std::true_type{});
        else if (wide) of_kind(std::true_type{}, std::false_type{});
        else if (d.full) of_kind(std::false_type{}, std::true_type{});
        else of_kind(std::false_type{}, std::false_type{});
    });
    check_last_launch("block_norm_backward");
    if (folds > 0) {
        launch_kernel(ctx, fold_kernel, dim3(static_cast<unsigned>(ceil_div(p.width, 32)), fold.vectors + groups), 32 * kFoldShares, 0, fold);
        check_last_launch("block_norm_backward");
    }
    ctx->count_launch(folds > 0 ? 2 : 1);
}

}  // namespace

void check_block_norm(const b200_block_norm_args& a) {
    int columns = -1;
    (void)check_forward(a, columns);
}
void check_block_norm_backward(const b200_block_norm_grad_args& a) {
    const Shape p = check_backward(a);
    if (a.workspace != nullptr && p.s.rows != 0 && p.width != 0) check_workspace(a.workspace, a.workspace_bytes, divide(a, p, sm_count()).bytes);
}

}  // namespace b200

using namespace b200;

extern "C" {

int b200_block_norm(b200_ctx* ctx, const b200_block_norm_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_forward(ctx, *args); });
}

int b200_block_norm_backward(b200_ctx* ctx, const b200_block_norm_grad_args* args) {
    if (ctx == nullptr || args == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(ctx, [&] { launch_backward(ctx, *args); });
}

int b200_block_norm_backward_workspace(const b200_block_norm_grad_args* args, size_t* nbytes) {
    if (args == nullptr || nbytes == nullptr) return B200_INVALID_ARGUMENT;
    return guarded_operator(nullptr, [&] {
        const Shape p = check_backward(*args);
        *nbytes = p.s.rows == 0 || p.width == 0 ? 0 : divide(*args, p, sm_count()).bytes;
    });
}

}  // extern "C"
