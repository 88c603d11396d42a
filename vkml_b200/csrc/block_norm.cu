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
// in the registers of the threads that share it, 8 elements of each tensor to a thread for each of its NV pieces, and what is summed over the
// row goes through shuffles and shared memory.
#include "operators.cuh"

#include <algorithm>

namespace b200 {
namespace {

constexpr int64_t kMostWidth = 16384;
constexpr int kWarpRows = 8;  // rows to a block where a row is a warp's

// A vector over the columns (a weight, a bias, the gate), F32 or F16.
struct Columns {
    const void* p;
    int64_t pitch;  // of the gate's rows, in elements
};

// Element e of piece v of thread t of `threads` that share a row: pieces of 8 neighbours where WIDE, else neighbours to neighbouring threads.
template <bool WIDE>
__device__ __forceinline__ int column_of(int v, int e, int t, int threads) {
    return WIDE ? (v * threads + t) * 8 + e : (v * 8 + e) * threads + t;
}

template <typename T, bool WIDE>
__device__ __forceinline__ void read_piece(float (&x)[8], const char* row, int v, int t, int threads, int width) {
    const T* p = reinterpret_cast<const T*>(row);
    if constexpr (WIDE) {
        const int c = column_of<true>(v, 0, t, threads);
        Raw8<T> raw = {};
        if (c < width) load8(raw, p + c);
        unpack8(raw, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = column_of<false>(v, e, t, threads);
            x[e] = c < width ? to_float(p[c]) : 0.f;
        }
    }
}

template <typename T, bool WIDE>
__device__ __forceinline__ void write_piece(char* row, const float (&x)[8], int v, int t, int threads, int width) {
    T* p = reinterpret_cast<T*>(row);
    if constexpr (WIDE) {
        const int c = column_of<true>(v, 0, t, threads);
        if (c < width) store8(p + c, x);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = column_of<false>(v, e, t, threads);
            if (c < width) p[c] = from_float<T>(x[e]);
        }
    }
}

// The piece of a vector over the columns; `absent` where there is none.
template <bool WIDE>
__device__ __forceinline__ void read_columns(float (&x)[8], const void* p, bool half, float absent, int v, int t, int threads, int width) {
    if (p == nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = absent;
    } else if (half) {
        read_piece<__half, WIDE>(x, static_cast<const char*>(p), v, t, threads, width);
    } else {
        read_piece<float, WIDE>(x, static_cast<const char*>(p), v, t, threads, width);
    }
}

// Sums of two values over the threads of a row, the same bits in each of them.  `slot` alternates between calls, so that one barrier is enough.
template <bool WARP>
__device__ __forceinline__ float2 row_sum(float2 x, float2 (&part)[2][32], int& slot) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) {
        x.x += __shfl_xor_sync(0xffffffffu, x.x, d);
        x.y += __shfl_xor_sync(0xffffffffu, x.y, d);
    }
    if constexpr (!WARP) {
        const int lane = threadIdx.x % 32, warps = blockDim.x / 32;
        if (lane == 0) part[slot][threadIdx.x / 32] = x;
        __syncthreads();
        x = lane < warps ? part[slot][lane] : make_float2(0.f, 0.f);
#pragma unroll
        for (int d = 16; d > 0; d /= 2) {
            x.x += __shfl_xor_sync(0xffffffffu, x.x, d);
            x.y += __shfl_xor_sync(0xffffffffu, x.y, d);
        }
        slot ^= 1;
    }
    return x;
}

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
__device__ __forceinline__ float2 norm_of(const float (&x)[NV][8], bool layer, float eps, float share, int t, int threads, int width,
                                          float2 (&part)[2][32], int& slot) {
    float mean = 0.f;
    if (layer) {
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) s.x += x[v][e];
        mean = row_sum<WARP>(s, part, slot).x * share;
    }
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float d = column_of<WIDE>(v, e, t, threads) < width ? x[v][e] - mean : 0.f;
            s.x += d * d;
        }
    return make_float2(mean, 1.f / sqrtf(row_sum<WARP>(s, part, slot).x * share + eps));
}

template <typename TH, typename TY, int NV, bool WIDE, bool WARP>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : 1024)
norm_kernel(const ForwardArgs k) {
    __shared__ float2 part[2][32];
    pdl_prologue();
    int slot = 0;
    const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x % 32 : threadIdx.x;
    const uint32_t r = WARP ? blockIdx.x * kWarpRows + threadIdx.x / 32 : blockIdx.x;
    if (r >= k.rows) return;  // (a whole warp, or a whole block)
    float h[NV][8], y[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) h[v][e] = y[v][e] = 0.f;
        if (k.residual.base != nullptr) read_piece<TH, WIDE>(h[v], row_at(k.residual, k.inner, r), v, t, threads, k.width);
        if (k.branch.base != nullptr) read_piece<TY, WIDE>(y[v], row_at(k.branch, k.inner, r), v, t, threads, k.width);
    }
    float2 post = make_float2(0.f, 0.f), pre = make_float2(0.f, 0.f);
    if (k.post) post = norm_of<WARP, WIDE, NV>(y, k.layer, k.eps, k.share, t, threads, k.width, part, slot);
    const char* gate = static_cast<const char*>(k.gate);
    if (gate != nullptr) gate += int64_t(k.gate_rows.div(r)) * k.gate_pitch;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        if (k.branch.base != nullptr) {
            float w[8], b[8], g[8];
            read_columns<WIDE>(g, gate, k.half_columns, 1.f, v, t, threads, k.width);
            if (k.post) {
                read_columns<WIDE>(w, k.post_weight, k.half_columns, 1.f, v, t, threads, k.width);
                read_columns<WIDE>(b, k.post_bias, k.half_columns, 0.f, v, t, threads, k.width);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[v][e] = (y[v][e] - post.x) * post.y * w[e] + b[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[v][e] = k.a * h[v][e] + k.b * (g[e] * y[v][e]);
                if (column_of<WIDE>(v, e, t, threads) >= k.width) h[v][e] = 0.f;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[v][e] *= k.a;
        }
        if (k.out.base != nullptr) write_piece<TH, WIDE>(row_at(k.out, k.inner, r), h[v], v, t, threads, k.width);
    }
    if (k.normed.base != nullptr) {
        pre = norm_of<WARP, WIDE, NV>(h, k.layer, k.eps, k.share, t, threads, k.width, part, slot);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float w[8], b[8];
            read_columns<WIDE>(w, k.pre_weight, k.half_columns, 1.f, v, t, threads, k.width);
            read_columns<WIDE>(b, k.pre_bias, k.half_columns, 0.f, v, t, threads, k.width);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[v][e] = (h[v][e] - pre.x) * pre.y * w[e] + b[e];
            write_piece<TY, WIDE>(row_at(k.normed, k.inner, r), h[v], v, t, threads, k.width);
        }
    }
    if (k.stats != nullptr && t == 0) k.stats[r] = make_float4(post.x, post.y, pre.x, pre.y);
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
    FastDiv inner;
    uint32_t group_rows, pieces;  // rows to a gate, and how many items they are divided into
    uint32_t items;
    int width;
    float a, b, share;
    bool layer, post, half_columns;
};

// A block takes items one after another: item i is piece i % pieces of the rows of gate i / pieces.  The gate's sums are left behind after each
// item, the others once, in the block's own row of the partial sums; fold_kernel adds those up in order, so that no result depends on timing.
// REGS: the sums stay in the threads' registers; else in the partial sums themselves (each thread its own columns).
template <typename TH, typename TY, int NV, bool WIDE, bool WARP, bool REGS>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : REGS ? 512 : 1024)
norm_backward_kernel(const BackwardArgs k) {
    __shared__ float2 part[2][32];
    pdl_prologue();
    int slot = 0;
    const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x % 32 : threadIdx.x;
    const int own = WARP ? blockIdx.x * kWarpRows + threadIdx.x / 32 : blockIdx.x;  // whose partial sums
    const int owners = WARP ? gridDim.x * kWarpRows : gridDim.x;
    float sum[REGS ? kSums : 1][REGS ? NV : 1][8];
    auto clear = [&](int which) {
        if constexpr (REGS) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[which][v][e] = 0.f;
        }
    };
    auto each_column = [&](float* to, auto&& f) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = column_of<WIDE>(v, e, t, threads);
                if (c < k.width) f(to[c], v, e);
            }
    };
    auto row_of = [&](int which, uint32_t item) { return k.partial[which] + int64_t(which == kGate ? item : uint32_t(own)) * k.width; };
    auto begin = [&](int which, uint32_t item) {
        if constexpr (REGS) clear(which);
        else if (k.partial[which] != nullptr) each_column(row_of(which, item), [](float& x, int, int) { x = 0.f; });
    };
    auto end = [&](int which, uint32_t item) {
        if constexpr (REGS) {
            if (k.partial[which] != nullptr) each_column(row_of(which, item), [&](float& x, int v, int e) { x = sum[which][v][e]; });
        }
    };
#pragma unroll
    for (int s = kPostWeight; s < kSums; ++s) begin(s, 0);
    for (uint32_t item = own; item < k.items; item += owners) {
        const uint32_t group = item / k.pieces, piece = item % k.pieces;
        const uint32_t r0 = group * k.group_rows + static_cast<uint32_t>(uint64_t(k.group_rows) * piece / k.pieces);
        const uint32_t r1 = group * k.group_rows + static_cast<uint32_t>(uint64_t(k.group_rows) * (piece + 1) / k.pieces);
        const char* gate = static_cast<const char*>(k.gate);
        if (gate != nullptr) gate += int64_t(group) * k.gate_pitch;
        begin(kGate, item);
        for (uint32_t r = r0; r < r1; ++r) {
            float s[NV][8], dn[NV][8], ds[NV][8], y[NV][8];
            const bool pre = k.normed_grad.base != nullptr;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
#pragma unroll
                for (int e = 0; e < 8; ++e) s[v][e] = dn[v][e] = ds[v][e] = y[v][e] = 0.f;
                if (pre) {
                    read_piece<TH, WIDE>(s[v], row_at(k.out, k.inner, r), v, t, threads, k.width);
                    read_piece<TY, WIDE>(dn[v], row_at(k.normed_grad, k.inner, r), v, t, threads, k.width);
                }
                if (k.out_grad.base != nullptr) read_piece<TH, WIDE>(ds[v], row_at(k.out_grad, k.inner, r), v, t, threads, k.width);
                if (k.branch.base != nullptr) read_piece<TY, WIDE>(y[v], row_at(k.branch, k.inner, r), v, t, threads, k.width);
            }
            const float4 st = k.stats != nullptr ? k.stats[r] : make_float4(0.f, 1.f, 0.f, 1.f);
            auto add = [&](int which, int v, const float (&x)[8]) {
                if constexpr (REGS) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum[which][v][e] += x[e];
                } else if (k.partial[which] != nullptr) {
                    float* to = row_of(which, item);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int c = column_of<WIDE>(v, e, t, threads);
                        if (c < k.width) to[c] += x[e];
                    }
                }
            };
            if (pre) {
                float2 m = make_float2(0.f, 0.f);
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    float w[8], x[8];
                    read_columns<WIDE>(w, k.pre_weight, k.half_columns, 1.f, v, t, threads, k.width);
                    add(kPreBias, v, dn[v]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        s[v][e] = (s[v][e] - st.z) * st.w;
                        x[e] = dn[v][e] * s[v][e];
                        dn[v][e] *= w[e];
                        m.x += dn[v][e] * s[v][e];
                        m.y += dn[v][e];
                    }
                    add(kPreWeight, v, x);
                }
                m = row_sum<WARP>(m, part, slot);
                m.x *= k.share;
                m.y = k.layer ? m.y * k.share : 0.f;
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int e = 0; e < 8; ++e) ds[v][e] += st.w * (dn[v][e] - m.y - s[v][e] * m.x);
            }
            if (k.residual_grad.base != nullptr) {
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = k.a * ds[v][e];
                    write_piece<TH, WIDE>(row_at(k.residual_grad, k.inner, r), x, v, t, threads, k.width);
                }
            }
            if (k.branch.base == nullptr && k.branch_grad.base == nullptr) continue;
            float2 m = make_float2(0.f, 0.f);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                float w[8], b[8], g[8], x[8];
                read_columns<WIDE>(g, gate, k.half_columns, 1.f, v, t, threads, k.width);
                read_columns<WIDE>(w, k.post_weight, k.half_columns, 1.f, v, t, threads, k.width);
                read_columns<WIDE>(b, k.post_bias, k.half_columns, 0.f, v, t, threads, k.width);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (k.post) y[v][e] = (y[v][e] - st.x) * st.y;
                    ds[v][e] *= k.b;
                    x[e] = ds[v][e] * (y[v][e] * w[e] + b[e]);
                    ds[v][e] *= g[e];  // du
                }
                add(kGate, v, x);
                add(kPostBias, v, ds[v]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = ds[v][e] * y[v][e];
                    ds[v][e] *= w[e];
                    m.x += ds[v][e] * y[v][e];
                    m.y += ds[v][e];
                }
                add(kPostWeight, v, x);
            }
            if (k.branch_grad.base == nullptr) continue;
            if (k.post) {
                m = row_sum<WARP>(m, part, slot);
                m.x *= k.share;
                m.y = k.layer ? m.y * k.share : 0.f;
            }
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (k.post) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) ds[v][e] = st.y * (ds[v][e] - m.y - y[v][e] * m.x);
                }
                write_piece<TY, WIDE>(row_at(k.branch_grad, k.inner, r), ds[v], v, t, threads, k.width);
            }
        }
        end(kGate, item);
    }
#pragma unroll
    for (int s = kPostWeight; s < kSums; ++s) end(s, 0);
}

struct Fold {
    const float* from;   // [groups * parts][width]
    void* to;            // [groups][width], dense
    uint32_t groups, parts;
};
struct FoldArgs {
    Fold f[kSums];
    int width;
    bool half;
};

// to[g][c] = sum over p of from[g * parts + p][c]: 32 columns to a block, 8 threads to a column, each with an eighth of the parts in order.
__global__ void __launch_bounds__(256) fold_kernel(const FoldArgs k) {
    __shared__ float part[8][33];
    pdl_prologue();
    const Fold& f = k.f[blockIdx.y];
    const int x = threadIdx.x % 32, y = threadIdx.x / 32, c = blockIdx.x * 32 + x;
    for (uint32_t g = blockIdx.z; g < f.groups; g += gridDim.z) {
        const uint32_t p0 = f.parts * y / 8, p1 = f.parts * (y + 1) / 8;
        float sum = 0.f;
        if (c < k.width) {
            const float* from = f.from + (int64_t(g) * f.parts) * k.width + c;
            uint32_t p = p0;
            for (; p + 8 <= p1; p += 8) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = from[int64_t(p + i) * k.width];
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += v[i];
            }
            for (; p < p1; ++p) sum += from[int64_t(p) * k.width];
        }
        part[y][x] = sum;
        __syncthreads();
        if (y == 0 && c < k.width) {
            float total = part[0][x];
#pragma unroll
            for (int i = 1; i < 8; ++i) total += part[i][x];
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
            if (n.t->data == nullptr && n.t->ndim == 0) continue;
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
    if (!present(a.branch) && (present(a.gate) || (a.flags & B200_NORM_POST) != 0)) fail(B200_INVALID_ARGUMENT, "block_norm: a gate or a norm of an absent branch");
    if ((a.flags & B200_NORM_POST) == 0 && (present(a.post_weight) || present(a.post_bias))) fail(B200_INVALID_ARGUMENT, "block_norm: weights of a norm that is not applied");
    if (!present(a.normed) && (present(a.pre_weight) || present(a.pre_bias))) fail(B200_INVALID_ARGUMENT, "block_norm: weights of a norm that is not applied");
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
    const unsigned blocks = static_cast<unsigned>(warp ? ceil_div(p.s.rows, kWarpRows) : p.s.rows);
    ProfScope scope(ctx, "block_norm");
    with_types(p, [&](auto th, auto ty) {
        using TH = decltype(th);
        using TY = decltype(ty);
        auto go = [&](auto kernel) { launch_kernel(ctx, kernel, blocks, threads, 0, k); };
        if (wide) go(warp ? norm_kernel<TH, TY, 1, true, true> : pieces == 1 ? norm_kernel<TH, TY, 1, true, false> : norm_kernel<TH, TY, 2, true, false>);
        else go(warp ? norm_kernel<TH, TY, 1, false, true> : pieces == 1 ? norm_kernel<TH, TY, 1, false, false> : norm_kernel<TH, TY, 2, false, false>);
    });
    check_last_launch("block_norm");
    ctx->count_launch();
}

// How a backward call is divided.
struct Division {
    uint32_t blocks, threads, owners, pieces, items;
    bool warp, regs;
    int nv;
    int64_t partial_floats[kSums];
    size_t bytes;
};

Division divide(const b200_block_norm_grad_args& a, const Shape& p, int sms) {
    Division d{};
    d.warp = p.width <= 256;
    d.nv = p.width <= 4096 ? 1 : 2;
    d.regs = d.nv == 1;
    d.threads = d.warp ? kWarpRows * 32 : static_cast<uint32_t>(ceil_div(p.width, int64_t(8) * d.nv * 32)) * 32;
    const int64_t group_rows = p.s.rows / p.gates;
    // as many blocks as the registers of an SM hold at once
    const int64_t resident = int64_t(sms) * std::max<int64_t>(1, (d.regs ? 512 : 1024) / d.threads);
    const int64_t workers = d.warp ? resident * kWarpRows : resident;
    // a gate's rows in as many pieces as leave the longest worker the least to do
    int64_t best = INT64_MAX;
    d.pieces = 1;
    for (int64_t n = 1; n <= std::min(group_rows, workers) && (n == 1 || p.gates * n < 2 * workers + p.gates); ++n) {
        const int64_t longest = ceil_div(p.gates * n, workers) * ceil_div(group_rows, n);
        if (longest < best) best = longest, d.pieces = static_cast<uint32_t>(n);
    }
    d.items = static_cast<uint32_t>(p.gates * d.pieces);
    const int64_t needed = std::min<int64_t>(workers, d.items);
    d.blocks = static_cast<uint32_t>(d.warp ? ceil_div(needed, kWarpRows) : needed);
    d.owners = d.warp ? d.blocks * kWarpRows : d.blocks;
    const b200_tensor* wanted[kSums] = {&a.gate_grad, &a.post_weight_grad, &a.post_bias_grad, &a.pre_weight_grad, &a.pre_bias_grad};
    for (int s = 0; s < kSums; ++s) {
        if (!present(*wanted[s])) continue;
        d.partial_floats[s] = (s == kGate ? int64_t(d.items) : int64_t(d.owners)) * p.width;
        d.bytes += (static_cast<size_t>(d.partial_floats[s]) * sizeof(float) + 255) / 256 * 256;
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
    const bool post = (a.flags & B200_NORM_POST) != 0, pre = present(a.normed_grad);
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
    const b200_tensor* vectors[kSums] = {&a.gate_grad, &a.post_weight_grad, &a.post_bias_grad, &a.pre_weight_grad, &a.pre_bias_grad};
    if (p.width == 0) return;
    wait_for_tensors(ctx, {&a.out, &a.branch, &a.stats, &a.out_grad, &a.normed_grad, &a.post_weight, &a.post_bias, &a.gate, &a.pre_weight, &a.residual_grad, &a.branch_grad,
                           &a.post_weight_grad, &a.post_bias_grad, &a.pre_weight_grad, &a.pre_bias_grad, &a.gate_grad});
    if (p.s.rows == 0) {  // sums of nothing
        for (const b200_tensor* t : vectors) {
            if (present(*t)) B200_CUDA_CHECK(cudaMemsetAsync(t->data, 0, static_cast<size_t>(numel_of(*t)) * dtype_size(t->dtype), ctx->stream));
        }
        return;
    }
    const Division d = divide(a, p, sm_count());
    char* scratch = operator_workspace(ctx, a.workspace, a.workspace_bytes, d.bytes);
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
    unsigned folds = 0, groups = 1;
    for (int s = 0; s < kSums; ++s) {
        if (!present(*vectors[s])) continue;
        k.partial[s] = reinterpret_cast<float*>(scratch);
        scratch += (static_cast<size_t>(d.partial_floats[s]) * sizeof(float) + 255) / 256 * 256;
        fold.f[folds++] = Fold{k.partial[s], vectors[s]->data, static_cast<uint32_t>(s == kGate ? p.gates : 1), s == kGate ? d.pieces : d.owners};
        if (s == kGate) groups = static_cast<unsigned>(std::min<int64_t>(p.gates, 4096));
        fold.half = vectors[s]->dtype == B200_F16;
    }
    k.inner = FastDiv(static_cast<uint32_t>(p.s.inner));
    k.group_rows = static_cast<uint32_t>(p.s.rows / p.gates);
    k.pieces = d.pieces;
    k.items = d.items;
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
        auto go = [&](auto kernel) { launch_kernel(ctx, kernel, d.blocks, d.threads, 0, k); };
        if (wide) go(d.warp ? norm_backward_kernel<TH, TY, 1, true, true, true> : d.regs ? norm_backward_kernel<TH, TY, 1, true, false, true>
                                                                                         : norm_backward_kernel<TH, TY, 2, true, false, false>);
        else go(d.warp ? norm_backward_kernel<TH, TY, 1, false, true, true> : d.regs ? norm_backward_kernel<TH, TY, 1, false, false, true>
                                                                                     : norm_backward_kernel<TH, TY, 2, false, false, false>);
    });
    check_last_launch("block_norm_backward");
    if (folds > 0) {
        launch_kernel(ctx, fold_kernel, dim3(static_cast<unsigned>(ceil_div(p.width, 32)), folds, groups), 256, 0, fold);
        check_last_launch("block_norm_backward");
    }
    ctx->count_launch(folds > 0 ? 2 : 1);
}

}  // namespace

void check_block_norm(const b200_block_norm_args& a) {
    int columns = -1;
    (void)check_forward(a, columns);
}
void check_block_norm_backward(const b200_block_norm_grad_args& a) { (void)check_backward(a); }

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
