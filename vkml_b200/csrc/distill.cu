// Distillation from a teacher's top logits, with a share of cross-entropy on labels, forward and backward.
//
// For a row z of V logits, the teacher's logits t at K columns k_j, temperature T and hard weight c:
//
//   p = softmax(t / T)        q = softmax(z / T)        h = softmax(z)
//   loss = (1 - c) T^2 sum_j p_j (log p_j - log q_{k_j}) + c (log sum exp z - z_label)
//   grad = w [ (1 - c) T (q - p at k) + c (h - 1 at the label) ]
//
// Bound by memory: z read once and, with a gradient, as much written.  A block takes a row.  One pass over it keeps the running maximum and the
// running sums of exp((z - max) / T) and exp(z - max); the gradient's pass writes q and h in every column, and the K + 1 columns that
// the teacher or the label adds to are written again afterwards.
#include "operators.cuh"

#include <algorithm>
#include <cmath>

namespace b200 {
namespace {

constexpr int kThreads = 512;
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
    bool wide_ids, wide_labels, half_teacher;
    bool soft, hard;      // which parts have a weight
    float temperature, inverse, hard_weight, grad_scale;
};

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Running maximum and sums of a part of a row.  A maximum of -inf (nothing but -inf so far) has sums of 0.
struct Running {
    float top, soft, hard;
};

__device__ __forceinline__ float shift_of(float top) { return top == -INFINITY ? 0.f : top; }

template <typename F>
__device__ __forceinline__ float block_reduce(float x, float* part, F&& join, float empty) {
#pragma unroll
    for (int d = 16; d > 0; d /= 2) x = join(x, __shfl_xor_sync(0xffffffffu, x, d));
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = x;
    __syncthreads();
    x = threadIdx.x % 32 < kThreads / 32 ? part[threadIdx.x % 32] : empty;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) x = join(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
}

// Elements of a row that lie before its first 16-byte boundary, and how many vectors of 16 bytes follow.
template <typename T>
__device__ __forceinline__ int64_t head_of(const T* row, int64_t n) {
    const int64_t head = (16 - (reinterpret_cast<uintptr_t>(row) & 15)) % 16 / int64_t(sizeof(T));
    return head < n ? head : n;
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

template <typename T>
__device__ __forceinline__ uint4 pack(const float (&x)[16 / sizeof(T)]) {
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
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, bool FORWARD, bool GRAD>
__global__ void __launch_bounds__(kThreads)
distill_kernel(const Args k) {
    constexpr int E = 16 / sizeof(T);
    extern __shared__ char shared[];
    float* const p = reinterpret_cast<float*>(shared);        // [top]: the teacher's probabilities
    float* const zk = p + k.top;                              // [top + 1]: the logits at its columns, and at the label's
    int* const col = reinterpret_cast<int*>(zk + k.top + 1);  // [top + 1]: the columns, -1: none
    __shared__ float part[32];
    pdl_prologue();
    const int tid = threadIdx.x;
    const uint32_t r = blockIdx.x;
    const T* const z = reinterpret_cast<const T*>(row_at(k.logits, k.inner, r));

    // the teacher's distribution and the logits at its columns
    float top_t = -INFINITY;
    if (k.soft) {
        const char* ids = row_at(k.ids, k.inner, r);
        const char* t = row_at(k.teacher, k.inner, r);
        for (int j = tid; j < k.top; j += kThreads) {
            const int64_t id = load_index(ids + int64_t(j) * (k.wide_ids ? 8 : 4), k.wide_ids);
            const bool in = id >= 0 && id < k.vocab;
            if (id >= k.vocab) atomicOr(k.status, kStatusIndexOutOfRange);
            col[j] = in ? static_cast<int>(id) : -1;
            p[j] = in ? (k.half_teacher ? __half2float(reinterpret_cast<const __half*>(t)[j]) : reinterpret_cast<const float*>(t)[j]) : -INFINITY;
            zk[j] = in ? to_float(z[id]) : 0.f;
            top_t = fmaxf(top_t, p[j]);
        }
    }
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
    bool taught = false;  // whether the row has a teacher's entry
    float log_sum = 0.f;
    if (k.soft) {
        top_t = block_reduce(top_t, part, [](float a, float b) { return fmaxf(a, b); }, -INFINITY);
        float sum = 0.f;
        for (int j = tid; j < k.top; j += kThreads) sum += col[j] >= 0 ? expf((p[j] - shift_of(top_t)) * k.inverse) : 0.f;
        sum = block_reduce(sum, part, [](float a, float b) { return a + b; }, 0.f);
        taught = !(sum == 0.f);
        log_sum = logf(sum);
        if constexpr (!FORWARD) {
            for (int j = tid; j < k.top; j += kThreads) p[j] = taught && col[j] >= 0 ? expf((p[j] - shift_of(top_t)) * k.inverse - log_sum) : 0.f;
        }
    }

    // the row's log sums of exponentials
    const float c_soft = k.inverse * kLog2e;
    const int64_t head = head_of(z, k.vocab), vectors = (k.vocab - head) / E, tail = head + vectors * E;
    // q = exp((z - at) / T - log_soft), h = exp(z - at - log_hard).  The maximum and the logarithms stay apart: their sum would lose the
    // logarithm in a row whose logits are all the type's lowest value.
    float at = 0.f, log_soft = 0.f, log_hard = 0.f;
    if constexpr (FORWARD) {
        Running run = {-INFINITY, 0.f, 0.f};
        auto take = [&](const float* x, int n) {
            float top = x[0];
            for (int e = 1; e < n; ++e) top = fmaxf(top, x[e]);
            if (top > run.top) {
                const float at = shift_of(top);
                run.soft *= fast_exp2((run.top - at) * c_soft);
                run.hard *= fast_exp2((run.top - at) * kLog2e);
                run.top = top;
            }
            const float at = shift_of(run.top);
            if (k.soft) {
                for (int e = 0; e < n; ++e) run.soft += fast_exp2((x[e] - at) * c_soft);
            }
            if (k.hard) {
                for (int e = 0; e < n; ++e) run.hard += fast_exp2((x[e] - at) * kLog2e);
            }
        };
        for (int64_t i = tid; i < head; i += kThreads) {
            const float x = to_float(z[i]);
            take(&x, 1);
        }
        for (int64_t i = tail + tid; i < k.vocab; i += kThreads) {
            const float x = to_float(z[i]);
            take(&x, 1);
        }
        const uint4* const zv = reinterpret_cast<const uint4*>(z + head);
#pragma unroll 4
        for (int64_t i = tid; i < vectors; i += kThreads) {
            float x[E];
            unpack<T>(zv[i], x);
            take(x, E);
        }
        const float top = block_reduce(run.top, part, [](float a, float b) { return fmaxf(a, b); }, -INFINITY);
        at = shift_of(top);
        auto add = [](float a, float b) { return a + b; };
        if (k.soft) log_soft = logf(block_reduce(run.soft * fast_exp2((run.top - at) * c_soft), part, add, 0.f));
        if (k.hard) log_hard = logf(block_reduce(run.hard * fast_exp2((run.top - at) * kLog2e), part, add, 0.f));
        if (tid == 0 && k.stats != nullptr) k.stats[r] = make_float4(top, log_soft, log_hard, 0.f);
        // a row of nothing but -inf: the sums are 0 and their logarithms -inf, which stay out of the differences so that q = 0, log q = -inf
        log_soft = shift_of(log_soft), log_hard = shift_of(log_hard);
        float kl = 0.f;
        if (k.soft) {
            for (int j = tid; j < k.top; j += kThreads) {
                const float lp = (p[j] - shift_of(top_t)) * k.inverse - log_sum;
                const float pj = taught && col[j] >= 0 ? expf(lp) : 0.f;
                p[j] = pj;
                if (pj != 0.f) kl += pj * (lp - ((zk[j] - at) * k.inverse - log_soft));
            }
            kl = block_reduce(kl, part, add, 0.f);
        }
        if (tid == 0 && k.losses != nullptr) {
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
        __syncthreads();  // (p, zk and col of the other threads; and z is written from here on where the gradient lies on it)
        T* const g = reinterpret_cast<T*>(row_at(k.grad, k.inner, r));
        const float w = k.grad_scale * (k.weights.base != nullptr ? *reinterpret_cast<const float*>(row_at(k.weights, k.inner, r)) : 1.f);
        const bool hard_there = k.hard && col[k.top] >= 0;
        const float ws = taught ? w * (1.f - k.hard_weight) * k.temperature : 0.f;
        const float wh = hard_there ? w * k.hard_weight : 0.f;
        const float soft2 = log_soft * kLog2e, hard2 = log_hard * kLog2e;
        auto value = [&](float x) {
            float y = 0.f;
            if (ws != 0.f) y += ws * fast_exp2(fmaf(x - at, c_soft, -soft2));
            if (wh != 0.f) y += wh * fast_exp2(fmaf(x - at, kLog2e, -hard2));
            return y;
        };
        for (int64_t i = tid; i < head; i += kThreads) g[i] = from_float<T>(value(to_float(z[i])));
        for (int64_t i = tail + tid; i < k.vocab; i += kThreads) g[i] = from_float<T>(value(to_float(z[i])));
        const uint4* const zv = reinterpret_cast<const uint4*>(z + head);
        if ((reinterpret_cast<uintptr_t>(g + head) & 15) == 0) {
#pragma unroll 4
            for (int64_t i = tid; i < vectors; i += kThreads) {
                float x[E];
                unpack<T>(zv[i], x);
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = value(x[e]);
                reinterpret_cast<uint4*>(g + head)[i] = pack<T>(x);
            }
        } else {
            for (int64_t i = head + tid; i < tail; i += kThreads) g[i] = from_float<T>(value(to_float(z[i])));
        }
        __syncthreads();
        // the columns that p or the label adds to, each by the first entry that names it
        for (int j = tid; j <= k.top; j += kThreads) {
            const int c = j < k.top && !k.soft ? -1 : col[j];
            if (c < 0) continue;
            bool first = true;
            float minus = 0.f;
            if (k.soft) {
                for (int i = 0; i < k.top; ++i) {
                    if (col[i] != c) continue;
                    if (i < j) first = false;
                    if (ws != 0.f) minus += ws * p[i];
                }
            }
            if (!first) continue;
            if (col[k.top] == c) minus += wh;
            g[c] = from_float<T>(value(zk[j]) - minus);
        }
    }
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
};

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
    if (!(a.temperature > 0.f) || std::isinf(a.temperature)) fail(B200_INVALID_ARGUMENT, "distill_loss: the temperature is not above 0 and finite");
    if (!(a.hard_weight >= 0.f && a.hard_weight <= 1.f)) fail(B200_INVALID_ARGUMENT, "distill_loss: the hard weight is not in 0..1");
    const bool labelled = a.labels.data != nullptr || a.labels.ndim != 0;
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
    const Plan plan{axes, vocab, top, s, labelled};
    if (s.rows == 0) return plan;
    if (labelled && !present(a.labels)) fail(B200_INVALID_ARGUMENT, "labels have no storage");
    if (forward && !present(a.losses) && !present(a.stats) && !present(a.grad)) fail(B200_INVALID_ARGUMENT, "distill_loss: no result is asked for");
    if (!forward && (!present(a.grad) || !present(a.stats))) fail(B200_INVALID_ARGUMENT, "distill_loss_backward: grad and the forward call's stats are needed");
    if (a.hard_weight > 0.f && !labelled) fail(B200_INVALID_ARGUMENT, "distill_loss: a hard weight without labels");
    return plan;
}

void launch_distill(b200_ctx* ctx, const b200_distill_args& a, bool forward) {
    const Plan plan = check_distill(a, forward);
    const auto& [axes, vocab, top, s, labelled] = plan;
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
    const size_t shared = (3 * static_cast<size_t>(top) + 2) * 4;
    const unsigned blocks = static_cast<unsigned>(s.rows);
    auto go = [&](auto kernel) { launch_kernel(ctx, kernel, blocks, kThreads, shared, k); };
    const bool half = a.logits.dtype == B200_F16;
    if (!forward) go(half ? distill_kernel<__half, false, true> : distill_kernel<float, false, true>);
    else if (present(a.grad)) go(half ? distill_kernel<__half, true, true> : distill_kernel<float, true, true>);
    else go(half ? distill_kernel<__half, true, false> : distill_kernel<float, true, false>);
    check_last_launch("distill_loss");
    ctx->count_launch();
}

}  // namespace

void check_distill_loss(const b200_distill_args& a, bool forward) { (void)check_distill(a, forward); }

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
